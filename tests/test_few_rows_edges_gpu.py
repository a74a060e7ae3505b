"""GPU: inputs at the edges of what the few-row operators take: activations beside an outlier, infinite weights, logits far below
zero, two host threads at once, the gradient's graph kept, traced quantising."""

import threading

import pytest
import torch

from primus_turbo_b200 import _lib
from primus_turbo_b200.pytorch.core.int4_weight import Int4Weight
from primus_turbo_b200.pytorch.ops import dequantize_int4, gemm_int4, quantize_int4

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16


def weight(shape, group, zeros, seed=0, codes=None):
    g = torch.Generator(DEV).manual_seed(seed)
    groups = (*shape[:-1], -(-shape[-1] // group))
    drawn = torch.randint(0, 16, shape, generator=g, device=DEV, dtype=torch.uint8)
    scale = ((torch.rand(groups, generator=g, device=DEV) + 0.5) * shape[-1] ** -0.5).to(BF)
    zero = torch.randint(0, 16, groups, generator=g, device=DEV, dtype=torch.uint8) if zeros else None
    return Int4Weight.from_codes(drawn if codes is None else codes, scale, zero, group_size=group)


# ---- the host side ----------------------------------------------------------------------------------------------------------------
def test_two_threads_launch_one_kernel_with_different_sizes():
    """Calls of the same kernels with more and with less shared memory, from two threads that do not wait for each other (a call of
    the C interface lets the interpreter go)."""
    q, k = weight((64, 4096), 64, False), 4096
    x = torch.randn(32, k, device=DEV, dtype=BF)
    need = _lib.lib.ptb_gemm_int4_workspace(_lib.PTB_BF16, 32, k, 64)
    sizes = ((32, 8), (17, 1))  # rows of the two threads: the kernel of more rows, and that of a few
    streams = [torch.cuda.Stream() for _ in sizes]
    want = [[gemm_int4(x[:m], q) for m in ms] for ms in sizes]
    out = [[torch.empty(m, 64, device=DEV, dtype=BF) for m in ms] for ms in sizes]
    space = [torch.empty(need, device=DEV, dtype=torch.uint8) for _ in sizes]
    torch.cuda.synchronize()
    failed = [0, 0]

    def work(i):
        torch.cuda.set_device(x.device)
        calls = [(x.data_ptr(), _lib.PTB_BF16, k, m, 64, k, q.qdata.data_ptr(), q.scale.data_ptr(), None, 64, None, space[i].data_ptr(), y.data_ptr(),
                  streams[i].cuda_stream) for m, y in zip(sizes[i], out[i])]
        for _ in range(20000):
            for c in calls:
                failed[i] += _lib.lib.ptb_gemm_int4(*c) != 0

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert failed == [0, 0]
    assert all(torch.equal(a, b) for o, w in zip(out, want) for a, b in zip(o, w))


def test_traced_quantising_runs_again_on_new_inputs():
    w, x, other = quantize_int4(torch.randn(72, 256, device=DEV, dtype=BF), 128), *(torch.randn(3, 256, device=DEV, dtype=BF) for _ in range(2))
    for f in (lambda x: x @ dequantize_int4(w).T, lambda x: quantize_int4(x, 32).qdata, lambda x: dequantize_int4(quantize_int4(x, 32, False))):
        traced = torch.jit.trace(f, (x,), check_trace=False)
        assert torch.equal(traced(other), f(other)) and torch.equal(traced(x), f(x))
