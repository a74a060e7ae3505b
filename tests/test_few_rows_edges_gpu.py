"""GPU: inputs at the edges of what the few-row operators take: activations beside an outlier, infinite weights, logits far below
zero, two host threads at once, the gradient's graph kept, traced quantising."""

import math
import threading

import pytest
import torch

from primus_turbo_b200 import _lib, _native
from primus_turbo_b200.pytorch.core.int4_weight import Int4Weight
from primus_turbo_b200.pytorch.core.low_precision import Float8QuantConfig, ScalingGranularity
from primus_turbo_b200.pytorch.core.quantized_tensor import create_quantized_weight
from primus_turbo_b200.pytorch.ops import dequantize_int4, gemm_int4, quantize_int4
from primus_turbo_b200.pytorch.ops.moe import moe_few_tokens, topk_router

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16


def spread(t, group, k):
    return t.repeat_interleave(group, dim=-1)[..., :k]


def weight(shape, group, zeros, seed=0, codes=None):
    g = torch.Generator(DEV).manual_seed(seed)
    groups = (*shape[:-1], -(-shape[-1] // group))
    drawn = torch.randint(0, 16, shape, generator=g, device=DEV, dtype=torch.uint8)
    scale = ((torch.rand(groups, generator=g, device=DEV) + 0.5) * shape[-1] ** -0.5).to(BF)
    zero = torch.randint(0, 16, groups, generator=g, device=DEV, dtype=torch.uint8) if zeros else None
    return Int4Weight.from_codes(drawn if codes is None else codes, scale, zero, group_size=group)


def parts(q):
    """(values, scales, zero points) of every code, in 64 bits"""
    k = q.shape[-1]
    z = torch.full(q.shape, 8.0, device=DEV, dtype=torch.float64) if q.zero is None else spread(q.zero, q.group_size, k).double()
    s = spread(q.scale, q.group_size, k).double()
    return (q.codes().double() - z) * s, s, z


def at_zero_point(q, channels):
    """The weight with its codes of some channels at the zero point: what x holds there meets a value of zero."""
    codes = q.codes()
    codes[..., channels] = parts(q)[2][..., channels].to(torch.uint8)
    return Int4Weight.from_codes(codes, q.scale, q.zero, group_size=q.group_size)


# ---- outliers -----------------------------------------------------------------------------------------------------------------
def product_bound(x, q, dtype):
    """What a product of 4-bit weights may be off by.  x is held to 2^-22 of the largest of its 128 or better; bare codes, up to 15, are added up
    exactly or in 32 bits, and zero (up to 15) times the sum of x is taken off: 12 operations of a group on sums of that size; then the
    blocks of a warp (K / 1024 + 1), the warps and halves (20), each within 2^-23; one rounding to the output."""
    w, s, _ = parts(q)
    xd, k = x.double(), x.shape[-1]
    want = xd @ w.T
    ops = k / 1024 + 31
    size = xd.abs() @ w.abs().T * ops + xd.abs() @ s.T * (30 * 12)
    pad = lambda t: torch.nn.functional.pad(t, (0, -k % 128)).unflatten(-1, (-1, 128))  # noqa: E731
    held = (pad(xd.abs()).amax(-1) @ pad(w.abs()).sum(-1).T) * 2.0**-22
    return want, size * 2.0**-23 + held + want.abs() * torch.finfo(dtype).eps / 2


@pytest.mark.parametrize("m", [1, 2, 3, 5, 8, 9, 16, 24])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("dtype,outlier", [(torch.float16, 1000.0), (BF, 1000.0), (BF, 32768.0)])
def test_small_activations_beside_an_outlier(m, group, zeros, dtype, outlier):
    """A channel of 1000 among others of one, whose weights are zero: the result is that of the others, as exact as without it."""
    k = 520
    q = at_zero_point(weight((272, k), group, zeros, seed=group), [5, 130, 519])
    x = torch.randn(m, k, device=DEV, generator=torch.Generator(DEV).manual_seed(m)).to(dtype)
    x[:, [5, 130, 519]] = torch.tensor([outlier, -outlier, outlier / 3], device=DEV).to(dtype)
    want, bound = product_bound(x, q, dtype)
    y = gemm_int4(x, q).double()
    assert bool(((y - want).abs() <= bound).all()), ((y - want).abs() / bound).max()


def test_a_row_is_as_exact_in_a_small_batch_as_in_a_larger_one():
    k = 2048
    q = at_zero_point(weight((1024, k), 128, False), [77])
    x = torch.randn(9, k, device=DEV, generator=torch.Generator(DEV).manual_seed(1)).to(torch.float16)
    x[:, 77] = 3000.0
    want = x.double() @ parts(q)[0].T
    off = [((gemm_int4(x[:m], q).double() - want[:m]).norm() / want[:m].norm()).item() for m in (1, 8, 9)]
    # rounding to fp16 leaves at most 2^-11 of each value; values held to 2^-22 of 3000 add at most 3000 x 2^-22 = 2^-10.4 of 1 to a sixteenth of the
    # channels, a quarter of that in the norm, and fp32 sums beside it 12 x 30 / 4.6 x 2^-23 x 3000 / sqrt(2048) = 2^-10.7 at the very worst
    assert all(o <= 2.0**-11 + 2.0**-12 + 2.0**-10 for o in off), off


@pytest.mark.parametrize("T", [1, 2, 8, 9])
@pytest.mark.parametrize("dtype", [BF, torch.float16])
@pytest.mark.parametrize("where", ["x", "h"])
def test_a_layer_beside_an_outlier(T, dtype, where):
    """An outlier among the activations, or among what lies between the two products, at a channel whose weights are zero."""
    E, H, I, k, group = 4, 384, 256, 2, 64
    g = torch.Generator(DEV).manual_seed(T)
    w1, w2 = weight((E, 2 * I, H), group, False, seed=1), weight((E, H, I), group, False, seed=2)
    x = torch.randn(T, H, device=DEV, generator=g).to(dtype)
    ids = torch.rand(T, E, device=DEV, generator=g).argsort(1)[:, :k].contiguous()
    probs = torch.rand(T, k, device=DEV, generator=g) + 0.1
    if where == "x":
        w1, x[:, 9] = at_zero_point(w1, [9]), 1000.0
    else:
        scale = w1.scale.clone()
        scale[:, I + 33] *= 1024  # of an up channel
        w1, w2 = Int4Weight(w1.qdata, scale, None, w1.shape, group), at_zero_point(w2, [33])
    (v1, s1, _), (v2, s2, _) = parts(w1), parts(w2)
    y = moe_few_tokens(x, ids, probs, w1, w2).double()
    eps = torch.finfo(dtype).eps / 2
    blocks = lambda t: torch.nn.functional.pad(t, (0, -t.shape[-1] % 128)).unflatten(-1, (-1, 128))  # noqa: E731
    held = lambda v, a: (blocks(v.abs()).sum(-1) * blocks(a).amax(-1)).sum(-1)  # noqa: E731  (sum of |v| of a block times its largest |a|)
    for t in range(T):
        want, bound = 0.0, 0.0
        for j, e in enumerate(ids[t].tolist()):
            xd, p = x[t].double(), probs[t, j].double()
            u = v1[e] @ xd
            du = (v1[e].abs() @ xd.abs() * 31 + s1[e] @ xd.abs() * (30 * 12)) * 2.0**-23 + held(v1[e], xd.abs()) * 2.0**-22
            a, b = u[:I], u[I:]
            h = a * torch.sigmoid(a) * b
            # silu's slope is at most 1.1; between the products h is held to 2^-12 of itself or 2^-22 of the block's largest (a half-block's in
            # larger batches), and silu and the products are within 8 roundings
            dh = 1.1 * du[:I] * (b.abs() + du[I:]) + (a * torch.sigmoid(a)).abs() * du[I:] + h.abs() * (2.0**-12 + 8 * 2.0**-23)
            dy = v2[e].abs() @ (dh + h.abs() * 91 * 2.0**-23) + (s2[e] @ h.abs()) * (30 * 12 * 2.0**-23) + held(v2[e], h.abs()) * 2.0**-22
            want, bound = want + p * (v2[e] @ h), bound + p * dy
        off, bound = (y[t] - want).abs(), bound + want.abs() * eps + torch.finfo(dtype).smallest_normal
        assert bool((off <= bound).all()), (off / bound).max()


# ---- infinite weights -----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("T", [1, 2, 3, 4, 5, 8, 9, 20])
@pytest.mark.parametrize("dtype", [BF, torch.float16])
def test_an_infinite_weight_of_16_bits_is_infinite_in_any_batch(T, dtype):
    """An infinity in the up projection: in bf16 the same signed infinities whatever the number of tokens, and nothing where it takes no part.
    In fp16 the down projection's weights are the sum of two bf16, of either sign: an infinity times one less an infinity times the other is NaN."""
    E, H, I = 3, 256, 128
    g = torch.Generator(DEV).manual_seed(T)
    w1, w2 = (torch.randn(E, 2 * I, H, device=DEV, generator=g) / 16).to(dtype), (torch.randn(E, H, I, device=DEV, generator=g) / 11).to(dtype)
    w1[1, I + 3, 40] = math.inf
    w1[1, 3] = w1[1, 3].abs()  # its gate is positive for positive x
    x = (torch.rand(T, H, device=DEV, generator=g) + 0.5).to(dtype)
    ids = (torch.arange(T, device=DEV) % 3)[:, None].flip(0).contiguous()
    if T == 1:
        ids[0] = 1
    y = moe_few_tokens(x, ids, torch.ones(T, 1, device=DEV), w1, w2)
    sign = torch.sign(w2[1, :, 3].double())
    for t in range(T):
        if ids[t, 0] == 1:
            if dtype == BF:
                assert torch.equal(y[t].double()[sign != 0], (sign * math.inf)[sign != 0])
            else:
                assert not y[t].isfinite().any()
        else:
            assert bool(y[t].isfinite().all())


@pytest.mark.parametrize("kind", ["raw", "e5m2", "int4"])
@pytest.mark.parametrize("T", [1, 2, 3, 8, 9])
def test_an_infinite_weight_shows_where_it_takes_part(kind, T):
    """In the down projection: infinite or NaN in its output column for the tokens of its expert, nothing else touched."""
    E, H, I = 4, 256, 256
    g = torch.Generator(DEV).manual_seed(T)
    w1, w2 = (torch.randn(E, 2 * I, H, device=DEV, generator=g) / 16).to(BF), (torch.randn(E, H, I, device=DEV, generator=g) / 16).to(BF)
    if kind == "int4":
        w1, w2 = quantize_int4(w1, 64), quantize_int4(w2, 64)
    elif kind == "e5m2":
        cfg = Float8QuantConfig(granularity=ScalingGranularity.BLOCKWISE, block_size=128)
        w1, w2 = (create_quantized_weight(w, torch.float8_e5m2, cfg)[0] for w in (w1, w2))
    x = torch.randn(T, H, device=DEV, generator=g).to(BF)
    ids = torch.rand(T, E, device=DEV, generator=g).argsort(1)[:, :2].contiguous()
    ids[0, 0], ids[0, 1] = 1, 2
    probs = torch.rand(T, 2, device=DEV, generator=g) + 0.1
    before = moe_few_tokens(x, ids, probs, w1, w2)
    if kind == "int4":
        w2.scale[1, 77, 3] = math.inf
    elif kind == "e5m2":
        w2.qdata.view(torch.uint8)[1, 77, 200] = 0x7C
    else:
        w2[1, 77, 200] = math.inf
    y = moe_few_tokens(x, ids, probs, w1, w2)
    hit = torch.zeros(T, H, dtype=torch.bool, device=DEV)
    hit[:, 77] = (ids == 1).any(1)
    assert not y[hit].isfinite().any() and torch.equal(y[~hit], before[~hit])


# ---- router: rows of very negative logits -----------------------------------------------------------------------------------------
@pytest.mark.parametrize("E", [4, 16, 64])
@pytest.mark.parametrize("base", [-12.0, -33.0, -46.0, -62.0, -80.0, -86.0, -95.0])
@pytest.mark.parametrize("bias", [False, True])
def test_close_sigmoid_scores_far_below_zero(E, base, bias):
    """Two groups of two whose logits are units of the last place away and add up to the same: what counts are the sums of the 64-bit scores."""
    g = torch.Generator(DEV).manual_seed(E)
    T, size = 1 << 18, E // 2
    i, j = (torch.randint(0, 2048, (T,), device=DEV, generator=g) for _ in range(2))
    d = torch.randint(1, 32, (T,), device=DEV, generator=g)
    unit = 2.0 ** (math.floor(math.log2(-base)) - 23)
    l = torch.full((T, E), 2 * base, device=DEV, dtype=torch.float64)
    for e, v in ((0, i), (size - 1, j), (size, i + d), (E - 1, j - d)):
        l[:, e] = base + v * unit
    l = l.float()
    s = 1 / (1 + torch.exp(-l.double()))
    best = s.view(T, 2, size).sort(dim=2, descending=True).values[:, :, :2].sum(2)
    other = (best[:, 1] > best[:, 0])[:, None].expand(T, E).clone()
    other[:, size:] = ~other[:, size:]
    want = s.masked_fill(other, -1.0).sort(dim=1, descending=True, stable=True).indices[:, :2]
    _, ids = topk_router(l, 2, score_function="sigmoid", expert_bias=torch.zeros(E, device=DEV) if bias else None, num_groups=2, topk_groups=1)
    assert torch.equal(ids, want), (ids != want).any(1).sum()


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


@pytest.mark.parametrize("native", [True, False])
def test_create_graph_is_taken_and_its_derivative_refused(monkeypatch, native):
    if not native:
        monkeypatch.setattr(_native, "usable", lambda t: False)
    logits = torch.randn(5, 16, device=DEV, requires_grad=True)
    probs, _ = topk_router(logits, 3)
    (want,) = torch.autograd.grad(probs.square().sum(), logits)
    probs, _ = topk_router(logits, 3)
    (g,) = torch.autograd.grad(probs.square().sum(), logits, create_graph=True)
    assert torch.equal(g, want)
    with pytest.raises(RuntimeError, match="twice"):
        torch.autograd.grad(g.sum(), logits, retain_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        torch.autograd.grad(probs.sum() + g.norm(), logits)


def test_scales_that_want_a_gradient_are_refused():
    q = weight((16, 64), 64, False)
    learned = Int4Weight(q.qdata, q.scale.clone().requires_grad_(), None, q.shape, 64)
    x = torch.randn(3, 64, device=DEV, dtype=BF)
    layer = [weight(s, 64, False) for s in ((2, 64, 64), (2, 64, 32))]
    grown = [Int4Weight(w.qdata, w.scale.clone().requires_grad_(), None, w.shape, 64) for w in layer]
    ids, probs = torch.zeros(3, 1, dtype=torch.int64, device=DEV), torch.ones(3, 1, device=DEV)
    for call, same in ((lambda: gemm_int4(x, learned), lambda: gemm_int4(x, q)), (lambda: dequantize_int4(learned), lambda: dequantize_int4(q)),
                       (lambda: moe_few_tokens(x, ids, probs, grown[0], layer[1]), lambda: moe_few_tokens(x, ids, probs, *layer)),
                       (lambda: moe_few_tokens(x, ids, probs, layer[0], grown[1]), lambda: moe_few_tokens(x, ids, probs, *layer))):
        with pytest.raises(NotImplementedError, match="no backward"):
            call()
        with torch.no_grad():
            assert torch.equal(call(), same())


def test_traced_quantising_runs_again_on_new_inputs():
    w, x, other = quantize_int4(torch.randn(72, 256, device=DEV, dtype=BF), 128), *(torch.randn(3, 256, device=DEV, dtype=BF) for _ in range(2))
    for f in (lambda x: x @ dequantize_int4(w).T, lambda x: quantize_int4(x, 32).qdata, lambda x: dequantize_int4(quantize_int4(x, 32, False))):
        traced = torch.jit.trace(f, (x,), check_trace=False)
        assert torch.equal(traced(other), f(other)) and torch.equal(traced(x), f(x))
