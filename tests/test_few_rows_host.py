"""CPU: what the routing, 4-bit and few-token ops refuse and how they say it, the packed layout of 4-bit codes, the C ABI's own
argument errors, and the shapes that tracing sees.  Nothing here reaches a device."""

import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from primus_turbo_b200 import _lib
from primus_turbo_b200.pytorch.core.int4_weight import Int4Weight
from primus_turbo_b200.pytorch.kernels import custom_ops as C
from primus_turbo_b200.pytorch.kernels.few_rows_impl import ExpertWeightArg
from primus_turbo_b200.pytorch.ops import dequantize_int4, gemm_int4, quantize_int4
from primus_turbo_b200.pytorch.ops.moe import moe_few_tokens, topk_router, topk_routing_map

BF = torch.bfloat16


def int4(shape, group=64, zeros=False):
    groups = (*shape[:-1], -(-shape[-1] // group))
    zero = torch.full(groups, 8, dtype=torch.uint8) if zeros else None
    return Int4Weight.from_codes(torch.zeros(shape, dtype=torch.uint8), torch.ones(groups), zero, group_size=group)


# ---- layout ---------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("shape", [(1, 8), (3, 128), (5, 264), (2, 3, 1000)])
def test_codes_there_and_back(shape):
    codes = torch.randint(0, 16, shape, dtype=torch.uint8)
    w = Int4Weight.from_codes(codes, torch.ones((*shape[:-1], -(-shape[-1] // 32))), group_size=32)
    assert torch.equal(w.codes(), codes) and w.qdata.shape[-1] == -(-shape[-1] // 128) * 64


def test_packed_layout_is_the_documented_one():
    codes = torch.randint(0, 16, (2, 300), dtype=torch.uint8)[:, :296]
    w = Int4Weight.from_codes(codes, torch.ones(2, 3), group_size=128)
    for n in range(2):
        for k in range(296):
            b, r = divmod(k, 128)
            q, r = divmod(r, 32)
            t, i = divmod(r, 8)
            byte = w.qdata[n, b * 64 + (t * 4 + q) * 4 + i % 4].item()
            assert byte >> 4 * (i // 4) & 15 == codes[n, k].item()
    used = torch.zeros(2, 384, dtype=torch.uint8)
    used[:, :296] = codes
    assert torch.equal(Int4Weight.from_codes(used, torch.ones(2, 3), group_size=128).qdata, w.qdata)  # codes past the end are 0


def test_weight_parts_are_checked():
    w = int4((4, 256))
    good = dict(qdata=w.qdata, scale=w.scale, zero=None, shape=(4, 256), group_size=64)
    Int4Weight(**good)
    for change in (dict(group_size=48), dict(group_size=128), dict(shape=(4, 264)), dict(shape=(4, 250)), dict(shape=(1024,)),
                   dict(scale=w.scale.float()), dict(qdata=w.qdata.to(torch.int8)), dict(zero=w.scale), dict(qdata=w.qdata[:, :64]),
                   dict(scale=w.scale.t().contiguous().t())):
        with pytest.raises(AssertionError):
            Int4Weight(**{**good, **change})
    with pytest.raises(AssertionError):
        Int4Weight.from_codes(torch.zeros(4, 12, dtype=torch.uint8), torch.ones(4, 1), group_size=32)


# ---- refusals ---------------------------------------------------------------------------------------------------------
def test_router_refusals():
    l = torch.zeros(4, 64)
    for args, kw in (
        ((l[0], 2), {}), ((l.double(), 2), {}), ((l, 0), {}), ((l, 65), {}), ((l, 33), {}), ((torch.zeros(2, 1025), 2), {}), ((torch.zeros(2, 0), 1), {}),
        ((l, 2), dict(score_function="tanh")), ((l, 2), dict(num_groups=5)), ((l, 2), dict(num_groups=0)), ((l, 2), dict(num_groups=64)),
        ((l, 2), dict(num_groups=8, topk_groups=9)), ((l, 2), dict(num_groups=8, topk_groups=0)), ((l, 9), dict(num_groups=8, topk_groups=1)),
    ):
        for op in (topk_router, topk_routing_map):
            with pytest.raises(ValueError):
                op(*args, **kw)
    with pytest.raises(_lib.PtbError, match="CPU"):
        topk_router(l, 2)


def test_int4_refusals():
    x, w = torch.zeros(3, 256, dtype=BF), int4((16, 256))
    for bad in (lambda: quantize_int4(torch.zeros(8)), lambda: quantize_int4(torch.zeros(2, 8, dtype=torch.float64)), lambda: quantize_int4(torch.zeros(2, 12)),
                lambda: quantize_int4(torch.zeros(2, 64), group_size=16), lambda: dequantize_int4(w, torch.float8_e4m3fn),
                lambda: gemm_int4(x[:, :128], w), lambda: gemm_int4(x.float(), w), lambda: gemm_int4(x, int4((2, 16, 256))),
                lambda: gemm_int4(x, w, bias=torch.zeros(15, dtype=BF)), lambda: gemm_int4(x, w, bias=torch.zeros(16)),
                lambda: gemm_int4(x, w, bias=torch.zeros(32, dtype=BF)[::2]), lambda: gemm_int4(torch.zeros((), dtype=BF), w)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: gemm_int4(x, torch.zeros(16, 256, dtype=BF)), lambda: dequantize_int4(x)):
        with pytest.raises(TypeError):
            bad()
    for call in (lambda: quantize_int4(torch.zeros(2, 64, dtype=BF)), lambda: dequantize_int4(w), lambda: gemm_int4(x, w)):
        with pytest.raises(_lib.PtbError, match="CPU"):
            call()


def test_moe_refusals():
    E, H, I, T, k = 4, 64, 32, 3, 2
    w1, w2 = torch.zeros(E, 2 * I, H, dtype=BF), torch.zeros(E, H, I, dtype=BF)
    x, ids, p = torch.zeros(T, H, dtype=BF), torch.zeros(T, k, dtype=torch.int64), torch.zeros(T, k)
    many = torch.zeros(129, H, dtype=BF)
    for args in ((x[0], ids, p, w1, w2), (x.float(), ids, p, w1, w2), (x, ids.int(), p, w1, w2), (x, ids[:2], p[:2], w1, w2), (x, ids, p[:, :1], w1, w2),
                 (x, ids, p.double(), w1, w2), (x, ids[:, :0], p[:, :0], w1, w2), (x, ids, p, w1.half(), w2.half()), (x, ids, p, w1, w2[:3]),
                 (x, ids, p, w1[:, :60], w2), (x, ids, p, w1[..., :56], w2), (x, ids, p, w1[0], w2), (x, ids, p, int4((E, 2 * I, H)), w2),
                 (x, ids, p, int4((E, 2 * I, H), 64), int4((E, H, I), 32)), (many, ids.new_zeros(129, k), p.new_zeros(129, k), w1, w2),
                 (many[:64], ids.new_zeros(64, 17), p.new_zeros(64, 17), w1, w2), (x[:, :60], ids, p, w1[..., :60], w2[:, :60])):
        with pytest.raises(ValueError):
            moe_few_tokens(*args)
    with pytest.raises(_lib.PtbError, match="CPU"):
        moe_few_tokens(x, ids, p, w1, w2)


def test_calls_that_would_need_a_gradient_are_refused():
    import torch.autograd.forward_ad as fwAD

    w = int4((16, 64))
    x = torch.zeros(2, 64, dtype=BF, requires_grad=True)
    ids, p = torch.zeros(2, 1, dtype=torch.int64), torch.zeros(2, 1, requires_grad=True)
    w1, w2 = torch.zeros(1, 64, 64, dtype=BF), torch.zeros(1, 64, 32, dtype=BF)
    calls = (lambda: gemm_int4(x, w), lambda: gemm_int4(x.detach(), w, bias=torch.zeros(16, dtype=BF, requires_grad=True)), lambda: quantize_int4(x),
             lambda: moe_few_tokens(x, ids, p.detach(), w1, w2), lambda: moe_few_tokens(x.detach(), ids, p, w1, w2),
             lambda: moe_few_tokens(x.detach(), ids, p.detach(), w1, w2.clone().requires_grad_(True)))
    for call in calls:
        with pytest.raises(NotImplementedError, match="no backward"):
            call()
        with torch.no_grad(), pytest.raises(_lib.PtbError, match="CPU"):
            call()
    with fwAD.dual_level(), torch.no_grad():
        d = fwAD.make_dual(torch.zeros(2, 64, dtype=BF), torch.ones(2, 64, dtype=BF))
        with pytest.raises(NotImplementedError, match="forward mode"):
            gemm_int4(d, w)
        with pytest.raises((NotImplementedError, RuntimeError), match="(?i)jvp|forward mode|CPU"):
            topk_router(d, 2)


# ---- C ABI --------------------------------------------------------------------------------------------------------------
def test_argument_errors_are_codes():
    L, p = _lib.lib, 0x1000
    bf, f32 = _lib.PTB_BF16, _lib.PTB_F32
    router = lambda T=4, E=64, stride=64, k=2, score=0, groups=1, tg=1, dt=f32, ids=p, probs=p, table=None, m=None: L.ptb_topk_router(  # noqa: E731
        p, dt, T, E, stride, k, score, None, groups, tg, 0, 1.0, ids, probs, table, m, None)
    assert router(T=0) == 0 and router(T=-1) == -1 and router(E=0) == -1 and router(k=65) == -1 and router(k=0) == -1
    assert router(E=1025, stride=2000) == -5 and router(k=33) == -5 and router(stride=63) == -1 and router(score=2) == -1 and router(dt=_lib.PTB_E4M3) == -1
    assert router(groups=5) == -1 and router(groups=64, tg=64) == -1 and router(groups=8, tg=9) == -1 and router(groups=32, tg=1, k=3) == -1
    assert router(ids=None) == -1 and router(probs=None) == -1 and router(table=p) == -1 and router(table=p + 4, m=p) == -3
    bwd = lambda T=4, out=p, k=2: L.ptb_topk_router_bwd(p, f32, T, 64, 64, k, 0, 0, 1.0, p, p, 2, 0, out, None)  # noqa: E731
    assert bwd(T=0) == 0 and bwd(out=None) == -1 and bwd(out=p + 8) == -3 and bwd(k=40) == -5
    quant = lambda w=p, dt=bf, rows=4, K=128, g=64, codes=p: L.ptb_quant_int4(w, dt, rows, K, g, codes, p, None, None)  # noqa: E731
    assert quant(rows=0) == 0 and quant(rows=-1) == -1 and quant(dt=3) == -1 and quant(g=16) == -1 and quant(K=12) == -3 and quant(w=p + 2) == -3
    assert quant(codes=p + 4) == -3 and quant(w=None) == -1 and quant(K=1 << 25) == -5
    deq = lambda codes=p, K=128, g=64, out=p, dt=bf, rows=4: L.ptb_dequant_int4(codes, p, None, rows, K, g, out, dt, None)  # noqa: E731
    assert deq(rows=0) == 0 and deq(codes=None) == -1 and deq(K=4) == -3 and deq(g=0) == -1 and deq(out=p + 2) == -3 and deq(dt=4) == -1
    gemm = lambda x=p, dt=bf, ld=128, M=2, N=16, K=128, codes=p, g=64, ws=p: L.ptb_gemm_int4(x, dt, ld, M, N, K, codes, p, None, g, None, ws, p, None)  # noqa: E731
    assert gemm(M=0) == 0 and gemm(N=0) == 0 and gemm(K=0) == -1 and gemm(dt=f32) == -1 and gemm(ld=127) == -3 and gemm(ld=120) == -1 and gemm(K=12) == -3
    assert gemm(x=p + 2) == -3 and gemm(codes=p + 8) == -3 and gemm(g=256) == -1 and gemm(x=None) == -1 and gemm(M=1 << 21) == -5 and gemm(ws=None) == -1 and gemm(ws=p + 8) == -3
    need = L.ptb_gemm_int4_workspace
    assert need(bf, 2, 200, 64) >= 2 * 2 * 256 and need(_lib.PTB_F16, 1, 128, 128) >= 2 * 128 and need(f32, 1, 128, 64) == -1 and need(bf, 1, 128, 16) == -1


def test_moe_argument_errors_are_codes():
    L, p, bf = _lib.lib, 0x1000, _lib.PTB_BF16
    w = lambda data=p, scale=p, gran=0, group=0: ExpertWeightArg(data, scale, None, gran, group)  # noqa: E731

    def call(dt=bf, ld=64, T=2, H=64, I=32, E=4, k=2, fmt=bf, a=None, b=None, x=p, ws=p):
        a, b = a or w(), b or w()
        return L.ptb_moe_few_tokens(x, dt, ld, T, H, I, E, p, p, k, fmt, ctypes.addressof(a), ctypes.addressof(b), ws, p, None)

    assert call(T=0) == 0 and call(T=-1) == -1 and call(H=0) == -1 and call(k=0) == -1 and call(dt=0) == -1 and call(fmt=_lib.PTB_F16) == -1 and call(fmt=9) == -1
    assert call(T=129) == -5 and call(T=100, k=11) == -5 and call(E=1025) == -5 and call(H=60) == -3 and call(H=72, ld=72, fmt=3) == -3 and call(ld=56) == -3
    assert call(x=None) == -1 and call(x=p + 2) == -3 and call(ws=p + 8) == -3 and call(ws=None) == -1 and call(a=w(data=None)) == -1 and call(b=w(data=p + 4)) == -3
    assert call(fmt=3, a=w(scale=None)) == -1 and call(fmt=5) == -1 and call(fmt=5, a=w(group=32), b=w(group=64)) == -1
    need = L.ptb_moe_few_tokens_workspace
    assert need(bf, 2, 64, 32, 2, bf) >= 2 * 2 * 32 * 4 and need(bf, 16, 64, 32, 4, 3) >= 64 * (2 * 128 + 64 * 4) + 16 * 2 * 128
    assert need(bf, 129, 8, 8, 1, bf) == -1 and need(bf, 128, 8, 8, 9, bf) == -1 and need(bf, 0, 8, 8, 1, bf) >= 0


# ---- tracing ------------------------------------------------------------------------------------------------------------
def test_fake_shapes():
    with FakeTensorMode():
        l = torch.empty(5, 64, dtype=BF, device="cuda")
        ids, probs, table = C.topk_router(l, 3, 0, None, 1, 1, True, 1.0, False)
        assert ids.shape == probs.shape == (5, 3) and ids.dtype == torch.int64 and probs.dtype == torch.float32
        ids, probs, table = C.topk_router(l, 3, 0, None, 1, 1, True, 1.0, True)
        assert probs.shape == table.shape == (5, 64) and table.dtype == torch.bool
        assert C.topk_router_bwd(l, ids, probs, 0, True, 1.0, True).shape == (5, 64)
        q, s, z = C.quant_int4(torch.empty(3, 16, 200, dtype=BF, device="cuda"), 64, False)
        assert q.shape == (3, 16, 128) and s.shape == z.shape == (3, 16, 4)
        assert C.dequant_int4(q, s, z, 200, 64, BF).shape == (3, 16, 200)
        x = torch.empty(7, 200, dtype=BF, device="cuda")
        assert C.gemm_int4(x, q[0], s[0], z[0], 64, None).shape == (7, 16)
        w = torch.empty(4, 64, 200, dtype=BF, device="cuda")
        assert C.moe_few_tokens(x, ids, probs, w, None, None, w, None, None, 32, 0, 0).shape == (7, 200)
