"""``moe_few_tokens`` against a plain form in 64 bits, for each way of keeping the weights: token counts around the eights, widths that
end inside a block, experts without tokens, tokens without experts, the same expert twice, strides, special values; and the layer
as it is used, behind the router and from weights quantised by the framework."""

import math

import pytest
import torch

from primus_turbo_b200.pytorch.core.int4_weight import Int4Weight
from primus_turbo_b200.pytorch.core.low_precision import Float8QuantConfig, Format, ScalingGranularity as G
from primus_turbo_b200.pytorch.core.quantized_tensor import create_quantized_weight
from primus_turbo_b200.pytorch.ops import grouped_gemm_fp8, quantize_int4
from primus_turbo_b200.pytorch.ops.activation import swiglu_with_probs
from primus_turbo_b200.pytorch.ops.moe import moe_few_tokens, token_permute, token_unpermute, topk_router, topk_routing_map

pytestmark = pytest.mark.gpu
DEV = "cuda"
FORMATS = ["raw", "tensor", "row", "block", "e5m2", "int4_32", "int4_64", "int4_128", "int4_zeros"]


def kept(w, fmt):
    """(weight as it is kept, its values in 64 bits)"""
    if fmt == "raw":
        return w, w.double()
    if fmt.startswith("int4"):
        q = quantize_int4(w, int(fmt[5:]) if fmt != "int4_zeros" else 64, symmetric=fmt != "int4_zeros")
        k = w.shape[-1]
        z = 8.0 if q.zero is None else q.zero.double().repeat_interleave(q.group_size, -1)[..., :k]
        s = q.scale.double().repeat_interleave(q.group_size, -1)[..., :k]
        v = (q.codes().double() - z) * s
        v.steps = s
        return q, v
    gran = {"tensor": G.TENSORWISE, "row": G.ROWWISE, "block": G.BLOCKWISE, "e5m2": G.BLOCKWISE}[fmt]
    cfg = Float8QuantConfig(granularity=gran, block_size=128 if gran == G.BLOCKWISE else None)
    q, _ = create_quantized_weight(w, torch.float8_e5m2 if fmt == "e5m2" else torch.float8_e4m3fn, cfg)
    s = q.scale_inv.double()
    if gran == G.BLOCKWISE:
        s = s.repeat_interleave(128, 1)[:, : w.shape[1]].repeat_interleave(128, 2)[:, :, : w.shape[2]]
    v = q.qdata.double() * s
    v.steps = None
    return q, v


def layer(E, H, I, fmt, dtype=torch.bfloat16, seed=0):
    g = torch.Generator(DEV).manual_seed(seed)
    w1 = (torch.randn(E, 2 * I, H, generator=g, device=DEV) * H**-0.5).to(dtype)
    w2 = (torch.randn(E, H, I, generator=g, device=DEV) * I**-0.5).to(dtype)
    return kept(w1, fmt), kept(w2, fmt)


def detour(v, e, x):
    """What 4-bit weights add: x is a 16-bit integer in units of at most 2^-14 of the largest of its block, off by up to half of one; bare
    codes, up to 15, are added up, and zero (up to 15) times the sum of x is taken off: at most 24 operations on sums of that size.  With
    FP8 weights x is fp16, which holds values below 2^-27 of the largest less exactly."""
    if not hasattr(v, "steps"):
        return 0.0
    if v.steps is None:
        return v[e].abs().sum(1) * x.abs().max() * 2.0**-37
    return v.steps[e] @ x.abs() * (30 * 24 * 2.0**-23) + v[e].abs().sum(1) * x.abs().max() * 2.0**-15


def reference(x, ids, probs, v1, v2):
    """(y, bound of the error) in 64 bits."""
    T, H = x.shape
    E, _, I = v2.shape
    y = torch.zeros(T, H, dtype=torch.float64, device=DEV)
    err = torch.zeros_like(y)
    add = 2.0**-23  # an addition, where the MMA may cut instead of rounding
    for t in range(T):
        for j, e in enumerate(ids[t].tolist()):
            if not 0 <= e < E:
                continue
            xd, p = x[t].double(), probs[t, j].double()
            u, size = v1[e] @ xd, v1[e].abs() @ xd.abs()
            du = size * (H / 1024 + 30) * add + detour(v1, e, xd)  # a term passes through the sums of a scale, of a warp's blocks and of the warps
            a, b = u[:I], u[I:]
            s = torch.sigmoid(a)
            h = a * s * b
            # silu's slope is at most 1.1; expf, the division and the products within 8 roundings; two bf16 parts leave 2^-17,
            # one fp16 (FP8 weights) 2^-11; what integers (4-bit weights) leave is in detour
            dh = 1.1 * du[:I] * (b.abs() + du[I:]) + (a * s).abs() * du[I:] + h.abs() * ((2.0**-11 if hasattr(v1, "steps") else 2.0**-17) + 8 * add)
            y[t] += p * (v2[e] @ h)
            # the second product: two MMAs an octet, at worst all of an expert's blocks in one warp, 16 warps, the experts of a token
            err[t] += p.abs() * (v2[e].abs() @ (dh + h.abs() * (I / 8 + 60) * add) + detour(v2, e, h))
    return y, err + y.abs() * torch.finfo(x.dtype).eps / 2 + torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps


def assert_layer(x, ids, probs, w1, w2):
    y = moe_few_tokens(x, ids, probs, w1[0], w2[0])
    want, bound = reference(x, ids, probs, w1[1], w2[1])
    assert y.shape == x.shape and y.dtype == x.dtype and y.is_contiguous()
    assert bool(((y.double() - want).abs() <= bound).all()), ((y.double() - want).abs() / bound).max()
    return y


def routed(T, E, k, seed=0):
    g = torch.Generator(DEV).manual_seed(seed)
    ids = torch.rand(T, E, generator=g, device=DEV).argsort(1)[:, :k].contiguous()
    return ids, torch.rand(T, k, generator=g, device=DEV) + 0.1


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,E,k,H,I", [(1, 8, 2, 256, 128), (1, 4, 4, 528, 144), (3, 16, 8, 384, 400), (8, 2, 1, 272, 272), (9, 3, 2, 640, 96),
                                       (17, 5, 3, 144, 32), (40, 4, 2, 288, 528), (100, 3, 2, 160, 160)])
def test_layer(fmt, dtype, T, E, k, H, I):
    w1, w2 = layer(E, H, I, fmt, dtype, seed=T)
    ids, probs = routed(T, E, k, seed=T)
    assert_layer(torch.randn(T, H, device=DEV).to(dtype), ids, probs, w1, w2)


@pytest.mark.parametrize("fmt", ["raw", "int4_32", "int4_zeros"])
@pytest.mark.parametrize("H,I", [(8, 8), (8, 136), (136, 8), (264, 1000), (1000, 264)])
def test_widths_of_eights(fmt, H, I):
    w1, w2 = layer(3, H, I, fmt)
    ids, probs = routed(5, 3, 2)
    assert_layer(torch.randn(5, H, device=DEV, dtype=torch.bfloat16), ids, probs, w1, w2)


@pytest.mark.parametrize("fmt", ["block", "int4_128", "raw"])
def test_a_model_sized_layer(fmt):
    w1, w2 = layer(16, 2048, 768, fmt)
    for T in (1, 2, 24):
        ids, probs = routed(T, 16, 8, seed=T)
        assert_layer(torch.randn(T, 2048, device=DEV, dtype=torch.bfloat16), ids, probs, w1, w2)


@pytest.mark.parametrize("fmt", ["raw", "block", "int4_64"])
def test_unused_places(fmt):
    """Padding, ids that name no expert, an expert named twice, one expert for all, none at all."""
    w1, w2 = layer(6, 256, 128, fmt)
    x = torch.randn(12, 256, device=DEV, dtype=torch.bfloat16)
    ids, probs = routed(12, 6, 3)
    ids[0] = -1
    ids[1, 1] = 6
    ids[2, 0] = 2**40
    ids[3, 2] = -(2**40)
    ids[4] = torch.tensor([5, 5, 5], device=DEV)
    ids[5] = torch.tensor([1, 2, 1], device=DEV)
    probs[6] = 0.0
    probs[7] = -probs[7]
    y = assert_layer(x, ids, probs, w1, w2)
    assert not y[0].any() and not y[6].any()
    probs[0] = math.nan  # belongs to nobody
    assert torch.equal(moe_few_tokens(x, ids, probs, w1[0], w2[0]), y)
    assert_layer(x, torch.full_like(ids, 3), probs.nan_to_num(1.0), w1, w2)
    assert not moe_few_tokens(x, torch.full_like(ids, -1), probs, w1[0], w2[0]).any()
    assert moe_few_tokens(x[:0], ids[:0], probs[:0], w1[0], w2[0]).shape == (0, 256)


def test_the_most_tokens_and_experts():
    w1, w2 = layer(1024, 64, 32, "raw")
    for T, k in ((128, 8), (32, 32), (128, 1)):
        ids, probs = routed(T, 1024, k, seed=k)
        assert_layer(torch.randn(T, 64, device=DEV, dtype=torch.bfloat16), ids, probs, w1, w2)
    w1, w2 = layer(1, 64, 32, "int4_32")
    ids, probs = routed(128, 1, 1)
    assert_layer(torch.randn(128, 64, device=DEV, dtype=torch.bfloat16), ids, probs, w1, w2)


def test_strides():
    w1, w2 = layer(4, 256, 128, "block")
    base = torch.randn(30, 600, device=DEV, dtype=torch.bfloat16)
    ids, probs = routed(10, 4, 2)
    wide_ids, wide_probs = ids.repeat(1, 2)[:, ::1], probs.repeat(1, 2)
    for x in (base[:10, :256], base[:10, 8:264], base[:10, 3:259], base[::3, :256], torch.randn(256, 10, device=DEV, dtype=torch.bfloat16).t(),
              base[:1, :256].expand(10, 256)):
        y = assert_layer(x, ids, probs, w1, w2)
        assert torch.equal(y, moe_few_tokens(x, wide_ids[:, :2], wide_probs[:, :2], w1[0], w2[0]))
        assert_layer(x, ids, probs.to(torch.bfloat16), w1, w2)


@pytest.mark.parametrize("fmt", ["raw", "block", "int4_64"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_special_values_stay_with_their_token(fmt, dtype):
    w1, w2 = layer(4, 256, 128, fmt, dtype)
    x = torch.randn(11, 256, device=DEV).to(dtype)
    ids, probs = routed(11, 4, 2)
    y = moe_few_tokens(x, ids, probs, w1[0], w2[0])
    x[2, 9] = math.nan
    x[9, 200] = math.inf
    z = moe_few_tokens(x, ids, probs, w1[0], w2[0])
    assert bool(z[2].isnan().all()) and not bool(z[9].isfinite().any())
    keep = [i for i in range(11) if i not in (2, 9)]
    assert torch.equal(z[keep], y[keep])


def test_an_fp8_nan_shows():
    w1, w2 = layer(4, 256, 128, "block")
    x = torch.randn(6, 256, device=DEV, dtype=torch.bfloat16)
    ids, probs = routed(6, 4, 2)
    w2[0].qdata.view(torch.uint8)[1, 77, 5] = 0x7F
    y = moe_few_tokens(x, ids, probs, w1[0], w2[0])
    hit = (ids == 1).any(1)
    assert bool(y[hit, 77].isnan().all()) and not y[~hit].isnan().any() and not y[:, :77].isnan().any()


def test_repeatable_captured_and_side_by_side():
    """Equal bits every time; two captured graphs replayed at once on two streams do not disturb each other."""
    w1, w2 = layer(32, 1024, 512, "int4_128")
    xs = [torch.randn(16, 1024, device=DEV, dtype=torch.bfloat16) for _ in range(2)]
    ids, probs = routed(16, 32, 4)
    want = [moe_few_tokens(x, ids, probs, w1[0], w2[0]) for x in xs]
    graphs, outs = [], []
    for x in xs:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(moe_few_tokens(x, ids, probs, w1[0], w2[0]))
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, gr in zip(streams, graphs):
            with torch.cuda.stream(s):
                gr.replay()
    torch.cuda.synchronize()
    for y, w in zip(outs, want):
        assert torch.equal(y, w)
    # other routing through the same graph
    ids2, probs2 = routed(16, 32, 4, seed=9)
    ids2[3] = -1
    ids.copy_(ids2)
    probs.copy_(probs2)
    graphs[0].replay()
    assert torch.equal(outs[0], moe_few_tokens(xs[0], ids2, probs2, w1[0], w2[0]))


def test_large_offsets():
    """An expert whose weights lie past 2^32 bytes."""
    E, H, I = 104, 7168, 2048
    one = torch.zeros(1, 2 * I, H, device=DEV, dtype=torch.bfloat16)
    w1 = torch.zeros(E, 2 * I, H, device=DEV, dtype=torch.bfloat16)
    w2 = torch.zeros(E, H, I, device=DEV, dtype=torch.bfloat16)
    w1[-1, 5, 7], w1[-1, I + 5, 7], w2[-1, H - 1, 5] = 1.0, 2.0, 3.0
    x = torch.zeros(1, H, device=DEV, dtype=torch.bfloat16)
    x[0, 7] = 1.0
    ids, probs = torch.tensor([[E - 1, 0]], device=DEV), torch.tensor([[0.5, 0.5]], device=DEV)
    want = torch.sigmoid(torch.tensor(1.0, dtype=torch.float64)) * 3.0
    del one
    y = moe_few_tokens(x, ids, probs, w1, w2)
    assert abs(y[0, -1].item() - want.item()) <= want.item() * 2.0**-8 and not y[0, :-1].any()


@pytest.mark.parametrize("fmt", ["block", "int4_64"])
def test_router_and_layer_together(fmt):
    """A decoding step as it is run: router, then the layer, on one stream without a wait; against the same steps in 64 bits."""
    E, H, I, k, T = 16, 512, 256, 4, 6
    w1, w2 = layer(E, H, I, fmt)
    wr = torch.randn(E, H, device=DEV, dtype=torch.bfloat16) * H**-0.5
    for step in range(10):
        x = torch.randn(T, H, device=DEV, dtype=torch.bfloat16, generator=torch.Generator(DEV).manual_seed(step))
        logits = x @ wr.T
        logits[step % T, : E - 2] = -math.inf  # two experts left for one token
        probs, ids = topk_router(logits, k, normalize=True)
        y = moe_few_tokens(x, ids, probs, w1[0], w2[0])
        want, bound = reference(x, ids, probs, w1[1], w2[1])
        assert int((ids[step % T] < 0).sum()) == k - 2
        assert bool(((y.double() - want).abs() <= bound).all())


def test_the_same_layer_as_in_training():
    """The few-token layer and the training path (permute, FP8 grouped GEMMs, SwiGLU, unpermute) on the same FP8 weights: they differ
    by the activations that training quantises to FP8 in both products (2^-4 a value at worst, a few per cent of a row's norm)."""
    E, H, I, k, T = 8, 512, 256, 2, 32
    cfg = Float8QuantConfig(format=Format.E4M3, granularity=G.BLOCKWISE, block_size=128)
    (w1, _), (w2, _) = layer(E, H, I, "block")
    x = torch.randn(T, H, device=DEV, dtype=torch.bfloat16)
    logits = torch.randn(T, E, device=DEV)
    probs, ids = topk_router(logits, k, normalize=True)
    table, routing = topk_routing_map(logits, k, normalize=True)
    rows, p, idx, lens = token_permute(x, T * k, probs=table, routing_map=routing)
    h = swiglu_with_probs(grouped_gemm_fp8(rows, w1, lens, trans_b=True, config=cfg), p)
    want = token_unpermute(grouped_gemm_fp8(h, w2, lens, trans_b=True, config=cfg), idx, restore_shape=x.shape, routing_map=routing)
    y = moe_few_tokens(x, ids, probs, w1, w2)
    off = (y.double() - want.double()).norm(dim=1) / want.double().norm(dim=1)
    assert bool((off < 2 * 2.0**-4).all())


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_an_expert_with_most_of_the_tokens(fmt, dtype):
    """Fewer columns a pass than an expert has tokens, where the others have few."""
    w1, w2 = layer(8, 272, 144, fmt, dtype)
    ids = torch.full((60, 1), 3, device=DEV)
    ids[::7] = 5
    assert_layer(torch.randn(60, 272, device=DEV).to(dtype), ids, torch.rand(60, 1, device=DEV) + 0.1, w1, w2)


@pytest.mark.parametrize("fmt", ["raw", "block", "int4_32"])
def test_batches_in_two_graphs_and_between_them(fmt):
    w1, w2 = layer(6, 512, 256, fmt)
    ids, probs = routed(40, 6, 2)
    xs = [torch.randn(40, 512, device=DEV, dtype=torch.bfloat16) for _ in range(3)]
    want = [moe_few_tokens(x, ids, probs, w1[0], w2[0]) for x in xs]
    held, outs, graphs = [x.clone() for x in xs[:2]], [], []
    for x in held:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(moe_few_tokens(x, ids, probs, w1[0], w2[0]))
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(5):
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        with torch.cuda.stream(streams[2]):
            y = moe_few_tokens(xs[2], ids, probs, w1[0], w2[0])
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1]) and torch.equal(y, want[2])


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("T,E,k,H,I", [(9, 2, 1, 1168, 656), (12, 4, 2, 2000, 1040), (40, 2, 2, 4112, 528)])
def test_few_experts_share_k(fmt, T, E, k, H, I):
    """So few experts that the CTAs of a cluster share k, in parts that end inside a run of blocks."""
    dtype = torch.float16 if T == 12 else torch.bfloat16
    w1, w2 = layer(E, H, I, fmt, dtype, seed=T)
    ids, probs = routed(T, E, k, seed=T)
    x = torch.randn(T, H, device=DEV).to(dtype)
    y = assert_layer(x, ids, probs, w1, w2)
    assert torch.equal(y, moe_few_tokens(x, ids, probs, w1[0], w2[0]))
