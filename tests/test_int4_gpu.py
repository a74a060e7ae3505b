"""4-bit weights against a plain form in 64 bits: codes, scales and zero points equal, products to the accuracy of fp32 sums
and one rounding.  Every group size and row tail, row counts on both sides of the eights, strides, special values."""

import math

import pytest
import torch

from primus_turbo_b200.pytorch.core.int4_weight import Int4Weight
from primus_turbo_b200.pytorch.ops import dequantize_int4, gemm_int4, quantize_int4

pytestmark = pytest.mark.gpu
DEV = "cuda"


def spread(t, group, k):
    return t.repeat_interleave(group, dim=-1)[..., :k]


def reference_quant(w, group, symmetric):
    """(codes, scale, zero) of a finite weight, in 64 bits."""
    k = w.shape[-1]
    wide = torch.nn.functional.pad(w.double(), (0, -k % group)).unflatten(-1, (-1, group))
    lo, hi = wide.amin(-1).clamp(max=0), wide.amax(-1).clamp(min=0)
    scale = ((torch.maximum(hi, -lo) / 7) if symmetric else (hi - lo) / 15).to(torch.bfloat16)
    s = scale.double()
    zero = torch.full_like(s, 8) if symmetric else torch.where(s > 0, (-lo / s).round().clamp(0, 15), 0.0)
    steps = torch.where(s[..., None] > 0, wide / s[..., None], 0.0).round()
    codes = (steps + zero[..., None]).clamp(0, 15).flatten(-2)[..., :k].to(torch.uint8)
    return codes, scale, zero.to(torch.uint8)


@pytest.mark.parametrize("shape", [(1, 8), (3, 32), (5, 40), (7, 120), (4, 128), (9, 136), (17, 1000), (2, 3, 264), (33, 4096)])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_quantise(shape, group, symmetric, dtype):
    torch.manual_seed(shape[-1] + group)
    w = (torch.randn(shape, device=DEV) * torch.rand((*shape[:-1], 1), device=DEV)).to(dtype)
    q = quantize_int4(w, group_size=group, symmetric=symmetric)
    codes, scale, zero = reference_quant(w, group, symmetric)
    assert torch.equal(q.scale, scale)
    if symmetric:
        assert q.zero is None
    else:
        assert torch.equal(q.zero, zero)
    assert torch.equal(q.codes(), codes)
    # the stored form is the one that from_codes makes, padding included
    assert torch.equal(Int4Weight.from_codes(codes, scale, q.zero, group_size=group).qdata, q.qdata)
    for out in (torch.float32, dtype):
        z = spread(zero, group, shape[-1]).double()
        want = ((codes.double() - z) * spread(scale, group, shape[-1]).double()).to(out)
        assert torch.equal(dequantize_int4(q, out), want)


def test_quantise_fp32_is_within_half_a_step():
    torch.manual_seed(0)
    w = torch.randn(64, 520, device=DEV)
    for symmetric in (True, False):
        q = quantize_int4(w, group_size=64, symmetric=symmetric)
        s = spread(q.scale, 64, 520).double()
        # half a step, and what the clamp takes where the scale's rounding (2^-8 of 7 or 15 steps) or the zero point's (half a step) cut the range
        assert bool(((dequantize_int4(q, torch.float32).double() - w.double()).abs() <= s * (0.5 + (0.03 if symmetric else 0.56))).all())


@pytest.mark.parametrize("symmetric", [True, False])
def test_quantise_special_values(symmetric):
    w = torch.zeros(6, 128, device=DEV, dtype=torch.bfloat16)
    w[1, 5] = math.nan
    w[2, 40] = math.inf
    w[3, 70] = -math.inf
    w[4, :] = 1e-38  # the scale of its groups is subnormal
    w[5, 0], w[5, 1] = torch.finfo(torch.bfloat16).max / 2, torch.finfo(torch.bfloat16).min / 2
    q = quantize_int4(w, group_size=32, symmetric=symmetric)
    v = dequantize_int4(q, torch.float32)
    assert not v[0].any() and not v[1, 32:].any() and bool(v[1, :32].isnan().all())
    assert bool(v[2, 32:64].isnan().all()) and not v[2, :32].any() and bool(v[3, 64:96].isnan().all())
    assert bool(((v[4] - 1e-38).abs() < 1e-39).all())
    assert bool(v[5].isfinite().all()) and v[5, 0] > 1.5e38 and v[5, 1] < -1.5e38
    assert bool((q.codes()[0] == (8 if symmetric else 0)).all())


def test_ties_go_to_the_even_code():
    w = torch.tensor([[7.0, 0.5, 1.5, 2.5, -0.5, -1.5, -2.5, 3.5]], device=DEV, dtype=torch.bfloat16)
    q = quantize_int4(w, group_size=32)
    assert q.scale.item() == 1.0 and q.codes().tolist() == [[15, 8, 10, 10, 8, 6, 6, 12]]


def weight(shape, group, zeros, seed=0):
    g = torch.Generator(DEV).manual_seed(seed)
    k = shape[-1]
    groups = (*shape[:-1], -(-k // group))
    codes = torch.randint(0, 16, shape, generator=g, device=DEV, dtype=torch.uint8)
    scale = (torch.rand(groups, generator=g, device=DEV) + 0.5).to(torch.bfloat16) * k**-0.5
    zero = torch.randint(0, 16, groups, generator=g, device=DEV, dtype=torch.uint8) if zeros else None
    return Int4Weight.from_codes(codes, scale, zero, group_size=group)


def values(q):
    k = q.shape[-1]
    z = 8.0 if q.zero is None else spread(q.zero, q.group_size, k).double()
    return (q.codes().double() - z) * spread(q.scale, q.group_size, k).double()


def assert_product(y, x, q, bias=None):
    w, xd = values(q), x.double()
    want, size = xd @ w.T, xd.abs() @ w.abs().T
    if bias is not None:
        want, size = want + bias.double(), size + bias.double().abs()
    # a product passes through the sums of a group (8), of the blocks of a warp (K / 1024 + 1), of the warps and halves (20) and the bias, each
    # within 2^-23 (the MMA may cut where it does not round) of a partial sum; then one rounding to the output
    k = x.shape[-1]
    s = spread(q.scale, q.group_size, k).double()
    # a group's sum is that of bare codes, up to 15, from which zero (up to 15) times the sum of x is taken: 12 operations on sums of that size
    size = size + xd.abs() @ s.T * (30 * 12 / (k / 1024 + 31))
    # x is a 16-bit integer in units of at most 2^-14 of the largest of its 128: off by up to half of one
    size = size + xd.abs().amax(1, keepdim=True) * w.abs().sum(1) * (2.0**8 / (k / 1024 + 31))
    tol = size * (k / 1024 + 31) * 2.0**-23 + want.abs() * torch.finfo(y.dtype).eps / 2 + torch.finfo(y.dtype).smallest_normal * torch.finfo(y.dtype).eps
    assert bool(((y.double() - want).abs() <= tol).all()), ((y.double() - want).abs() / tol).max()


@pytest.mark.parametrize("m", [1, 2, 7, 8, 9, 16, 17, 31, 32, 33, 64, 65, 100, 130])
@pytest.mark.parametrize("n,k", [(1, 8), (16, 128), (37, 520), (300, 1152), (129, 2880)])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_product(m, n, k, group):
    dtype = torch.float16 if (m + n) % 2 else torch.bfloat16
    q = weight((n, k), group, zeros=(m % 3 == 0), seed=m)
    x = torch.randn(m, k, device=DEV).to(dtype)
    bias = torch.randn(n, device=DEV).to(dtype) if m % 2 else None
    assert_product(gemm_int4(x, q, bias), x, q, bias)


@pytest.mark.parametrize("m,n,k", [(1, 4096, 14336), (5, 14336, 4096), (64, 8192, 8192), (24, 5760, 2880), (48, 1000, 14328)])
def test_product_of_large_weights(m, n, k):
    q = weight((n, k), 128, zeros=True, seed=k)
    x = torch.randn(m, k, device=DEV, dtype=torch.bfloat16)
    assert_product(gemm_int4(x, q), x, q)


def test_product_shapes_and_strides():
    q = weight((48, 264), 64, True)
    base = torch.randn(40, 400, device=DEV, dtype=torch.bfloat16)
    for x in (base[:9, :264], base[:9, 8:272], base[:9, 1:265], base[::3, :264], torch.randn(264, 9, device=DEV, dtype=torch.bfloat16).t(),
              base[:1, :264].expand(5, 264), torch.randn(2, 3, 264, device=DEV, dtype=torch.bfloat16), base[0, :264], base[:0, :264]):
        y = gemm_int4(x, q)
        assert y.shape == (*x.shape[:-1], 48) and y.is_contiguous()
        assert_product(y.reshape(-1, 48), x.reshape(-1, 264), q)
    # codes that start in the middle of a 16-byte piece
    raw = torch.empty(q.qdata.numel() + 4, dtype=torch.uint8, device=DEV)
    part = raw[4:].view(q.qdata.shape)
    part.copy_(q.qdata)
    q2 = Int4Weight(part, q.scale, q.zero, q.shape, q.group_size)
    assert torch.equal(gemm_int4(base[:9, :264], q2), gemm_int4(base[:9, :264], q))
    assert torch.equal(dequantize_int4(q2), dequantize_int4(q))


def test_product_special_values():
    """A NaN or an infinity stays in its row of x and its row of the weight."""
    q = weight((40, 256), 64, True)
    x = torch.randn(11, 256, device=DEV, dtype=torch.bfloat16)
    want = gemm_int4(x, q)
    x2 = x.clone()
    x2[3, 100] = math.nan
    x2[10, 7] = math.inf
    y = gemm_int4(x2, q)
    assert bool(y[3].isnan().all()) and not bool(y[10].isfinite().any())
    keep = [i for i in range(11) if i not in (3, 10)]
    assert torch.equal(y[keep], want[keep])
    scale = q.scale.clone()
    scale[5, 1] = math.nan
    y = gemm_int4(x, Int4Weight(q.qdata, scale, q.zero, q.shape, 64))
    assert bool(y[:, 5].isnan().all()) and torch.equal(y[:, [i for i in range(40) if i != 5]], want[:, [i for i in range(40) if i != 5]])


def test_product_is_repeatable_and_captured():
    q = weight((2048, 4096), 128, False)
    x = torch.randn(8, 4096, device=DEV, dtype=torch.bfloat16)
    y = gemm_int4(x, q)
    assert torch.equal(y, gemm_int4(x, q))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        z = gemm_int4(x, q)
        d = dequantize_int4(q)
        r = quantize_int4(d)
    x.copy_(torch.randn_like(x))
    graph.replay()
    assert torch.equal(z, gemm_int4(x, q)) and torch.equal(d, dequantize_int4(q)) and torch.equal(r.qdata, quantize_int4(d).qdata)


def test_a_weight_is_ready_for_the_product_that_follows():
    """Quantise and multiply in a row, without a wait between: the product reads what the quantiser wrote."""
    x = torch.randn(4, 512, device=DEV, dtype=torch.bfloat16)
    for seed in range(20):
        w = torch.randn(256, 512, device=DEV, dtype=torch.bfloat16, generator=torch.Generator(DEV).manual_seed(seed))
        y = gemm_int4(x, quantize_int4(w, 64))
        q = quantize_int4(w, 64)
        torch.cuda.synchronize()
        assert torch.equal(y, gemm_int4(x, q))


def test_offsets_past_32_bits():
    n, k = 70000, 65536  # 2.3 GB of codes, 4.6 G values
    q = quantize_int4(torch.zeros(1, k, device=DEV, dtype=torch.bfloat16), 128)
    codes = q.qdata.repeat(n, 1)
    scale = torch.full((n, k // 128), 1.0, device=DEV, dtype=torch.bfloat16)
    last = torch.full((1, k), 8, device=DEV, dtype=torch.uint8)
    last[0, 2] = 9  # one
    codes[-1:] = Int4Weight.from_codes(last, scale[:1], group_size=128).qdata
    big = Int4Weight(codes, scale, None, torch.Size((n, k)), 128)
    x = torch.zeros(1, k, device=DEV, dtype=torch.bfloat16)
    x[0, 2] = 3.0
    y = gemm_int4(x, big)
    assert y[0, -1] == 3.0 and not y[0, :-1].any()
    v = dequantize_int4(big)
    assert v[-1, 2] == 1.0 and v[-1].sum() == 1.0
    again = quantize_int4(v, 128)
    assert torch.equal(again.codes()[-1, :4].cpu(), torch.tensor([8, 8, 15, 8], dtype=torch.uint8)) and bool((again.qdata[:-1] == q.qdata).all())


@pytest.mark.parametrize("m", [13, 24, 64])
def test_a_batch_is_repeatable_and_captured(m):
    """Rows of x that share k among the CTAs of a cluster."""
    q = weight((520, 6152), 32, True)
    x = torch.randn(m, 6152, device=DEV, dtype=torch.float16)
    y = gemm_int4(x, q)
    assert_product(y, x, q)
    assert all(torch.equal(y, gemm_int4(x, q)) for _ in range(5))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        z = gemm_int4(x, q)
    x.copy_(torch.randn_like(x))
    graph.replay()
    with torch.cuda.stream(torch.cuda.Stream()):
        y = gemm_int4(x, q)
        torch.cuda.synchronize()
    assert torch.equal(z, y)


def test_scales_that_start_anywhere():
    """Groups whose scales and zero points lie at odd places of their memory."""
    for group in (32, 64):
        q = weight((64, 1024), group, True)
        x = torch.randn(20, 1024, device=DEV, dtype=torch.bfloat16)
        s, z = torch.empty(q.scale.numel() + 1, device=DEV, dtype=torch.bfloat16), torch.empty(q.zero.numel() + 1, device=DEV, dtype=torch.uint8)
        s[1:].copy_(q.scale.flatten())
        z[1:].copy_(q.zero.flatten())
        other = Int4Weight(q.qdata, s[1:].view(q.scale.shape), z[1:].view(q.zero.shape), q.shape, group)
        for rows in (1, 20):
            assert torch.equal(gemm_int4(x[:rows], other), gemm_int4(x[:rows], q))


@pytest.mark.parametrize("m", [1, 8, 9, 40])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_zero_points_of_any_byte(m, group, dtype):
    q = weight((72, 520), group, True)
    zero = (torch.arange(q.zero.numel(), device=DEV) * 37 % 256).to(torch.uint8).view(q.zero.shape)
    q = Int4Weight(q.qdata, q.scale, zero, q.shape, group)
    w = values(q)
    for t in (torch.bfloat16, torch.float16, torch.float32):
        v = dequantize_int4(q, t).double()
        assert bool(((v - w).abs() <= w.abs() * torch.finfo(t).eps / 2).all())  # values below 2^-14 do not occur: scales are 2^-6 and more
    x = torch.randn(m, 520, device=DEV).to(dtype)
    xd, s = x.double(), spread(q.scale, group, 520).double()
    want = xd @ w.T
    # as in assert_product, with zero points up to 255 in the place of 15: sums of codes and zero times the sum of x, up to 270 steps together
    size = (xd.abs() @ w.abs().T) * (520 / 1024 + 31) + xd.abs() @ s.T * (270 * 12)
    tol = size * 2.0**-23 + xd.abs().amax(1, keepdim=True) * w.abs().sum(1) * 2.0**-15 + want.abs() * torch.finfo(dtype).eps / 2
    y = gemm_int4(x, q).double()
    assert bool(((y - want).abs() <= tol).all()), ((y - want).abs() / tol).max()
