"""Top-k routing against a plain form in 64 bits: choices equal, probabilities and gradients to fp32 accuracy.  Widths around the
lane's share of experts, ties, masked experts, groups, biases, strides."""

import math

import pytest
import torch

from primus_turbo_b200.pytorch.ops.moe import token_permute, token_unpermute, topk_router, topk_routing_map

pytestmark = pytest.mark.gpu
DEV = "cuda"


def reference(l, k, score="softmax", bias=None, groups=1, topk_groups=1, normalize=False, scaling=1.0):
    """(probs [T, k], ids) in 64 bits; l [T, E] double, may require grad."""
    T, E = l.shape
    gone = l.detach() == -math.inf
    s = torch.softmax(l, 1) if score == "softmax" else torch.sigmoid(l)
    c = s.detach() if bias is not None or groups > topk_groups else l.detach()
    if bias is not None:
        c = c + bias.double()
    c = c.masked_fill(gone, -math.inf)
    if groups > topk_groups:
        two = c.view(T, groups, -1).sort(dim=2, descending=True).values[:, :, :2]
        second = two[:, :, 1] if two.shape[2] > 1 else torch.zeros_like(two[:, :, 0])
        best = two[:, :, 0] + torch.where(second == -math.inf, 0.0, second)
        kept = best.sort(dim=1, descending=True, stable=True).indices[:, :topk_groups]
        keep = torch.zeros(T, groups, dtype=torch.bool, device=l.device).scatter_(1, kept, True) & (best > -math.inf)
        c = c.masked_fill(~keep.repeat_interleave(E // groups, 1), -math.inf)
    top = c.sort(dim=1, descending=True, stable=True)
    ids, there = top.indices[:, :k], top.values[:, :k] > -math.inf
    p = torch.where(there, s.gather(1, ids), 0.0)
    if normalize:
        p = torch.softmax(l.gather(1, ids).masked_fill(~there, -math.inf), 1) if score == "softmax" else p / (p.sum(1, keepdim=True) + 1e-20)
        p = torch.where(there, p, 0.0)
    return p * scaling, torch.where(there, ids, -1)


def check(l, k, **kw):
    opts = dict(score_function=kw.get("score", "softmax"), expert_bias=kw.get("bias"), num_groups=kw.get("groups", 1),
                topk_groups=kw.get("topk_groups", 1), normalize=kw.get("normalize", False), scaling_factor=kw.get("scaling", 1.0))
    leaf = l.detach().requires_grad_(True)
    probs, ids = topk_router(leaf, k, **opts)
    ld = l.detach().double().requires_grad_(True)
    want, want_ids = reference(ld, k, **kw)
    assert torch.equal(ids, want_ids)
    # exp, a sum over at most 1024 scores by halves, two divisions and a product: within 16 roundings of 2^-24, and exp's own 2 ulp
    # on an argument rounded to 2^-24 of up to |l - max| <= 64
    tol = 2.0**-18
    torch.testing.assert_close(probs.double(), want, rtol=tol, atol=1e-30)
    g = torch.randn(probs.shape, device=DEV, generator=torch.Generator(DEV).manual_seed(5))
    (dl,) = torch.autograd.grad(probs, leaf, g)
    (wd,) = torch.autograd.grad(want, ld, g.double())
    wd = torch.where((l == -math.inf).all(1, keepdim=True), 0.0, wd)  # a row of nothing: 0 / 0 in the plain form
    size = (g.abs() * want.detach().abs()).sum(1, keepdim=True) + wd.abs()  # what the differences are taken between
    half = torch.finfo(l.dtype).eps / 2
    assert bool(((dl.double() - wd).abs() <= wd.abs() * half + size * tol + torch.finfo(l.dtype).smallest_normal * torch.finfo(l.dtype).eps).all())
    # the tables are the same numbers
    leaf2 = l.detach().requires_grad_(True)
    table, chosen = topk_routing_map(leaf2, k, **opts)
    there = ids >= 0
    assert torch.equal(table.gather(1, ids.clamp(min=0))[there], probs.detach()[there])
    assert torch.equal(chosen.sum(1), there.sum(1)) and bool(chosen.gather(1, ids.clamp(min=0))[there].all())
    assert not table[~chosen].any()
    dense = torch.full_like(table, 7.0).scatter_(1, ids.clamp(min=0), g)  # what lies elsewhere is not read
    dense = torch.where(chosen, torch.zeros_like(table).scatter_add_(1, ids.clamp(min=0), torch.where(there, g, 0.0)), dense)
    (dl2,) = torch.autograd.grad(table, leaf2, dense)
    assert torch.equal(dl2, dl)
    return probs, ids


@pytest.mark.parametrize("E", [1, 2, 7, 31, 32, 33, 64, 96, 100, 128, 160, 256, 257, 384, 512, 1000, 1024])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("normalize", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_widths(E, score, normalize, dtype):
    torch.manual_seed(E)
    l = (torch.randn(37, E, device=DEV) * 2).to(dtype)
    for k in sorted({1, min(2, E), min(8, E), min(32, E)}):
        if normalize and k == 1:
            continue  # one normalised probability is constant: its gradient is rounding
        check(l, k, score=score, normalize=normalize, scaling=2.5)


@pytest.mark.parametrize("E,groups,topk_groups", [(256, 8, 4), (256, 8, 1), (64, 8, 3), (128, 2, 1), (160, 8, 3), (36, 6, 2), (12, 12, 5), (1024, 32, 7), (32, 4, 4), (60, 4, 2)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", [False, True])
def test_groups_and_bias(E, groups, topk_groups, score, bias):
    torch.manual_seed(E + groups)
    l = torch.randn(200, E, device=DEV) * 1.5
    b = torch.randn(E, device=DEV) * 0.1 if bias else None
    k = min(8, E // groups * topk_groups)
    check(l, k, score=score, bias=b, groups=groups, topk_groups=topk_groups, normalize=k > 1)


def test_ties_go_to_the_lowest_expert():
    l = torch.zeros(5, 100, device=DEV, dtype=torch.bfloat16)
    l[1, 50:] = 1
    l[2, 3] = -0.0
    l[3, 99] = l[3, 7] = 2
    _, ids = check(l, 6, score="sigmoid")
    assert ids[0].tolist() == [0, 1, 2, 3, 4, 5] and ids[1].tolist() == [50, 51, 52, 53, 54, 55]
    assert ids[2].tolist() == [0, 1, 2, 3, 4, 5] and ids[3].tolist() == [7, 99, 0, 1, 2, 3]
    check(l, 6, score="softmax", bias=torch.zeros(100, device=DEV))
    check(l, 6, score="sigmoid", groups=10, topk_groups=2)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("normalize", [False, True])
@pytest.mark.parametrize("bias", [False, True])
def test_masked_experts(score, normalize, bias):
    torch.manual_seed(1)
    l = torch.randn(6, 64, device=DEV)
    l[0] = -math.inf  # nothing is available
    l[1, 1:] = -math.inf
    l[2, 5:] = -math.inf
    l[3, ::2] = -math.inf
    l[4] = torch.finfo(torch.float32).min  # the lowest value is a value
    b = torch.rand(64, device=DEV) if bias else None
    probs, ids = check(l, 8, score=score, normalize=normalize, bias=b)
    assert ids[0].tolist() == [-1] * 8 and not probs[0].any()
    assert ids[1].tolist() == [0] + [-1] * 7 and set(ids[2, 5:].tolist()) == {-1} and bool((ids[4] >= 0).all())
    if bias:
        check(l, 4, score=score, bias=b, groups=8, topk_groups=2)


def test_nan_and_infinity_show():
    l = torch.randn(3, 40, device=DEV)
    l[0, 17] = math.nan
    l[1, 3] = math.inf
    for score in ("softmax", "sigmoid"):
        probs, ids = topk_router(l, 4, score_function=score, normalize=True)
        assert ids[0, 0] == 17 and bool(probs[0].isnan().all()) and not probs[2].isnan().any()
        assert ids[1, 0] == 3 and bool((ids < 40).all()) and bool((ids >= 0).all())
        probs, ids = topk_router(l, 4, score_function=score, expert_bias=torch.zeros(40, device=DEV), num_groups=4, topk_groups=1)
        assert (score == "softmax" or ids[0, 0] == 17) and bool(((ids >= 0) & (ids < 40)).all())


def test_large_differences():
    """Scores that underflow in 32 bits keep their order and, normalised over the chosen, their probabilities."""
    l = torch.tensor([[0.0, -90.0, -91.0, -120.0, -119.0, 60.0]], device=DEV)
    check(l, 6, score="softmax", normalize=True)
    check(l, 2, score="sigmoid", bias=torch.tensor([0.0, 5.0, 5.0, 5.0, 5.0, 0.0], device=DEV))
    p, ids = topk_router(l, 2, score_function="softmax", normalize=True, expert_bias=torch.tensor([0.0, 5.0, 5.0, 0.0, 0.0, 0.0], device=DEV))
    assert ids.tolist() == [[1, 2]]
    torch.testing.assert_close(p.double(), torch.softmax(l[:, 1:3].double(), 1), rtol=1e-6, atol=0)


@pytest.mark.parametrize("T", [0, 1, 7, 8, 9, 4000])
def test_token_counts(T):
    torch.manual_seed(T)
    l = torch.randn(T, 128, device=DEV, dtype=torch.bfloat16)
    if T:
        check(l, 8, normalize=True)
    else:
        p, ids = topk_router(l.requires_grad_(True), 8)
        assert p.shape == ids.shape == (0, 8)
        assert torch.autograd.grad(p.sum(), l)[0].shape == (0, 128)


def test_strides():
    torch.manual_seed(0)
    wide = torch.randn(33, 300, device=DEV)
    for l in (wide[:, :128], wide[:, 1:129], wide[::2, 4:132], torch.randn(128, 33, device=DEV).t(), torch.randn(1, 64, device=DEV).expand(5, 64)):
        check(l, 4)
        leaf = l.detach().clone().requires_grad_(True)
        p, ids = topk_router(l, 4)
        q, jds = topk_router(l.contiguous(), 4)
        assert torch.equal(p, q) and torch.equal(ids, jds)
        probs, _ = topk_router(leaf, 4)
        probs.sum().backward()  # an expanded gradient
        probs.t()
        assert leaf.grad is not None


def test_gradient_against_differences():
    torch.manual_seed(2)
    for score, normalize in (("softmax", False), ("softmax", True), ("sigmoid", False), ("sigmoid", True)):
        l = torch.randn(4, 16, device=DEV, requires_grad=True)
        g = torch.randn(4, 3, device=DEV)
        p, ids = topk_router(l, 3, score_function=score, normalize=normalize)
        (dl,) = torch.autograd.grad(p, l, g)
        h = 2.0**-7
        for e in range(16):
            d = torch.zeros_like(l)
            d[:, e] = h
            a, ia = topk_router((l + d).detach(), 3, score_function=score, normalize=normalize)
            b, ib = topk_router((l - d).detach(), 3, score_function=score, normalize=normalize)
            same = (ia == ids).all(1) & (ib == ids).all(1)
            diff = ((a - b) * g).sum(1) / (2 * h)
            # third derivative of order one: h^2 / 6 = 1e-5 relative to the gradients' size; fp32 noise 2^-23 / h = 1.5e-5
            assert bool(((diff - dl[:, e]).abs() <= 3e-4 * (1 + g.abs().sum(1)))[same].all())


def test_tables_feed_the_permutation():
    """Router -> token_permute -> token_unpermute: with the identity in between, a token comes back times its probabilities' sum, and
    the gradient reaches the logits."""
    torch.manual_seed(3)
    T, E, H, k = 50, 12, 64, 3
    l = torch.randn(T, E, device=DEV, requires_grad=True)
    x = torch.randn(T, H, device=DEV, dtype=torch.bfloat16)
    probs, routing = topk_routing_map(l, k, score_function="sigmoid", scaling_factor=0.5)
    rows, _, idx, _ = token_permute(x, T * k, routing_map=routing)
    y = token_unpermute(rows, idx, merging_probs=probs, restore_shape=x.shape, routing_map=routing)
    torch.testing.assert_close(y.double(), x.double() * probs.double().sum(1, keepdim=True), rtol=2.0**-7, atol=1e-6)
    gy = torch.randn_like(y)
    (dl,) = torch.autograd.grad(y, l, gy)
    dot = (gy.double() * x.double()).sum(1, keepdim=True)
    s = torch.sigmoid(l.detach().double())
    want = torch.where(routing, 0.5 * s * (1 - s) * dot, 0.0)
    torch.testing.assert_close(dl.double(), want, rtol=1e-4, atol=1e-4)


def test_captured_and_other_stream():
    torch.manual_seed(4)
    l = torch.randn(64, 128, device=DEV, requires_grad=True)
    g = torch.randn(64, 8, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            p, ids = topk_router(l, 8)
            (dl,) = torch.autograd.grad(p, l, g)
        del p, dl, ids
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        p, ids = topk_router(l, 8)
        (dl,) = torch.autograd.grad(p, l, g)
    with torch.no_grad():
        l.copy_(torch.randn_like(l))
    graph.replay()
    q, jds = topk_router(l, 8)
    (wl,) = torch.autograd.grad(q, l, g)
    assert torch.equal(p, q) and torch.equal(ids, jds) and torch.equal(dl, wl)
