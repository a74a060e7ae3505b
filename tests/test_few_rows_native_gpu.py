"""GPU: the native host path of the router, the 4-bit product and the few-token MoE layer gives what the Python form gives, takes the
calls it is meant for, and leaves those to Python that only that can refuse or record."""

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from primus_turbo_b200 import _lib, _native
from primus_turbo_b200.pytorch.core.low_precision import ScalingGranularity, ScalingRecipe
from primus_turbo_b200.pytorch.core.quantized_tensor import QuantizedTensor
from primus_turbo_b200.pytorch.ops import dequantize_int4, gemm_int4, quantize_int4
from primus_turbo_b200.pytorch.ops.moe import moe_few_tokens, topk_router, topk_routing_map

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _randn(*shape, dtype=torch.bfloat16, seed=1):
    return torch.randn(*shape, device=DEV, generator=torch.Generator(DEV).manual_seed(seed)).to(dtype)


def _both(monkeypatch, f):
    """f() by the native path, which has to take it, and by the Python form."""
    before = _native.ext.calls()
    native = f()
    assert _native.ext.calls() > before
    with monkeypatch.context() as m:
        m.setattr(_native, "usable", lambda t: False)
        before = _native.ext.calls()
        python = f()
        assert _native.ext.calls() == before
    return native, python


def _same(a, b):
    return a.dtype == b.dtype and a.shape == b.shape and torch.equal(a.view(torch.uint8) if a.dtype == torch.bool else a, b.view(torch.uint8) if b.dtype == torch.bool else b)


def _layer(kind, dtype=torch.bfloat16, E=6, H=256, I=128):
    w1, w2 = _randn(E, 2 * I, H, dtype=dtype, seed=3) / 16, _randn(E, H, I, dtype=dtype, seed=4) / 11
    if kind == "int4":
        return quantize_int4(w1, 64, False), quantize_int4(w2, 64, False)
    if kind == "fp8":
        recipe = ScalingRecipe(use_2d_block=True)
        return tuple(QuantizedTensor.quantize(w, torch.float8_e4m3fn, ScalingGranularity.BLOCKWISE, axis=-1, block_size=128, scaling_recipe=recipe) for w in (w1, w2))
    return w1, w2


def _routed(T, E=6, k=2):
    return topk_router(_randn(T, E, dtype=torch.float32, seed=5), k, normalize=True)


# ---- the same results ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("shape", [(1, 256), (3, 256), (40, 256), (2, 5, 256), (256,)])
@pytest.mark.parametrize("bias", [False, True])
def test_product(monkeypatch, shape, bias):
    w = quantize_int4(_randn(72, 256), 32, symmetric=bias)
    x, b = _randn(*shape, seed=2), _randn(72, seed=6) if bias else None
    assert _same(*_both(monkeypatch, lambda: gemm_int4(x, w, b)))


def test_product_of_rows_of_a_wider_tensor(monkeypatch):
    w, x = quantize_int4(_randn(72, 256), 128), _randn(5, 320, seed=2)
    assert _same(*_both(monkeypatch, lambda: gemm_int4(x[:, 64:], w)))


@pytest.mark.parametrize("symmetric", [False, True])
def test_quantise_and_back(monkeypatch, symmetric):
    w = _randn(2, 24, 136)
    a, b = _both(monkeypatch, lambda: quantize_int4(w, 32, symmetric))
    assert _same(a.qdata, b.qdata) and _same(a.scale, b.scale) and (a.zero is None) == symmetric and (symmetric or _same(a.zero, b.zero))
    assert _same(*_both(monkeypatch, lambda: dequantize_int4(a, torch.float16)))


@pytest.mark.parametrize("kind", ["raw", "fp8", "int4"])
@pytest.mark.parametrize("T", [1, 20])
def test_layer(monkeypatch, kind, T):
    w1, w2 = _layer(kind)
    (probs, ids), x = _routed(T), _randn(T, 256, seed=7)
    assert _same(*_both(monkeypatch, lambda: moe_few_tokens(x, ids, probs, w1, w2)))


@pytest.mark.parametrize("route", [topk_router, topk_routing_map])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_router_and_its_gradient(monkeypatch, route, dtype):
    logits, bias = _randn(33, 24, dtype=dtype), _randn(24, dtype=torch.float32, seed=2) / 10
    grad = _randn(33, 24 if route is topk_routing_map else 3, dtype=torch.float32, seed=3)

    def f():
        l = logits.clone().requires_grad_()
        probs, chosen = route(l, 3, score_function="sigmoid", expert_bias=bias, num_groups=4, topk_groups=2, normalize=True, scaling_factor=2.5)
        assert probs.requires_grad and not chosen.requires_grad
        return probs.detach(), chosen, torch.autograd.grad(probs, l, grad)[0]

    for a, b in zip(*_both(monkeypatch, f)):
        assert _same(a, b)


# ---- calls that stay with Python ------------------------------------------------------------------------------------
def test_gradients_and_tangents_are_refused():
    w, x = quantize_int4(_randn(72, 256), 128), _randn(3, 256)
    (probs, ids), (w1, w2) = _routed(3), _layer("int4")
    calls = [lambda x: gemm_int4(x, w), lambda x: moe_few_tokens(x, ids, probs, w1, w2)]
    for call in calls:
        with pytest.raises(NotImplementedError):
            call(x.clone().requires_grad_())
        with torch.no_grad():
            call(x.clone().requires_grad_())
        with fwAD.dual_level(), pytest.raises(NotImplementedError, match="jvp"):
            call(fwAD.make_dual(x, torch.ones_like(x)))
    with pytest.raises(NotImplementedError):
        gemm_int4(x, w, torch.zeros(72, device=DEV, dtype=torch.bfloat16, requires_grad=True))
    with pytest.raises(NotImplementedError):
        quantize_int4(_randn(8, 64).requires_grad_())
    logits = _randn(3, 8, dtype=torch.float32)
    with fwAD.dual_level(), pytest.raises((NotImplementedError, RuntimeError), match="(?i)jvp|forward mode|forward AD"):
        topk_router(fwAD.make_dual(logits, torch.ones_like(logits)), 2)


def test_the_gradient_of_the_routers_gradient_is_refused():
    logits = _randn(3, 8, dtype=torch.float32).requires_grad_()
    probs, _ = topk_router(logits, 2)
    with pytest.raises((NotImplementedError, RuntimeError)):
        g = torch.autograd.grad(probs.square().sum(), logits, create_graph=True)[0]
        torch.autograd.grad(g.sum(), logits)


def test_traced_calls_run_again_on_new_inputs():
    w, x, other = quantize_int4(_randn(72, 256), 128), _randn(3, 256), _randn(3, 256, seed=9)
    (probs, ids), (w1, w2) = _routed(3), _layer("int4")
    for f in (lambda x: gemm_int4(x, w), lambda x: moe_few_tokens(x, ids, probs, w1, w2), lambda x: topk_router(x, 2)[0]):
        traced = torch.jit.trace(f, (x,), check_trace=False)
        assert torch.equal(traced(other), f(other)) and torch.equal(traced(x), f(x))


def test_recorded_calls_name_their_entries():
    w, x = quantize_int4(_randn(72, 256), 128), _randn(3, 256)
    (probs, ids), (w1, w2) = _routed(3), _layer("raw")
    with _lib.record_kernel_times() as rec:
        a, b = gemm_int4(x, w), moe_few_tokens(x, ids, probs, w1, w2)
    assert set(rec.durations_ms()) == {"ptb_gemm_int4", "ptb_moe_few_tokens"}
    assert torch.equal(a, gemm_int4(x, w)) and torch.equal(b, moe_few_tokens(x, ids, probs, w1, w2))


def test_unfit_arguments_get_the_python_forms_errors():
    w, x = quantize_int4(_randn(72, 256), 128), _randn(3, 256)
    (probs, ids), (w1, w2) = _routed(3), _layer("raw")
    with pytest.raises(ValueError, match="contraction"):
        gemm_int4(x[:, :128], w)
    with pytest.raises(ValueError, match="bias"):
        gemm_int4(x, w, torch.zeros(71, device=DEV, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="do not fit"):
        moe_few_tokens(x, ids, probs, w1[:, :, :128].contiguous(), w2)
    with pytest.raises(ValueError, match="int64"):
        moe_few_tokens(x, ids.int(), probs, w1, w2)
    with pytest.raises(ValueError, match="topk"):
        topk_router(_randn(3, 8), 9)
