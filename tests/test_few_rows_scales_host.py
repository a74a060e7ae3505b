"""CPU: scales of a quantised weight that would need a gradient are refused, by the ops that would silently give a constant."""

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from primus_turbo_b200 import _lib
from primus_turbo_b200.pytorch.core.int4_weight import Int4Weight
from primus_turbo_b200.pytorch.core.low_precision import ScalingGranularity
from primus_turbo_b200.pytorch.core.quantized_tensor import QuantizedTensor
from primus_turbo_b200.pytorch.ops import dequantize_int4, gemm_int4
from primus_turbo_b200.pytorch.ops.moe import moe_few_tokens

BF = torch.bfloat16


def int4(shape, scale=None):
    return Int4Weight.from_codes(torch.zeros(shape, dtype=torch.uint8), torch.ones((*shape[:-1], 1), dtype=BF) if scale is None else scale, group_size=64)


def fp8(shape, learned):
    return QuantizedTensor(torch.zeros(shape).to(torch.float8_e4m3fn), torch.ones((), requires_grad=learned), shape=torch.Size(shape), orig_dtype=BF,
                           dest_dtype=torch.float8_e4m3fn, granularity=ScalingGranularity.TENSORWISE)


def calls(scales):
    """Calls of every op, one weight of each with the scales that scales(shape) makes."""
    x, ids, p = torch.zeros(3, 64, dtype=BF), torch.zeros(3, 1, dtype=torch.int64), torch.ones(3, 1)
    w, up, down = (int4(s, scales((*s[:-1], 1))) for s in ((16, 64), (2, 64, 64), (2, 64, 32)))
    return (lambda: gemm_int4(x, w), lambda: dequantize_int4(w), lambda: moe_few_tokens(x, ids, p, up, int4((2, 64, 32))),
            lambda: moe_few_tokens(x, ids, p, int4((2, 64, 64)), down))


def test_learned_scales_are_refused():
    x, ids, p = torch.zeros(3, 64, dtype=BF), torch.zeros(3, 1, dtype=torch.int64), torch.ones(3, 1)
    eight = [lambda a=a, b=b: moe_few_tokens(x, ids, p, fp8((2, 64, 64), a), fp8((2, 64, 32), b)) for a, b in ((True, False), (False, True))]
    for call in (*calls(lambda shape: torch.ones(shape, dtype=BF, requires_grad=True)), *eight):
        with pytest.raises(NotImplementedError, match="no backward"):
            call()
        with torch.no_grad(), pytest.raises(_lib.PtbError, match="CPU"):
            call()


def test_scales_with_a_tangent_are_refused():
    with fwAD.dual_level():
        for call in calls(lambda shape: fwAD.make_dual(torch.ones(shape, dtype=BF), torch.ones(shape, dtype=BF))):
            with pytest.raises(NotImplementedError, match="forward mode"):
                call()


# ---- from_codes takes what it can hold -----------------------------------------------------------------------------------------
def test_from_codes_refuses_scales_that_would_be_rounded():
    codes = torch.randint(0, 16, (4, 64), dtype=torch.uint8)
    for dtype in (torch.float16, torch.float32, torch.float64):
        held = torch.tensor([[0.5], [1.0078125], [float("nan")], [float("inf")]], dtype=dtype)
        assert torch.equal(Int4Weight.from_codes(codes, held, group_size=64).scale.double().nan_to_num(7.0), held.double().nan_to_num(7.0))
        for bad in (1.0009765625, 65504.0, 0.1):
            scale = held.clone()
            scale[1, 0] = bad
            with pytest.raises(AssertionError, match="bfloat16"):
                Int4Weight.from_codes(codes, scale, group_size=64)
            rounded = scale.to(BF)
            assert torch.equal(Int4Weight.from_codes(codes, rounded, group_size=64).scale[:2], rounded[:2])


def test_from_codes_refuses_codes_of_more_than_four_bits():
    codes = torch.zeros(2, 3, 64, dtype=torch.uint8)
    scale = torch.ones(2, 3, 1, dtype=BF)
    Int4Weight.from_codes(codes, scale, group_size=64)
    codes[1, 2, 63] = 16
    with pytest.raises(AssertionError, match="15"):
        Int4Weight.from_codes(codes, scale, group_size=64)
    assert Int4Weight.from_codes(codes[:0], scale[:0], group_size=64).shape == (0, 3, 64)
    assert Int4Weight.from_codes(codes.to("meta"), scale.to("meta"), group_size=64).shape == (2, 3, 64)


def test_from_codes_of_stand_ins():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        codes, scale = torch.empty(4, 64, dtype=torch.uint8), torch.empty(4, 1, dtype=torch.float16)
        assert Int4Weight.from_codes(codes, scale, group_size=64).scale.dtype == BF
