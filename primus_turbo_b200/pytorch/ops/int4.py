"""4-bit weights with group scales: ``quantize_int4``, ``dequantize_int4`` and ``gemm_int4``, the product of a few rows of
activations with one.  For serving: a weight is quantised once, when a model is loaded, and each token then reads a quarter of
the bytes.  None of the three has a gradient; a call that would need one, of the activations or of the scales, is refused.

The reference has no 4-bit integer format; names and argument order follow its FP8 ops (ops/quantization.py:52-269,
ops/gemm_fp8.py:658 there).
"""

from __future__ import annotations

from typing import Optional

import torch

from primus_turbo_b200 import _native
from primus_turbo_b200._lib import PtbError, require_cuda
from primus_turbo_b200.pytorch.core.int4_weight import INT4_GROUP_SIZES, Int4Weight
from primus_turbo_b200.pytorch.kernels import custom_ops as _ops

__all__ = ["quantize_int4", "dequantize_int4", "gemm_int4"]

_WIDE = (torch.bfloat16, torch.float16, torch.float32)


def refuse_gradient(name: str, *tensors: Optional[torch.Tensor]) -> None:
    """Raise where a call would have to be differentiated: its result would silently be a constant."""
    for t in tensors:
        if t is None:
            continue
        if t.requires_grad and torch.is_grad_enabled():
            raise NotImplementedError(f"{name} has no backward pass: call it under torch.no_grad() or on detached tensors")
        if torch.autograd.forward_ad._current_level >= 0 and torch.autograd.forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f"{name} has no forward mode derivative (jvp)")


def quantize_int4(w: torch.Tensor, group_size: int = 128, symmetric: bool = True) -> Int4Weight:
    """``w`` [N, K] or [E, N, K] (bf16, fp16 or fp32, K a multiple of 8) in 4 bits, groups of ``group_size`` (32, 64 or 128) along K.

    ``symmetric``: ``scale = max |w| / 7`` and codes around 8; otherwise the range of a group, 0 included, in 15 steps from a
    zero point.  The scale is rounded to bf16 before the codes are chosen.  A group that holds a NaN or an infinity becomes
    NaN as a whole.  ``w`` is taken as it is: no gradient flows through (pass a detached tensor, or call under ``no_grad``)."""
    if _native.usable(w) and type(group_size) is int:
        parts = _native.ext.quant_int4(w, group_size, bool(symmetric))
        if parts is not None:
            return Int4Weight(*parts, w.shape, group_size)
    refuse_gradient("quantize_int4", w)
    if w.dim() not in (2, 3):
        raise ValueError(f"a 4-bit weight is 2D or 3D, got {w.dim()}D")
    if w.dtype not in _WIDE:
        raise ValueError(f"quantize_int4 takes bf16, fp16 or fp32, got {w.dtype}")
    if group_size not in INT4_GROUP_SIZES:
        raise ValueError(f"group_size must be one of {INT4_GROUP_SIZES}, got {group_size}")
    if w.shape[-1] % 8 != 0:
        raise ValueError(f"the row length must be a multiple of 8, got {w.shape[-1]}")
    require_cuda(w)
    codes, scale, zero = _ops.quant_int4(w, int(group_size), bool(symmetric))
    return Int4Weight(codes, scale, None if symmetric else zero, w.shape, int(group_size))


def dequantize_int4(w: Int4Weight, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values ``(code - zero) * scale`` of ``w``, computed in fp32 and rounded once to ``out_dtype``."""
    if not isinstance(w, Int4Weight):
        raise TypeError(f"dequantize_int4 takes an Int4Weight, got {type(w).__name__}")
    if out_dtype not in _WIDE:
        raise ValueError(f"dequantize_int4 gives bf16, fp16 or fp32, not {out_dtype}")
    if _native.usable(w.qdata):
        out = _native.ext.dequant_int4(w.qdata, w.scale, w.zero, w.shape[-1], w.group_size, out_dtype)
        if out is not None:
            return out
    refuse_gradient("dequantize_int4", w.scale)
    require_cuda(w.qdata)
    return _ops.dequant_int4(w.qdata, w.scale, w.zero, w.shape[-1], w.group_size, out_dtype)


def gemm_int4(x: torch.Tensor, w: Int4Weight, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x @ dequantised(w).T (+ bias)`` for ``x`` [..., K] (bf16 or fp16) and a 4-bit weight [N, K]; result [..., N] in x's type.

    Activations are held to 2^-22 of the largest of their 128 neighbours along K or better (what is above 2^-11 of it is exact), sums in
    fp32; the weight is never written out.  Made for few rows (a token, a decoding
    batch): 32 rows are taken at a time, and beyond some hundreds ``dequantize_int4`` with a library product is the faster way.  A row
    of ``x`` that holds a NaN or an infinity gives NaN and infinities, other rows are not touched by it."""
    if not isinstance(w, Int4Weight):
        raise TypeError(f"gemm_int4 takes an Int4Weight, got {type(w).__name__}")
    if _native.usable(x):
        y = _native.ext.gemm_int4(x, w.qdata, w.scale, w.zero, w.shape[-1], w.group_size, bias)
        if y is not None:
            return y
    refuse_gradient("gemm_int4", x, bias, w.scale)
    if w.ndim != 2:
        raise ValueError(f"gemm_int4 takes a 2D weight, got {w.ndim}D")
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"gemm_int4 takes bf16 or fp16 activations, got {x.dtype}")
    n, k = w.shape
    if x.dim() < 1 or x.shape[-1] != k:
        raise ValueError(f"contraction sizes differ: x {tuple(x.shape)}, weight {tuple(w.shape)}")
    if k == 0:
        raise ValueError("the contraction is empty")
    if bias is not None and (tuple(bias.shape) != (n,) or bias.dtype != x.dtype or not bias.is_contiguous()):
        raise ValueError(f"bias must be a contiguous vector of {n} in x's type")
    require_cuda(x, w.qdata, bias)
    if x.device != w.device or (bias is not None and bias.device != x.device):
        raise PtbError("gemm_int4: x, the weight and the bias must be on one device")
    y = _ops.gemm_int4(x if x.dim() == 2 else x.reshape(-1, k), w.qdata, w.scale, w.zero, w.group_size, bias)
    return y if x.dim() == 2 else y.view(*x.shape[:-1], n)
