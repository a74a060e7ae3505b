"""``moe_few_tokens``: the whole feed-forward part of an MoE layer for a handful of tokens, straight from the weights a model is
kept in.  What ``token_permute``, two grouped GEMMs, ``swiglu_with_probs`` and ``token_unpermute`` do for a training batch costs a
decoding step more in launches and row padding than its weights take to read; here it is two kernels (a token or a few) or four that read the
experts that are hit once.  For inference: there is no backward pass.  The reference has no counterpart.
"""

from __future__ import annotations

from typing import Union

import torch

from primus_turbo_b200 import _native
from primus_turbo_b200._lib import PtbError, require_cuda
from primus_turbo_b200.pytorch.core.int4_weight import Int4Weight
from primus_turbo_b200.pytorch.core.low_precision import ScalingGranularity
from primus_turbo_b200.pytorch.core.quantized_tensor import QuantizedTensor
from primus_turbo_b200.pytorch.kernels import custom_ops as _ops
from primus_turbo_b200.pytorch.ops.int4 import refuse_gradient

__all__ = ["moe_few_tokens"]

MAX_TOKENS, MAX_PAIRS, MAX_EXPERTS = 128, 1024, 1024
Weight = Union[torch.Tensor, QuantizedTensor, Int4Weight]


def _parts(name: str, w: Weight, dtype: torch.dtype):
    """(kind, data, scales, zero points, granularity, group size) of an expert weight [E, rows, K]."""
    if len(w.shape) != 3:
        raise ValueError(f"{name} must be [experts, rows, K], got {len(w.shape)}D")
    if isinstance(w, Int4Weight):
        return "int4", w.qdata, w.scale, w.zero, 0, w.group_size
    if isinstance(w, QuantizedTensor):
        E, rows, K = w.shape
        g, data, scale = w.granularity, w.qdata, w.scale_inv
        cd = lambda n: (n + 127) // 128  # noqa: E731
        if g == ScalingGranularity.TENSORWISE:
            want = 1
        elif g == ScalingGranularity.ROWWISE and w.quantized_axis == 2:
            want = E * rows
        elif g == ScalingGranularity.BLOCKWISE and w.scaling_recipe is not None and w.scaling_recipe.use_2d_block and w.block_size == 128:
            want = E * cd(rows) * cd(K)
        else:
            raise NotImplementedError(
                f"moe_few_tokens: {name} must have tensorwise scales, rowwise ones along K, or blockwise ones per 128 x 128 tile"
            )
        if tuple(data.shape) != tuple(w.shape) or scale.numel() != want or scale.dtype != torch.float32:
            raise ValueError(f"moe_few_tokens: {name}: {scale.numel()} scales of {scale.dtype} do not fit {tuple(w.shape)} {g.name}")
        return "fp8", data, scale, None, g.value, 0
    if w.dtype != dtype:
        raise ValueError(f"{name} must have the activations' type {dtype}, or be quantised; got {w.dtype}")
    return "raw", w.contiguous(), None, None, 0, 0


def _native_layer(x, ids, probs, w1, w2):
    """The call through the native host path; ``None`` where it has to run in Python."""
    if type(w1) is Int4Weight and type(w2) is Int4Weight:
        if x.dim() != 2 or len(w1.shape) != 3 or len(w2.shape) != 3 or w1.group_size != w2.group_size or w1.shape[2] != x.shape[-1]:
            return None
        return _native.ext.moe_few_tokens(x, ids, probs, w1.qdata, w1.scale, w1.zero, w2.qdata, w2.scale, w2.zero, w2.shape[2], 0, w1.group_size)
    if isinstance(w1, QuantizedTensor) and isinstance(w2, QuantizedTensor):
        if w1.requires_grad or w2.requires_grad:
            return None
        kind, d1, s1, _, g1, _ = _parts("w_gate_up", w1, x.dtype)
        _, d2, s2, _, g2, _ = _parts("w_down", w2, x.dtype)
        return _native.ext.moe_few_tokens(x, ids, probs, d1, s1, None, d2, s2, None, w2.shape[2], g1, 0) if g1 == g2 else None
    if _native.usable(w1) and _native.usable(w2) and w2.dim() == 3:
        return _native.ext.moe_few_tokens(x, ids, probs, w1, None, None, w2, None, None, w2.shape[2], 0, 0)
    return None


def moe_few_tokens(
    x: torch.Tensor, topk_ids: torch.Tensor, topk_probs: torch.Tensor, w_gate_up: Weight, w_down: Weight
) -> torch.Tensor:
    """``y[t] = sum_j topk_probs[t, j] * w_down[e] @ (silu(gate) * up)`` with ``e = topk_ids[t, j]`` and
    ``[gate, up] = w_gate_up[e] @ x[t]``.

    ``x`` [T, H] bf16 or fp16, T at most 128; ``topk_ids`` int64 and ``topk_probs`` [T, k] as ``topk_router`` gives them, T * k at most
    1024 (an id outside [0, E) contributes nothing: padding, or a token with too few experts); ``w_gate_up`` [E, 2 I, H]
    with the gate rows first and ``w_down`` [E, H, I], both plain tensors of x's type, both FP8 ``QuantizedTensor`` (tensorwise, rowwise
    or 128 x 128 blockwise scales, of one kind), or both ``Int4Weight`` of one group size.  H and I are multiples of 8, of 16 for FP8.
    Weights are read where they lie if they are contiguous and start on 16 bytes; a plain tensor that is not (a transposed view of
    another layout) is copied whole in every call, so lay such a weight out once.

    Activations are not quantised: with FP8 and 4-bit weights they are held to 2^-22 of the largest of their 128 neighbours or better
    (what is above 2^-11 of it is exact), with 16-bit weights as they are.  Sums are kept in fp32, and the activation between the two
    products in more than bf16; the result is rounded once to x's type.  What an infinite weight or scale takes part in is infinite or NaN.
    Equal inputs give equal bits.  Every call allocates its own workspace, so calls on
    several streams or in several captured graphs do not share any."""
    if _native.usable(x):
        y = _native_layer(x, topk_ids, topk_probs, w_gate_up, w_down)
        if y is not None:
            return y
    refuse_gradient("moe_few_tokens", x, topk_probs, *(w for w in (w_gate_up, w_down) if isinstance(w, torch.Tensor)))
    if x.dim() != 2 or x.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"x must be [tokens, hidden] in bf16 or fp16, got {x.dim()}D {x.dtype}")
    T, H = x.shape
    if topk_ids.dim() != 2 or topk_ids.shape[0] != T or topk_ids.shape[1] < 1 or topk_ids.dtype != torch.int64:
        raise ValueError(f"topk_ids must be int64 [{T}, k]")
    if topk_probs.shape != topk_ids.shape or topk_probs.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise ValueError(f"topk_probs must be floating point {tuple(topk_ids.shape)}")
    k = topk_ids.shape[1]
    if T > MAX_TOKENS or T * k > MAX_PAIRS:
        raise ValueError(f"moe_few_tokens takes at most {MAX_TOKENS} tokens and {MAX_PAIRS} (token, expert) pairs, got {T} x {k}")
    kind, d1, s1, z1, g1, group1 = _parts("w_gate_up", w_gate_up, x.dtype)
    kind2, d2, s2, z2, g2, group2 = _parts("w_down", w_down, x.dtype)
    if (kind, g1, group1) != (kind2, g2, group2) or (kind == "fp8" and d1.dtype != d2.dtype):
        raise ValueError("w_gate_up and w_down must be kept in the same format")
    E, rows, width = w_gate_up.shape
    inter = w_down.shape[2]
    if width != H or rows != 2 * inter or tuple(w_down.shape) != (E, H, inter):
        raise ValueError(f"x {tuple(x.shape)}, w_gate_up {tuple(w_gate_up.shape)} and w_down {tuple(w_down.shape)} do not fit")
    if not 1 <= E <= MAX_EXPERTS:
        raise ValueError(f"1 to {MAX_EXPERTS} experts are supported, got {E}")
    step = 16 if kind == "fp8" else 8
    if H < 1 or inter < 1 or H % step or inter % step:
        raise ValueError(f"the hidden and intermediate widths must be multiples of {step}, got {H} and {inter}")
    refuse_gradient("moe_few_tokens", s1, s2)
    require_cuda(x, topk_ids, topk_probs, d1, d2)
    if any(t is not None and t.device != x.device for t in (topk_ids, topk_probs, d1, s1, z1, d2, s2, z2)):
        raise PtbError("moe_few_tokens: all tensors must be on one device")
    return _ops.moe_few_tokens(x, topk_ids.contiguous(), topk_probs.to(torch.float32).contiguous(), d1, s1, z1, d2, s2, z2, inter, g1, group1)
