"""Thin torch layer over the routing, 4-bit weight and few-token MoE entry points of the C ABI: allocation and the call, on plain
tensors.  The checks of what a user passes are in ``pytorch/ops``."""

from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch

from primus_turbo_b200 import _lib
from primus_turbo_b200._lib import dtype_code, ptr, stream_of

PTB_INT4 = 5
SCORE_FUNCTIONS = {"softmax": 0, "sigmoid": 1}


class ExpertWeightArg(ctypes.Structure):
    """PtbExpertWeight of include/ptb.h"""

    _fields_ = [("data", ctypes.c_void_p), ("scale", ctypes.c_void_p), ("zero", ctypes.c_void_p), ("granularity", ctypes.c_int),
                ("group", ctypes.c_int)]


def _cdiv(a: int, b: int) -> int:
    return (a + b - 1) // b


# ---- routing ----------------------------------------------------------------------------------------------------------
def topk_router_impl(
    logits: torch.Tensor, topk: int, score_function: int, expert_bias: Optional[torch.Tensor], num_groups: int, topk_groups: int,
    normalize: bool, scaling_factor: float, dense: bool,
) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """-> (ids [T, k] int64, probs fp32 [T, k], or [T, E] if dense, routing map [T, E] bool, or [0])"""
    T, E = logits.shape
    dev = logits.device
    if logits.stride(1) != 1 or (T > 1 and logits.stride(0) < E):
        logits = logits.contiguous()
    ids = torch.empty((T, topk), dtype=torch.int64, device=dev)
    probs = torch.empty((T, E) if dense else (T, topk), dtype=torch.float32, device=dev)
    table = torch.empty((T, E) if dense else (0,), dtype=torch.bool, device=dev)
    with torch.cuda.device(dev):
        _lib.call("ptb_topk_router", ptr(logits), dtype_code(logits.dtype), T, E, logits.stride(0), topk, score_function,
                  ptr(expert_bias), num_groups, topk_groups, int(normalize), scaling_factor, ptr(ids), None if dense else ptr(probs),
                  ptr(probs) if dense else None, ptr(table) if dense else None, stream_of(logits))
    return ids, probs, table


def topk_router_bwd_impl(
    logits: torch.Tensor, ids: torch.Tensor, grad: torch.Tensor, score_function: int, normalize: bool, scaling_factor: float, dense: bool
) -> torch.Tensor:
    T, E = logits.shape
    if logits.stride(1) != 1 or (T > 1 and logits.stride(0) < E):
        logits = logits.contiguous()
    if grad.dtype != torch.float32:
        grad = grad.to(torch.float32)
    if grad.stride(1) != 1:
        grad = grad.contiguous()
    out = torch.empty((T, E), dtype=logits.dtype, device=logits.device)
    with torch.cuda.device(logits.device):
        _lib.call("ptb_topk_router_bwd", ptr(logits), dtype_code(logits.dtype), T, E, logits.stride(0), ids.shape[1], score_function,
                  int(normalize), scaling_factor, ptr(ids), ptr(grad), grad.stride(0), int(dense), ptr(out), stream_of(logits))
    return out


# ---- 4-bit weights ------------------------------------------------------------------------------------------------------
def quant_int4_impl(w: torch.Tensor, group_size: int, symmetric: bool) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """-> (codes, scales, zero points, or [0] if symmetric)"""
    w = _aligned(w.contiguous())
    lead, k = w.shape[:-1], w.shape[-1]
    rows = lead.numel()
    codes = torch.empty((*lead, _cdiv(k, 128) * 64), dtype=torch.uint8, device=w.device)
    scale = torch.empty((*lead, _cdiv(k, group_size)), dtype=torch.bfloat16, device=w.device)
    zero = torch.empty((0,) if symmetric else scale.shape, dtype=torch.uint8, device=w.device)
    with torch.cuda.device(w.device):
        _lib.call("ptb_quant_int4", ptr(w), dtype_code(w.dtype), rows, k, group_size, ptr(codes), ptr(scale),
                  None if symmetric else ptr(zero), stream_of(w))
    return codes, scale, zero


def dequant_int4_impl(
    codes: torch.Tensor, scale: torch.Tensor, zero: Optional[torch.Tensor], k: int, group_size: int, out_dtype: torch.dtype
) -> torch.Tensor:
    lead = codes.shape[:-1]
    codes = _aligned(codes)
    out = torch.empty((*lead, k), dtype=out_dtype, device=codes.device)
    with torch.cuda.device(codes.device):
        _lib.call("ptb_dequant_int4", ptr(codes), ptr(scale), ptr(zero), lead.numel(), k, group_size, ptr(out), dtype_code(out_dtype),
                  stream_of(codes))
    return out


def gemm_int4_impl(
    x: torch.Tensor, codes: torch.Tensor, scale: torch.Tensor, zero: Optional[torch.Tensor], group_size: int, bias: Optional[torch.Tensor]
) -> torch.Tensor:
    x, codes = _rows(x), _aligned(codes)
    m, k = x.shape
    n = codes.shape[0]
    out = torch.empty((m, n), dtype=x.dtype, device=x.device)
    ws = torch.empty(_lib.lib.ptb_gemm_int4_workspace(dtype_code(x.dtype), m, k, group_size), dtype=torch.uint8, device=x.device)
    with torch.cuda.device(x.device):
        _lib.call("ptb_gemm_int4", ptr(x), dtype_code(x.dtype), x.stride(0), m, n, k, ptr(codes), ptr(scale), ptr(zero), group_size,
                  ptr(bias), ptr(ws), ptr(out), stream_of(x))
    return out


# ---- MoE layer for a few tokens ---------------------------------------------------------------------------------------------
def moe_few_tokens_impl(
    x: torch.Tensor, ids: torch.Tensor, probs: torch.Tensor, w1: torch.Tensor, w1_scale: Optional[torch.Tensor],
    w1_zero: Optional[torch.Tensor], w2: torch.Tensor, w2_scale: Optional[torch.Tensor], w2_zero: Optional[torch.Tensor],
    inter: int, granularity: int, group_size: int,
) -> torch.Tensor:
    """``group_size`` > 0: 4-bit codes; FP8 payloads otherwise by their type, with scales of ``granularity``."""
    x = _rows(x)
    w1, w2 = _aligned(w1), _aligned(w2)
    (T, H), k, E = x.shape, ids.shape[1], w1.shape[0]
    fmt = PTB_INT4 if group_size else dtype_code(w1.dtype)
    need = _lib.lib.ptb_moe_few_tokens_workspace(dtype_code(x.dtype), T, H, inter, k, fmt)
    out = torch.empty((T, H), dtype=x.dtype, device=x.device)
    ws = torch.empty(max(need, 0), dtype=torch.uint8, device=x.device)
    a = ExpertWeightArg(ptr(w1), ptr(w1_scale), ptr(w1_zero), granularity, group_size)
    b = ExpertWeightArg(ptr(w2), ptr(w2_scale), ptr(w2_zero), granularity, group_size)
    with torch.cuda.device(x.device):
        _lib.call("ptb_moe_few_tokens", ptr(x), dtype_code(x.dtype), x.stride(0), T, H, inter, E, ptr(ids), ptr(probs), k, fmt,
                  ctypes.addressof(a), ctypes.addressof(b), ptr(ws), ptr(out), stream_of(x))
    return out


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """A contiguous tensor whose first byte the kernels' 16-byte loads may start at (a view into the middle of another may not)."""
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _rows(x: torch.Tensor) -> torch.Tensor:
    """Rows of 16-bit values that can be read 16 bytes at a time, or a copy that can."""
    fits = x.stride(1) == 1 and x.data_ptr() % 16 == 0 and (x.shape[0] <= 1 or (x.stride(0) % 8 == 0 and x.stride(0) >= x.shape[1]))
    return x if fits else x.contiguous() if not x.is_contiguous() else x.clone()
