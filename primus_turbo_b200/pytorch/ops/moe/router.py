"""Top-k routing of an MoE layer: which experts a token goes to, and with what probability.

``topk_router`` gives the compact form (``probs`` and expert ids ``[T, k]``, what ``moe_few_tokens`` takes), ``topk_routing_map`` the
tables ``probs`` / ``routing_map`` ``[T, E]`` that ``token_permute`` and ``token_unpermute`` take.  Both are differentiable in the
logits.  The reference has this step as ops/moe/fused_moe_router.py, under other names and with an auxiliary score that is not made here.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from primus_turbo_b200 import _native
from primus_turbo_b200._lib import PtbError, require_cuda
from primus_turbo_b200.pytorch.kernels import custom_ops as _ops
from primus_turbo_b200.pytorch.kernels.few_rows_impl import SCORE_FUNCTIONS

__all__ = ["topk_router", "topk_routing_map"]

_MAX_EXPERTS, _MAX_TOPK, _MAX_GROUPS = 1024, 32, 32


class _NoSecondDerivative(torch.autograd.Function):
    """The gradient itself, kept in the graph (create_graph) as a function of the logits whose derivative is refused."""

    @staticmethod
    def forward(ctx, dl, logits):
        return dl.view_as(dl)

    @staticmethod
    def backward(ctx, _):
        raise RuntimeError("trying to differentiate topk_router twice: its gradient has no derivative")


class _TopkRouter(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, topk, score, bias, num_groups, topk_groups, normalize, scaling_factor, dense):
        ids, probs, table = _ops.topk_router(logits, topk, score, bias, num_groups, topk_groups, normalize, scaling_factor, dense)
        ctx.save_for_backward(logits, ids)
        ctx.options = (score, normalize, scaling_factor, dense)
        chosen = table if dense else ids
        ctx.mark_non_differentiable(chosen)
        return probs, chosen

    @staticmethod
    def backward(ctx, grad, _):
        logits, ids = ctx.saved_tensors
        with torch.no_grad():
            dl = _ops.topk_router_bwd(logits, ids, grad, *ctx.options)
        if torch.is_grad_enabled() and not torch.compiler.is_compiling():
            dl = _NoSecondDerivative.apply(dl, logits)
        return (dl,) + (None,) * 8


def _route(logits, topk, score_function, expert_bias, num_groups, topk_groups, normalize, scaling_factor, dense):
    if _native.usable(logits) and type(topk) is type(num_groups) is type(topk_groups) is int and score_function in SCORE_FUNCTIONS:
        out = _native.ext.topk_router(logits, expert_bias, topk, SCORE_FUNCTIONS[score_function], num_groups, topk_groups, bool(normalize),
                                      float(scaling_factor), dense)
        if out is not None:
            return out
    if logits.dim() != 2:
        raise ValueError(f"logits must be [tokens, experts], got {logits.dim()}D")
    if logits.dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise ValueError(f"logits must be fp32, fp16 or bf16, got {logits.dtype}")
    if score_function not in SCORE_FUNCTIONS:
        raise ValueError(f"score_function must be one of {tuple(SCORE_FUNCTIONS)}, got {score_function!r}")
    E = logits.shape[1]
    if not 1 <= E <= _MAX_EXPERTS:
        raise ValueError(f"1 to {_MAX_EXPERTS} experts are supported, got {E}")
    if not 1 <= num_groups <= _MAX_GROUPS or E % num_groups != 0:
        raise ValueError(f"num_groups must divide the {E} experts and be at most {_MAX_GROUPS}, got {num_groups}")
    if not 1 <= topk_groups <= num_groups:
        raise ValueError(f"topk_groups must be between 1 and num_groups, got {topk_groups}")
    if not 1 <= topk <= min(_MAX_TOPK, E // num_groups * topk_groups):
        raise ValueError(f"topk must be between 1 and {min(_MAX_TOPK, E // num_groups * topk_groups)}, got {topk}")
    require_cuda(logits, expert_bias)
    if expert_bias is not None:
        if tuple(expert_bias.shape) != (E,) or expert_bias.dtype != torch.float32:
            raise ValueError(f"expert_bias must be fp32 [{E}]")
        if expert_bias.device != logits.device:
            raise PtbError("topk_router: logits and expert_bias must be on one device")
        expert_bias = expert_bias.detach().contiguous()
    args = (logits, int(topk), SCORE_FUNCTIONS[score_function], expert_bias, int(num_groups), int(topk_groups), bool(normalize),
            float(scaling_factor), dense)
    return _TopkRouter.apply(*args)


def topk_router(
    logits: torch.Tensor,
    topk: int,
    *,
    score_function: str = "softmax",
    expert_bias: Optional[torch.Tensor] = None,
    num_groups: int = 1,
    topk_groups: int = 1,
    normalize: bool = False,
    scaling_factor: float = 1.0,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(probs fp32 [T, k], expert ids int64 [T, k])`` of the ``topk`` experts of every token, best first.

    ``score_function``: "softmax" over the experts or "sigmoid" of each logit.  ``expert_bias`` (fp32 [E]) is added to the scores when
    experts are chosen, not to the probabilities, and has no gradient.  With ``num_groups`` > 1 only the ``topk_groups`` groups of
    neighbouring experts whose two best add up to most take part.  ``normalize``: probabilities relative to their sum over the
    chosen experts (a sigmoid's sum plus 1e-20).  ``scaling_factor`` multiplies them.

    Ties go to the lowest expert.  A logit of -inf makes an expert unavailable; a token with fewer than ``topk`` available
    experts has id -1 and probability 0 in its last places.  A NaN logit counts as the largest, so that it shows."""
    return _route(logits, topk, score_function, expert_bias, num_groups, topk_groups, normalize, scaling_factor, False)


def topk_routing_map(
    logits: torch.Tensor,
    topk: int,
    *,
    score_function: str = "softmax",
    expert_bias: Optional[torch.Tensor] = None,
    num_groups: int = 1,
    topk_groups: int = 1,
    normalize: bool = False,
    scaling_factor: float = 1.0,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(probs fp32 [T, E], routing_map bool [T, E])``: ``topk_router`` as the tables that ``token_permute`` takes; probabilities
    of experts that were not chosen are 0.  The gradient reads the table's gradient at the chosen experts."""
    return _route(logits, topk, score_function, expert_bias, num_groups, topk_groups, normalize, scaling_factor, True)
