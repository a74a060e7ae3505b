"""``Int4Weight``: a weight of 4-bit codes with a scale (and optionally a zero point) per group of a row.

``value[..., n, k] = (code - zero) * scale`` with one bf16 ``scale`` and one byte ``zero`` (any; 8 where there are none) per
``group_size`` neighbouring ``k`` of a row.  ``qdata`` holds the codes as the kernels read them, ``ceil(K / 128) * 64`` bytes a
row (the order is described in ``include/ptb.h``); ``from_codes`` and ``codes`` convert from and to one code a byte.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch

INT4_GROUP_SIZES = (32, 64, 128)
INT4_BLOCK = 128  # values per block of the packed layout
INT4_BLOCK_BYTES = INT4_BLOCK // 2


def _packed_bytes(k: int) -> int:
    return (k + INT4_BLOCK - 1) // INT4_BLOCK * INT4_BLOCK_BYTES


def _has_values(t: torch.Tensor) -> bool:
    """Not a stand-in of a tensor, as while tracing."""
    plain = type(t) in (torch.Tensor, torch.nn.Parameter) and not t.is_meta
    return plain and not torch.compiler.is_compiling() and torch._C._len_torch_dispatch_stack() == 0


@dataclass(frozen=True)
class Int4Weight:
    """``[N, K]`` or ``[E, N, K]``; made by ``quantize_int4`` or ``from_codes``."""

    qdata: torch.Tensor  # uint8 [..., N, ceil(K / 128) * 64]
    scale: torch.Tensor  # bfloat16 [..., N, ceil(K / group_size)]
    zero: Optional[torch.Tensor]  # uint8, like scale
    shape: torch.Size
    group_size: int

    def __post_init__(self):
        object.__setattr__(self, "shape", torch.Size(self.shape))
        assert self.group_size in INT4_GROUP_SIZES, f"group_size must be one of {INT4_GROUP_SIZES}, got {self.group_size}"
        assert len(self.shape) in (2, 3), f"a 4-bit weight is 2D or 3D, got {len(self.shape)}D"
        k = self.shape[-1]
        assert k % 8 == 0, f"the row length of a 4-bit weight must be a multiple of 8, got {k}"
        lead = tuple(self.shape[:-1])
        want = (*lead, _packed_bytes(k))
        assert self.qdata.dtype == torch.uint8 and tuple(self.qdata.shape) == want, f"qdata must be uint8 {want}"
        groups = (*lead, (k + self.group_size - 1) // self.group_size)
        assert self.scale.dtype == torch.bfloat16 and tuple(self.scale.shape) == groups, f"scale must be bfloat16 {groups}"
        parts = [self.qdata, self.scale]
        if self.zero is not None:
            assert self.zero.dtype == torch.uint8 and tuple(self.zero.shape) == groups, f"zero must be uint8 {groups}"
            parts.append(self.zero)
        for t in parts:
            assert t.is_contiguous() and t.device == self.qdata.device, "the parts of a 4-bit weight are contiguous and on one device"

    @property
    def device(self) -> torch.device:
        return self.qdata.device

    @property
    def ndim(self) -> int:
        return len(self.shape)

    def size(self, dim: int) -> int:
        return self.shape[dim]

    def to(self, device) -> "Int4Weight":
        zero = None if self.zero is None else self.zero.to(device)
        return Int4Weight(self.qdata.to(device), self.scale.to(device), zero, self.shape, self.group_size)

    @classmethod
    def from_codes(
        cls, codes: torch.Tensor, scale: torch.Tensor, zero: Optional[torch.Tensor] = None, *, group_size: int
    ) -> "Int4Weight":
        """From codes 0 .. 15, one a byte, ``[..., N, K]``; ``scale`` and ``zero`` ``[..., N, ceil(K / group_size)]``.

        Scales are kept in bfloat16.  Others are taken where bfloat16 holds every one of them exactly; where it does not, rounding them
        (``scale.to(torch.bfloat16)``, up to 2^-8 of each weight) is left to the caller.  For these checks the codes and such scales are read
        back: this is for loading a model, not for a captured graph."""
        assert codes.dtype == torch.uint8, "codes must be uint8, one code (0 .. 15) a byte"
        k = codes.shape[-1]
        assert k % 8 == 0, f"the row length of a 4-bit weight must be a multiple of 8, got {k}"
        if _has_values(codes) and codes.numel() > 0:
            assert int(codes.max()) <= 15, f"codes must be 0 .. 15, got {int(codes.max())}"
        if scale.dtype != torch.bfloat16 and _has_values(scale):
            kept = (scale.to(torch.bfloat16).to(scale.dtype) == scale) | scale.isnan()
            assert bool(kept.all()), f"these {scale.dtype} scales are not bfloat16 numbers: pass scale.to(torch.bfloat16) to have them rounded"
        padded = torch.nn.functional.pad(codes, (0, -k % INT4_BLOCK)) if k % INT4_BLOCK else codes
        octets = padded.unflatten(-1, (-1, 4, 4, 8)).transpose(-2, -3)  # [..., block, t, q, 8]
        qdata = (octets[..., :4] & 15 | octets[..., 4:] << 4).flatten(-4).contiguous()
        return cls(qdata, scale.to(torch.bfloat16).contiguous(), None if zero is None else zero.contiguous(), codes.shape, group_size)

    def codes(self) -> torch.Tensor:
        """The codes, one a byte, ``[..., N, K]``."""
        words = self.qdata.unflatten(-1, (-1, 4, 4, 4))  # [..., block, t, q, byte]
        octets = torch.cat([words & 15, words >> 4], dim=-1)
        return octets.transpose(-2, -3).flatten(-4)[..., : self.shape[-1]].contiguous()

    def __repr__(self) -> str:
        kind = "symmetric" if self.zero is None else "zero points"
        return f"Int4Weight(shape={tuple(self.shape)}, group_size={self.group_size}, {kind}, device={self.device})"


__all__ = ["Int4Weight", "INT4_GROUP_SIZES"]
