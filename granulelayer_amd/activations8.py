"""Activations kept in 8 bits between forward and backward.

``pack_activation(x)`` puts a tensor into 8 bits and ``PackedActivation.unpack()`` reads it back.
Along the last dimension blocks of 32 values share a power of two ``step``, the smallest (from 2^-126
to 2^121) that holds every ``rint(x / step)`` in [-127, 127], and every value is such a quotient:
``|x - unpack(x)| <= step / 2``, at most 1/127 of the block's largest magnitude, and 1 + 1/32 bytes a value.
(Values within 1/256 of the largest fp32 number are cut to 127 steps.)
Unpacked values have 7 significant bits and are exact in bf16 and fp32; putting them into 8 bits again
changes nothing.  A block that holds an infinity or a NaN reads back as NaN.

``activation_checkpoint="int8"`` of ``DenseProjection``, ``SparsePoolingLayer`` and
``CoverTopK16Layer`` keeps what their backward needs in this form.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from .backend import backend_for

ACTIVATION_CHECKPOINTS = ("exact", "int8")
BLOCK = 32


def check_activation_checkpoint(kind: str) -> str:
    if kind not in ACTIVATION_CHECKPOINTS:
        raise ValueError(f"activation_checkpoint must be one of {ACTIVATION_CHECKPOINTS} (got {kind!r})")
    return kind


@dataclass(frozen=True)
class PackedActivation:
    """A tensor in 8 bits: ``codes`` [rows, round_up(features, 32)] int8, zeros behind the features, and
    ``exponents`` [rows, ceil(features / 32)] uint8, of a tensor of ``shape`` and ``dtype``."""

    codes: torch.Tensor
    exponents: torch.Tensor
    shape: Tuple[int, ...]
    dtype: torch.dtype

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + self.exponents.numel()

    def unpack(self, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        """The values the codes stand for, of ``dtype`` (float32 or bfloat16; the packed tensor's own)."""
        x = backend_for(self.codes.device).unpack8(self.codes, self.exponents, self.shape[-1], dtype or self.dtype)
        return x.view(self.shape)


def pack_activation(x: torch.Tensor) -> PackedActivation:
    """``x`` [..., features] (float32 or bfloat16, on a ROCm GPU) in 8 bits.  Not differentiable: the
    result is storage."""
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"x must be [..., features] with at least one feature (got {tuple(x.shape)})")
    x2 = x.detach().reshape(-1, x.shape[-1]) if x.dim() != 2 else x.detach()
    codes, exponents = backend_for(x.device).pack8(x2)
    return PackedActivation(codes, exponents, tuple(x.shape), x.dtype)
