"""Rows in e4m3: what the products of 8-bit weights and activations exchange (the form is spelled out in csrc/kernels/rows_e4m3.cuh)."""
from __future__ import annotations

from dataclasses import dataclass

import torch

BLOCK = 128                    # columns that share a scale
TOP = 448.0                    # the largest e4m3 number
LEAST = 2.0 ** -100            # a block's maximum counts as at least this


@dataclass
class RowsE4M3:
    """Rows [T, K] as e4m3 codes and an fp32 scale for each 128 columns, block by block: `codes` [T, K] float8_e4m3fn, `scale`
    [ceil(K / 128), T]; column k of row t stands for codes[t, k] * scale[k // 128, t]."""
    codes: torch.Tensor
    scale: torch.Tensor

    def __post_init__(self):
        if self.codes.dim() != 2 or self.codes.dtype is not torch.float8_e4m3fn:
            raise ValueError(f"rows in e4m3 have codes [T, K] in float8_e4m3fn, not {tuple(self.codes.shape)} in {self.codes.dtype}")
        T, K = self.codes.shape
        if self.scale.shape != (-(-K // BLOCK), T) or self.scale.dtype is not torch.float32 or self.scale.device != self.codes.device:
            raise ValueError(f"{T} rows of {K} columns need fp32 scales [{-(-K // BLOCK)}, {T}] on their device, not "
                             f"{tuple(self.scale.shape)} in {self.scale.dtype}")

    @classmethod
    def of(cls, codes, scale) -> "RowsE4M3":
        """Rows that were made to fit, unchecked."""
        q = cls.__new__(cls)
        q.codes, q.scale = codes, scale
        return q

    @property
    def shape(self):
        return self.codes.shape

    @property
    def device(self):
        return self.codes.device

    @property
    def is_cuda(self) -> bool:
        return self.codes.is_cuda

    def numel(self) -> int:
        return self.codes.numel()

    def values(self) -> torch.Tensor:
        """What the codes stand for, in fp32."""
        return self.codes.float() * self.scale.t().repeat_interleave(BLOCK, 1)[:, :self.codes.shape[1]]
