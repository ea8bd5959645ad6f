"""Matrices in 8 bits: e4m3 values with one fp32 scale per block of 128."""
from __future__ import annotations

from dataclasses import dataclass

import torch

BLOCK = 128


@dataclass
class Fp8Rows:
    """Rows in 8 bits: row r, column c is ``data[r, c] * scales[r, c // 128]``."""
    data: torch.Tensor     # float8_e4m3fn [R, K]
    scales: torch.Tensor   # fp32 [R, ceil(K / 128)]
    dtype: torch.dtype     # 16-bit type of the products
