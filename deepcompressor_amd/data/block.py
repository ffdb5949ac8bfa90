"""A matrix held in 8 bits: e4m3 codes with a float32 scale for each block of 128, value = code * scale.

What the fake quantizer computes for ``sfp8_e4m3_nan`` with float32 scales and group shapes (1, 128) or (128, 128), kept
as the codes themselves (the reference de-quantizes and has no such tensor).
"""

from __future__ import annotations

import math
from dataclasses import dataclass, field

import torch

from ..engine_fp8 import checked_codes, quantize_blocks

__all__ = ["BlockScaledTensor"]


@dataclass(eq=False, slots=True)
class BlockScaledTensor:
    """``codes``: float8_e4m3fn [rows][cols], rows starting at multiples of 16 bytes; ``scales``: float32 [ceil(rows /
    block_rows)][ceil(cols / 128)], of any strides; ``block_rows``: 1 (activations, a scale per row) or 128 (weights);
    ``shape``: the tensor's shape, its leading axes flattened into the rows.  ``looked_over``: the codes, if it is known that
    memory can be read up to the next multiple of 16 bytes behind their last row; the product looks itself otherwise."""

    codes: torch.Tensor
    scales: torch.Tensor
    block_rows: int
    shape: torch.Size
    looked_over: torch.Tensor | None = field(default=None, repr=False)

    @staticmethod
    def quantize(x: torch.Tensor, block_rows: int = 1) -> "BlockScaledTensor":
        """float32 / float16 / bfloat16 [..., cols] -> scale = max|block| / 448 (0 -> 1), code = nearest e4m3 value of
        x / scale, a tie to the upper one.  NaN becomes the NaN code (and does not count for the scale); an infinity makes
        its block's scale infinite, so the whole block de-quantizes to NaN.  No host check is made of either."""
        if x.ndim == 0:
            raise ValueError("expected at least one dimension")
        shape = x.shape
        if x.ndim != 2:
            x = x.reshape(math.prod(shape[:-1]), shape[-1])
        codes, scales = quantize_blocks(x, block_rows)
        return BlockScaledTensor(codes, scales, block_rows, shape, codes)

    @staticmethod
    def from_codes(codes: torch.Tensor, scales: torch.Tensor, block_rows: int = 1) -> "BlockScaledTensor":
        """Codes and scales made elsewhere.  The codes are used where they are if their rows start at multiples of 16 bytes
        (and the last row's memory reaches to the next multiple), and copied otherwise."""
        checked = checked_codes(codes, scales, block_rows)
        return BlockScaledTensor(checked, scales, block_rows, codes.shape, checked)

    @staticmethod
    def from_quantized(quantized, block_rows: int = 128) -> "BlockScaledTensor":
        """From a ``QuantTensor`` with codes (``Quantizer.quantize(weight, return_with_dequant=False, return_with_quant=True)``:
        asked for together, the codes share memory with the de-quantized tensor) of a quantizer with
        dtype ``sfp8_e4m3_nan``, float32 scales and group shapes ((block_rows, 128),): calibrated weights."""
        codes = quantized.qdata
        if codes is None or quantized.scale is None:
            raise ValueError("the quantized tensor holds no codes: ask for return_with_dequant=False, return_with_quant=True")
        codes = codes.reshape(-1, codes.shape[-1])
        grid = (-(-codes.shape[0] // block_rows), -(-codes.shape[1] // 128))
        scales = quantized.scale.data
        # (groups along an axis come with an axis of size 1 behind them; the last pair belongs to the columns)
        columns = scales.shape[-2] if scales.ndim > 2 else scales.shape[-1] if scales.ndim else 1
        if scales.numel() != grid[0] * grid[1] or columns != grid[1]:
            raise ValueError(f"scales of shape {tuple(scales.shape)}, {grid[0]} x {grid[1]} blocks of {block_rows} x 128")
        if quantized.zero is not None and bool(torch.as_tensor(quantized.zero).ne(0).any()):
            raise ValueError("the quantized tensor has zero points")
        narrow = codes.to(torch.float8_e4m3fn)
        if not torch.equal(narrow.to(codes.dtype), codes):
            raise ValueError("the codes are not values of e4m3")
        return BlockScaledTensor.from_codes(narrow, scales.reshape(grid).to(torch.float32), block_rows)
