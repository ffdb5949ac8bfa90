"""Linear layers that run on 8-bit values (no counterpart in the reference, whose quantized linears multiply
de-quantized weights): ``block_scaled_linear`` and the module that stands in for an ``nn.Linear``."""

from __future__ import annotations

import torch
import torch.nn as nn

from ...data.block import BlockScaledTensor
from ...engine_fp8 import block_product, look_over

__all__ = ["block_scaled_linear", "Fp8BlockLinear"]


def block_scaled_linear(x: torch.Tensor | BlockScaledTensor, weight: BlockScaledTensor, bias: torch.Tensor | None = None,
                        *, dtype: torch.dtype | None = None) -> torch.Tensor:
    """``x @ weight.T + bias`` on the codes: x [..., K] in 1 x 128 blocks (a plain tensor is quantized first), weight [N][K]
    in 128 x 128 blocks.  Each block's products are summed on the matrix cores and scaled and added in float32; the sum is
    rounded once to ``dtype`` (default: x's own type, bfloat16 if x comes quantized).  For 16-bit results the matrix cores cut
    products off below 2^-13 of the largest of each eight (about 1.5e-5 of the sums for normally distributed codes); for
    float32 the block's sums are full float32, at half the rate."""
    if not isinstance(x, BlockScaledTensor):
        dtype = x.dtype if dtype is None else dtype
        x = BlockScaledTensor.quantize(x)
    if x.block_rows != 1 or weight.block_rows != 128:
        raise ValueError("x has a scale for each row and 128 columns, weight for each 128 x 128 block")
    x_codes, w_codes = x.codes, weight.codes
    if x.looked_over is not x_codes or weight.looked_over is not w_codes:
        look_over(x_codes, w_codes)
    y = block_product(x_codes, x.scales, w_codes, weight.scales, bias, torch.bfloat16 if dtype is None else dtype)
    return y if len(x.shape) == 2 else y.view(*x.shape[:-1], y.shape[-1])


class Fp8BlockLinear(nn.Module):
    """A linear whose weight is kept as e4m3 codes in 128 x 128 blocks and whose input is quantized in 1 x 128 blocks."""

    def __init__(self, weight: BlockScaledTensor, bias: torch.Tensor | None = None) -> None:
        super().__init__()
        if weight.block_rows != 128:
            raise ValueError("the weight has a scale for each 128 x 128 block")
        self.out_features, self.in_features = weight.codes.shape
        # bytes: a module's .half() or .to(dtype) converts its floating-point buffers, and e4m3 counts as one
        pitch = -(-self.in_features // 16) * 16
        codes = torch.zeros((self.out_features, pitch), dtype=torch.uint8, device=weight.codes.device)
        codes[:, :self.in_features] = weight.codes.view(torch.uint8)
        self.register_buffer("codes", codes)
        self.register_buffer("scales", weight.scales.contiguous())
        self.bias = None if bias is None else nn.Parameter(bias.detach().clone(), requires_grad=False)

    def _apply(self, fn, recurse=True):
        def bits(t):
            if t is not self.scales and t is not self.codes:
                return fn(t)
            held = t.view(torch.int32) if t is self.scales else t
            moved = fn(held)
            if moved.dtype != held.dtype:
                raise TypeError(f"the codes and scales of an 8-bit linear cannot become {moved.dtype}: convert with .to(), which leaves them as they are")
            return moved.view(t.dtype)

        return super()._apply(bits, recurse)

    @property
    def weight(self) -> BlockScaledTensor:
        codes = self.codes.view(torch.float8_e4m3fn)[:, :self.in_features]
        return BlockScaledTensor(codes, self.scales, 128, codes.shape, codes)

    @staticmethod
    def from_linear(linear: nn.Linear) -> "Fp8BlockLinear":
        bias = None if linear.bias is None else linear.bias.data
        return Fp8BlockLinear(BlockScaledTensor.quantize(linear.weight.data, block_rows=128), bias)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return block_scaled_linear(x, self.weight, self.bias)
