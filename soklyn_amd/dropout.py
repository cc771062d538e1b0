"""Dropout without a stored mask, over skl_dropout: an element is kept, times 1 / (1 - p), or becomes 0 as
the seed and its row and column say, drawn as a DeviceBlock's forward draws its own."""
from __future__ import annotations

import torch

from . import abi


def apply(ctx: abi.Context, src: torch.Tensor, out: torch.Tensor, p: float, seed: int) -> torch.Tensor:
    """The elements of src [rows x cols] (fp16 or fp32) that stay, in out, which may be src.  On the gradient of
    out, with the same p and seed, this is its own backward."""
    if src.dtype not in (torch.float16, torch.float32):
        raise ValueError(f"fp16 or fp32 values are wanted, got {src.dtype}")
    rows, cols = src.shape
    abi.call("skl_dropout", ctx.h, int(src.dtype is torch.float16), rows, cols, p, seed & 0xFFFFFFFF,
             abi.need("src", src, src.dtype, (rows, cols), ctx.device), abi.need("out", out, src.dtype, (rows, cols), ctx.device))
    return out
