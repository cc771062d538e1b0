"""Dropout without a stored mask, over skl_dropout: an element is kept, times 1 / (1 - p), or becomes 0 as
the seed and its row and column say, drawn as a DeviceBlock's forward draws its own."""
from __future__ import annotations

import torch

from . import abi


def apply(ctx: abi.Context, src: torch.Tensor, out: torch.Tensor, p: float, seed: int) -> torch.Tensor:
    """The elements of src [rows x cols] (fp16 or fp32) that stay, in out, which may be src.  On the gradient of
    out, with the same p and seed, this is its own backward."""
    t, shape, dev = src.dtype, src.shape, ctx.device
    if t is not torch.float16 and t is not torch.float32:
        raise ValueError(f"fp16 or fp32 values are wanted, got {t}")
    rows, cols = shape
    rc = abi.load().skl_dropout(ctx.h, t is torch.float16, rows, cols, p, seed & 0xFFFFFFFF, abi.need("src", src, t, shape, dev),
                                abi.need("out", out, t, shape, dev))
    if rc:
        raise abi.SklError("skl_dropout", rc)
    return out
