"""Matrices as 4-bit microscaled floats (MXFP4) and layers that are served with 4-bit weights, over
skl_mxfp4_quantise, skl_mxfp4_dequantise and skl_dense_forward_mxfp4.

A matrix of n vectors of k elements is held as codes, uint8 [n x kp / 2], and scales, uint8
[n x kp / 32], kp = k rounded up to 128: two e2m1 floats to a byte, the first in its low half, and
2^(byte - 127) for each block of 32.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import abi
from .devblock import _ptr


def shapes(rows: int, cols: int, down: bool = False) -> tuple[tuple[int, int], tuple[int, int]]:
    """The shapes of the codes and scales of a [rows x cols] matrix whose vectors are its rows, or
    (down) its columns."""
    n, k = (cols, rows) if down else (rows, cols)
    kp = -(-k // 128) * 128
    return (n, kp // 2), (n, kp // 32)


def _type(t: torch.Tensor) -> int:
    if t.dtype not in (torch.float16, torch.float32):
        raise ValueError(f"fp16 or fp32 values are wanted, got {t.dtype}")
    return abi.F16 if t.dtype is torch.float16 else abi.F32


def quantise(ctx: abi.Context, src: torch.Tensor, *, down: bool = False, codes: torch.Tensor | None = None,
             scales: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """src [rows x cols] (fp16 or fp32) in 4 bits, along its rows or (down) its columns."""
    rows, cols = src.shape
    dev, (cs, ss) = ctx.device, shapes(rows, cols, down)
    dtype, p = _type(src), abi.need("src", src, src.dtype, (rows, cols), ctx.device)
    codes = torch.empty(cs, dtype=torch.uint8, device=src.device) if codes is None else codes
    scales = torch.empty(ss, dtype=torch.uint8, device=src.device) if scales is None else scales
    abi.call("skl_mxfp4_quantise", ctx.h, p, dtype, rows, cols, int(down),
             abi.need("codes", codes, torch.uint8, cs, dev), abi.need("scales", scales, torch.uint8, ss, dev))
    return codes, scales


def dequantise(ctx: abi.Context, codes: torch.Tensor, scales: torch.Tensor, out: torch.Tensor, *,
               down: bool = False) -> torch.Tensor:
    """The values of codes and scales, rounded to out's type, in out [rows x cols]."""
    rows, cols = out.shape
    dev, (cs, ss) = ctx.device, shapes(rows, cols, down)
    abi.call("skl_mxfp4_dequantise", ctx.h, abi.need("codes", codes, torch.uint8, cs, dev),
             abi.need("scales", scales, torch.uint8, ss, dev), rows, cols, int(down),
             abi.need("out", out, out.dtype, (rows, cols), dev), _type(out))
    return out


class Layer:
    """A layer that is only used, its weights in 4 bits: codes and scales of W [inputs x outputs],
    quantised down, with the bias, norm and activation of a DeviceBlock.  Holds the output, the
    norm's caches and a workspace, so its calls follow each other on one stream."""

    def __init__(self, ctx: abi.Context, inputs: int, outputs: int, max_batch: int, codes: torch.Tensor,
                 scales: torch.Tensor, *, half: bool = False, norm: int = abi.NORM_DISABLED,
                 act: int = abi.ACT_IDENTITY, leaky: float = 0.0, b: torch.Tensor | None = None,
                 norm_w: torch.Tensor | None = None, norm_b: torch.Tensor | None = None,
                 out: torch.Tensor | None = None):
        self.ctx, self.inputs, self.outputs, self.max_batch = ctx, inputs, outputs, max_batch
        self.dtype = t = torch.float16 if half else torch.float32
        dev, m, n = ctx.device, max_batch, outputs
        cs, ss = shapes(inputs, outputs, True)
        abi.need("codes", codes, torch.uint8, cs, dev)
        abi.need("scales", scales, torch.uint8, ss, dev)

        def own(name, given, shape, make):
            if given is None:
                return make(shape, device=f"cuda:{dev}", dtype=t)
            abi.need(name, given, t, shape, dev)
            return given

        self.codes, self.scales = codes, scales
        self.b = own("b", b, (1, n), torch.zeros)
        self.out = own("out", out, (m, n), torch.zeros)
        self.norm_w = self.norm_b = self.prenorm = self.centered = self.preact = self.predrop = self.norm_rstd = None
        if norm:
            self.norm_w = own("norm_w", norm_w, (1, n), torch.ones)
            self.norm_b = own("norm_b", norm_b, (1, n), torch.zeros)
            for cache in ("prenorm", "centered", "preact", "predrop"):
                setattr(self, cache, own(cache, None, (m, n), torch.zeros))
            self.norm_rstd = own("norm_rstd", None, (max(m, n),), torch.zeros)
        size = abi.load().skl_mxfp4_work_bytes(inputs, outputs, max_batch)
        self.work = torch.empty(size, device=f"cuda:{dev}", dtype=torch.uint8)
        d = self._desc = abi.SklDenseDesc()
        d.dtype, d.inputs, d.outputs, d.max_batch = abi.F16 if half else abi.F32, inputs, outputs, max_batch
        d.norm, d.act, d.leaky = norm, act, leaky
        for name in ("b", "out", "norm_w", "norm_b", "prenorm", "centered", "preact", "predrop", "norm_rstd"):
            setattr(d, name, _ptr(getattr(self, name)))
        self._ref = C.byref(d)

    def forward(self, x: torch.Tensor, batch: int) -> torch.Tensor:
        """The outputs of the first `batch` rows of x, in the first `batch` rows of out."""
        rows, cols = x.shape
        abi.call("skl_dense_forward_mxfp4", self.ctx.h, self._ref,
                 abi.need("x", x, self.dtype, (rows, cols), self.ctx.device), rows, cols, batch,
                 self.codes.data_ptr(), self.scales.data_ptr(), self.work.data_ptr() or None, self.work.numel())
        return self.out
