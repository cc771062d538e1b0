"""Joins between the blocks of a residual network, over skl_residual_forward / _backward, and the
projection into its stream, over skl_dense_forward_residual / skl_dense_residual_error.

    u = post(y);  h = scale * x + gate_act(gate) * u;  n = pre(h)

`y` is the output of a block, `x` and `h` the residual stream before and behind it and `n` the
input of the next block.

    h = scale * stream + drop(act(x W + b))

All calls run on the context's stream; tensors are contiguous and on
its GPU, as for a DeviceBlock.
"""
from __future__ import annotations

import ctypes as C
import threading

import torch

from . import abi

_NONE, _RMS, _LAYER = abi.NORM_DISABLED, abi.NORM_RMS, abi.NORM_LAYER


class Join:
    """One join: its norms' parameters (tensors [1 x cols] of the blocks' type, held by reference and
    read at each call, so an update in place is seen), gate activation and residual scale.  Calls of
    one Join that are given no workspace share its own and follow each other on one stream."""

    def __init__(self, ctx: abi.Context, cols: int, *, half: bool = False, half_stream: bool = False,
                 post_norm: int = _NONE, pre_norm: int = _RMS, gate_act: int = abi.ACT_IDENTITY, scale: float = 1.0,
                 post_w: torch.Tensor | None = None, post_b: torch.Tensor | None = None,
                 pre_w: torch.Tensor | None = None, pre_b: torch.Tensor | None = None):
        self.ctx, self.cols = ctx, cols
        self.half, self.half_stream = half, half_stream
        self.post_norm, self.pre_norm, self.gate_act, self.scale = post_norm, pre_norm, gate_act, scale
        self.dtype = torch.float16 if half else torch.float32
        self.stream_dtype = torch.float16 if half_stream else torch.float32
        self.post_w, self.post_b, self.pre_w, self.pre_b = post_w, post_b, pre_w, pre_b
        self._call = abi.load().skl_residual_forward, abi.load().skl_residual_backward
        self._work = []
        for name, t in zip(("post_w", "post_b", "pre_w", "pre_b"), (post_w, post_b, pre_w, pre_b)):
            if t is not None:
                abi.need(name, t, self.dtype, (1, cols), ctx.device)

    def _params(self):
        return [None if t is None else t.data_ptr() for t in (self.post_w, self.post_b, self.pre_w, self.pre_b)]

    def _addresses(self, tensors):
        """The tensors' addresses (None for None), each (name, tensor, type, shape) as it is wanted."""
        dev = self.ctx.device
        got = []
        for name, t, dtype, shape in tensors:
            if t is None:
                got.append(None)
            elif t.dtype is dtype and t.shape == shape and t.is_contiguous() and t.get_device() == dev:
                got.append(t.data_ptr())
            else:
                abi.need(name, t, dtype, shape, dev)   # raises
        return got

    def _gate_rows(self, gate, rows):
        if gate is None:
            return 0
        n = gate.shape[0]
        if n != 1 and n != rows:
            raise ValueError(f"gate: 1 or {rows} rows are wanted, got {n}")
        return n

    def forward(self, x: torch.Tensor | None, y: torch.Tensor | None, gate: torch.Tensor | None = None, *,
                h: torch.Tensor | None = None, n: torch.Tensor | None = None, stats: torch.Tensor | None = None):
        """Writes h (the stream's type), n (the blocks' type) and stats (fp32 [4 x rows], what the
        backward reads), those that are given; h may be x and n may be y."""
        first = x if x is not None else y
        if first is None:
            raise ValueError("x, y or both are wanted")
        rows, cols, t, r = first.shape[0], self.cols, self.dtype, self.stream_dtype
        wide, gates = (rows, cols), self._gate_rows(gate, rows)
        px, py, pg, ph, pn, ps = self._addresses((("x", x, r, wide), ("y", y, t, wide), ("gate", gate, t, (gates, cols)),
                                                  ("h", h, r, wide), ("n", n, t, wide),
                                                  ("stats", stats, torch.float32, (4, rows))))
        rc = self._call[0](self.ctx.h, self.half, self.half_stream, rows, cols, self.post_norm if py else _NONE,
                           self.pre_norm, self.gate_act, gates, self.scale, px, py, pg, *self._params(), ph, pn, ps)
        if rc:
            raise abi.SklError("skl_residual_forward", rc)
        return h, n

    def backward(self, h: torch.Tensor | None, y: torch.Tensor | None, gate: torch.Tensor | None, stats: torch.Tensor,
                 dn: torch.Tensor | None, dh: torch.Tensor | None, *, dx: torch.Tensor | None = None,
                 dy: torch.Tensor | None = None, dgate: torch.Tensor | None = None,
                 dparam: torch.Tensor | None = None, work: torch.Tensor | None = None):
        """Writes those of dx, dy, dgate (of gate's shape) and dparam ([4 x cols]: post_w, post_b,
        pre_w, pre_b) that are given, all fp32, from dn and dh (fp32).  work: a float tensor of at
        least skl_residual_work_bytes, where not the Join's own."""
        rows, cols, f32 = stats.shape[1], self.cols, torch.float32
        wide, gates = (rows, cols), self._gate_rows(gate, rows)
        if dgate is not None and gate is None:
            raise ValueError("dgate: there is no gate")
        size = 0
        if dparam is not None or (dgate is not None and gates == 1):
            size = abi.load().skl_residual_work_bytes(rows, cols)
            if work is None:
                if not self._work or self._work[-1].numel() * 4 < size:
                    # (smaller ones stay: calls in flight and captured ones write there)
                    self._work.append(torch.empty(size // 4, device=f"cuda:{self.ctx.device}", dtype=f32))
                work = self._work[-1]
            size = work.numel() * 4
        ph, py, pg, ps, pdn, pdh, pdx, pdy, pdg, pdp, pw = self._addresses((
            ("h", h, self.stream_dtype, wide), ("y", y, self.dtype, wide), ("gate", gate, self.dtype, (gates, cols)),
            ("stats", stats, f32, (4, rows)), ("dn", dn, f32, wide), ("dh", dh, f32, wide), ("dx", dx, f32, wide),
            ("dy", dy, f32, wide), ("dgate", dgate, f32, (gates, cols)), ("dparam", dparam, f32, (4, cols)),
            ("work", work if size else None, f32, (size // 4,))))
        post_w, post_b, pre_w, _ = self._params()
        rc = self._call[1](self.ctx.h, self.half, self.half_stream, rows, cols, self.post_norm if py else _NONE,
                           self.pre_norm, self.gate_act, gates, self.scale, ph, py, pg, post_w, post_b, pre_w, ps, pdn,
                           pdh, pdx, pdy, pdg, pdp, pw, size)
        if rc:
            raise abi.SklError("skl_residual_backward", rc)


class Projection(abi.Tracked):
    """A layer whose result, with dropout, is added to the stream: weights w [inputs x outputs] and bias b
    [1 x outputs] (or None) of the blocks' type, held by reference.  No mask is stored: the backward draws
    it again from the seed.  w may be None where only the backward is called.  Calls share a workspace and
    follow each other on one stream; the object, which holds it, outlives the graphs that its calls were
    captured into."""

    def __init__(self, ctx: abi.Context, w: torch.Tensor | None, b: torch.Tensor | None = None, *, outputs: int,
                 half: bool = False, act: int = abi.ACT_IDENTITY, leaky: float = 0.0, dropout: float = 0.0,
                 scale: float = 1.0):
        self.ctx, self.outputs, self.half, self.act, self.leaky = ctx, outputs, half, act, leaky
        self.dropout, self.scale = dropout, scale
        self.dtype = torch.float16 if half else torch.float32
        self.inputs = 1 if w is None else w.shape[0]
        self.w, self.b, self.work = w, b, abi.Workspace(ctx)
        self._weights()
        self._call = abi.load().skl_dense_forward_residual, abi.load().skl_dense_residual_error
        self._local = threading.local()   # descriptors, one per thread

    def _weights(self):
        """The addresses of w and b, looked at each time: a tensor held by reference may have become another."""
        t, n, dev, w, b = self.dtype, self.outputs, self.ctx.device, self.w, self.b
        return (None if w is None else abi.need("w", w, t, (self.inputs, n), dev),
                None if b is None else abi.need("b", b, t, (1, n), dev))

    def _desc(self, rows: int) -> abi.SklDenseDesc:
        own = self._local.__dict__
        key = rows, self.changes
        if own.get("key") != key:
            d = own["desc"] = abi.SklDenseDesc()
            own["ref"] = C.byref(d)
            d.dtype, d.inputs, d.outputs, d.max_batch = int(self.half), self.inputs, self.outputs, rows
            d.act, d.leaky, d.mask_coeff, d.is_training = self.act, self.leaky, self.dropout, 1
            own["key"] = key
        d = own["desc"]
        d.w, d.b = self._weights()
        return d

    def forward(self, x: torch.Tensor, stream: torch.Tensor | None, h: torch.Tensor, *, preact: torch.Tensor | None = None,
                seed: int = 0) -> torch.Tensor:
        """h [rows x outputs] (fp32, or fp16 with fp16 layers) from x [rows x inputs] and the stream of h's type;
        h may be stream.  preact [rows x outputs], where given, keeps x W + b for the backward."""
        rows, dev, r = x.shape[0], self.ctx.device, h.dtype
        wide = (rows, self.outputs)
        if r is not torch.float32 and r is not self.dtype:
            raise ValueError(f"h: {torch.float32} or {self.dtype} is wanted, got {r}")
        d = self._desc(rows)
        d.preact = None if preact is None else abi.need("preact", preact, self.dtype, wide, dev)
        work = self.work.product(int(self.half), rows, self.inputs, self.outputs, 1)
        rc = self._call[0](self.ctx.h, self._local.ref, abi.need("x", x, self.dtype, (rows, self.inputs), dev), rows,
                           self.inputs, rows, self.dropout != 0.0, seed & 0xFFFFFFFF, r is torch.float16, self.scale,
                           None if stream is None else abi.need("stream", stream, r, wide, dev),
                           abi.need("h", h, r, wide, dev), *work)
        if rc:
            raise abi.SklError("skl_dense_forward_residual", rc)
        return h

    def error(self, dh: torch.Tensor, preact: torch.Tensor | None, d_prenorm: torch.Tensor, *,
              d_prenorm_h: torch.Tensor | None = None, dx: torch.Tensor | None = None, seed: int = 0):
        """From dh (fp32), the gradient of h: that of x W + b in d_prenorm (fp32) and, for fp16 layers, its copy
        d_prenorm_h; dx = scale * dh where given (it may be dh)."""
        rows, dev, f32 = dh.shape[0], self.ctx.device, torch.float32
        wide = (rows, self.outputs)
        d = self._desc(rows)
        d.preact = None if preact is None else abi.need("preact", preact, self.dtype, wide, dev)
        d.d_prenorm = abi.need("d_prenorm", d_prenorm, f32, wide, dev)
        d.d_prenorm_h = None if d_prenorm_h is None else abi.need("d_prenorm_h", d_prenorm_h, torch.float16, wide, dev)
        rc = self._call[1](self.ctx.h, self._local.ref, abi.need("dh", dh, f32, wide, dev), rows, self.dropout != 0.0,
                           seed & 0xFFFFFFFF, self.scale, None if dx is None else abi.need("dx", dx, f32, wide, dev))
        if rc:
            raise abi.SklError("skl_dense_residual_error", rc)
