"""Joins between the blocks of a residual network, over skl_residual_forward / _backward.

    u = post(y);  h = scale * x + gate_act(gate) * u;  n = pre(h)

`y` is the output of a block, `x` and `h` the residual stream before and behind it and `n` the
input of the next block.  All calls run on the context's stream; tensors are contiguous and on
its GPU, as for a DeviceBlock.
"""
from __future__ import annotations

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
