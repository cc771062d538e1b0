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
    """One join: its norms' parameters (tensors [1 x cols] of the blocks' type, held by reference:
    an update in place is seen by the next call), gate activation and residual scale.  Calls of one
    Join share its workspace and follow each other on one stream."""

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
        self._work = None

    def _param(self, name: str, wanted: bool) -> int | None:
        t = getattr(self, name)
        return abi.need(name, t, self.dtype, (1, self.cols), self.ctx.device) if wanted and t is not None else None

    def _params(self):
        post, pre = self.post_norm, self.pre_norm
        return (self._param("post_w", post != _NONE), self._param("post_b", post == _LAYER),
                self._param("pre_w", pre != _NONE), self._param("pre_b", pre == _LAYER))

    def _maybe(self, name, t, dtype, shape):
        return None if t is None else abi.need(name, t, dtype, shape, self.ctx.device)

    def _gate(self, gate, rows):
        if gate is None:
            return None, 0
        if gate.shape[0] not in (1, rows):
            raise ValueError(f"gate: 1 or {rows} rows are wanted, got {gate.shape[0]}")
        return abi.need("gate", gate, self.dtype, (gate.shape[0], self.cols), self.ctx.device), gate.shape[0]

    def forward(self, x: torch.Tensor | None, y: torch.Tensor | None, gate: torch.Tensor | None = None, *,
                h: torch.Tensor | None = None, n: torch.Tensor | None = None, stats: torch.Tensor | None = None):
        """Writes h (the stream's type), n (the blocks' type) and stats (fp32 [4 x rows], what the
        backward reads), those that are given; h may be x and n may be y."""
        first = x if x is not None else y
        if first is None:
            raise ValueError("x, y or both are wanted")
        rows = first.shape[0]
        wide = (rows, self.cols)
        g, gate_rows = self._gate(gate, rows)
        abi.call("skl_residual_forward", self.ctx.h, int(self.half), int(self.half_stream), rows, self.cols,
                 self.post_norm if y is not None else _NONE, self.pre_norm, self.gate_act, gate_rows, self.scale,
                 self._maybe("x", x, self.stream_dtype, wide), self._maybe("y", y, self.dtype, wide), g,
                 *self._params(), self._maybe("h", h, self.stream_dtype, wide),
                 self._maybe("n", n, self.dtype, wide), self._maybe("stats", stats, torch.float32, (4, rows)))
        return h, n

    def backward(self, h: torch.Tensor | None, y: torch.Tensor | None, gate: torch.Tensor | None, stats: torch.Tensor,
                 dn: torch.Tensor | None, dh: torch.Tensor | None, *, dx: torch.Tensor | None = None,
                 dy: torch.Tensor | None = None, dgate: torch.Tensor | None = None,
                 dparam: torch.Tensor | None = None, work: torch.Tensor | None = None):
        """Writes those of dx, dy, dgate (of gate's shape) and dparam ([4 x cols]: post_w, post_b,
        pre_w, pre_b) that are given, all fp32, from dn and dh (fp32).  work: a float tensor of at
        least skl_residual_work_bytes, where not the Join's own."""
        rows = stats.shape[1]
        wide, f32 = (rows, self.cols), torch.float32
        g, gate_rows = self._gate(gate, rows)
        if dgate is not None and gate is None:
            raise ValueError("dgate: there is no gate")
        size = 0
        if dparam is not None or (dgate is not None and gate_rows == 1):
            size = abi.load().skl_residual_work_bytes(rows, self.cols)
            if work is None:
                if self._work is None or self._work.numel() * 4 < size:
                    if self._work is not None:
                        self.ctx.synchronize()   # a call may still write the smaller one
                    self._work = torch.empty(size // 4, device=f"cuda:{self.ctx.device}", dtype=f32)
                work = self._work
            size = work.numel() * 4
        post_w, post_b, pre_w, _ = self._params()
        abi.call("skl_residual_backward", self.ctx.h, int(self.half), int(self.half_stream), rows, self.cols,
                 self.post_norm if y is not None else _NONE, self.pre_norm, self.gate_act, gate_rows, self.scale,
                 self._maybe("h", h, self.stream_dtype, wide), self._maybe("y", y, self.dtype, wide), g, post_w,
                 post_b, pre_w, abi.need("stats", stats, f32, (4, rows), self.ctx.device),
                 self._maybe("dn", dn, f32, wide), self._maybe("dh", dh, f32, wide), self._maybe("dx", dx, f32, wide),
                 self._maybe("dy", dy, f32, wide), self._maybe("dgate", dgate, f32, (gate_rows, self.cols)),
                 self._maybe("dparam", dparam, f32, (4, self.cols)),
                 None if not size else abi.need("work", work, f32, (size // 4,), self.ctx.device), size)
