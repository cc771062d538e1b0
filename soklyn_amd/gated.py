"""Gated feed-forward blocks, over skl_gated_forward and its backward calls.

    a = x Wg + bg;  u = x Wu + bu;  out = act(a) * u

`Gated` works on tensors at hand; `GatedBlock` on two DeviceBlocks, whose weights their own backward
updates.  All calls run on the context's stream; tensors are contiguous and on its GPU.
"""
from __future__ import annotations

import ctypes as C
import threading

import torch

from . import abi
from .devblock import DeviceBlock

_F32, _F16 = torch.float32, torch.float16


class Gated(abi.Tracked):
    """The weights wg and wu [inputs x outputs] and biases [1 x outputs] (or None) of both projections, held by
    reference; act is the gate's activation.  The weights may be None where only error_from_sum and hidden_error
    are called.  Calls share a workspace and follow each other on one stream; the object, which holds it,
    outlives the graphs that its calls were captured into."""

    def __init__(self, ctx: abi.Context, wg: torch.Tensor | None, wu: torch.Tensor | None, bg: torch.Tensor | None = None,
                 bu: torch.Tensor | None = None, *, outputs: int, half: bool = False, act: int = abi.ACT_SILU,
                 leaky: float = 0.0):
        self.ctx, self.outputs, self.half, self.act, self.leaky = ctx, outputs, half, act, leaky
        self.dtype = _F16 if half else _F32
        self.inputs = 1 if wg is None else wg.shape[0]
        self.wg, self.wu, self.bg, self.bu, self.work = wg, wu, bg, bu, abi.Workspace(ctx)
        self._weights()
        lib = abi.load()
        self._call = lib.skl_gated_forward, lib.skl_gated_error_from_sum, lib.skl_gated_hidden_error, lib.skl_gated_input_grad
        self._local = threading.local()   # descriptors, one set per thread

    def _weights(self):
        """The addresses of wg, wu, bg and bu, looked at each time: a tensor held by reference may have become another."""
        t, n, dev, need = self.dtype, self.outputs, self.ctx.device, abi.need
        wg, wu, bg, bu = self.wg, self.wu, self.bg, self.bu
        wide, row = (self.inputs, n), (1, n)
        return (None if wg is None else need("wg", wg, t, wide, dev), None if wu is None else need("wu", wu, t, wide, dev),
                None if bg is None else need("bg", bg, t, row, dev), None if bu is None else need("bu", bu, t, row, dev))

    def _descs(self, rows: int, weights: bool = True):
        """This thread's descriptors of gate, up and the layer above; weights: with the weights as they are now."""
        own = self._local.__dict__
        key = rows, self.changes
        if own.get("key") != key:
            if not own:
                own["d"] = tuple(abi.SklDenseDesc() for _ in range(3))
                own["refs"] = tuple(C.byref(x) for x in own["d"])
            for d in own["d"]:
                d.is_training, d.dtype, d.inputs, d.outputs, d.max_batch = 1, int(self.half), self.inputs, self.outputs, rows
            own["d"][0].act, own["d"][0].leaky = self.act, self.leaky
            own["key"] = key
        gate, up, above = own["d"]
        if weights:
            gate.w, up.w, gate.b, up.b = self._weights()
        return gate, up, above, own["refs"]

    def _at(self, name, t, dtype, shape):
        return None if t is None else abi.need(name, t, dtype, shape, self.ctx.device)

    def forward(self, x: torch.Tensor, out: torch.Tensor, *, a: torch.Tensor | None = None,
                u: torch.Tensor | None = None) -> torch.Tensor:
        """out [rows x outputs] from x [rows x inputs]; a and u (of out's shape), where given, are kept for the
        backward."""
        ctx, rows, t, k, n, need = self.ctx, x.shape[0], self.dtype, self.inputs, self.outputs, abi.need
        dev, wide = ctx.device, (rows, n)
        gate, up, _, (rg, ru, _) = self._descs(rows)
        gate.preact = None if a is None else need("a", a, t, wide, dev)
        up.preact = None if u is None else need("u", u, t, wide, dev)
        rc = self._call[0](ctx.h, rg, ru, need("x", x, t, (rows, k), dev), rows, k, rows,
                           None if out is None else need("out", out, t, wide, dev),
                           *self.work.product(int(self.half), rows, k, n, 2))
        if rc:
            raise abi.SklError("skl_gated_forward", rc)
        return out

    def _errors(self, rows, a, u, dg, du, dg_h, du_h):
        t, wide = self.dtype, (rows, self.outputs)
        gate, up, above, refs = self._descs(rows, False)
        for d, kept, g, h, n in ((gate, a, dg, dg_h, ("a", "dg", "dg_h")), (up, u, du, du_h, ("u", "du", "du_h"))):
            d.preact = self._at(n[0], kept, t, wide)
            d.d_prenorm = self._at(n[1], g, _F32, wide)
            d.d_prenorm_h = self._at(n[2], h, _F16, wide)
        return above, refs

    def error_from_sum(self, s: torch.Tensor, a: torch.Tensor, u: torch.Tensor, *, dg: torch.Tensor, du: torch.Tensor,
                       dg_h: torch.Tensor | None = None, du_h: torch.Tensor | None = None):
        """The gradients of both projections' results, dg and du (fp32; fp16 blocks also their copies), from s, that
        of out, and the kept a and u."""
        rows = s.shape[0]
        _, (rg, ru, _) = self._errors(rows, a, u, dg, du, dg_h, du_h)
        rc = self._call[1](self.ctx.h, rg, ru, self._at("s", s, _F32, (rows, self.outputs)), rows)
        if rc:
            raise abi.SklError("skl_gated_error_from_sum", rc)

    def hidden_error(self, above_d: torch.Tensor, above_w: torch.Tensor, a: torch.Tensor, u: torch.Tensor, *,
                     dg: torch.Tensor, du: torch.Tensor, dg_h: torch.Tensor | None = None,
                     du_h: torch.Tensor | None = None):
        """The same from the layer above: its gradient above_d [rows x n] and weights above_w [outputs x n], of the
        blocks' type."""
        (rows, n), t = above_d.shape, self.dtype
        above, (rg, ru, rn) = self._errors(rows, a, u, dg, du, dg_h, du_h)
        above.inputs, above.outputs = self.outputs, n
        above.w = self._at("above_w", above_w, t, (self.outputs, n))
        d = self._at("above_d", above_d, t, (rows, n))
        above.d_prenorm, above.d_prenorm_h = (None, d) if self.half else (d, None)
        rc = self._call[2](self.ctx.h, rg, ru, rn, rows, *self.work.gradient(int(self.half), rows, n, self.outputs, 1))
        if rc:
            raise abi.SklError("skl_gated_hidden_error", rc)

    def input_grad(self, dg: torch.Tensor, du: torch.Tensor, dx: torch.Tensor) -> torch.Tensor:
        """dx [rows x inputs] (fp32) from the gradients of both projections' results, of the blocks' type."""
        ctx, rows, t, n, half, need = self.ctx, dg.shape[0], self.dtype, self.outputs, self.half, abi.need
        dev, wide = ctx.device, (rows, n)
        gate, up, _, (rg, ru, _) = self._descs(rows)
        pg, pu = need("dg", dg, t, wide, dev), None if du is None else need("du", du, t, wide, dev)
        gate.d_prenorm, gate.d_prenorm_h, up.d_prenorm, up.d_prenorm_h = (None, pg, None, pu) if half else (pg, None, pu, None)
        rc = self._call[3](ctx.h, rg, ru, rows,
                           None if dx is None else need("dx", dx, _F32, (rows, self.inputs), dev),
                           *self.work.gradient(int(half), rows, n, self.inputs, 2))
        if rc:
            raise abi.SklError("skl_gated_input_grad", rc)
        return dx


class GatedBlock:
    """A gated block over two DeviceBlocks of one size without norms: the gate with its activation, up with
    Identity.  The kept a and u are their preact, the errors their d_prenorm."""

    def __init__(self, gate: DeviceBlock, up: DeviceBlock):
        self.ctx, self.gate, self.up, self.work = gate.ctx, gate, up, abi.Workspace(gate.ctx)

    def forward(self, x: torch.Tensor, batch: int, out: torch.Tensor, *, keep: bool = True) -> torch.Tensor:
        """out [batch x outputs] from the first `batch` rows of x; keep: a and u stay for the backward."""
        g, (rows, cols), dev = self.gate, x.shape, self.ctx.device
        how = "project" if keep else "serve"
        abi.call("skl_gated_forward", self.ctx.h, g._fill(how), self.up._fill(how),
                 abi.need("x", x, g.tdtype, (rows, cols), dev), rows, cols, batch,
                 abi.need("out", out, g.tdtype, (batch, g.outputs), dev),
                 *self.work.product(int(g.half), batch, g.inputs, g.outputs, 2))
        return out

    def error_from_sum(self, s: torch.Tensor, batch: int):
        g = self.gate
        abi.call("skl_gated_error_from_sum", self.ctx.h, g._fill("unproject"), self.up._fill("unproject"),
                 abi.need("s", s, _F32, (batch, g.outputs), self.ctx.device), batch)

    def hidden_error(self, nxt: DeviceBlock, batch: int):
        g = self.gate
        abi.call("skl_gated_hidden_error", self.ctx.h, g._fill("unproject"), self.up._fill("unproject"), nxt._fill("above"),
                 batch, *self.work.gradient(int(g.half), batch, nxt.outputs, g.outputs, 1))

    def input_grad(self, batch: int, out: torch.Tensor | None = None) -> torch.Tensor:
        g, dev = self.gate, self.ctx.device
        if out is None:
            out = torch.empty((batch, g.inputs), device=g.w.device, dtype=_F32)
        abi.call("skl_gated_input_grad", self.ctx.h, g._fill("above"), self.up._fill("above"), batch,
                 abi.need("out", out, _F32, (batch, g.inputs), dev),
                 *self.work.gradient(int(g.half), batch, g.outputs, g.inputs, 2))
        return out

    def backward(self, x: torch.Tensor, tc: abi.SklTrainCtx, step: int):
        """Both projections' weight gradients and updates, from the errors."""
        self.gate.backward(x, tc, step)
        self.up.backward(x, tc, step)
