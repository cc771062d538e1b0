"""Products of gated blocks and projections whose operands lie differently: one of them alone an element off its
boundary, as views of one flat buffer of parameters are.  Even widths, so that the rows' pitch hides nothing.  Against
64 bits, with the bounds of ffn_helpers."""
from __future__ import annotations

import pytest
import torch

from soklyn_amd import abi
from soklyn_amd.gated import Gated
from soklyn_amd.residual import Projection
from tests.ffn_helpers import LEAKY, check, filled, gated_ref, odd_base, product, ungate_ref, values, within
from tests.test_gpu_gated import routed

pytestmark = pytest.mark.gpu
F16, F32 = torch.float16, torch.float32

# the form through registers on each of its tiles, as planned on each (few rows over a long k, 16, 32, 64 and a pair's
# 64x32 tiles, 128x128 and 256x256 direct-to-LDS ones), and copies
FORMS = [("wave:16:16", 20, 40, 24), ("wave:32:8", 70, 200, 68), ("wave:64:4", 70, 200, 68), (None, 1, 4096, 264), (None, 3, 40, 24),
         (None, 200, 128, 256), (None, 200, 600, 260), (None, 500, 1024, 1026), (None, 3000, 1024, 1024), (None, 8192, 256, 1024),
         ("copied", 130, 80, 132)]
IDS = [f"{r or 'planned'}-{m}x{k}x{n}" for r, m, k, n in FORMS]


def on(monkeypatch, ctx, route):
    return routed(monkeypatch, ctx, route) if route else ctx


# the epilogue's own tensors leave the product's form as it is
FORWARD = ([(*f, off) for f in FORMS for off in ("x", "wg", "wu")] +
           [(*f, off) for f in FORMS if f[0] is None for off in ("bg", "bu", "out", "a", "u")])


@pytest.mark.parametrize("route,m,k,n,off", FORWARD)
def test_gated_forward(monkeypatch, ctx, route, m, k, n, off):
    t = {"x": values((m, k), F16, 1), "wg": values((k, n), F16, 2, k ** -0.5), "wu": values((k, n), F16, 3, k ** -0.5),
         "bg": values((1, n), F16, 4, 0.3), "bu": values((1, n), F16, 5, 0.3)} | {v: filled((m, n), F16) for v in ("out", "a", "u")}
    t[off] = odd_base(t[off])
    assert t[off].data_ptr() % 4 == 2 and all(v.data_ptr() % 16 == 0 for name, v in t.items() if name != off)
    op = Gated(on(monkeypatch, ctx, route), t["wg"], t["wu"], t["bg"], t["bu"], outputs=n, half=True, act=abi.ACT_SILU)
    op.forward(t["x"], t["out"], a=t["a"], u=t["u"])
    torch.cuda.synchronize()
    for name, ref in gated_ref(t["x"], t["wg"], t["wu"], t["bg"], t["bu"], abi.ACT_SILU).items():
        check(t[name], ref, F16, name)


@pytest.mark.parametrize("off", ["dg", "du", "wg", "wu"])
@pytest.mark.parametrize("route,m,n,k", FORMS, ids=IDS)   # columns and k change places
def test_gated_input_grad(monkeypatch, ctx, route, m, n, k, off):
    t = {"dg": values((m, n), F16, 1, 64.0), "du": values((m, n), F16, 2, 64.0), "wg": values((k, n), F16, 3, k ** -0.5),
         "wu": values((k, n), F16, 4, k ** -0.5)}
    t[off] = odd_base(t[off])
    dx = filled((m, k), F32)
    Gated(on(monkeypatch, ctx, route), t["wg"], t["wu"], outputs=n, half=True).input_grad(t["dg"], t["du"], dx)
    torch.cuda.synchronize()
    want, bound = product(torch.cat([t["dg"], t["du"]], 1), torch.cat([t["wg"], t["wu"]], 1).t())
    within(dx, want, bound, "dx")


@pytest.mark.parametrize("off", ["d", "w"])
@pytest.mark.parametrize("route,m,k,n", FORMS, ids=IDS)
def test_gated_hidden_error(monkeypatch, ctx, route, m, k, n, off):
    t = {"d": values((m, k), F16, 1, 64.0), "w": values((n, k), F16, 2, k ** -0.5)}
    t[off] = odd_base(t[off])
    a, u = values((m, n), F16, 3), values((m, n), F16, 4)
    to = {v: filled((m, n), F32) for v in ("dg", "du")} | {v: filled((m, n), F16) for v in ("dg_h", "du_h")}
    Gated(on(monkeypatch, ctx, route), None, None, outputs=n, half=True, act=abi.ACT_SILU).hidden_error(t["d"], t["w"], a, u, **to)
    torch.cuda.synchronize()
    ref = ungate_ref(*product(t["d"], t["w"].t()), a, u, abi.ACT_SILU)
    for name in ("dg", "du"):
        check(to[name], ref[name], F32, name)


@pytest.mark.parametrize("off", ["x", "w"])
@pytest.mark.parametrize("route,m,k,n", FORMS, ids=IDS)
def test_projection(monkeypatch, ctx, route, m, k, n, off):
    t = {"x": values((m, k), F16, 1), "w": values((k, n), F16, 2, k ** -0.5)}
    t[off] = odd_base(t[off])
    h = filled((m, n), F32)
    Projection(on(monkeypatch, ctx, route), t["w"], outputs=n, half=True, leaky=LEAKY).forward(t["x"], None, h)
    torch.cuda.synchronize()
    check(h, product(t["x"], t["w"]), F32, "h")
