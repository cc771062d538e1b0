"""Gated blocks, projections and dropout past 2^32 elements: the rows at the far end come out as the same rows by
themselves do, or as the formula has them."""
from __future__ import annotations

import pytest
import torch

from soklyn_amd import abi, dropout
from soklyn_amd.gated import Gated
from soklyn_amd.residual import Projection
from tests.ffn_helpers import ACTS, U, check, half_step, slope, ungate_ref, within

pytestmark = pytest.mark.gpu
FAR = (1 << 32) + 12345
F16, F32 = torch.float16, torch.float32


@pytest.fixture(autouse=True)
def memory():
    if torch.cuda.mem_get_info()[0] < 200 << 30:
        pytest.skip("needs 200 GB of free GPU memory")
    yield
    torch.cuda.synchronize()
    torch.cuda.empty_cache()


def rows_of(cols):
    return -(-FAR // cols)


def far(rows, cols, dtype, seed, std=1.0):
    """Zeros, random in the first and last 4 rows."""
    v = torch.zeros((rows, cols), dtype=dtype, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(seed)
    for at in (slice(0, 4), slice(rows - 4, rows)):
        v[at] = (torch.randn((4, cols), generator=g, device="cuda") * std).to(dtype)
    return v


def ends(t):
    return torch.cat([t[:4], t[-4:]])


def drawn(rows, at, cols, p, seed):
    """The dropout factors of rows `at`, by the formula."""
    r = torch.tensor(at, dtype=torch.int64)[:, None]
    c = torch.arange(cols, dtype=torch.int64)[None, :]
    low = 0xFFFFFFFF
    s = (r * 1103515245 & low) ^ (seed + 7 * r & low) ^ (c * 0x4C957F2D & low)
    s = s ^ (s >> 17)
    s = s * 1103515245 + 12345 & low
    s = (s ^ (s >> 15)).float() / 2.0 ** 32
    q = torch.tensor(p)
    return torch.where(s >= q, 1.0 / (1.0 - q.double()), 0.0)


def last(rows):
    return list(range(4)) + list(range(rows - 4, rows))


@pytest.mark.parametrize("cols", [8192, 8191])
def test_dropout(ctx, cols):
    rows = rows_of(cols)
    x = far(rows, cols, F16, 1)
    want = ends(x).double().cpu() * drawn(rows, last(rows), cols, 0.25, 9)
    dropout.apply(ctx, x, x, 0.25, 9)
    torch.cuda.synchronize()
    check(ends(x), (want, 2 * U * want.abs()), F16, "out")


@pytest.mark.parametrize("cols", [4096, 4095])
def test_error_of_a_projection(ctx, cols):
    rows = rows_of(cols)
    dh, z = far(rows, cols, F32, 1, 64.0), far(rows, cols, F16, 2)
    d, d_h = torch.empty_like(dh), torch.empty_like(z)
    Projection(ctx, None, outputs=cols, half=True, act=abi.ACT_SILU, dropout=0.25).error(dh, z, d, d_prenorm_h=d_h, seed=9)
    torch.cuda.synchronize()
    g, zz = ends(dh).double().cpu() * drawn(rows, last(rows), cols, 0.25, 9), ends(z).double().cpu()
    check(ends(d), (g * slope(abi.ACT_SILU, zz), g.abs() * 4 * (16 + 4 * zz.abs()) * U * (1 + zz.abs())), F32, "d")
    assert torch.equal(ends(d_h), ends(d).half())


def test_forward(ctx):
    """Output and caches past 2^32 elements on the kernels of large batches; K 64."""
    k, n = 64, 8192
    rows = -(-rows_of(n) // 256) * 256
    x = far(rows, k, F16, 1)
    g = torch.Generator(device="cuda").manual_seed(5)
    wg, wu = (torch.randn((k, n), generator=g, device="cuda").to(F16) / 8 for _ in range(2))
    out, a, u = (torch.empty((rows, n), dtype=F16, device="cuda") for _ in range(3))
    Gated(ctx, wg, wu, outputs=n, half=True).forward(x, out, a=a, u=u)
    h = torch.empty((rows, n), dtype=F16, device="cuda")
    Projection(ctx, wg, outputs=n, half=True, dropout=0.25).forward(x, a, h, seed=9)
    torch.cuda.synchronize()
    za, zu = (ends(x).double() @ w.double() for w in (wg, wu))
    size = ends(x).double().abs() @ wg.double().abs()
    bound = (k + 64) * U * size
    within(ends(a), za, bound + half_step(za, F16), "a")
    want = ACTS[abi.ACT_SILU](za, 0) * zu
    within(ends(out), want, 2 * (1.1 * bound * zu.abs() + za.abs() * bound + 64 * U * (1 + za.abs()) * zu.abs()) + half_step(want, F16), "out")
    f = drawn(rows, last(rows), n, 0.25, 9).cuda()
    want = ends(a).double() + f * za
    within(ends(h), want, f * bound + 8 * U * (want.abs() + za.abs()) + half_step(want, F16) * 1.01, "h")
    assert not bool(out[4:-4].any()) and not bool(u[4:-4].any())   # rows of zeros


def test_error_from_the_layer_above(ctx):
    k, n = 64, 4096
    rows = -(-rows_of(n) // 256) * 256
    d, a, u = far(rows, k, F16, 1, 8.0), far(rows, n, F16, 2), far(rows, n, F16, 3)
    g = torch.Generator(device="cuda").manual_seed(5)
    w = torch.randn((n, k), generator=g, device="cuda").to(F16) / 8
    dg, du = (torch.empty((rows, n), device="cuda") for _ in range(2))
    dg_h, du_h = (torch.empty((rows, n), dtype=F16, device="cuda") for _ in range(2))
    Gated(ctx, None, None, outputs=n, half=True).hidden_error(d, w, a, u, dg=dg, du=du, dg_h=dg_h, du_h=du_h)
    torch.cuda.synchronize()
    s, ds = ends(d).double() @ w.double().t().contiguous(), (k + 64) * U * (ends(d).double().abs() @ w.double().t().contiguous().abs())
    ref = ungate_ref(s, ds, ends(a), ends(u), abi.ACT_SILU)
    for name, got, h in (("dg", dg, dg_h), ("du", du, du_h)):
        check(ends(got), ref[name], F32, name)
        assert torch.equal(ends(h), ends(got).half()) and not bool(got[4:-4].any())
