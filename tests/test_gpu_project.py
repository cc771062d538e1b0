"""The projection into the residual stream and dropout without a mask, against 64 bits and against the blocks'
own dropout; bounds as in ffn_helpers."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from soklyn_amd import abi, dropout
from soklyn_amd.devblock import DeviceBlock
from soklyn_amd.residual import Projection
from tests.ffn_helpers import ACTS, LEAKY, U, act_off, check, factors, filled, half_step, keeps, odd_base, product, slope, values, within
from tests.test_gpu_gated import FEW_ROWS, KERNELS, routed

pytestmark = pytest.mark.gpu
F32, F16 = torch.float32, torch.float16
PAIRS = [(F32, F32), (F16, F32), (F16, F16)]
IDS = ["f32", "f16_f32", "f16"]
TYPES = [F32, F16]


def project_case(ctx, m, k, n, t, r, act=abi.ACT_IDENTITY, bias=True, drop=0.25, scale=0.75, stream=True, keep=True,
                 in_place=False, place=lambda v: v, seed=0xDEADBEEF):
    w, b = place(values((k, n), t, m + n, k ** -0.5)), place(values((1, n), t, 5, 0.3)) if bias else None
    x, s = place(values((m, k), t, 7)), place(values((m, n), r, 8, 3.0)) if stream else None
    was = None if s is None else s.clone()
    h = s if in_place else place(filled((m, n), r))
    pre = place(filled((m, n), t))
    p = Projection(ctx, w, b, outputs=n, half=t == F16, act=act, leaky=LEAKY, dropout=drop, scale=scale)
    p.forward(x, s, h, preact=pre if keep else None, seed=seed)
    torch.cuda.synchronize()
    z, dz = product(x, w, b)
    z, dz = z.cpu(), dz.cpu()
    f = factors(m, n, drop, seed) if drop else torch.ones((m, n), dtype=torch.float64)
    v = ACTS[act](z, LEAKY) * f
    want = v + (scale * was.double().cpu() if stream else 0.0)
    check(h, (want, act_off(z, dz) * f + 4 * U * (v.abs() + want.abs() + (want - v).abs())), r, "h")
    if keep:
        check(pre, (z, dz), t, "preact")
    else:
        assert bool((pre == -7).all())


@pytest.mark.parametrize("t,r", PAIRS, ids=IDS)
@pytest.mark.parametrize("m,k,n", [(1, 1, 1), (1, 64, 64), (1, 129, 200), (2, 33, 65), (3, 5, 7), (5, 4096, 40), (16, 96, 80),
                                   (17, 31, 16), (33, 250, 100), (130, 257, 129), (256, 128, 256), (300, 72, 250),
                                   (1000, 65, 66)])
def test_forward_sizes(ctx, m, k, n, t, r):
    project_case(ctx, m, k, n, t, r, bias=n % 2 == 0, drop=0.25 if m % 2 else 0.0)


@pytest.mark.parametrize("t,r", PAIRS, ids=IDS)
@pytest.mark.parametrize("act", list(ACTS))
def test_forward_activations(ctx, act, t, r):
    project_case(ctx, 37, 64, 72, t, r, act=act)


@pytest.mark.parametrize("t,r", PAIRS, ids=IDS)
def test_forward_forms(ctx, t, r):
    project_case(ctx, 21, 40, 36, t, r, in_place=True)
    project_case(ctx, 21, 40, 37, t, r, in_place=True, keep=False)
    project_case(ctx, 21, 40, 36, t, r, stream=False)
    project_case(ctx, 21, 40, 35, t, r, stream=False, drop=0.0, keep=False)
    project_case(ctx, 20, 40, 24, t, r, place=odd_base)
    project_case(ctx, 9, 40, 24, t, r, drop=0.999, seed=1)


@pytest.mark.parametrize("route,t,m,k,n", KERNELS)
def test_forward_kernels(monkeypatch, ctx, route, t, m, k, n):
    c = routed(monkeypatch, ctx, route)
    if route == "dma":
        n *= 2   # one matrix fills the grid that two do
    for r in (F32, F16) if t is F16 else (F32,):
        project_case(c, m, k, n, t, r, act=abi.ACT_SILU)


@pytest.mark.parametrize("t,r", PAIRS, ids=IDS)
@pytest.mark.parametrize("m,k,n", FEW_ROWS)
def test_forward_few_rows(ctx, m, k, n, t, r):
    k *= 2 if k < 3000 else 1
    project_case(ctx, m, k, n, t, r, act=abi.ACT_SILU, bias=n % 3 == 0, drop=0.25 if m % 2 else 0.0, keep=m % 2 == 0,
                 in_place=n % 2 == 0)


def unproject_case(ctx, m, n, t, act=abi.ACT_IDENTITY, drop=0.25, scale=0.75, dx="own", place=lambda v: v, seed=77):
    dh, z = place(values((m, n), F32, 1, 64.0)), place(values((m, n), t, 2))
    was = dh.double().cpu()
    half = t == F16
    d, d_h = place(filled((m, n), F32)), place(filled((m, n), F16)) if half else None
    to = {"own": place(filled((m, n), F32)), "same": dh, "none": None}[dx]
    p = Projection(ctx, None, outputs=n, half=half, act=act, leaky=LEAKY, dropout=drop, scale=scale)
    p.error(dh, z if act else None, d, d_prenorm_h=d_h, dx=to, seed=seed)
    torch.cuda.synchronize()
    f = factors(m, n, drop, seed) if drop else torch.ones((m, n), dtype=torch.float64)
    want = was * f * slope(act, z)
    z = z.double().cpu()
    check(d, (want, was.abs() * f * 4 * (16 + 4 * z.abs()) * U * (1 + z.abs())), F32, "d")
    assert bool((d[f.cuda() == 0] == 0).all())
    if half:
        assert torch.equal(d_h, d.half())
    if to is not None:
        check(to, (scale * was, 2 * U * (scale * was).abs()), F32, "dx")


@pytest.mark.parametrize("t", TYPES, ids=["f32", "f16"])
@pytest.mark.parametrize("m,n", [(1, 1), (1, 8), (3, 5), (7, 129), (64, 64), (33, 777), (1000, 3), (500, 96)])
def test_error(ctx, m, n, t):
    unproject_case(ctx, m, n, t)
    unproject_case(ctx, m, n, t, act=abi.ACT_TANH, dx="same")
    unproject_case(ctx, m, n, t, act=abi.ACT_SILU, drop=0.0, dx="none", place=odd_base)


@pytest.mark.parametrize("t", TYPES, ids=["f32", "f16"])
@pytest.mark.parametrize("act", list(ACTS))
def test_error_activations(ctx, act, t):
    unproject_case(ctx, 37, 72, t, act=act)


def test_dropped_gradients_are_0_whatever_they_were(ctx):
    m, n, p, seed = 16, 40, 0.5, 3
    keep = keeps(m, n, p, seed).cuda()
    dh = torch.where(keep, 1.0, float("nan")).contiguous()
    z = torch.where(keep, 0.5, float("inf")).contiguous()
    d = filled((m, n), F32)
    Projection(ctx, None, outputs=n, act=abi.ACT_SILU, dropout=p).error(dh, z, d, seed=seed)
    out = dropout.apply(ctx, dh, torch.empty_like(dh), p, seed)
    torch.cuda.synchronize()
    assert bool((d[~keep] == 0).all()) and bool(torch.isfinite(d).all())
    assert bool((out[~keep] == 0).all()) and bool((out[keep] == 2).all())


def drop_case(ctx, m, n, t, p, seed, in_place=False, place=lambda v: v):
    x = place(values((m, n), t, m + n))
    was = x.clone()
    out = x if in_place else place(filled((m, n), t))
    got = dropout.apply(ctx, x, out, p, seed)
    torch.cuda.synchronize()
    assert got is out
    f = factors(m, n, p, seed)
    want = was.double().cpu() * f
    check(out, (want, 2 * U * want.abs()), t, "out")
    assert bool(((out.cpu() != 0) == ((f != 0) & (was.cpu() != 0))).all())


@pytest.mark.parametrize("t", TYPES, ids=["f32", "f16"])
@pytest.mark.parametrize("m,n", [(1, 1), (1, 7), (5, 1), (3, 9), (64, 777), (130, 64), (2000, 3), (1, 100000)])
def test_dropout(ctx, m, n, t):
    drop_case(ctx, m, n, t, 0.2, 12345)
    drop_case(ctx, m, n, t, 0.5, 0xFFFFFFFF, in_place=True)
    drop_case(ctx, m, n, t, 0.9, 0, place=odd_base)


@pytest.mark.parametrize("p", [0.0, 1e-8, 2.0 ** -32, 0.1, 1.0 - 2.0 ** -24])
def test_dropout_probabilities(ctx, p):
    drop_case(ctx, 300, 50, F32, p, 99)


def test_dropout_of_nothing(ctx):
    for shape in ((0, 5), (5, 0)):
        x = torch.empty(shape, device="cuda")
        dropout.apply(ctx, x, x, 0.5, 1)


@pytest.mark.parametrize("half", [False, True])
def test_same_draw_as_a_block(ctx, half):
    """A block's dropout, with its stored mask, and these from the same seed and place."""
    m, k, n, p, seed = 70, 40, 67, 0.3, 0xABCDEF01
    w = np.random.default_rng(1).standard_normal((k, n)).astype(np.float32) / 6
    b = DeviceBlock(ctx, k, n, m, w, half=half, act=abi.ACT_TANH, mask_coeff=p)
    t = F16 if half else F32
    x = values((m, k), t, 2)
    b.forward(x, m, use_dropout=True, seed=seed)
    h = filled((m, n), t)
    b2 = DeviceBlock(ctx, k, n, m, w, half=half, act=abi.ACT_TANH, mask_coeff=p)
    b2.forward_residual(x, m, None, h, use_dropout=True, seed=seed)
    ones = torch.ones((m, n), dtype=t, device="cuda")
    mask = dropout.apply(ctx, ones, torch.empty_like(ones), p, seed)
    b.error_from_sum(torch.ones((m, n), device="cuda"), m)
    b2.residual_error(torch.ones((m, n), device="cuda"), m, use_dropout=True, seed=seed)
    torch.cuda.synchronize()
    assert torch.equal(mask, b.mask) and torch.equal(h == 0, b.out == 0)
    assert torch.equal(b2.d_prenorm == 0, b.d_prenorm == 0)
    # the block rounds z before its activation, this one does not: a step of z and one of the result
    step = half_step(b.preact.double(), t) * 2 + half_step(b.out.double(), t) * 2 + 64 * U
    within(h, b.out.double(), step / (1 - p) + 64 * U, "h")


def test_rows_behind_the_batch_stay(ctx):
    m, batch, k, n = 30, 17, 24, 28
    b = DeviceBlock(ctx, k, n, m, np.random.default_rng(1).standard_normal((k, n)).astype(np.float32) / 5, half=True,
                    act=abi.ACT_SILU, mask_coeff=0.2)
    for name in ("preact", "d_prenorm", "d_prenorm_h", "grad", "mask", "out"):
        getattr(b, name).fill_(-7.0)
    x = values((m, k), F16, 2)
    x[batch:] = float("nan")
    stream, h, dh = values((m, n), F32, 3), filled((m, n), F32), values((m, n), F32, 4)
    b.forward_residual(x, batch, stream[:batch], h[:batch], use_dropout=True, seed=4)
    b.residual_error(dh[:batch], batch, use_dropout=True, seed=4)
    torch.cuda.synchronize()
    assert bool((h[batch:] == -7).all()) and bool(torch.isfinite(h).all())
    for name in ("preact", "d_prenorm", "d_prenorm_h"):
        v = getattr(b, name)
        assert bool((v[batch:] == -7).all()) and not bool((v[:batch] == -7).any())
    for name in ("grad", "mask", "out"):
        assert bool((getattr(b, name) == -7).all())


def test_gradient_against_differences(ctx):
    """The loss's slope in a direction of w by the backward (d_prenorm summed over rows in 64 bits) and by central
    differences of the formula (step 1e-4, third derivatives below 100)."""
    m, k, n, p, seed = 11, 16, 12, 0.25, 9
    w, b, x = values((k, n), F32, 1, 0.25), values((1, n), F32, 2), values((m, k), F32, 3)
    s, dh, way = values((m, n), F32, 4), values((m, n), F32, 5), values((k, n), F32, 6)
    pre, h, d = (filled((m, n), F32) for _ in range(3))
    op = Projection(ctx, w, b, outputs=n, act=abi.ACT_MISH, dropout=p, scale=0.5)
    op.forward(x, s, h, preact=pre, seed=seed)
    op.error(dh, pre, d, seed=seed)
    torch.cuda.synchronize()
    f = factors(m, n, p, seed).cuda()

    def loss(v):
        z = x.double() @ v + b.double()
        return ((0.5 * s.double() + f * ACTS[abi.ACT_MISH](z, 0.0)) * dh.double()).sum()

    step = 1e-4
    want = (loss(w.double() + step * way.double()) - loss(w.double() - step * way.double())) / (2 * step)
    dw = x.double().t().contiguous() @ d.double()
    got, size = (dw * way.double()).sum(), ((x.double().abs().t().contiguous() @ d.double().abs()) * way.double().abs()).sum()
    assert abs(got - want) <= 1e-6 * 100 * m + 4 * (k + 64) * U * size * 8
