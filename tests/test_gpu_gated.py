"""Gated feed-forward blocks against 64 bits: every kernel and its edges, the backward against the formula and
against differences, bounds as in ffn_helpers."""
from __future__ import annotations

import pytest
import torch

from soklyn_amd import abi
from soklyn_amd.devblock import DeviceBlock
from soklyn_amd.gated import Gated, GatedBlock
from tests.ffn_helpers import ACTS, LEAKY, U, check, filled, gated_ref, half_step, odd_base, product, ungate_ref, values, within

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16]
IDS = ["f32", "f16"]


def weights(k, n, t, seed, bias):
    return (values((k, n), t, seed, k ** -0.5), values((k, n), t, seed + 1, k ** -0.5),
            values((1, n), t, seed + 2, 0.3) if bias else None, values((1, n), t, seed + 3, 0.3) if bias else None)


def forward_case(ctx, m, k, n, t, act, bias, keep, place=lambda v: v):
    wg, wu, bg, bu = (None if v is None else place(v) for v in weights(k, n, t, m + n, bias))
    x = place(values((m, k), t, 7))
    out, a, u = (place(filled((m, n), t)) for _ in range(3))
    Gated(ctx, wg, wu, bg, bu, outputs=n, half=t == torch.float16, act=act, leaky=LEAKY).forward(
        x, out, a=a if keep else None, u=u if keep else None)
    torch.cuda.synchronize()
    ref = gated_ref(x, wg, wu, bg, bu, act)
    check(out, ref["out"], t, "out")
    if keep:
        check(a, ref["a"], t, "a")
        check(u, ref["u"], t, "u")
    else:
        assert bool((a == -7).all()) and bool((u == -7).all())


@pytest.mark.parametrize("t", TYPES, ids=IDS)
@pytest.mark.parametrize("m,k,n", [(1, 1, 1), (1, 64, 64), (1, 200, 129), (2, 33, 65), (3, 5, 7), (5, 4096, 40), (16, 96, 80),
                                   (17, 31, 16), (33, 250, 100), (64, 64, 256), (130, 257, 129), (200, 128, 36),
                                   (256, 128, 128), (300, 72, 250), (1000, 65, 66)])
def test_forward_sizes(ctx, m, k, n, t):
    forward_case(ctx, m, k, n, t, abi.ACT_SILU, n % 2 == 0, m % 2 == 0)


@pytest.mark.parametrize("t", TYPES, ids=IDS)
@pytest.mark.parametrize("act", list(ACTS))
def test_forward_activations(ctx, act, t):
    forward_case(ctx, 37, 64, 72, t, act, True, True)


@pytest.mark.parametrize("t", TYPES, ids=IDS)
@pytest.mark.parametrize("m,k,n", [(1, 64, 64), (20, 40, 24), (130, 64, 128)])
def test_forward_bases_off_their_boundaries(ctx, m, k, n, t):
    forward_case(ctx, m, k, n, t, abi.ACT_TANH, True, True, odd_base)


def routed(monkeypatch, ctx, route):
    """A context whose products take this kernel or fail, on the stream of the others."""
    monkeypatch.setenv("SOKLYN_GEMM_ROUTE", route)
    c = abi.Context(0, 16, stream=torch.cuda.current_stream().cuda_stream)
    monkeypatch.delenv("SOKLYN_GEMM_ROUTE")
    return c


WAVES16 = ["wave:16:16", "wave:32:4", "wave:64:2", "wave:64:4"]
WAVES32 = ["wave:16:16", "wave:32:8", "wave:64:8", "wave:64:4", "wave:64:2", "wave:64:1"]
WAVES_ODD = ["wave:16:16", "wave:32:8", "wave:64:4"]
# (rows, k, columns): whole tiles, ragged ones, and for padded copies grids of 192 tiles
KERNELS = ([(r, torch.float16, 70, 200, 68) for r in WAVES16] + [(r, torch.float16, 70, 77, 67) for r in WAVES_ODD] +
           [(r, torch.float32, 70, 203, 67) for r in WAVES32] + [(r, torch.float32, 130, 64, 64) for r in WAVES32] +
           [("copied", torch.float16, 300, 77, 131), ("copied", torch.float16, 129, 1001, 259)] +
           [("dma128", torch.float16, 256, 128, 256), ("dma128", torch.float16, 300, 72, 130),
            ("dma128", torch.float16, 129, 200, 264), ("dma", torch.float16, 4096, 128, 1536),
            ("dma", torch.float16, 4000, 100, 1500), ("dma", torch.float16, 4096, 65, 1531)])


@pytest.mark.parametrize("route,t,m,k,n", KERNELS)
def test_forward_kernels(monkeypatch, ctx, route, t, m, k, n):
    forward_case(routed(monkeypatch, ctx, route), m, k, n, t, abi.ACT_SILU, True, True)


@pytest.mark.parametrize("m,k,n", [(200, 80, 131), (130, 77, 132), (257, 75, 260)])
@pytest.mark.parametrize("place", [lambda v: v, odd_base], ids=["aligned", "off"])
def test_forward_copies_of_one_operand(monkeypatch, ctx, m, k, n, place):
    """Odd rows of the weights alone, part of a 16-byte piece of k alone, and bases off their boundaries."""
    forward_case(routed(monkeypatch, ctx, "copied"), m, k, n, torch.float16, abi.ACT_SILU, False, True, place)


# up to 16 rows over a long k: eight slices of it (up to 4096 columns of fp16, 2048 of fp32), four, two, one; k
# that ends inside a step, slices without any, and sizes on both sides of the rule's borders
FEW_ROWS = [(1, 3000, 256), (3, 4096, 1000), (16, 3008, 2056), (16, 1500, 260), (17, 3000, 264), (2, 3001, 264), (5, 2999, 256),
            (9, 1504, 8200), (1, 1500, 16400), (7, 1512, 32776), (16, 40000, 256), (1, 6004, 252),
            (32, 3000, 256), (31, 1504, 4104), (18, 3008, 1000), (32, 1500, 16388), (33, 3000, 256),
            (64, 3008, 264), (49, 4000, 4000)]


@pytest.mark.parametrize("t", TYPES, ids=IDS)
@pytest.mark.parametrize("m,k,n", FEW_ROWS)
def test_forward_few_rows(ctx, m, k, n, t):
    forward_case(ctx, m, k, n, t, abi.ACT_SILU, n % 3 == 0, m % 2 == 0)
    if n < 300:
        forward_case(ctx, m, k, n, t, abi.ACT_SILU, True, True, odd_base)


def test_forward_few_rows_beside_nan(ctx):
    """Rows past the batch, which follow the last one in memory, are not read into its sums."""
    k, n, t = 3004, 256, torch.float32
    wg, wu, _, _ = weights(k, n, t, 1, False)
    for m in (1, 4):
        x = values((16, k), t, 2)
        x[m:] = float("nan")
        out = filled((m, n), t)
        Gated(ctx, wg, wu, outputs=n).forward(x[:m], out)
        torch.cuda.synchronize()
        check(out, gated_ref(x[:m], wg, wu, None, None, abi.ACT_SILU)["out"], t, "out")


def error_case(ctx, m, n, above, t, act, place=lambda v: v):
    a, u = place(values((m, n), t, 3)), place(values((m, n), t, 4))
    half = t == torch.float16
    to = {k: place(filled((m, n), torch.float32)) for k in ("dg", "du")}
    to |= {k: place(filled((m, n), torch.float16)) if half else None for k in ("dg_h", "du_h")}
    g = Gated(ctx, None, None, outputs=n, half=half, act=act, leaky=LEAKY)
    if above:
        d, w = place(values((m, above), t, 5, 64.0)), place(values((n, above), t, 6, above ** -0.5))
        g.hidden_error(d, w, a, u, **to)
        s, ds = product(d, w.t())
    else:
        s = place(values((m, n), torch.float32, 5, 64.0))
        g.error_from_sum(s, a, u, **to)
        s, ds = s.double(), torch.zeros_like(s, dtype=torch.float64)
    torch.cuda.synchronize()
    ref = ungate_ref(s, ds, a, u, act)
    for k in ("dg", "du"):
        check(to[k], ref[k], torch.float32, k)
        if half:   # the copies hold the rounded gradients
            assert torch.equal(to[k + "_h"], to[k].half()), k


@pytest.mark.parametrize("t", TYPES, ids=IDS)
@pytest.mark.parametrize("m,n", [(1, 1), (1, 64), (3, 5), (7, 129), (64, 64), (33, 777), (500, 96)])
def test_error_from_sum(ctx, m, n, t):
    error_case(ctx, m, n, 0, t, abi.ACT_SILU)
    error_case(ctx, m, n, 0, t, abi.ACT_TANH, odd_base)


@pytest.mark.parametrize("t", TYPES, ids=IDS)
@pytest.mark.parametrize("act", list(ACTS))
def test_error_activations(ctx, act, t):
    error_case(ctx, 37, 72, 0, t, act)
    error_case(ctx, 37, 72, 40, t, act)


@pytest.mark.parametrize("t", TYPES, ids=IDS)
@pytest.mark.parametrize("m,n,above", [(1, 1, 1), (1, 64, 10), (2, 65, 33), (16, 80, 96), (33, 100, 250), (130, 129, 257),
                                       (256, 256, 128), (300, 250, 72), (1000, 66, 65)])
def test_hidden_error_sizes(ctx, m, n, above, t):
    error_case(ctx, m, n, above, t, abi.ACT_SILU)


@pytest.mark.parametrize("t", TYPES, ids=IDS)
def test_hidden_error_bases_off_their_boundaries(ctx, t):
    error_case(ctx, 20, 24, 40, t, abi.ACT_SIGMOID, odd_base)


@pytest.mark.parametrize("route,t,m,k,n", KERNELS)
def test_hidden_error_kernels(monkeypatch, ctx, route, t, m, k, n):
    if route == "dma":
        n *= 2   # one matrix fills the grid that two do
    error_case(routed(monkeypatch, ctx, route), m, n, k, t, abi.ACT_SILU)


def grad_case(ctx, m, k, n, t, place=lambda v: v):
    wg, wu, _, _ = weights(k, n, t, m + n, False)
    wg, wu, dg, du = place(wg), place(wu), place(values((m, n), t, 3, 64.0)), place(values((m, n), t, 4, 64.0))
    dx = place(filled((m, k), torch.float32))
    Gated(ctx, wg, wu, outputs=n, half=t == torch.float16).input_grad(dg, du, dx)
    torch.cuda.synchronize()
    want, bound = product(torch.cat([dg, du], 1), torch.cat([wg, wu], 1).t())
    within(dx, want, bound, "dx")


@pytest.mark.parametrize("t", TYPES, ids=IDS)
@pytest.mark.parametrize("m,k,n", [(1, 1, 1), (1, 64, 64), (1, 200, 129), (3, 5, 7), (16, 96, 80), (33, 250, 100), (64, 64, 33),
                                   (130, 257, 129), (256, 256, 64), (256, 256, 192), (300, 72, 250), (129, 66, 72),
                                   (1000, 66, 65)])
def test_input_grad_sizes(ctx, m, k, n, t):
    grad_case(ctx, m, k, n, t)
    if m < 100:
        grad_case(ctx, m, k, n, t, odd_base)


# columns and k change places; parts of whole k-tiles (64) and others
@pytest.mark.parametrize("route,t,m,n,k", KERNELS + [("dma", torch.float16, 4096, 64, 3200), ("dma", torch.float16, 4096, 192, 3200)])
def test_input_grad_kernels(monkeypatch, ctx, route, t, m, n, k):
    grad_case(routed(monkeypatch, ctx, route), m, 2 * k if route == "dma" else k, n, t)


def test_rows_behind_the_batch_stay(ctx):
    m, batch, k, n = 40, 23, 48, 52
    g = torch.Generator().manual_seed(1)
    blocks = [DeviceBlock(ctx, k, n, m, (torch.randn((k, n), generator=g) / 7).numpy(), half=True, act=act)
              for act in (abi.ACT_SILU, abi.ACT_IDENTITY)]
    nxt = DeviceBlock(ctx, n, 30, m, (torch.randn((n, 30), generator=g) / 7).numpy(), half=True)
    nxt.d_prenorm_h.copy_(values((m, 30), torch.float16, 5))
    for b in blocks:
        for name in ("preact", "d_prenorm", "d_prenorm_h", "grad", "predrop", "out"):
            getattr(b, name).fill_(-7.0)
    block = GatedBlock(*blocks)
    x = values((m, k), torch.float16, 2)
    x[batch:] = float("nan")          # rows behind the batch are not read
    nxt.d_prenorm_h[batch:] = float("inf")
    out = filled((m, n), torch.float16)
    dx = filled((m, k), torch.float32)
    block.forward(x, batch, out[:batch])
    block.hidden_error(nxt, batch)
    block.input_grad(batch, dx[:batch])
    torch.cuda.synchronize()
    ref = gated_ref(x[:batch], blocks[0].w, blocks[1].w, blocks[0].b, blocks[1].b, abi.ACT_SILU)
    check(out[:batch], ref["out"], torch.float16, "out")
    for b in blocks:
        for name in ("preact", "d_prenorm", "d_prenorm_h"):
            t = getattr(b, name)
            assert bool((t[batch:] == -7).all()) and bool(torch.isfinite(t[:batch]).all()) and not bool((t[:batch] == -7).all())
        for name in ("grad", "predrop", "out"):   # not this call's
            assert bool((getattr(b, name) == -7).all())
    assert bool((out[batch:] == -7).all()) and bool((dx[batch:] == -7).all()) and bool(torch.isfinite(dx[:batch]).all())


def test_block_trains_as_its_formula_says(ctx):
    """Both updates and dx of one step in fp32 against autograd in 64 bits: d_prenorm (off by `ungate` of the
    sums' bound) summed over the rows for each weight, off by another (m + 64) u of the terms."""
    m, k, n, lr = 50, 40, 56, 0.5
    g = torch.Generator().manual_seed(3)
    ws = [torch.randn((k, n), generator=g) / k ** 0.5 for _ in range(2)]
    bs = [torch.randn((1, n), generator=g) * 0.2 for _ in range(2)]
    blocks = [DeviceBlock(ctx, k, n, m, w.numpy(), b=b.numpy(), act=act)
              for w, b, act in zip(ws, bs, (abi.ACT_SILU, abi.ACT_IDENTITY))]
    block = GatedBlock(*blocks)
    x = torch.randn((m, k), generator=g)
    s = torch.randn((m, n), generator=g) * 512
    out, xd = filled((m, n), torch.float32), x.cuda()
    block.forward(xd, m, out)
    block.error_from_sum(s.cuda(), m)
    dx = block.input_grad(m)
    block.backward(xd, abi.train_ctx(abi.sgd(), abi.sgd(), m, lr), 1)
    torch.cuda.synchronize()
    leaves = [v.double().requires_grad_() for v in (x, *ws, *bs)]
    x64, wg, wu, bg, bu = leaves
    y = ACTS[abi.ACT_SILU](x64 @ wg + bg, 0.0) * (x64 @ wu + bu)
    grads = torch.autograd.grad((y * s.double()).sum(), leaves)
    # every term of a gradient is at most 512 x 8 (the largest deviates of s, x, a, u and w) and all its steps are
    # within 4 (k + n + m + 128) u of it
    terms = 4 * (k + n + m + 128) * U * 512 * 8 * 8
    within(dx, grads[0], torch.full_like(grads[0], terms * 2 * n ** 0.5), "dx")
    for b, w, bias, dw, db in zip(blocks, ws, bs, grads[1:3], grads[3:5]):
        for got, was, d in ((b.w, w, dw), (b.b, bias, db)):
            want = was.double() - lr * d / 512 / m
            within(got, want, torch.full_like(want, lr * terms / 512 + 4 * U), "update")


def test_gradient_against_differences(ctx):
    """d out / d x in a direction, by the backward in fp32 and by central differences in 64 bits of the forward's
    formula (step 1e-4: off by 1e-8 of third derivatives, which are below 100 here)."""
    m, k, n = 9, 24, 20
    wg, wu, bg, bu = weights(k, n, torch.float32, 5, True)
    x, s, way = (values(sh, torch.float32, 8 + i) for i, sh in enumerate([(m, k), (m, n), (m, k)]))
    g = Gated(ctx, wg, wu, bg, bu, outputs=n, act=abi.ACT_MISH)
    out, a, u, dg, du = (filled((m, n), torch.float32) for _ in range(5))
    dx = filled((m, k), torch.float32)
    g.forward(x, out, a=a, u=u)
    g.error_from_sum(s, a, u, dg=dg, du=du)
    g.input_grad(dg, du, dx)
    torch.cuda.synchronize()

    def loss(v):
        return (gated_ref(v, wg, wu, bg, bu, abi.ACT_MISH)["out"][0] * s.double()).sum()

    h = 1e-4
    want = (loss(x.double() + h * way.double()) - loss(x.double() - h * way.double())) / (2 * h)
    got = (dx.double() * way.double()).sum()
    size = (dx.double() * way.double()).abs().sum()
    assert abs(got - want) <= 1e-6 * 100 * m + 4 * (k + 2 * n + 64) * U * size * 8


@pytest.mark.parametrize("t", TYPES, ids=IDS)
def test_infinities_and_nan_keep_to_their_rows(ctx, t):
    m, k, n = 40, 64, 48
    wg, wu, bg, bu = weights(k, n, t, 1, True)
    x = values((m, k), t, 2)
    x[3, 5], x[17, 0] = float("nan"), float("inf")
    out, a, u = (filled((m, n), t) for _ in range(3))
    Gated(ctx, wg, wu, bg, bu, outputs=n, half=t == torch.float16, act=abi.ACT_SIGMOID).forward(x, out, a=a, u=u)
    torch.cuda.synchronize()
    rest = [i for i in range(m) if i not in (3, 17)]
    ref = gated_ref(x[rest], wg, wu, bg, bu, abi.ACT_SIGMOID)
    check(out[rest], ref["out"], t, "out")
    assert bool(torch.isnan(out[3]).all()) and bool(torch.isnan(a[3]).all())
    assert bool(torch.isinf(a[17]).all()) and bool(torch.isinf(u[17]).all())


def test_workspace_makes_no_difference_but_for_order(ctx):
    """A ragged product that is given no workspace for its padded copies takes another kernel."""
    m, k, n = 4001, 130, 1500
    t = torch.float16
    assert abi.load().skl_product_work_bytes(1, m, k, n, 2) > 0
    wg, wu, _, _ = weights(k, n, t, 1, False)
    x = values((m, k), t, 2)
    g = Gated(ctx, wg, wu, outputs=n, half=True)
    got = []
    for work in (True, False):
        if not work:
            g.work.product = lambda *size: (None, 0)
        out = filled((m, n), t)
        g.forward(x, out)
        torch.cuda.synchronize()
        got.append(out)
    ref = gated_ref(x, wg, wu, None, None, abi.ACT_SILU)["out"]
    for out in got:
        check(out, ref, t, "out")
    within(got[0], got[1].double(), 2 * ref[1] + 2 * half_step(ref[0], t), "both")


@pytest.mark.parametrize("t", TYPES, ids=IDS)
def test_few_rows_with_a_workspace_too_small(ctx, t):
    """... and so does one of few rows, whose sums over slices of k do not fit; what lies behind the given bytes stays."""
    m, k, n = 7, 4096, 520
    need = abi.load().skl_product_work_bytes(int(t == torch.float16), m, k, n, 2)
    wg, wu, _, _ = weights(k, n, t, 1, False)
    x = values((m, k), t, 2)
    g = Gated(ctx, wg, wu, outputs=n, half=t == torch.float16)
    work = torch.full((need + 4096,), 171, dtype=torch.uint8, device="cuda")
    for size in (0, 16, need - 16, need):
        g.work.product = lambda *_: (work.data_ptr(), size)
        out = filled((m, n), t)
        g.forward(x, out)
        torch.cuda.synchronize()
        check(out, gated_ref(x, wg, wu, None, None, abi.ACT_SILU)["out"], t, "out")
        assert bool((work[size:] == 171).all()), size
