"""skl_dense_distill_error against the formulas in 64 bits, on the CPU.

Tolerances count roundings, u = 2^-24.  exp2((z - m) k): the difference, k and the product are off
by u each, so the exponent by 3 u |arg| and the value by 3 u |arg| ln 2 + 2 u (the hardware exp2's
last place) relative.  A sum over n classes adds at most n / 64 + 40 times (each thread's share,
lanes, waves), so a probability is off by (3 |arg| + n / 64 + 48) u relative, a teacher's share by
the same with n = top.  The gradient adds those, scaled, with a few roundings of its own; the loss
adds its logarithms' absolute errors (an exponent's 3 u |arg| and a logarithm's place).  The fp16
copy rounds once more: 2^-11 relative or 2^-25.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from soklyn_amd import abi
from soklyn_amd.devblock import DeviceBlock, distill_error
from tests.helpers import he_normal, rng

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
INF = float("inf")


def inputs(rows, n, top, half, seed, std=2.5):
    g = torch.Generator().manual_seed(seed)
    z = (torch.randn(rows, n, generator=g) * std).to(torch.float16 if half else torch.float32)
    value = torch.randn(rows, top, generator=g) * std
    index = torch.stack([torch.randperm(n, generator=g)[:top] for _ in range(rows)]) if top else torch.zeros(rows, 0)
    label = torch.randint(0, n, (rows,), generator=g)
    return z, index.int(), value, label.int()


def softmax_err(arg, n):
    return (3 * arg.abs() + n / 64 + 48) * U


def reference(z, index, value, label, tau, alpha):
    z = z.double()
    rows, n = z.shape
    top = index.shape[1]
    grad, tol = torch.zeros_like(z), torch.zeros_like(z)
    loss, ltol = torch.zeros(rows, dtype=torch.float64), torch.zeros(rows, dtype=torch.float64)
    for r in range(rows):
        if torch.isinf(z[r]).all() and (z[r] < 0).all():
            continue
        held = [j for j in range(top) if 0 <= index[r, j] < n and value[r, j] > -INF]
        if alpha > 0 and held:
            v = value[r, held].double() / tau
            at = index[r, held].long()
            lq, arg_q = torch.log_softmax(v, 0), v - v.max()
            q = lq.exp()
            lq = torch.stack([lq[at == c].logsumexp(0) for c in at])   # of the class: all of its slots' shares
            lp = torch.log_softmax(z[r] / tau, 0)
            arg = (z[r] - z[r].max()) / tau
            p = lp.exp()
            share = torch.zeros(n, dtype=torch.float64).index_add_(0, at, q)
            eq = torch.zeros(n, dtype=torch.float64).index_add_(0, at, q * softmax_err(arg_q, top))
            grad[r] += alpha * tau * (p - share)
            fine = torch.where(arg.isinf(), 0.0, arg)
            tol[r] += alpha * tau * (p * softmax_err(fine, n) + eq + 4 * U * (p + share))
            loss[r] += alpha * tau * tau * (q * (lq - lp[at])).sum()
            err = (4 * arg_q.abs() + 4 * fine[at].abs() + n / 64 + 4 * top + 64) * U
            ltol[r] += alpha * tau * tau * (q * (err * (1 + (lq - lp[at]).abs()))).sum()
        if alpha < 1 and 0 <= label[r] < n:
            lp = torch.log_softmax(z[r], 0)
            arg = z[r] - z[r].max()
            fine = torch.where(arg.isinf(), 0.0, arg)
            p = lp.exp()
            y = int(label[r])
            grad[r] += (1 - alpha) * p
            grad[r, y] -= 1 - alpha
            tol[r] += (1 - alpha) * p * (softmax_err(fine, n) + 4 * U)
            tol[r, y] += (1 - alpha) * 4 * U
            loss[r] -= (1 - alpha) * lp[y]
            ltol[r] += (1 - alpha) * (4 * fine[y].abs() + n / 64 + 64) * U * 2
    return 512 * grad, 512 * (tol + 4 * U * grad.abs()) + 1e-30, loss, ltol + 4 * U * loss.abs() + 1e-30


def run(ctx, z, index, value, label, tau, alpha, offset=0):
    rows, n = z.shape
    guard = 64

    def out(shape, dtype):
        e = int(np.prod(shape))
        b = torch.full((e + 2 * guard + offset,), 7.0, dtype=dtype, device="cuda")
        return b, b[guard + offset:guard + offset + e].view(shape)

    half = z.dtype is torch.float16
    bufs = [out((rows, n), torch.float32), out((rows, n), torch.float32), out((rows,), torch.float32)]
    if half:
        bufs.append(out((rows, n), torch.float16))
    zb = torch.empty(z.numel() + offset, dtype=z.dtype, device="cuda")[offset:].view(z.shape)
    zb.copy_(z)
    grad, dp, loss = (v for _, v in bufs[:3])
    distill_error(ctx, zb, index.cuda(), value.cuda(), None if label is None else label.cuda(), temperature=tau,
                  alpha=alpha, grad=grad, d_prenorm=dp, d_prenorm_h=bufs[3][1] if half else None, loss=loss)
    torch.cuda.synchronize()
    for b, v in bufs:
        at = v.storage_offset()
        assert (b[:at] == 7).all() and (b[at + v.numel():] == 7).all(), "written outside the output"
    assert torch.equal(grad, dp) or torch.isnan(grad).any()
    if half and torch.isfinite(grad).all():
        assert torch.equal(bufs[3][1], grad.half())
    assert torch.equal(zb.cpu(), z) or torch.isnan(z).any()
    return grad.cpu().double(), loss.cpu().double()


def check(ctx, z, index, value, label, tau, alpha, offset=0):
    g, l = run(ctx, z, index, value, label, tau, alpha, offset)
    rg, tg, rl, tl = reference(z, index, value, label if label is not None else torch.full((z.shape[0],), -1), tau, alpha)
    d = (g - rg).abs()
    assert (d <= tg).all(), f"gradient: {(d / tg).max().item():.3g} of its tolerance"
    same = rl.float() == l.float()   # infinities: fp32's, where the loss is past its largest (3.4e38)
    e = (l - rl).abs()
    assert (same | (e <= tl)).all(), f"loss: {torch.where(same, 0, e / tl).max().item():.3g} of its tolerance"
    return g, l


@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("rows,n,top", [(1, 1, 1), (5, 2, 2), (7, 10, 4), (3, 511, 9), (4, 512, 16), (6, 513, 1), (5, 1000, 33),
                                        (2, 1024, 64), (3, 1025, 64), (2, 2048, 7), (3, 2049, 100), (2, 8191, 128),
                                        (1, 16384, 5), (2, 16385, 64), (2, 50257, 64), (1, 65536, 3), (1, 65537, 300),
                                        (1, 131072, 64), (1, 131075, 64), (1, 300001, 1024)])
def test_sizes(ctx, half, rows, n, top):
    print(f"distill {rows}x{n} top={top} half={half}", flush=True)
    z, index, value, label = inputs(rows, n, top, half, rows + n)
    check(ctx, z, index, value, label, 2.0, 0.75)


# the last width of each form and the next, rows that start at every remainder of 4
@pytest.mark.parametrize("n", [61, 62, 63, 253, 254, 509, 510, 1021, 1022, 2045, 2046, 4093, 4094, 8189, 8190, 16381, 16382, 32765, 32766,
                               65533, 65534])
def test_edges_of_the_forms(ctx, n):
    print(f"distill {n}", flush=True)
    for half in (True, False):
        z, index, value, label = inputs(6, n, 11, half, n)
        check(ctx, z, index, value, label, 1.5, 0.25)


@pytest.mark.parametrize("n", [61, 253, 257, 500, 509, 1000, 1021, 1999, 2045, 3000])
def test_enough_rows_to_fill_the_gpu(ctx, n):
    """Where rows are many a wave, or a quarter, has each of them by itself; every 97th is compared."""
    rows = 4113
    for half in (True, False):
        z, index, value, label = inputs(rows, n, 7, half, n)
        g, l = run(ctx, z, index, value, label, 2.0, 0.5)
        some = slice(n % 97, rows, 97)
        rg, tg, rl, tl = reference(z[some], index[some], value[some], label[some], 2.0, 0.5)
        assert ((g[some] - rg).abs() <= tg).all() and ((l[some] - rl).abs() <= tl).all()


@pytest.mark.parametrize("tau", [0.25, 1.0, 7.5])
@pytest.mark.parametrize("alpha", [0.0, 0.3, 1.0])
def test_temperatures_and_mixtures(ctx, tau, alpha):
    for half, n in ((True, 777), (False, 40), (True, 5000)):
        z, index, value, label = inputs(9, n, 12, half, 3)
        check(ctx, z, index, value, label if alpha < 1 else None, tau, alpha)


@pytest.mark.parametrize("n", [12, 900, 3001])
def test_slots_without_class_and_rows_without_teacher_or_label(ctx, n):
    z, index, value, label = inputs(12, n, 6, True, 5)
    index[0] = -1                       # no teacher
    index[1, 2:] = -1
    index[2, ::2] = n                   # past the classes: empty
    index[3] = 2 ** 31 - 1
    value[4] = -INF                     # held, and without mass
    value[5, 1:] = -INF
    value[6, 0] = -3.4028234663852886e38
    value[1, 3] = float("nan")          # in an empty slot
    label[7] = -1
    label[8] = n
    label[0] = -1                       # neither
    g, l = check(ctx, z, index, value, label, 2.0, 0.5)
    assert (g[0] == 0).all() and l[0] == 0
    check(ctx, z, torch.zeros(12, 0, dtype=torch.int32), torch.zeros(12, 0), label, 1.0, 0.5)


@pytest.mark.parametrize("n", [10, 700, 4000])
def test_a_class_named_twice_adds_its_shares(ctx, n):
    z, index, value, label = inputs(6, n, 8, True, 6)
    index[0] = 3
    index[1, 4:] = index[1, :4]
    index[2, 7] = index[2, 0]
    label[0] = 3
    label[1] = index[1, 0]
    check(ctx, z, index, value, label, 2.0, 0.5)


# each form of the kernel, with a table of the columns and without
@pytest.mark.parametrize("n,top", [(1, 2), (10, 4), (60, 33), (250, 64), (700, 8), (2000, 128), (4000, 64), (8000, 64), (9001, 300),
                                   (40000, 64), (70001, 1024), (5, 1024), (60, 65), (300, 1000), (3000, 1024)])
def test_the_loss_is_a_divergence_where_classes_repeat(ctx, n, top):
    """sum Q (log Q - log p) over the classes, Q a class's shares added up: 0 where the layer has the
    teacher's distribution, and never below."""
    rows = 7
    z, index, value, label = inputs(rows, n, min(top, n), False, n + top)
    g = torch.Generator().manual_seed(n)
    index, value = torch.zeros(rows, top, dtype=torch.int32), torch.randn(rows, top, generator=g)
    index[1:] = torch.randint(0, n, (rows - 1, top), generator=g)      # some twice
    index[2] = torch.randint(0, min(n, 3), (top,), generator=g)        # each many times
    index[3, ::2] = index[3, 0]
    value[3, top // 2:] -= 90.0                                        # shares that vanish beside the others
    index[4, 1::2] = -1
    value[5, ::2] = -INF
    index[6, top // 2:] = (index[6, : top - top // 2] + 1) % n         # neighbours: one vector's columns
    z[0] = -INF
    z[0, 0] = 1.5                                                      # one class, the teacher's
    _, l = check(ctx, z, index, value, None, 1.0, 1.0)
    assert l[0].abs() <= (4 * top + 64) * U                            # (two sums of the same terms, in other orders)
    check(ctx, z, index, value, label, 2.0, 0.5)
    check(ctx, z.half(), index, value, label, 2.0, 0.5)
    for tau in (0.5, 1.0, 4.0):
        # the teacher's own distribution over its classes, mixed from all of its slots
        same = torch.full((rows, n), -INF)
        for r in range(rows):
            v = torch.where(index[r] >= 0, value[r], -INF).double() / tau
            for c in set(index[r].tolist()) - {-1}:
                same[r, c] = (tau * v[index[r] == c].logsumexp(0)).float()
        _, l = check(ctx, same, index, value, None, tau, 1.0)
        # the logits round by u each, and the tolerance of a loss near 0 is that of its logarithms
        assert (l.abs() <= tau * tau * (4 * top + n / 64 + 64 + 4 * 100 / tau) * U + tau * U * same.where(same > -INF, 0.0).abs().amax(1)).all()


@pytest.mark.parametrize("n", [16, 1000, 3000, 20000])
def test_logits_that_are_masked_or_not_finite(ctx, n):
    z, index, value, label = inputs(8, n, 4, True, 7)
    z[0] = -INF                          # nothing left: no loss, no gradient
    z[1, 1:] = -INF                      # one class left
    index[1, 0], label[1] = 0, 0
    value[1, 1:] = -INF
    z[2] = -65504.0                      # the type's lowest everywhere: uniform
    z[3, index[3, 0].long()] = -INF      # the teacher's class is masked: an infinite loss
    clean = z.clone()
    g, l = check(ctx, z, index, value, label, 1.0, 0.5)
    assert (g[0] == 0).all() and l[0] == 0 and l[3] == INF and torch.isfinite(g).all()
    clean[4, 3] = float("nan")
    clean[5, 2] = INF
    clean[6] = float("nan")
    value[7, 0] = float("nan")
    index[7, 0] = 1
    g2, l2 = run(ctx, clean, index, value, label, 1.0, 0.5)
    for row in (4, 5, 6):
        assert torch.isnan(l2[row]) and torch.isnan(g2[row]).any()
    assert torch.isnan(g2[4]).all() and torch.isnan(g2[6]).all() and torch.isnan(l2[7])
    assert torch.equal(g2[:4], g[:4])


@pytest.mark.parametrize("offset", [1, 3])
def test_any_alignment(ctx, offset):
    for half, n in ((True, 640), (True, 4096), (False, 1000)):
        z, index, value, label = inputs(5, n, 8, half, 8)
        check(ctx, z, index, value, label, 2.0, 0.5, offset)


def test_many_rows_twice(ctx):
    z, index, value, label = inputs(3000, 130, 5, True, 9)
    a = run(ctx, z, index, value, label, 2.0, 0.5)
    b = run(ctx, z, index, value, label, 2.0, 0.5)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    few = run(ctx, z[1500:1520].contiguous(), index[1500:1520], value[1500:1520], label[1500:1520], 2.0, 0.5)
    assert torch.equal(few[0], a[0][1500:1520]) and torch.equal(few[1], a[1][1500:1520])


def test_gradient_against_differences(ctx):
    """Central differences of the loss in fp64 logits are the reference's own; here the fp32 loss,
    step 2^-5: its rounding (100 u |loss| / step) and third-order term stay under 2e-3."""
    z, index, value, label = inputs(2, 9, 4, False, 10, std=1.0)
    g, _ = run(ctx, z, index, value, label, 2.0, 0.5)
    step = 2.0 ** -5
    for at in ((0, 0), (0, int(index[0, 0])), (1, int(label[1])), (1, 8)):
        zs = []
        for s in (step, -step):
            w = z.clone()
            w[at] += s
            zs.append(run(ctx, w, index, value, label, 2.0, 0.5)[1].sum())
        assert abs((zs[0] - zs[1]) / (2 * step) - g[at] / 512) < 2e-3


@pytest.mark.parametrize("n", [10, 300, 1000, 9000])
@pytest.mark.parametrize("std,tau", [(1e10, 1.0), (1e30, 2.0), (2.5, 2.0 ** -40), (2.5, 2.0 ** -60), (1e-3, 2.0 ** 60)])
def test_large_logits_and_extreme_temperatures(ctx, n, std, tau):
    """Exponents far past 2^31: the largest term is 1 all the same.  Beside a logit of 3e38, alpha tau^2
    (3e38 / tau) + (1 - alpha) 3e38 is 4.5e38 at tau = 2, so that row's loss rounds to infinity."""
    z, index, value, label = inputs(5, n, 4, False, 21, std)
    z[1, n // 2] = z[1, 3] = z[1].max()   # two largest
    z[2, 0] = 3e38
    check(ctx, z, index, value, label, tau, 0.5)


@pytest.mark.parametrize("half", [True, False])
def test_a_blocks_own_step(ctx, half):
    """forward, distill, backward of a DeviceBlock: the update is the one that the same gradient
    gives through skl_dense_error_from_sum; rows behind the batch stay as they were."""
    K, N, M, rows = 64, 48, 40, 33
    w = he_normal(rng(1), K, N)
    z, index, value, label = inputs(rows, N, 5, half, 11)
    x = torch.from_numpy(rng(2).standard_normal((rows, K)).astype(np.float32)).cuda()
    x = x.half() if half else x
    blocks = []
    for _ in range(2):
        b = DeviceBlock(ctx, K, N, M, w, half=half, master_w=w if half else None)
        b.forward(x, rows)
        blocks.append(b)
    a, b = blocks
    for n in ("grad", "d_prenorm", "d_prenorm_h"):
        for blk in blocks:
            if getattr(blk, n) is not None:
                getattr(blk, n).fill_(3.0)
    loss = torch.empty(rows, device="cuda")
    a.distill_error(index.cuda(), value.cuda(), label.cuda(), temperature=2.0, alpha=0.5, loss=loss)
    torch.cuda.synchronize()
    rg, tg, rl, tl = reference(a.out[:rows].cpu(), index, value, label, 2.0, 0.5)
    assert ((a.grad[:rows].cpu().double() - rg).abs() <= tg).all()
    assert ((loss.cpu().double() - rl).abs() <= tl).all()
    for n in ("grad", "d_prenorm", "d_prenorm_h"):
        if getattr(a, n) is not None:
            assert (getattr(a, n)[rows:] == 3.0).all(), n
    b.error_from_sum(a.grad[:rows].contiguous(), rows)
    opt = abi.adam()
    for blk in blocks:
        blk.backward(x, abi.train_ctx(opt, opt, rows, 1e-3), 1)
    torch.cuda.synchronize()
    for n in ("w", "master_w", "dm_w", "dv_w"):
        if getattr(a, n) is not None:
            assert torch.equal(getattr(a, n), getattr(b, n)), n
    # the bias sums add 33 terms in another order: 33 u of their magnitudes, |g| up to 512
    assert (a.dm_b - b.dm_b).abs().max() <= 0.1 * 33 * U * 33 * 512 / 512 / rows
    # a stale sum of the call before is not taken for this error's
    b.error_from_sum(torch.zeros(rows, N, device="cuda"), rows)
    b.distill_error(index.cuda(), value.cuda(), label.cuda(), temperature=2.0, alpha=0.5)
    before = b.dm_b.clone()
    b.backward(x, abi.train_ctx(opt, opt, rows, 1e-3), 2)
    torch.cuda.synchronize()
    want = 0.9 * before.double() + 0.1 * b.d_prenorm[:rows].double().sum(0, keepdim=True) / 512 / rows
    assert (b.dm_b.double() - want).abs().max() <= 64 * U * (before.abs().max() + 1)


def test_captured_and_replayed(ctx):
    z, index, value, label = inputs(20, 3000, 16, True, 12)
    side = torch.cuda.Stream()
    cap = abi.Context(0, 16, stream=side.cuda_stream)
    try:
        zb, ib, vb, lb = z.cuda(), index.cuda(), value.cuda(), label.cuda()
        out = dict(grad=torch.empty(20, 3000, device="cuda"), d_prenorm=torch.empty(20, 3000, device="cuda"),
                   d_prenorm_h=torch.empty(20, 3000, device="cuda", dtype=torch.float16), loss=torch.empty(20, device="cuda"))
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side, capture_error_mode="thread_local"):
            distill_error(cap, zb, ib, vb, lb, temperature=2.0, alpha=0.5, **out)
        for rep in range(3):
            zb.copy_(torch.randn(20, 3000, device="cuda") * (rep + 1))
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            want = {k: torch.empty_like(v) for k, v in out.items()}
            distill_error(ctx, zb, ib, vb, lb, temperature=2.0, alpha=0.5, **want)
            torch.cuda.synchronize()
            for k in out:
                assert torch.equal(out[k], want[k]), k
    finally:
        torch.cuda.synchronize()
        cap.close()
