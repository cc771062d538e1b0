"""skl_residual_forward / skl_residual_backward against the formulas in 64 bits, on the CPU.

Tolerances count roundings.  u = 2^-24 is half a step of fp32.  A row sum adds at most 16 terms in a
thread, 6 times across lanes and 16 times across waves: 38 roundings of at most u times the sum of
the terms' magnitudes.  A result a few operations behind two such sums is off by at most 128 u times
the same formula over magnitudes (64 for one sum, twice that behind the second); a column sum adds
up to 4 rows and 128 planes more, 512 u in all.  Results that are stored in fp16 round once more:
2^-11 relative, or half the smallest step, 2^-25.
"""
from __future__ import annotations

import pytest
import torch

from soklyn_amd import abi
from soklyn_amd.residual import Join

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
EPS = 1e-6
NONE, RMS, LAYER = abi.NORM_DISABLED, abi.NORM_RMS, abi.NORM_LAYER
IDENTITY, SIGMOID, TANH = abi.ACT_IDENTITY, abi.ACT_SIGMOID, abi.ACT_TANH
GUARD = 64


def guarded(shape, dtype, offset=0):
    """An output inside a larger buffer of 7s, `offset` elements off its alignment."""
    n = 1
    for s in shape:
        n *= s
    buf = torch.full((n + 2 * GUARD + offset,), 7.0, dtype=dtype, device="cuda")
    return buf, buf[GUARD + offset:GUARD + offset + n].view(shape)


def assert_guards(pairs):
    for buf, view in pairs:
        at = view.storage_offset()
        assert (buf[:at] == 7).all() and (buf[at + view.numel():] == 7).all(), "written outside the output"


def off_by(t, offset):
    """t at an address `offset` elements off its alignment."""
    buf = torch.empty(t.numel() + offset, dtype=t.dtype, device=t.device)
    v = buf[offset:].view(t.shape)
    v.copy_(t)
    return v


class Case:
    def __init__(self, ctx, rows, cols, half, half_stream, post, pre, gates, gate_act, scale, *, seed=1, offset=0,
                 with_x=True, with_y=True):
        g = torch.Generator().manual_seed(seed)
        self.t = t = torch.float16 if half else torch.float32
        self.r = r = torch.float16 if half_stream else torch.float32
        self.rows, self.cols, self.post, self.pre, self.act, self.scale = rows, cols, post, pre, gate_act, scale
        self.offset = offset

        def make(shape, dtype, std=1.0, mean=0.0):
            return off_by((torch.randn(shape, generator=g) * std + mean).to(dtype).cuda(), offset)

        self.x = make((rows, cols), r, 2.0, 0.5) if with_x else None
        self.y = make((rows, cols), t, 1.5, 0.25) if with_y else None
        self.gate = make((gates, cols), t, 0.7) if gates and with_y else None
        p = {"post_w": make((1, cols), t, 0.2, 1.0), "post_b": make((1, cols), t, 0.3),
             "pre_w": make((1, cols), t, 0.2, 1.0), "pre_b": make((1, cols), t, 0.3)}
        self.p = p
        self.dn, self.dh = make((rows, cols), torch.float32, 64.0), make((rows, cols), torch.float32, 64.0)
        self.join = Join(ctx, cols, half=half, half_stream=half_stream, post_norm=post if with_y else NONE, pre_norm=pre,
                         gate_act=gate_act, scale=scale, **p)

    def d(self, name):
        v = getattr(self, name) if hasattr(self, name) else self.p[name]
        return None if v is None else v.cpu().double()


def norm_parts(v, kind):
    """mean, 1/deviation, and the magnitudes that their roundings scale with."""
    z = torch.zeros(v.shape[0], 1, dtype=torch.float64)
    if kind == NONE:
        return z, z + 1, z
    mean = v.mean(1, keepdim=True) if kind == LAYER else z
    return mean, 1 / ((v - mean).square().mean(1, keepdim=True) + EPS).sqrt(), v.abs().mean(1, keepdim=True)


def gate_of(c):
    g = c.d("gate")
    if g is None:
        return torch.ones(1, c.cols, dtype=torch.float64), torch.zeros(1, c.cols, dtype=torch.float64)
    a = {IDENTITY: g, SIGMOID: torch.sigmoid(g), TANH: torch.tanh(g)}[c.act]
    return a, {IDENTITY: torch.ones_like(g), SIGMOID: a * (1 - a), TANH: 1 - a * a}[c.act]


def near(name, got, want, tol, dtype=torch.float32):
    if dtype is torch.float16:
        tol = tol + want.abs() * 2.0 ** -11 + 2.0 ** -25
    d = (got.cpu().double() - want).abs()
    worst = (d / tol.clamp(min=1e-300)).max().item() if d.numel() else 0.0
    assert not torch.isnan(d).any() and (d <= tol).all(), f"{name}: {worst:.3g} of its tolerance, off by {d.max().item():.3g}"


def forward_ref(c, h_stored):
    """h before it is rounded, n from h as stored, with their tolerances."""
    h = torch.zeros(c.rows, c.cols, dtype=torch.float64)
    mag = h.clone()
    if c.x is not None:
        h = c.scale * c.d("x")
        mag = h.abs()
    if c.y is not None:
        y = c.d("y")
        mean, r, m1 = norm_parts(y, c.post)
        u, um = (y - mean) * r, (y.abs() + m1) * r
        if c.post:
            u, um = u * c.d("post_w"), um * c.d("post_w").abs()
        if c.post == LAYER:
            u, um = u + c.d("post_b"), um + c.d("post_b").abs()
        a, _ = gate_of(c)
        h, mag = h + a * u, mag + a.abs() * um
    n = h_stored.cpu().double()
    mean, r, m1 = norm_parts(n, c.pre)
    nm = (n.abs() + m1) * r
    n = (n - mean) * r
    if c.pre:
        n, nm = n * c.d("pre_w"), nm * c.d("pre_w").abs()
    if c.pre == LAYER:
        n, nm = n + c.d("pre_b"), nm + c.d("pre_b").abs()
    return h, 64 * U * mag, n, 64 * U * nm


def check_forward(c):
    outs = [guarded((c.rows, c.cols), c.r, c.offset), guarded((c.rows, c.cols), c.t, c.offset),
            guarded((4, c.rows), torch.float32)]
    h, n, stats = (v for _, v in outs)
    c.join.forward(c.x, c.y, c.gate, h=h, n=n, stats=stats)
    torch.cuda.synchronize()
    assert_guards(outs)
    rh, th, rn, tn = forward_ref(c, h)
    near("h", h, rh, th, c.r)
    near("n", n, rn, tn, c.t)
    zero = torch.zeros(c.rows, 1, dtype=torch.float64)
    y = norm_parts(c.d("y"), c.post) if c.y is not None else (zero, zero + 1, zero)
    hs = norm_parts(h.cpu().double(), c.pre)
    want = torch.cat([y[0].t(), y[1].t(), hs[0].t(), hs[1].t()])
    near("stats", stats, want, 64 * U * (want.abs() + torch.cat([y[2].t(), y[1].t(), hs[2].t(), hs[1].t()])))
    return h, n, stats


def backward_ref(c, h, with_dn=True, with_dh=True):
    """The gradients and the same formulas over magnitudes."""
    z = torch.zeros(c.rows, c.cols, dtype=torch.float64)
    dh = c.d("dh") if with_dh else z
    d, dm = dh, dh.abs()
    out = {"post_w": z[:1], "post_b": z[:1], "pre_w": z[:1], "pre_b": z[:1]}
    out = {k: (v, v) for k, v in out.items()}
    if with_dn:
        dn, hs = c.d("dn"), h.cpu().double()
        mean, r, m1 = norm_parts(hs, c.pre)
        hat, hm = (hs - mean) * r, (hs.abs() + m1) * r
        if c.pre:
            w = c.d("pre_w")
            t, tm = dn * w, (dn * w).abs()
            step = t - hat * (t * hat).mean(1, keepdim=True)
            mag = tm + hm * (tm * hm).mean(1, keepdim=True)
            if c.pre == LAYER:
                step, mag = step - t.mean(1, keepdim=True), mag + tm.mean(1, keepdim=True)
                out["pre_b"] = (dn.sum(0, keepdim=True), dn.abs().sum(0, keepdim=True))
            out["pre_w"] = ((dn * hat).sum(0, keepdim=True), (dn.abs() * hm).sum(0, keepdim=True))
            d, dm = d + r * step, dm + r * mag
        else:
            d, dm = d + dn, dm + dn.abs()
    out["dx"] = (c.scale * d, abs(c.scale) * dm)
    if c.y is None:
        return out
    y = c.d("y")
    mean, r, m1 = norm_parts(y, c.post)
    hat, hm = (y - mean) * r, (y.abs() + m1) * r
    a, slope = gate_of(c)
    u, um = hat, hm
    if c.post:
        u, um = u * c.d("post_w"), um * c.d("post_w").abs()
    if c.post == LAYER:
        u, um = u + c.d("post_b"), um + c.d("post_b").abs()
    if c.gate is not None:
        dg, gm = d * u * slope, dm * um * (slope.abs() + 1)   # 1 - a a: off by u of 1
        if c.gate.shape[0] == 1:
            dg, gm = dg.sum(0, keepdim=True), gm.sum(0, keepdim=True)
        out["dgate"] = (dg, gm)
    du, dum = d * a, dm * a.abs()
    if c.post:
        w = c.d("post_w")
        out["post_w"] = ((du * hat).sum(0, keepdim=True), (dum * hm).sum(0, keepdim=True))
        if c.post == LAYER:
            out["post_b"] = (du.sum(0, keepdim=True), dum.sum(0, keepdim=True))
        b, bm = du * w, dum * w.abs()
        step, mag = b - hat * (b * hat).mean(1, keepdim=True), bm + hm * (bm * hm).mean(1, keepdim=True)
        if c.post == LAYER:
            step, mag = step - b.mean(1, keepdim=True), mag + bm.mean(1, keepdim=True)
        out["dy"] = (r * step, r * mag)
    else:
        out["dy"] = (du, dum)
    return out


def check_backward(c, h, stats, with_dn=True, with_dh=True):
    wide = (c.rows, c.cols)
    outs = {"dx": guarded(wide, torch.float32, c.offset), "dparam": guarded((4, c.cols), torch.float32, c.offset)}
    if c.y is not None:
        outs["dy"] = guarded(wide, torch.float32, c.offset)
    if c.gate is not None:
        outs["dgate"] = guarded(tuple(c.gate.shape), torch.float32, c.offset)
    c.join.backward(h, c.y, c.gate, stats, c.dn if with_dn else None, c.dh if with_dh else None,
                    **{k: v for k, (_, v) in outs.items()})
    torch.cuda.synchronize()
    assert_guards(outs.values())
    ref = backward_ref(c, h, with_dn, with_dh)
    for k in ("dx", "dy", "dgate"):
        if k in outs:
            near(k, outs[k][1], ref[k][0], (512 if k == "dgate" else 128) * U * ref[k][1])
    for i, k in enumerate(("post_w", "post_b", "pre_w", "pre_b")):
        near("d" + k, outs["dparam"][1][i:i + 1], ref[k][0], 512 * U * ref[k][1])
    return {k: v.clone() for k, (_, v) in outs.items()}


# every width class and its edges; rows that end inside a workgroup's four, one row, none aligned
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 2), (5, 511), (7, 512), (2, 513), (9, 777), (4, 1024), (3, 1025),
                                       (6, 2048), (3, 2049), (2, 4096), (3, 4099), (2, 8192), (1, 8191), (1300, 96)])
@pytest.mark.parametrize("half,half_stream", [(True, True), (True, False), (False, False)])
def test_widths(ctx, rows, cols, half, half_stream):
    print(f"join {rows}x{cols} half={half} half_stream={half_stream}", flush=True)
    c = Case(ctx, rows, cols, half, half_stream, LAYER, LAYER, 1, SIGMOID, 0.75, seed=rows + cols)
    h, _, stats = check_forward(c)
    check_backward(c, h, stats)


# the last width of each form and the next, in rows that end inside a workgroup and start at every remainder of 4
@pytest.mark.parametrize("rows,cols", [(33, 63), (17, 64), (19, 65), (1, 66), (9, 255), (5, 256), (6, 257), (2600, 61), (1300, 509),
                                       (530, 1023), (900, 1025), (300, 4095), (300, 4097)])
@pytest.mark.parametrize("half,half_stream", [(True, True), (True, False), (False, False)])
def test_edges_of_the_forms(ctx, rows, cols, half, half_stream):
    print(f"join {rows}x{cols} half={half} half_stream={half_stream}", flush=True)
    for norm, gates in ((LAYER, rows), (RMS, 1)):
        c = Case(ctx, rows, cols, half, half_stream, norm, norm, gates, TANH, 1.25, seed=rows + cols)
        h, _, stats = check_forward(c)
        check_backward(c, h, stats)


@pytest.mark.parametrize("rows,cols,post,pre,gates,half,half_stream", [
    (600, 5120, LAYER, LAYER, 1, True, True), (600, 5120, RMS, RMS, 1, True, False), (517, 8191, LAYER, RMS, 517, False, False),
    (530, 4101, NONE, LAYER, 1, True, True), (700, 6000, RMS, NONE, 1, False, False)])
def test_wide_rows_behind_each_other(ctx, rows, cols, post, pre, gates, half, half_stream):
    """Workgroups with several rows of more than 4096 columns, whose column sums go from row to row."""
    print(f"join {rows}x{cols} post={post} pre={pre}", flush=True)
    c = Case(ctx, rows, cols, half, half_stream, post, pre, gates, SIGMOID, 0.75, seed=rows + cols)
    h, _, stats = check_forward(c)
    first = check_backward(c, h, stats)
    second = check_backward(c, h, stats)
    for k in first:
        assert torch.equal(first[k], second[k]), k


@pytest.mark.parametrize("post", [NONE, RMS, LAYER])
@pytest.mark.parametrize("pre", [NONE, RMS, LAYER])
@pytest.mark.parametrize("gates,act", [(0, IDENTITY), (1, IDENTITY), (1, TANH), (11, SIGMOID), (11, IDENTITY)])
def test_forms(ctx, post, pre, gates, act):
    for half, half_stream in ((True, False), (False, False)):
        c = Case(ctx, 11, 300, half, half_stream, post, pre, gates, act, 1.0, seed=3 + post + pre)
        h, _, stats = check_forward(c)
        check_backward(c, h, stats)


@pytest.mark.parametrize("offset", [1, 3, 5])
def test_any_alignment(ctx, offset):
    for half, half_stream, cols in ((True, True, 640), (True, False, 2048), (False, False, 4096)):
        c = Case(ctx, 5, cols, half, half_stream, RMS, LAYER, 5, SIGMOID, 1.25, seed=offset, offset=offset)
        h, _, stats = check_forward(c)
        check_backward(c, h, stats)


def test_ends_of_a_network(ctx):
    """Without a stream (the first join), without a block (a norm alone), one gradient only."""
    c = Case(ctx, 6, 384, True, False, RMS, RMS, 1, TANH, 1.0, with_x=False)
    h, _, stats = check_forward(c)
    check_backward(c, h, stats, with_dn=False)
    check_backward(c, h, stats, with_dh=False)
    c = Case(ctx, 6, 384, True, False, NONE, LAYER, 0, IDENTITY, 0.5, with_y=False)
    h, _, stats = check_forward(c)
    check_backward(c, h, stats)


def test_in_place_and_partial_outputs(ctx):
    c = Case(ctx, 10, 1000, True, False, RMS, RMS, 1, IDENTITY, 1.0)
    h, n, stats = check_forward(c)
    x, y = c.x.clone(), c.y.clone()
    c.join.forward(x, y, c.gate, h=x, n=y)
    only = torch.empty_like(n)
    c.join.forward(c.x, c.y, c.gate, n=only)
    torch.cuda.synchronize()
    assert torch.equal(x, h) and torch.equal(y, n) and torch.equal(only, n)
    full = check_backward(c, h, stats)
    dh = c.dh.clone()
    c.join.backward(h, c.y, c.gate, stats, c.dn, dh, dx=dh)
    dg = torch.empty(1, 1000, device="cuda")
    c.join.backward(h, c.y, c.gate, stats, c.dn, c.dh, dgate=dg)
    torch.cuda.synchronize()
    assert torch.equal(dh, full["dx"]) and torch.equal(dg, full["dgate"])


def test_many_rows(ctx):
    """More rows than workgroups, in fp32 sums of thousands of terms, the same twice."""
    c = Case(ctx, 1500, 640, True, True, RMS, RMS, 1, IDENTITY, 1.0)
    h, _, stats = check_forward(c)
    first = check_backward(c, h, stats)
    second = check_backward(c, h, stats)
    for k in first:
        assert torch.equal(first[k], second[k]), k


def test_more_rows_than_workgroups(ctx):
    """Workgroups that go on to another row, with one sum (and one barrier) in each row."""
    rows, cols = (1 << 20) + 9, 1030
    g = torch.Generator(device="cuda").manual_seed(3)
    few = torch.randn(8, cols, generator=g, device="cuda").half()
    join = Join(ctx, cols, half=True, half_stream=True, pre_norm=RMS, pre_w=torch.ones(1, cols, device="cuda").half())
    want, got = torch.empty_like(few), torch.empty(rows, cols, dtype=torch.float16, device="cuda")
    y = few.repeat(-(-rows // 8), 1)[:rows].contiguous()
    join.forward(None, few, n=want)
    join.forward(None, y, n=got)
    torch.cuda.synchronize()
    whole = rows // 8 * 8
    assert (got[:whole].view(-1, 8, cols) == want).all() and torch.equal(got[whole:], want[:rows - whole])


def test_against_differences(ctx):
    """dx, dy, dgate and dparam against central differences of the fp32 forward: step 2^-6, whose
    third-order term and fp32 rounding (64 u |f| / step) stay under 1e-3 of the gradients' scale."""
    c = Case(ctx, 3, 40, False, False, LAYER, RMS, 1, SIGMOID, 0.75, seed=5)
    h, n, stats = check_forward(c)
    got = check_backward(c, h, stats)
    a, b = c.dn.cpu().double(), c.dh.cpu().double()

    def value():
        h, n = torch.empty_like(c.x), torch.empty_like(c.y)
        c.join.forward(c.x, c.y, c.gate, h=h, n=n)
        torch.cuda.synchronize()
        return (a * n.cpu().double()).sum() + (b * h.cpu().double()).sum()

    step = 2.0 ** -6
    grads = {"dx": c.x, "dy": c.y, "dgate": c.gate}
    for i, k in enumerate(("post_w", "post_b", "pre_w")):
        grads[i] = c.p[k]
    for k, t in grads.items():
        g = got["dparam"][k:k + 1] if isinstance(k, int) else got[k]
        for at in ((0, 0), (t.shape[0] - 1, 17), (0, 39)):
            old = t[at].item()
            t[at] = old + step
            up = value()
            t[at] = old - step
            down = value()
            t[at] = old
            assert abs((up - down) / (2 * step) - g[at].item()) <= 1e-3 * g.abs().max().item() + 0.5, (k, at)


def test_captured_and_replayed(ctx):
    """Forward and backward in one graph, replayed on new inputs with eager calls in between."""
    c = Case(ctx, 40, 1024, True, False, RMS, RMS, 1, SIGMOID, 1.0)
    side = torch.cuda.Stream()
    cap = abi.Context(0, 16, stream=side.cuda_stream)
    try:
        wide = (40, 1024)
        out = {"dx": torch.empty(wide, device="cuda"), "dy": torch.empty(wide, device="cuda"),
               "dgate": torch.empty(1, 1024, device="cuda"), "dparam": torch.empty(4, 1024, device="cuda")}
        h, n, stats = torch.empty_like(c.x), torch.empty_like(c.y), torch.empty(4, 40, device="cuda")
        work = torch.empty(abi.load().skl_residual_work_bytes(40, 1024) // 4, device="cuda")
        j = Join(cap, 1024, half=True, post_norm=RMS, pre_norm=RMS, gate_act=SIGMOID, **c.p)

        def both(join, h, n, stats, out, work):
            join.forward(c.x, c.y, c.gate, h=h, n=n, stats=stats)
            join.backward(h, c.y, c.gate, stats, c.dn, c.dh, work=work, **out)

        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side, capture_error_mode="thread_local"):
            both(j, h, n, stats, out, work)
        for rep in range(3):
            c.y.copy_(torch.randn(wide, device="cuda"))
            c.dn.copy_(torch.randn(wide, device="cuda") * (rep + 1))
            for v in out.values():
                v.fill_(float("nan"))
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            want = {k: torch.empty_like(v) for k, v in out.items()}
            eh, en, es = torch.empty_like(h), torch.empty_like(n), torch.empty_like(stats)
            both(c.join, eh, en, es, want, None)
            torch.cuda.synchronize()
            assert torch.equal(eh, h) and torch.equal(en, n) and torch.equal(es, stats)
            for k in out:
                assert torch.equal(want[k], out[k]), k
    finally:
        torch.cuda.synchronize()
        cap.close()


def test_a_captured_joins_own_workspace_outlives_larger_batches(ctx):
    """A Join whose own workspace grows behind a capture leaves the captured call's alone."""
    c = Case(ctx, 16, 512, True, True, RMS, RMS, 0, IDENTITY, 1.0)
    side = torch.cuda.Stream()
    cap = abi.Context(0, 16, stream=side.cuda_stream)
    try:
        j = Join(cap, 512, half=True, half_stream=True, post_norm=RMS, pre_norm=RMS, **c.p)
        h, n, stats, dparam = torch.empty_like(c.x), torch.empty_like(c.y), torch.empty(4, 16, device="cuda"), torch.empty(4, 512, device="cuda")
        torch.cuda.synchronize()
        j.forward(c.x, c.y, h=h, n=n, stats=stats)
        j.backward(h, c.y, None, stats, c.dn, c.dh, dparam=dparam)
        torch.cuda.synchronize()
        want, work = dparam.clone(), j._work[-1]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side, capture_error_mode="thread_local"):
            j.backward(h, c.y, None, stats, c.dn, c.dh, dparam=dparam)
        big = Case(ctx, 600, 512, True, True, RMS, RMS, 0, IDENTITY, 1.0)
        bh, bn, bs = torch.empty_like(big.x), torch.empty_like(big.y), torch.empty(4, 600, device="cuda")
        torch.cuda.synchronize()
        j.forward(big.x, big.y, h=bh, n=bn, stats=bs)
        j.backward(bh, big.y, None, bs, big.dn, big.dh, dparam=torch.empty(4, 512, device="cuda"))
        assert j._work[-1] is not work and j._work[0] is work
        for _ in range(3):
            dparam.fill_(float("nan"))
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(dparam, want)
    finally:
        torch.cuda.synchronize()
        cap.close()


def test_values_that_are_not_finite_stay_in_their_rows(ctx):
    c = Case(ctx, 4, 700, True, False, RMS, LAYER, 1, IDENTITY, 1.0)
    clean_h, clean_n, stats = check_forward(c)
    clean_h, clean_n = clean_h.clone(), clean_n.clone()
    c.y[1, 3] = float("nan")
    c.x[2, 5] = float("inf")
    h, n = torch.empty_like(c.x), torch.empty_like(c.y)
    c.join.forward(c.x, c.y, c.gate, h=h, n=n)
    torch.cuda.synchronize()
    assert torch.isnan(h[1]).all() and torch.isnan(n[1]).all() and torch.isnan(n[2, 5])
    for row in (0, 3):
        assert torch.equal(h[row], clean_h[row]) and torch.equal(n[row], clean_n[row])
    # a row of zeros: the root holds 1e-6
    c.y[:] = 0
    c.x[:] = 0
    c.join.forward(c.x, c.y, c.gate, h=h, n=n)
    torch.cuda.synchronize()
    assert (h == 0).all() and torch.equal(n, c.p["pre_b"].expand(4, 700))
