"""Gated blocks in a residual stream as they are trained and served: dropout of the input, then twice a join's norm,
a gated block and its projection back with dropout, a last norm and a head, one behind the other against the formula
in 64 bits, eager, captured, on streams of their own and one row at a time.

fp32: a run has 16 steps forward and back, each off by at most (F + 128) u of its terms' magnitudes (u = 2^-24;
products add up to F terms, a chain of two 2 F), which here are at most 8 times the largest result: 16 x 8 x
(2 F + 128) u of a result's largest element.  fp16: each step's result rounds to 2^-11 of itself, 16 x 8 steps of it.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from soklyn_amd import abi, dropout
from soklyn_amd.devblock import DeviceBlock
from soklyn_amd.gated import Gated, GatedBlock
from soklyn_amd.residual import Join, Projection
from tests.ffn_helpers import U, factors

pytestmark = pytest.mark.gpu
D, F, CLASSES, LAYERS, P, SCALE, LR = 72, 160, 30, 2, 0.25, 0.5, 0.25
TOL32, TOL16 = 16 * 8 * (2 * F + 128) * U, 16 * 8 * 2.0 ** -11
F32, F16 = torch.float32, torch.float16
SEEDS = [0x9E3779B9, 77, 0xFFFFFFF0]


class Stack:
    def __init__(self, ctx, rows, half, half_stream=False, max_batch=None):
        self.ctx, self.rows, self.half = ctx, rows, half
        m, g = max_batch or rows, np.random.default_rng(5)
        t, r = F16 if half else F32, F16 if half_stream else F32

        def make(shape, dtype, std, mean=0.0):
            return torch.from_numpy((g.standard_normal(shape) * std + mean).astype(np.float32)).to(dtype).cuda()

        def block(k, n, act, p=0.0):
            w = (g.standard_normal((k, n)) * k ** -0.5).astype(np.float16).astype(np.float32)
            b = (g.standard_normal((1, n)) * 0.2).astype(np.float16).astype(np.float32)
            return DeviceBlock(ctx, k, n, m, w, b=b, half=half, act=act, mask_coeff=p)

        def empty(*shape, dtype=F32):
            return torch.zeros(shape, dtype=dtype, device="cuda")

        self.x, self.up = make((rows, D), r, 1.0), make((rows, CLASSES), F32, 64.0)
        self.norms = [make((1, D), t, 0.2, 1.0) for _ in range(LAYERS + 1)]
        self.joins = [Join(ctx, D, half=half, half_stream=half_stream, pre_norm=abi.NORM_RMS, pre_w=w) for w in self.norms]
        self.gated = [GatedBlock(block(D, F, abi.ACT_SILU), block(D, F, abi.ACT_IDENTITY)) for _ in range(LAYERS)]
        self.down = [block(F, D, abi.ACT_TANH if i else abi.ACT_IDENTITY, P) for i in range(LAYERS)]
        self.head = block(D, CLASSES, abi.ACT_IDENTITY)
        self.h = [empty(rows, D, dtype=r) for _ in range(LAYERS + 1)]
        self.n = [empty(rows, D, dtype=t) for _ in range(LAYERS + 1)]
        self.mid = [empty(rows, F, dtype=t) for _ in range(LAYERS)]
        self.stats = [empty(4, rows) for _ in range(LAYERS + 1)]
        self.dn, self.dh = [[empty(rows, D) for _ in range(LAYERS + 1)] for _ in range(2)]
        self.dskip = [empty(rows, D) for _ in range(LAYERS)]
        self.dx, self.dw = empty(rows, D), [empty(4, D) for _ in range(LAYERS + 1)]
        size = abi.load().skl_residual_work_bytes(rows, D) // 4
        self.work = [empty(size) for _ in range(LAYERS + 1)]

    def forward(self):
        dropout.apply(self.ctx, self.x, self.h[0], P, SEEDS[2])
        for i in range(LAYERS):
            self.joins[i].forward(self.h[i], None, n=self.n[i], stats=self.stats[i])
            self.gated[i].forward(self.n[i], self.rows, self.mid[i])
            self.down[i].forward_residual(self.mid[i], self.rows, self.h[i], self.h[i + 1], scale=SCALE, use_dropout=True,
                                          seed=SEEDS[i])
        self.joins[LAYERS].forward(self.h[LAYERS], None, n=self.n[LAYERS], stats=self.stats[LAYERS])
        return self.head.forward(self.n[LAYERS], self.rows)

    def backward(self):
        """Errors and gradients; the weights stay."""
        self.head.error_from_sum_noalloc(self.up, self.rows)
        self.head.input_grad(self.rows, self.dn[LAYERS])
        self.joins[LAYERS].backward(self.h[LAYERS], None, None, self.stats[LAYERS], self.dn[LAYERS], None, dx=self.dh[LAYERS],
                                    dparam=self.dw[LAYERS], work=self.work[LAYERS])
        for i in reversed(range(LAYERS)):
            self.down[i].residual_error(self.dh[i + 1], self.rows, scale=SCALE, use_dropout=True, seed=SEEDS[i], dx=self.dskip[i])
            self.gated[i].hidden_error(self.down[i], self.rows)
            self.gated[i].input_grad(self.rows, self.dn[i])
            self.joins[i].backward(self.h[i], None, None, self.stats[i], self.dn[i], self.dskip[i], dx=self.dh[i],
                                   dparam=self.dw[i], work=self.work[i])
        dropout.apply(self.ctx, self.dh[0], self.dx, P, SEEDS[2])

    def update(self, tc):
        self.head.backward(self.n[LAYERS], tc, 1)
        for i in range(LAYERS):
            self.down[i].backward(self.mid[i], tc, 1)
            self.gated[i].backward(self.n[i], tc, 1)

    def blocks(self):
        return {"head": self.head} | {f"{n}{i}": b for i in range(LAYERS) for n, b in
                                      (("gate", self.gated[i].gate), ("up", self.gated[i].up), ("down", self.down[i]))}

    def results(self):
        return ({"logits": self.head.out[:self.rows], "dx": self.dx} | {f"dnorm{i}": w[2:3] for i, w in enumerate(self.dw)} |
                {f"{n}_d": b.d_prenorm[:self.rows] for n, b in self.blocks().items()})

    def leaves(self):
        named = {"x": self.x} | {f"norm{i}": w for i, w in enumerate(self.norms)}
        for n, b in self.blocks().items():
            named |= {n: b.w, n + "_b": b.b}
        return {k: v.cpu().double().requires_grad_() for k, v in named.items()}

    def formula(self, leaf):
        def rms(v, w):
            return v / (v.square().mean(1, keepdim=True) + 1e-6).sqrt() * w

        def layer(v, n):
            return v @ leaf[n] + leaf[n + "_b"]

        h = leaf["x"] * factors(self.rows, D, P, SEEDS[2])
        for i in range(LAYERS):
            n = rms(h, leaf[f"norm{i}"])
            a = layer(n, f"gate{i}")
            z = layer(a * torch.sigmoid(a) * layer(n, f"up{i}"), f"down{i}")
            h = SCALE * h + factors(self.rows, D, P, SEEDS[i]) * (torch.tanh(z) if i else z)
        return layer(rms(h, leaf[f"norm{LAYERS}"]), "head")


def near(name, got, want, tol):
    got, want = got.detach().cpu().double(), want.detach()
    off = ((got - want).abs().max() / want.abs().max()).item()
    print(f"{name}: {off:.2e} of the largest, {tol:.1e} allowed", flush=True)
    assert off <= tol, name


FORMS = [(False, False), (True, False), (True, True)]


@pytest.mark.parametrize("rows,max_batch", [(1, 1), (37, 64), (300, 300)])
@pytest.mark.parametrize("half,half_stream", FORMS)
def test_training_step(ctx, rows, max_batch, half, half_stream):
    t = Stack(ctx, rows, half, half_stream, max_batch)
    leaf = t.leaves()
    was = {n: ((b.master_w if half else b.w).clone(), (b.master_b if half else b.b).clone()) for n, b in t.blocks().items()}
    t.forward()
    t.backward()
    t.update(abi.train_ctx(abi.sgd(), abi.sgd(), rows, LR))
    torch.cuda.synchronize()
    z = t.formula(leaf)
    tol = TOL16 if half else TOL32
    near("logits", t.head.out[:rows], z, tol)
    (z * t.up.cpu().double()).sum().backward()
    near("dx", t.dx, leaf["x"].grad, tol)
    for i, w in enumerate(t.dw):
        near(f"norm{i}", w[2:3], leaf[f"norm{i}"].grad, tol)
    for n, b in t.blocks().items():
        for name, now, before in ((n, b.master_w if half else b.w, was[n][0]), (n + "_b", b.master_b if half else b.b, was[n][1])):
            # the step, lr / 512 / rows of the gradient, as the difference of two weights: half a step of each
            g = leaf[name].grad * (LR / 512 / rows)
            off = ((now.double() - before.double()).cpu() + g).abs().max()
            assert off <= tol * g.abs().max() + 2 * U * before.abs().max().item(), name


def test_captured_and_replayed(ctx):
    """One graph of the whole step, its products over padded copies among it, replayed on new inputs with eager
    steps in between."""
    side = torch.cuda.Stream()
    cap = abi.Context(0, 16, stream=side.cuda_stream)
    try:
        t, eager = Stack(cap, 130, True), Stack(ctx, 130, True)
        t.forward()
        t.backward()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side, capture_error_mode="thread_local"):
            t.forward()
            t.backward()
        for rep in range(3):
            v = torch.randn_like(t.x) * (rep + 1)
            t.x.copy_(v)
            eager.x.copy_(v)
            for r in t.results().values():
                r.fill_(float("nan"))
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            eager.forward()
            eager.backward()
            torch.cuda.synchronize()
            for k, r in eager.results().items():
                assert torch.equal(r, t.results()[k]), (rep, k)
    finally:
        torch.cuda.synchronize()
        cap.close()


def test_two_graphs_of_copied_operands(ctx):
    """Two captured products whose operands are copied into workspaces: each object has its own, so replays in
    flight together do not meet; a larger call in between leaves the captured workspace alone."""
    t, n = F16, 259
    streams = [torch.cuda.Stream() for _ in range(2)]
    cs = [abi.Context(0, 16, stream=s.cuda_stream) for s in streams]
    try:
        work = []
        for i, (c, s) in enumerate(zip(cs, streams)):
            g = torch.Generator(device="cuda").manual_seed(i)
            x, wg, wu = (torch.randn(sh, generator=g, device="cuda").to(t) * 0.1 for sh in ((4001, 131), (131, n), (131, n)))
            op, out = Gated(c, wg, wu, outputs=n, half=True), torch.empty((4001, n), dtype=t, device="cuda")
            torch.cuda.synchronize()
            op.forward(x, out)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=s, capture_error_mode="thread_local"):
                op.forward(x, out)
            big = torch.randn((9000, 131), generator=g, device="cuda").to(t)
            op.forward(big, torch.empty((9000, n), dtype=t, device="cuda"))
            torch.cuda.synchronize()
            work.append((graph, op, x, out, s))
        for rep in range(3):
            for _, _, x, out, _ in work:
                x.mul_(-1.5)
                out.fill_(float("nan"))
            torch.cuda.synchronize()
            for graph, _, _, _, s in work:
                with torch.cuda.stream(s):
                    graph.replay()
            torch.cuda.synchronize()
            for _, op, x, out, _ in work:
                want = torch.empty_like(out)
                op.forward(x, want)
                torch.cuda.synchronize()
                assert torch.equal(out, want), rep
    finally:
        torch.cuda.synchronize()
        for c in cs:
            c.close()


def test_graphs_of_few_rows(ctx):
    """The sums over slices of k are in workspaces: calls captured before any eager one, each object with its own,
    replayed in flight together, with larger and smaller eager calls of the same objects in between."""
    t, k, n = F16, 4096, 520
    streams = [torch.cuda.Stream() for _ in range(2)]
    cs = [abi.Context(0, 16, stream=s.cuda_stream) for s in streams]
    try:
        work = []
        for i, (c, s) in enumerate(zip(cs, streams)):
            g = torch.Generator(device="cuda").manual_seed(i)
            x, wg, wu, wp, x32 = (torch.randn(sh, generator=g, device="cuda").to(t) * 0.02
                                  for sh in ((3, k), (k, n), (k, n), (k, n), (32, k)))
            gate, project = Gated(c, wg, wu, outputs=n, half=True), Projection(c, wp, None, outputs=n, half=True, dropout=0.5)
            mid, h = torch.empty((3, n), dtype=t, device="cuda"), torch.randn((3, n), generator=g, device="cuda")
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=s, capture_error_mode="thread_local"):
                gate.forward(x, mid)
                project.forward(x, h, h, seed=i)
            work.append((graph, gate, project, x, mid, h, x32, s, i))
        for rep in range(4):
            want = []
            for _, gate, project, x, mid, h, x32, s, i in work:
                x.mul_(-1.25)
                torch.cuda.synchronize()
                a, b = torch.empty_like(mid), torch.empty_like(h)
                gate.forward(x, a)
                project.forward(x, h, b, seed=i)
                rows = 32 if rep % 2 else 1
                gate.forward(x32[:rows], torch.empty((rows, n), dtype=t, device="cuda"))
                want.append((a, b))
                mid.fill_(float("nan"))
            torch.cuda.synchronize()
            for graph, *_, s, _ in work:
                with torch.cuda.stream(s):
                    graph.replay()
            torch.cuda.synchronize()
            for (_, _, _, _, mid, h, *_), (a, b) in zip(work, want):
                assert torch.equal(mid, a) and torch.equal(h, b), rep
    finally:
        torch.cuda.synchronize()
        for c in cs:
            c.close()


def test_workspaces_belong_to_the_context_s_stream(ctx):
    """What a dropped object held goes to allocations of its context's stream alone, behind its last kernels."""
    side = torch.cuda.Stream()
    other = abi.Context(0, 16, stream=side.cuda_stream)
    try:
        size = 96 << 20
        piece = abi.Workspace(other)
        at, have = piece.get(size)
        assert have == size and piece.get(1000)[0] == at
        torch.cuda.synchronize()
        del piece
        elsewhere = torch.empty(size, dtype=torch.uint8, device="cuda")
        assert elsewhere.data_ptr() != at
        with torch.cuda.stream(side):
            assert torch.empty(size, dtype=torch.uint8, device="cuda").data_ptr() == at
    finally:
        torch.cuda.synchronize()
        other.close()


def test_weights_exchanged_for_others(ctx):
    """An object's weights may be exchanged; ones of another size, type or layout are refused."""
    wg, wu, w2 = (torch.randn((64, 40), device="cuda") for _ in range(3))
    x, out, h = torch.randn((5, 64), device="cuda"), torch.empty((5, 40), device="cuda"), torch.zeros((5, 40), device="cuda")
    op, pr = Gated(ctx, wg, wu, outputs=40, act=abi.ACT_IDENTITY), Projection(ctx, wg, None, outputs=40)
    op.wg = pr.w = w2
    op.forward(x, out)
    pr.forward(x, None, h)
    torch.cuda.synchronize()
    a, u = x.double() @ w2.double(), x.double() @ wu.double()
    size, other = x.double().abs() @ w2.double().abs(), x.double().abs() @ wu.double().abs()
    assert bool(((h.double() - a).abs() <= 128 * U * size).all())
    assert bool(((out.double() - a * u).abs() <= 4 * 128 * U * size * other).all())
    for bad in (w2[:32], w2.half(), w2.t(), torch.cat([w2, w2])):
        op.wg = pr.w = bad
        with pytest.raises(ValueError):
            op.forward(x, out)
        with pytest.raises(ValueError):
            pr.forward(x, None, h)
    op.wg, op.outputs = w2, 400
    with pytest.raises(ValueError):
        op.forward(x, torch.empty((5, 400), device="cuda"))


def test_weights_moved_in_place(ctx):
    """A weight whose memory is another one's now is read there."""
    wg, wu, other = (torch.randn((64, 40), device="cuda") for _ in range(3))
    x, got, want = torch.randn((5, 64), device="cuda"), torch.empty((5, 40), device="cuda"), torch.empty((5, 40), device="cuda")
    op, pr = Gated(ctx, wg, wu, outputs=40), Projection(ctx, wg, None, outputs=40)
    op.forward(x, got)
    pr.forward(x, None, got)
    torch.cuda.synchronize()
    wg.data = other.clone()
    torch.cuda.synchronize()
    for of, new in ((op, Gated(ctx, other, wu, outputs=40)), (pr, Projection(ctx, other, None, outputs=40))):
        args = (x, got) if of is op else (x, None, got)
        of.forward(*args)
        new.forward(*args[:-1], want)
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_two_contexts_at_once(ctx):
    """Steps of two contexts on streams of their own, in flight together, give what each gives alone."""
    side = torch.cuda.Stream()
    other = abi.Context(0, 16, stream=side.cuda_stream)
    try:
        stacks = [Stack(ctx, 200, True, True), Stack(other, 200, True, True)]
        stacks[1].x.mul_(2)
        torch.cuda.synchronize()
        alone = []
        for t in stacks:
            t.forward()
            torch.cuda.synchronize()
            alone.append([v.clone() for v in (*t.mid, *t.h, t.head.out)])
        for c in (ctx, other):
            c.set_sync(False)
        for _ in range(4):
            for t in stacks:
                t.forward()
        torch.cuda.synchronize()
        for t, want in zip(stacks, alone):
            for a, b in zip((*t.mid, *t.h, t.head.out), want):
                assert torch.equal(a, b)
    finally:
        torch.cuda.synchronize()
        ctx.set_sync(True)
        other.close()


@pytest.mark.parametrize("half", [False, True])
def test_served_row_by_row(ctx, half):
    """Single rows through Gated and Projection over the trained weights, nothing kept, against the same rows of the
    whole batch: the sums run in another order, so as near as two runs of a step may be."""
    rows, t = 9, F16 if half else F32
    s = Stack(ctx, rows, half)
    s.forward()
    torch.cuda.synchronize()
    b, down = s.gated[0], s.down[0]
    op = Gated(ctx, b.gate.w, b.up.w, b.gate.b, b.up.b, outputs=F, half=half, act=abi.ACT_SILU)
    proj = Projection(ctx, down.w, down.b, outputs=D, half=half, scale=SCALE)
    mid, h = torch.empty((1, F), dtype=t, device="cuda"), torch.empty((1, D), device="cuda")
    every = torch.empty((rows, D), device="cuda")
    proj.forward(s.mid[0], s.h[0], every)
    for i in range(rows):
        op.forward(s.n[0][i:i + 1], mid)
        near(f"gated {i}", mid, s.mid[0][i:i + 1].cpu().double(), 8 * 2.0 ** -11 if half else 8 * (D + 128) * U)
        proj.forward(s.mid[0][i:i + 1], s.h[0][i:i + 1], h)
        near(f"projection {i}", h, every[i:i + 1].cpu().double(), 8 * (F + 128) * U)
