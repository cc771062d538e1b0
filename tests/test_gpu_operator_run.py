"""A residual network as it is trained, distilled and then served in 4 bits: joins, blocks, the
distillation error and the 4-bit layers one behind the other, against the formulas in 64 bits.

fp32: a run has 12 steps forward and back, each off by at most (D + 128) u of its terms' magnitudes
(u = 2^-24; products add D terms, joins and the error 128), which here are at most 8 times the largest
result: 12 x 8 x 224 u = 1.3e-3 of a result's largest element.  fp16: each step's result rounds to
2^-11 of itself, 12 x 8 steps at most 4.7e-2 of the largest.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from soklyn_amd import abi, mxfp4
from soklyn_amd.devblock import DeviceBlock
from soklyn_amd.residual import Join
from tests.helpers import he_normal, rng

pytestmark = pytest.mark.gpu

NONE, RMS, LAYER = abi.NORM_DISABLED, abi.NORM_RMS, abi.NORM_LAYER
D, CLASSES, TOP = 96, 203, 9
TAU, ALPHA, SCALE = 2.0, 0.75, 0.5
TOL32, TOL16 = 12 * 8 * 224 * 2.0 ** -24, 12 * 8 * 2.0 ** -11


class Tower:
    """x -> [norm] -> block -> join -> block -> join -> head."""

    def __init__(self, ctx, rows, half, half_stream, max_batch=None):
        self.ctx, self.rows, self.half = ctx, rows, half
        g, M = rng(31), max_batch or rows
        t = torch.float16 if half else torch.float32
        r = torch.float16 if half_stream else torch.float32

        def make(shape, dtype, std, mean=0.0):
            return torch.from_numpy((g.standard_normal(shape) * std + mean).astype(np.float32)).to(dtype).cuda()

        def w(k, n):
            return he_normal(g, k, n).reshape(k, n).astype(np.float16).astype(np.float32)

        self.x = make((rows, D), r, 1.0)
        self.pre_w = [make((1, D), t, 0.2, 1.0) for _ in range(3)]
        self.pre_b = [make((1, D), t, 0.2) for _ in range(3)]
        self.post_w, self.post_b = make((1, D), t, 0.2, 1.0), make((1, D), t, 0.2)
        self.gates = [make((1, D), t, 0.7), make((rows, D), t, 0.7)]
        self.index = torch.from_numpy(np.stack([g.permutation(CLASSES)[:TOP] for _ in range(rows)]).astype(np.int32)).cuda()
        self.value = make((rows, TOP), torch.float32, 2.0)
        self.label = torch.from_numpy(g.integers(0, CLASSES, rows).astype(np.int32)).cuda()
        self.blocks = [DeviceBlock(ctx, D, D, M, w(D, D), half=half, act=abi.ACT_TANH),
                       DeviceBlock(ctx, D, D, M, w(D, D), half=half, act=abi.ACT_SILU),
                       DeviceBlock(ctx, D, CLASSES, M, w(D, CLASSES), half=half)]
        kind = dict(half=half, half_stream=half_stream)
        self.joins = [Join(ctx, D, pre_norm=RMS, pre_w=self.pre_w[0], **kind),
                      Join(ctx, D, post_norm=LAYER, pre_norm=RMS, gate_act=abi.ACT_SIGMOID, scale=SCALE, post_w=self.post_w,
                           post_b=self.post_b, pre_w=self.pre_w[1], **kind),
                      Join(ctx, D, pre_norm=LAYER, gate_act=abi.ACT_TANH, pre_w=self.pre_w[2], pre_b=self.pre_b[2], **kind)]

        def empty(shape, dtype=torch.float32):
            return torch.zeros(shape, dtype=dtype, device="cuda")

        self.h = [self.x, empty((rows, D), r), empty((rows, D), r)]
        self.n = [empty((rows, D), t) for _ in range(3)]
        self.stats = [empty((4, rows)) for _ in range(3)]
        self.loss = empty((rows,))
        self.dn = [empty((rows, D)) for _ in range(3)]
        self.dx = [empty((rows, D)) for _ in range(3)]
        self.dy = [None, empty((rows, D)), empty((rows, D))]
        self.dgate = [None, empty((1, D)), empty((rows, D))]
        self.dparam = [empty((4, D)) for _ in range(3)]
        size = abi.load().skl_residual_work_bytes(rows, D) // 4
        self.work = [empty((size,)) for _ in range(3)]

    def gate(self, i):
        return None if i == 0 else self.gates[i - 1]

    def forward(self):
        for i, (j, b) in enumerate(zip(self.joins, self.blocks)):
            y = self.blocks[i - 1].out[:self.rows] if i else None
            j.forward(self.h[i - 1] if i else self.x, y, self.gate(i), h=self.h[i] if i else None, n=self.n[i],
                      stats=self.stats[i])
            b.forward(self.n[i], self.rows)

    def backward(self, then=None):
        """then(block, its input): behind each block's error and the gradient of its input."""
        self.blocks[2].distill_error(self.index, self.value, self.label, temperature=TAU, alpha=ALPHA, loss=self.loss)
        for i in (2, 1, 0):
            b = self.blocks[i]
            if i < 2:
                b.error_from_sum_noalloc(self.dy[i + 1], self.rows)
            b.input_grad(self.rows, self.dn[i])
            if then:
                then(b, self.n[i])
            self.joins[i].backward(self.h[i], self.blocks[i - 1].out[:self.rows] if i else None, self.gate(i),
                                   self.stats[i], self.dn[i], self.dx[i + 1] if i < 2 else None, dx=self.dx[i],
                                   dy=self.dy[i], dgate=self.dgate[i], dparam=self.dparam[i], work=self.work[i])

    def results(self):
        got = {"loss": self.loss, "logits": self.blocks[2].out[:self.rows], "dx": self.dx[0]}
        for i in range(3):
            got |= {f"dparam{i}": self.dparam[i]} | ({f"dgate{i}": self.dgate[i]} if i else {})
        return got

    def leaves(self):
        named = {"x": self.x, "post_w": self.post_w, "post_b": self.post_b, "gate1": self.gates[0], "gate2": self.gates[1],
                 "pre_b2": self.pre_b[2]}
        named |= {f"pre_w{i}": w for i, w in enumerate(self.pre_w)} | {f"w{i}": b.w for i, b in enumerate(self.blocks)}
        return {k: v.cpu().double().requires_grad_() for k, v in named.items()}

    def formula(self, leaf):
        """Logits and loss [rows] of leaves, in 64 bits."""
        def rms(v, w):
            return v / (v.square().mean(1, keepdim=True) + 1e-6).sqrt() * w

        def layer(v, w, b):
            c = v - v.mean(1, keepdim=True)
            return rms(c, w) + b

        h = leaf["x"]
        y = torch.tanh(rms(h, leaf["pre_w0"]) @ leaf["w0"])
        h = SCALE * h + torch.sigmoid(leaf["gate1"]) * layer(y, leaf["post_w"], leaf["post_b"])
        z = rms(h, leaf["pre_w1"]) @ leaf["w1"]
        h = h + torch.tanh(leaf["gate2"]) * (z * torch.sigmoid(z))
        z = layer(h, leaf["pre_w2"], leaf["pre_b2"]) @ leaf["w2"]
        q = torch.log_softmax(self.value.cpu().double() / TAU, 1)
        p = torch.log_softmax(z / TAU, 1).gather(1, self.index.cpu().long())
        hard = torch.log_softmax(z, 1).gather(1, self.label.cpu().long()[:, None])[:, 0]
        return z, ALPHA * TAU ** 2 * (q.exp() * (q - p)).sum(1) - (1 - ALPHA) * hard


def near(name, got, want, tol):
    got, want = got.detach().cpu().double(), want.detach()
    off = ((got - want).abs().max() / want.abs().max()).item()
    print(f"{name}: {off:.2e} of the largest, {tol:.1e} allowed", flush=True)
    assert off <= tol, name


FORMS = [(False, False), (True, False), (True, True)]


@pytest.mark.parametrize("rows,max_batch", [(1, 1), (37, 64), (300, 300)])
@pytest.mark.parametrize("half,half_stream", FORMS)
def test_loss_and_gradients(ctx, rows, max_batch, half, half_stream):
    t = Tower(ctx, rows, half, half_stream, max_batch)
    tc = abi.train_ctx(abi.adam(), abi.adam(), rows, 0.0)
    leaf = t.leaves()
    t.forward()
    t.backward(lambda b, x: b.backward(x, tc, 1))
    torch.cuda.synchronize()
    z, loss = t.formula(leaf)
    loss.sum().backward()
    tol = TOL16 if half else TOL32
    near("logits", t.blocks[2].out[:rows], z, tol)
    near("loss", t.loss, loss, tol)
    want = {"dx": leaf["x"].grad, "dgate1": leaf["gate1"].grad, "dgate2": leaf["gate2"].grad}
    for k, g in want.items():
        near(k, t.results()[k] / 512, g, tol)
    for i, (row, k) in enumerate([(2, "pre_w0"), (0, "post_w"), (1, "post_b"), (2, "pre_w1"), (2, "pre_w2"), (3, "pre_b2")]):
        at = [0, 1, 1, 1, 2, 2][i]
        near(k, t.dparam[at][row:row + 1] / 512, leaf[k].grad, tol)
    for i, b in enumerate(t.blocks):   # Adam's first moment is the weights' gradient, to a factor
        m, g = b.dm_w.cpu().double(), leaf[f"w{i}"].grad
        near(f"w{i}", m * (g.norm() / m.norm()), g, 2 * tol)


def test_gradients_against_differences(ctx):
    """The change of the operators' own loss along the gradient is what the gradient says: both the
    losses' difference and its fp32 gradient are compared with those of the formula, so that the
    step's higher terms cancel."""
    t = Tower(ctx, 24, False, False)
    leaf = t.leaves()
    t.forward()
    t.backward()
    torch.cuda.synchronize()
    along = {"x": (t.x, t.dx[0]), "gate1": (t.gates[0], t.dgate[1]), "post_w": (t.post_w, t.dparam[1][0:1]),
             "pre_w1": (t.pre_w[1], t.dparam[1][2:3])}
    for k, (tensor, grad) in along.items():
        g = (grad / 512).clone()
        step = 0.05 / g.abs().max().item()
        kept, ends, refs = tensor.clone(), [], []
        for sign in (1, -1):
            tensor.copy_(kept + sign * step * g)
            t.forward()
            t.blocks[2].distill_error(t.index, t.value, t.label, temperature=TAU, alpha=ALPHA, loss=t.loss)
            torch.cuda.synchronize()
            ends.append(t.loss.cpu().double().sum().item())
            refs.append(t.formula(t.leaves())[1].sum().item())
        tensor.copy_(kept)
        got, want = (ends[0] - ends[1]) / (2 * step), (refs[0] - refs[1]) / (2 * step)
        z, loss = t.formula(leaf)
        exact = torch.autograd.grad(loss.sum(), leaf[k])[0]
        slope = (exact * g.cpu().double()).sum().item()
        rounding = TOL32 * abs(refs[0]) / step
        print(f"{k}: {got:.6g}, formula {want:.6g}, gradient {g.square().sum().item():.6g}", flush=True)
        assert abs(got - want) <= rounding
        assert abs(got - g.square().sum().item()) <= rounding + abs(want - slope) + TOL32 * abs(slope) * 2


def test_captured_and_replayed(ctx):
    """One graph of the whole step, replayed on new inputs with eager steps in between."""
    side = torch.cuda.Stream()
    cap = abi.Context(0, 16, stream=side.cuda_stream)
    try:
        t, eager = Tower(cap, 130, True, False), Tower(ctx, 130, True, False)
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


def test_two_contexts_at_once(ctx):
    """Steps of two contexts on streams of their own, in flight together, give what each gives alone."""
    side = torch.cuda.Stream()
    other = abi.Context(0, 16, stream=side.cuda_stream)
    try:
        towers = [Tower(ctx, 200, True, True), Tower(other, 200, True, True)]
        towers[1].x.mul_(2)
        torch.cuda.synchronize()
        alone = []
        for t in towers:
            t.forward()
            t.blocks[2].distill_error(t.index, t.value, t.label, temperature=TAU, alpha=ALPHA, loss=t.loss)
            torch.cuda.synchronize()
            alone.append([t.loss.clone(), t.blocks[2].out.clone(), t.blocks[2].grad.clone()])
        for c in (ctx, other):
            c.set_sync(False)
        for _ in range(4):
            for t in towers:
                t.loss.fill_(float("nan")) if t.ctx is ctx else None
                t.forward()
                t.blocks[2].distill_error(t.index, t.value, t.label, temperature=TAU, alpha=ALPHA, loss=t.loss)
        torch.cuda.synchronize()
        for t, want in zip(towers, alone):
            for a, b in zip((t.loss, t.blocks[2].out, t.blocks[2].grad), want):
                assert torch.equal(a, b)
    finally:
        torch.cuda.synchronize()
        ctx.set_sync(True)
        other.close()


@pytest.mark.parametrize("rows", [1, 16, 130])
@pytest.mark.parametrize("half,half_stream", FORMS)
def test_served_in_four_bits(ctx, rows, half, half_stream):
    """The trained blocks as 4-bit layers between the same joins: each layer against the product of the
    values that its codes and its input's stand for (fp32 sums of D terms, 2 D u of their magnitudes;
    the activations' own error 2^-20; a rounding to fp16), each join against the eager one on the
    same inputs."""
    t = Tower(ctx, rows, half, half_stream)
    layers = []
    for b, act in zip(t.blocks, (abi.ACT_TANH, abi.ACT_SILU, abi.ACT_IDENTITY)):
        codes, scales = mxfp4.quantise(ctx, b.w, down=True)
        layers.append(mxfp4.Layer(ctx, b.inputs, b.outputs, rows, codes, scales, half=half, act=act, b=b.b))
    acts = [torch.tanh, torch.nn.functional.silu, lambda z: z]
    y = None
    for i, (j, lay) in enumerate(zip(t.joins, layers)):
        j.forward(t.h[i - 1] if i else t.x, y, t.gate(i), h=t.h[i] if i else None, n=t.n[i])
        y = lay.forward(t.n[i], rows)
        codes, scales = mxfp4.quantise(ctx, t.n[i])
        x, w = torch.empty(rows, D, device="cuda"), torch.empty(D, lay.outputs, device="cuda")
        mxfp4.dequantise(ctx, codes, scales, x)
        mxfp4.dequantise(ctx, lay.codes, lay.scales, w, down=True)
        torch.cuda.synchronize()
        x, w = x.cpu().double(), w.cpu().double()
        z, mag = x @ w + lay.b.cpu().double(), x.abs() @ w.abs()
        want = acts[i](z)
        tol = 1.1 * 2 * D * 2.0 ** -24 * mag + 2.0 ** -20 * (1 + z.abs()) + (2.0 ** -11 * want.abs() + 2.0 ** -25 if half else 0)
        off = (y.cpu().double() - want).abs()
        assert (off <= tol).all(), f"layer {i}: {(off / tol).max().item():.3g} of its tolerance"
    # the network's answers are those of the blocks, to what 4 bits hold: an element is off by about
    # 0.11 of itself, two operands of three layers by 0.27 of the result, a cosine of 0.965
    t.forward()
    torch.cuda.synchronize()
    full, four = t.blocks[2].out.double(), y.double()
    assert torch.nn.functional.cosine_similarity(full.flatten(), four.flatten(), 0) > 0.9
