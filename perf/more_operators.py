"""Workloads of the gated feed-forward part of a residual network: its operators, forward and back.

The kinds of work:

  gated      out = act(x Wg + bg) * (x Wu + bu): both projections, the activation and the product
  ungate     its backward up to the two projections: the gradients of their results, from the layer
             above (its gradient times its weights) or from a gradient of out at hand
  pull       the gradient of x from those two: dg Wg^T + du Wu^T
  project    h = scale * stream + dropout(act(x W + b)): a product with all that follows it in its epilogue
  unproject  its backward up to the projection, the dropout's mask drawn again, and the stream's gradient
  dropout    of a matrix, from its seed and each element's place, with no mask kept

`run` computes them with the framework's kernels where `own` is true, else in elementary torch
operations in 32 bits, rounded once where a result is stored.
"""
from __future__ import annotations

import math

import torch

own = False

LOSS_SCALE = 512.0
ACTS = {"identity": 0, "sigmoid": 1, "tanh": 4, "silu": 6}
TYPES = {"f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # one row served: the weights of both projections are read once
        dict(name="gated_4096_8192_f16_b1", kind="gated", dtype="f16", rows=1, inputs=4096, outputs=8192, act="silu",
             bias=False, train=False),
        # a ragged block trained in 32 bits on an ordinary batch
        dict(name="gated_777_1531_f32_b500", kind="gated", dtype="f32", rows=500, inputs=777, outputs=1531,
             act="sigmoid", bias=True, train=True),
        # the benchmark's MLP width twice as wide inside, under its whole batch
        dict(name="gated_2048_4096_f16_b16384", kind="gated", dtype="f16", rows=16384, inputs=2048, outputs=4096,
             act="silu", bias=False, train=True),
        # odd widths on both sides, the layer above as odd
        dict(name="ungate_1531_777_f16_b2000", kind="ungate", dtype="f16", rows=2000, outputs=1531, above=777,
             act="tanh"),
        # the wide block's error from the projection above it
        dict(name="ungate_4096_2048_f16_b16384", kind="ungate", dtype="f16", rows=16384, outputs=4096, above=2048,
             act="silu"),
        # a small block in 32 bits on a minibatch of 64
        dict(name="pull_640_1024_f32_b64", kind="pull", dtype="f32", rows=64, inputs=640, outputs=1024),
        # the wide block's input gradient
        dict(name="pull_2048_4096_f16_b16384", kind="pull", dtype="f16", rows=16384, inputs=2048, outputs=4096),
        # the projection back into the stream, served to a handful of requests
        dict(name="project_8192_4096_f16_b16", kind="project", dtype="f16", stream="f32", rows=16, inputs=8192,
             outputs=4096, act="identity", bias=False, drop=0.0, scale=1.0, train=False),
        # the same of the benchmark's MLP width, trained with dropout
        dict(name="project_4096_2048_f16_b16384", kind="project", dtype="f16", stream="f32", rows=16384, inputs=4096,
             outputs=2048, act="identity", bias=True, drop=0.1, scale=1.0, train=True),
        # its backward, with an activation and a scaled stream
        dict(name="unproject_2048_f16_b16384", kind="unproject", dtype="f16", rows=16384, outputs=2048, act="silu",
             drop=0.1, scale=0.75),
        # the input of a small network: launch latency
        dict(name="dropout_777_f32_b64", kind="dropout", dtype="f32", rows=64, cols=777, drop=0.2),
        # the wide block's output under its whole batch
        dict(name="dropout_4096_f16_b16384", kind="dropout", dtype="f16", rows=16384, cols=4096, drop=0.1),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A layer width: mostly a multiple of 64 (as widths are chosen), else any number."""
    v = _log(rng, lo, hi)
    return v if rng.random() < 0.4 else max(64, (v + 32) // 64 * 64)


def draw(rng):
    kind = rng.choice(("gated", "gated", "ungate", "pull", "project", "project", "unproject", "dropout"))
    dtype = rng.choice(("f16", "f16", "f32"))
    most = 16384 * 2048 * 4096
    if kind == "dropout":
        cols = _width(rng, 16, 8192)
        return dict(kind=kind, dtype=dtype, rows=min(_log(rng, 1, 16384), 16384 * 4096 // cols), cols=cols,
                    drop=rng.choice((0.1, 0.2, 0.5)))
    outputs = _width(rng, 64, 8192)
    rows = min(_log(rng, 1, 16384), 16384 * 4096 // outputs)
    act = rng.choice(("silu", "silu", "sigmoid", "tanh", "identity"))
    if kind == "unproject":
        return dict(kind=kind, dtype=dtype, rows=min(rows, 16384 * 2048 // outputs), outputs=outputs, act=act,
                    drop=rng.choice((0.0, 0.1, 0.5)), scale=rng.choice((1.0, 0.75)))
    inputs = _width(rng, 64, 4096)
    rows = max(1, min(rows, most // (inputs * outputs)))
    if kind == "gated":
        return dict(kind=kind, dtype=dtype, rows=rows, inputs=inputs, outputs=outputs, act=act,
                    bias=rng.random() < 0.5, train=rng.random() < 0.6)
    if kind == "ungate":
        return dict(kind=kind, dtype=dtype, rows=rows, outputs=outputs, above=inputs if rng.random() < 0.7 else 0,
                    act=act)
    if kind == "pull":
        return dict(kind=kind, dtype=dtype, rows=rows, inputs=inputs, outputs=outputs)
    return dict(kind=kind, dtype=dtype, stream=rng.choice(("f32", dtype)), rows=rows, inputs=outputs, outputs=inputs,
                act=rng.choice(("identity", act)), bias=rng.random() < 0.5, drop=rng.choice((0.0, 0.1, 0.5)),
                scale=rng.choice((1.0, 0.75)), train=rng.random() < 0.6)


def work(case):
    c, t = case, 2 if case["dtype"] == "f16" else 4
    copy = 2 if t == 2 else 0   # fp16 blocks keep a copy of each gradient in fp16
    m = c["rows"]
    if c["kind"] == "dropout":
        return {"bytes": 2 * t * m * c["cols"], "flops": 2.0 * m * c["cols"]}
    n = c["outputs"]
    if c["kind"] == "unproject":   # dh and the cached result in, its gradient and the stream's out
        return {"bytes": m * n * (4 + t + 4 + copy + (4 if c["scale"] != 1.0 else 0)), "flops": 8.0 * m * n}
    if c["kind"] == "ungate":
        k = c["above"]
        src = t * (m * k + n * k) if k else 4 * m * n
        return {"bytes": src + m * n * 2 * (t + 4 + copy), "flops": 2.0 * m * n * k + 10.0 * m * n}
    k = c["inputs"]
    if c["kind"] == "gated":
        return {"bytes": t * (m * k + 2 * k * n + m * n * (3 if c["train"] else 1) + (2 * n if c["bias"] else 0)),
                "flops": 4.0 * m * n * k}
    if c["kind"] == "pull":
        return {"bytes": t * (2 * m * n + 2 * k * n) + 4 * m * k, "flops": 4.0 * m * n * k}
    s = 2 if c["stream"] == "f16" else 4
    return {"bytes": t * (m * k + k * n + (m * n if c["train"] else 0) + (n if c["bias"] else 0)) + 2 * s * m * n,
            "flops": 2.0 * m * n * k}


# ---- inputs ---------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    c, t = case, TYPES[case["dtype"]]
    half = t == torch.float16

    def normal(*shape, std=1.0, dtype=torch.float32):
        return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)

    def empty(*shape, dtype=torch.float32):
        return torch.empty(shape, device="cuda", dtype=dtype)

    def grads(name, *shape):
        return {name: empty(*shape), name + "_h": empty(*shape, dtype=t) if half else None}

    s = {"case": c, "seed": (int(seed) * 2654435761 + 12345) & 0xFFFFFFFF}
    m = c["rows"]
    if c["kind"] == "dropout":
        return dict(s, x=normal(m, c["cols"], dtype=t), out=empty(m, c["cols"], dtype=t))
    n = c["outputs"]
    if c["kind"] == "unproject":
        return dict(s, dh=normal(m, n, std=LOSS_SCALE / 8), preact=normal(m, n, dtype=t),
                    dx=empty(m, n) if c["scale"] != 1.0 else None, **grads("d", m, n))
    if c["kind"] == "ungate":
        k = c["above"]
        s.update(a=normal(m, n, dtype=t), u=normal(m, n, dtype=t), **grads("dg", m, n), **grads("du", m, n))
        if not k:
            return dict(s, s=normal(m, n, std=LOSS_SCALE / 8))
        return dict(s, above_d=normal(m, k, std=LOSS_SCALE / 8, dtype=t), above_w=normal(n, k, std=k ** -0.5, dtype=t))
    k = c["inputs"]
    if c["kind"] == "pull":
        return dict(s, dg=normal(m, n, std=LOSS_SCALE / 8, dtype=t), du=normal(m, n, std=LOSS_SCALE / 8, dtype=t),
                    wg=normal(k, n, std=k ** -0.5, dtype=t), wu=normal(k, n, std=k ** -0.5, dtype=t), dx=empty(m, k))

    def bias():
        return normal(1, n, std=0.1, dtype=t) if c["bias"] else None

    s.update(x=normal(m, k, dtype=t), keep=c["train"])
    if c["kind"] == "gated":
        return dict(s, wg=normal(k, n, std=k ** -0.5, dtype=t), wu=normal(k, n, std=k ** -0.5, dtype=t), bg=bias(),
                    bu=bias(), out=empty(m, n, dtype=t), a=empty(m, n, dtype=t) if c["train"] else None,
                    u=empty(m, n, dtype=t) if c["train"] else None)
    r = TYPES[c["stream"]]
    return dict(s, w=normal(k, n, std=k ** -0.5, dtype=t), b=bias(), stream=normal(m, n, std=3.0, dtype=r),
                h=empty(m, n, dtype=r), preact=empty(m, n, dtype=t) if c["train"] else None)


# ---- plain forms ------------------------------------------------------------------------
def _act(name, z):
    """The activation's value and its slope."""
    if name == "identity":
        return z, torch.ones_like(z)
    if name == "tanh":
        a = 2.0 / (1.0 + (-2.0 * z).exp()) - 1.0
        return a, 1.0 - a * a
    sig = 1.0 / (1.0 + (-z).exp())
    return (sig, sig * (1.0 - sig)) if name == "sigmoid" else (z * sig, sig * (1.0 + z * (1.0 - sig)))


def _kept(rows, cols, p, seed):
    """1 / (1 - p) where the element stays, else 0: a 32-bit mix of the seed and the element's row and
    column, as a number in [0, 1], is at least p."""
    low = 0xFFFFFFFF
    r = torch.arange(rows, device="cuda")[:, None]
    c = torch.arange(cols, device="cuda")[None, :]
    v = (r * 1103515245 & low) ^ (seed + 7 * r & low) ^ (c * 0x4C957F2D & low)
    v = v ^ (v >> 17)
    v = v * 1103515245 + 12345 & low
    v = (v ^ (v >> 15)).float() / 2.0 ** 32
    q = torch.tensor(p, device="cuda")
    return torch.where(v >= q, 1.0 / (1.0 - q), 0.0)


def _with_copy(s, name, v):
    return {name: v} | ({name + "_h": v.half()} if s[name + "_h"] is not None else {})


def _plain(s):
    c = s["case"]
    if c["kind"] == "dropout":
        return (s["x"].float() * _kept(c["rows"], c["cols"], c["drop"], s["seed"])).to(s["x"].dtype)
    if c["kind"] == "unproject":
        d = s["dh"] * _act(c["act"], s["preact"].float())[1]
        if c["drop"]:
            d = d * _kept(c["rows"], c["outputs"], c["drop"], s["seed"])
        return _with_copy(s, "d", d) | ({"dx": c["scale"] * s["dh"]} if s["dx"] is not None else {})
    if c["kind"] == "ungate":
        d = s["above_d"].float() @ s["above_w"].float().t() if c["above"] else s["s"]
        v, slope = _act(c["act"], s["a"].float())
        return _with_copy(s, "dg", d * s["u"].float() * slope) | _with_copy(s, "du", d * v)
    if c["kind"] == "pull":
        return s["dg"].float() @ s["wg"].float().t() + s["du"].float() @ s["wu"].float().t()
    x = s["x"].float()

    def product(w, b):
        z = x @ w.float()
        return z if b is None else z + b.float()

    if c["kind"] == "gated":
        a, u = product(s["wg"], s["bg"]), product(s["wu"], s["bu"])
        out = {"out": (_act(c["act"], a)[0] * u).to(s["x"].dtype)}
        return dict(out, a=a.to(s["x"].dtype), u=u.to(s["x"].dtype)) if s["keep"] else out
    z = product(s["w"], s["b"])
    v = _act(c["act"], z)[0]
    if c["drop"]:
        v = v * _kept(c["rows"], c["outputs"], c["drop"], s["seed"])
    out = {"h": (c["scale"] * s["stream"].float() + v).to(s["h"].dtype)}
    return dict(out, preact=z.to(s["x"].dtype)) if s["keep"] else out


# ---- the framework's kernels ------------------------------------------------------------
_context = None


def _ctx():
    """One context for the whole program, its calls ordered on its stream (no wait per call)."""
    global _context
    if _context is None:
        from soklyn_amd import abi
        _context = abi.Context(0, 16)
        _context.set_sync(False)
    return _context


def _results(s, *names):
    return {k: s[k] for k in names if s.get(k) is not None}


def _kernels(s):
    from soklyn_amd import dropout, gated, residual
    c = s["case"]
    if c["kind"] == "dropout":
        return dropout.apply(_ctx(), s["x"], s["out"], c["drop"], s["seed"])
    if c["kind"] in ("project", "unproject"):
        if "op" not in s:
            s["op"] = residual.Projection(_ctx(), s.get("w"), s.get("b"), outputs=c["outputs"], half=c["dtype"] == "f16",
                                          act=ACTS[c["act"]], dropout=c["drop"], scale=c["scale"])
        if c["kind"] == "project":
            s["op"].forward(s["x"], s["stream"], s["h"], preact=s["preact"], seed=s["seed"])
            return _results(s, "h", "preact")
        s["op"].error(s["dh"], s["preact"], s["d"], d_prenorm_h=s["d_h"], dx=s["dx"], seed=s["seed"])
        return _results(s, "d", "d_h", "dx")
    if "op" not in s:
        s["op"] = gated.Gated(_ctx(), s.get("wg"), s.get("wu"), s.get("bg"), s.get("bu"), outputs=c["outputs"],
                              half=c["dtype"] == "f16", act=ACTS[c.get("act", "identity")])
    if c["kind"] == "gated":
        s["op"].forward(s["x"], s["out"], a=s["a"], u=s["u"])
        return _results(s, "out", "a", "u")
    if c["kind"] == "pull":
        return s["op"].input_grad(s["dg"], s["du"], s["dx"])
    to = dict(dg=s["dg"], du=s["du"], dg_h=s["dg_h"], du_h=s["du_h"])
    if c["above"]:
        s["op"].hidden_error(s["above_d"], s["above_w"], s["a"], s["u"], **to)
    else:
        s["op"].error_from_sum(s["s"], s["a"], s["u"], **to)
    return _results(s, "dg", "dg_h", "du", "du_h")


def run(state):
    return _kernels(state) if own else _plain(state)


# ---- 64 bits ----------------------------------------------------------------------------
def _exact_kept(s):
    """The dropout's factors: the same mix, with the columns' 64-bit multiplier and in 64 bits."""
    c = s["case"]
    cols = c.get("cols") or c["outputs"]
    p = torch.tensor(c["drop"], dtype=torch.float32).double().item()

    def low(v):
        return v.remainder(2 ** 32)

    row = torch.arange(c["rows"], device="cuda")
    col = low(torch.arange(cols, device="cuda") * low(torch.tensor(6364136223846793005, device="cuda")))
    mix = (low(row * 1103515245) ^ low(row * 7 + s["seed"])).unsqueeze(1) ^ col
    mix = low((mix ^ mix // 2 ** 17) * 1103515245 + 12345)
    mix = (mix ^ mix // 2 ** 15).float().double()   # as a 32-bit float: nearest, ties to even
    return (mix >= p * 2 ** 32).double() / (1.0 - p)


def exact(case, seed):
    c, s = case, prepare(case, seed)
    acts = {"identity": lambda v: v, "sigmoid": torch.sigmoid, "tanh": torch.tanh, "silu": torch.nn.functional.silu}

    def both(name, v):
        return {name: v} | ({name + "_h": v} if s[name + "_h"] is not None else {})

    def layer(w, b):
        return torch.nn.functional.linear(s["x"].double(), w.double().t().contiguous(),
                                          None if b is None else b.double()[0])

    if c["kind"] == "dropout":
        return s["x"].double() * _exact_kept(s)
    if c["kind"] == "unproject":
        z = s["preact"].double().requires_grad_()
        x = torch.zeros_like(z, requires_grad=True)
        v = acts[c["act"]](z)
        h = c["scale"] * x + (v * _exact_kept(s) if c["drop"] else v)
        dz, dx = torch.autograd.grad(h, (z, x), s["dh"].double())
        return both("d", dz) | ({"dx": dx} if s["dx"] is not None else {})
    if c["kind"] == "ungate":
        a, u = (s[k].double().requires_grad_() for k in "au")
        d = torch.matmul(s["above_d"].double(), s["above_w"].double().t().contiguous()) if c["above"] else s["s"].double()
        da, du = torch.autograd.grad(acts[c["act"]](a) * u, (a, u), d)
        return both("dg", da) | both("du", du)
    if c["kind"] == "pull":
        both_d = torch.cat([s["dg"], s["du"]], 1).double()
        return both_d @ torch.cat([s["wg"], s["wu"]], 1).double().t().contiguous()
    if c["kind"] == "gated":
        a, u = layer(s["wg"], s["bg"]), layer(s["wu"], s["bu"])
        out = {"out": acts[c["act"]](a) * u}
        return dict(out, a=a, u=u) if c["train"] else out
    z = layer(s["w"], s["b"])
    v = acts[c["act"]](z) * (_exact_kept(s) if c["drop"] else 1.0)
    out = {"h": c["scale"] * s["stream"].double() + v}
    return dict(out, preact=z) if c["train"] else out
