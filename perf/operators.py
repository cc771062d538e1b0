"""Workloads of the operators around the DenseBlock path: residual joins, distillation, 4-bit layers.

The kinds of work:

  distill   the error of an output layer that learns from a teacher's top logits: per-row loss,
            the gradient (times the loss scale) in the buffers that the layer's backward reads
  join      the forward of a residual join: the norm behind a block, its gate, the scaled residual
            stream added, the norm before the next block
  unjoin    its backward: the gradients of the stream, the block's output, the gate and the norms
  quantise  a matrix to 4-bit microscaled floats (32 elements to a scale) and back to their values
  serve     a layer's forward with 4-bit weights: activations to 4 bits, product, bias, activation

`run` computes them with the framework's kernels where `own` is true, else in elementary torch
operations in 32 bits, rounded once where a result is stored.
"""
from __future__ import annotations

import math

import torch

own = False

LOSS_SCALE = 512.0
NORM_EPS = 1e-6
NORMS = {"none": 0, "rms": 1, "layer": 2}
ACTS = {"identity": 0, "sigmoid": 1, "tanh": 4, "silu": 6}
TYPES = {"f16": torch.float16, "f32": torch.float32}
VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)   # of the eight non-negative 4-bit codes


def listed():
    return [
        # the ten-class head of a small classifier on a minibatch: launch latency
        dict(name="distill_10_f32_b64", kind="distill", dtype="f32", rows=64, classes=10, top=4, temperature=2.0,
             alpha=0.5),
        # a 1000-class head on an ordinary minibatch, teacher and labels mixed
        dict(name="distill_1000_f16_b1024", kind="distill", dtype="f16", rows=1024, classes=1000, top=16,
             temperature=4.0, alpha=0.9),
        # a vocabulary-sized head of odd width, the teacher alone at its own temperature
        dict(name="distill_50257_f16_b2048", kind="distill", dtype="f16", rows=2048, classes=50257, top=64,
             temperature=1.0, alpha=1.0),
        # one row served: a join between two blocks
        dict(name="join_4096_f16_b1", kind="join", dtype="f16", stream="f32", rows=1, cols=4096, post="rms", pre="rms",
             gate="one", gate_act="identity", scale=1.0),
        # a training batch of the benchmark's wide block, the stream kept in 32 bits
        dict(name="join_4096_f16_b8192", kind="join", dtype="f16", stream="f32", rows=8192, cols=4096, post="rms",
             pre="rms", gate="each", gate_act="sigmoid", scale=1.0),
        # an odd width trained in 32 bits with LayerNorm on both sides
        dict(name="unjoin_777_f32_b500", kind="unjoin", dtype="f32", stream="f32", rows=500, cols=777, post="layer",
             pre="layer", gate="one", gate_act="tanh", scale=0.75),
        # the benchmark's MLP width under its whole batch
        dict(name="unjoin_2048_f16_b16384", kind="unjoin", dtype="f16", stream="f16", rows=16384, cols=2048, post="rms",
             pre="rms", gate="one", gate_act="identity", scale=1.0),
        # activations of an odd width, blocks along each row
        dict(name="quantise_12345x1531_f16", kind="quantise", dtype="f16", rows=12345, cols=1531, down=False),
        # the weights of the benchmark's wide block, blocks down each column
        dict(name="quantise_4096x4096_f32_down", kind="quantise", dtype="f32", rows=4096, cols=4096, down=True),
        # the wide layer served to a handful of requests: its weights are read once
        dict(name="serve_4096_4096_f16_b16", kind="serve", dtype="f16", batch=16, inputs=4096, outputs=4096,
             act="silu"),
        # a ragged layer on an ordinary batch
        dict(name="serve_777_1531_f32_b500", kind="serve", dtype="f32", batch=500, inputs=777, outputs=1531,
             act="tanh"),
        # the benchmark's wide layer under its whole batch
        dict(name="serve_4096_4096_f16_b8192", kind="serve", dtype="f16", batch=8192, inputs=4096, outputs=4096,
             act="silu"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A layer width: mostly a multiple of 64 (as widths are chosen), else any number."""
    v = _log(rng, lo, hi)
    return v if rng.random() < 0.4 else max(64, (v + 32) // 64 * 64)


def draw(rng):
    kind = rng.choice(("distill", "join", "unjoin", "quantise", "serve"))
    dtype = rng.choice(("f16", "f16", "f32"))
    if kind == "distill":
        classes = _log(rng, 2, 131072)
        rows = _log(rng, 1, 16384)
        rows = max(1, min(rows, int(2048 * 50257 * 10 / 12) // classes))
        return dict(kind=kind, dtype=dtype, rows=rows, classes=classes, top=min(classes, _log(rng, 1, 128)),
                    temperature=rng.choice((1.0, 2.0, 4.0, 0.5)), alpha=rng.choice((1.0, 0.5, 0.9, 0.0)))
    if kind in ("join", "unjoin"):
        cols = _width(rng, 16, 8192)
        rows = min(_log(rng, 1, 16384), 8192 * 2048 // cols)
        return dict(kind=kind, dtype=dtype, stream=rng.choice(("f32", dtype)), rows=rows, cols=cols,
                    post=rng.choice(("none", "rms", "layer")), pre=rng.choice(("rms", "layer")),
                    gate=rng.choice(("none", "one", "each")), gate_act=rng.choice(("identity", "sigmoid", "tanh")),
                    scale=rng.choice((1.0, 0.75)))
    if kind == "quantise":
        rows = _log(rng, 1, 16384)
        return dict(kind=kind, dtype=dtype, rows=rows, cols=_width(rng, 16, min(16384, 4096 * 4096 // rows)),
                    down=rng.random() < 0.5)
    return dict(kind=kind, dtype=dtype, batch=_log(rng, 1, 8192), inputs=_width(rng, 64, 4096),
                outputs=_width(rng, 64, 4096), act=rng.choice(("identity", "silu", "tanh")))


def _up(v, m):
    return -(-v // m) * m


def work(case):
    c, t = case, 2 if case["dtype"] == "f16" else 4
    if c["kind"] == "distill":
        e = c["rows"] * c["classes"]
        # logits in; grad, d_prenorm and, for fp16 layers, its fp16 copy out
        return {"bytes": e * (t + 8 + (2 if t == 2 else 0)) + c["rows"] * (8 * c["top"] + 8), "flops": 8.0 * e}
    if c["kind"] in ("join", "unjoin"):
        e, s = c["rows"] * c["cols"], 2 if c["stream"] == "f16" else 4
        gate = {"none": 0, "one": 0, "each": e}[c["gate"]]
        if c["kind"] == "join":   # stream and block output in, stream and normed out
            return {"bytes": e * 2 * (s + t) + gate * t + 16 * c["rows"], "flops": 12.0 * e}
        # stream, block output and two gradients in, two gradients out
        return {"bytes": e * (s + t + 16) + gate * (t + 4) + 16 * c["rows"], "flops": 30.0 * e}
    if c["kind"] == "quantise":
        n, k = (c["cols"], c["rows"]) if c["down"] else (c["rows"], c["cols"])
        return {"bytes": n * k * (t + 4) + n * _up(k, 128) * 17 / 32, "flops": 4.0 * n * k}
    m, k, n = c["batch"], c["inputs"], c["outputs"]
    return {"bytes": t * (m * k + m * n + n) + n * _up(k, 128) * 17 / 32, "flops": 2.0 * m * k * n}


# ---- inputs ---------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    c, t = case, TYPES[case["dtype"]]

    def normal(*shape, std=1.0, dtype=torch.float32):
        return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)

    def empty(*shape, dtype=torch.float32):
        return torch.empty(shape, device="cuda", dtype=dtype)

    s = {"case": c}
    if c["kind"] == "distill":
        m, n, k = c["rows"], c["classes"], c["top"]
        logits = normal(m, n, std=2.5, dtype=t)
        # a teacher near the student; some rows hold fewer than k of its logits, one in 16 none
        value, index = (logits.float() + normal(m, n)).topk(k, dim=1)
        held = torch.randint(1, k + 1, (m, 1), generator=g, device="cuda")
        held = torch.where(torch.rand((m, 1), generator=g, device="cuda") < 0.5, k, held)
        held = torch.where(torch.rand((m, 1), generator=g, device="cuda") < 1 / 16, 0, held)
        index = torch.where(torch.arange(k, device="cuda") < held, index, -1)
        label = torch.randint(0, n, (m,), generator=g, device="cuda")
        label = torch.where(torch.rand((m,), generator=g, device="cuda") < 1 / 8, -1, label)
        s.update(logits=logits, index=index.int(), value=value.contiguous(), label=label.int(), loss=empty(m),
                 grad=empty(m, n), d_prenorm=empty(m, n),
                 d_prenorm_h=empty(m, n, dtype=torch.float16) if t == torch.float16 else None)
    elif c["kind"] in ("join", "unjoin"):
        m, n, r = c["rows"], c["cols"], TYPES[c["stream"]]
        gates = {"none": 0, "one": 1, "each": m}[c["gate"]]
        s.update(y=normal(m, n, dtype=t), gate=normal(gates, n, std=0.5, dtype=t) if gates else None,
                 post_w=(1.0 + normal(1, n, std=0.1)).to(t), post_b=normal(1, n, std=0.1, dtype=t),
                 pre_w=(1.0 + normal(1, n, std=0.1)).to(t), pre_b=normal(1, n, std=0.1, dtype=t))
        stream = normal(m, n, std=3.0, dtype=r)
        if c["kind"] == "join":
            s.update(x=stream, h=empty(m, n, dtype=r), n=empty(m, n, dtype=t), stats=empty(4, m))
        else:
            post = _stats(s["y"].double(), c["post"])
            pre = _stats(stream.double(), c["pre"])
            s.update(h=stream, stats=torch.stack(post + pre).float().contiguous(),
                     dn=normal(m, n, std=LOSS_SCALE / 8), dh=normal(m, n, std=LOSS_SCALE / 8), dx=empty(m, n),
                     dy=empty(m, n), dgate=empty(gates, n) if gates else None, dparam=empty(4, n))
    elif c["kind"] == "quantise":
        n, k = (c["cols"], c["rows"]) if c["down"] else (c["rows"], c["cols"])
        # magnitudes that differ from row to row, as activations' do
        s.update(src=(normal(c["rows"], c["cols"]) * normal(c["rows"], 1).exp()).to(t),
                 codes=empty(n, _up(k, 128) // 2, dtype=torch.uint8),
                 scales=empty(n, _up(k, 128) // 32, dtype=torch.uint8), values=empty(c["rows"], c["cols"]))
    else:
        m, k, n = c["batch"], c["inputs"], c["outputs"]
        w = normal(k, n, std=math.sqrt(2.0 / k))
        codes, scales = _pack(*_to_codes(w.t()))
        s.update(x=normal(m, k, dtype=t), codes=codes, scales=scales, bias=normal(1, n, std=0.1, dtype=t),
                 out=empty(m, n, dtype=t))
    return s


# ---- plain forms ------------------------------------------------------------------------
def _distill(s):
    c, z = s["case"], s["logits"].float()
    tau, alpha = c["temperature"], c["alpha"]

    def log_softmax(v):
        v = v - v.amax(1, keepdim=True)
        return v - v.exp().sum(1, keepdim=True).log()

    held = s["index"] >= 0
    at = s["index"].clamp(min=0).long()
    some = held.any(1, keepdim=True)
    u = torch.where(held, s["value"] / tau, -math.inf)
    u = u - torch.where(some, u.amax(1, keepdim=True), 0.0)
    e = u.exp()
    total = e.sum(1, keepdim=True)
    q = torch.where(some, e / total.clamp(min=1e-30), 0.0)
    log_q = torch.where(held, u - total.clamp(min=1e-30).log(), 0.0)
    soft = log_softmax(z / tau)
    loss = alpha * tau * tau * (q * (log_q - soft.gather(1, at))).sum(1)
    p = torch.where(some, soft.exp(), 0.0)
    grad = (alpha * tau) * p.scatter_add(1, at, -q)
    if alpha < 1.0:
        hard, labelled = log_softmax(z), (s["label"] >= 0)[:, None]
        on = s["label"].clamp(min=0).long()[:, None]
        loss = loss - (1.0 - alpha) * torch.where(labelled, hard.gather(1, on), 0.0)[:, 0]
        g = hard.exp()
        g = g.scatter_add(1, on, torch.full_like(g[:, :1], -1.0))
        grad = grad + (1.0 - alpha) * torch.where(labelled, g, 0.0)
    grad = grad * LOSS_SCALE
    out = {"loss": loss, "grad": grad, "d_prenorm": grad}
    if s["d_prenorm_h"] is not None:
        out["d_prenorm_h"] = grad.half()
    return out


def _stats(v, norm):
    """Per-row mean and reciprocal deviation (0 and 1 where the norm has none)."""
    zero = torch.zeros_like(v[:, 0])
    if norm == "none":
        return [zero, zero + 1.0]
    mean = v.mean(1) if norm == "layer" else zero
    d = v - mean[:, None]
    return [mean, 1.0 / ((d * d).mean(1) + NORM_EPS).sqrt()]


def _gate(s):
    """The gate's value and its slope."""
    c = s["case"]
    if s["gate"] is None:
        return 1.0, 0.0
    g = s["gate"].float()
    if c["gate_act"] == "sigmoid":
        a = 1.0 / (1.0 + (-g).exp())
        return a, a * (1.0 - a)
    if c["gate_act"] == "tanh":
        a = 2.0 / (1.0 + (-2.0 * g).exp()) - 1.0
        return a, 1.0 - a * a
    return g, torch.ones_like(g)


def _affine(v, s, side):
    norm = s["case"][side]
    if norm != "none":
        v = v * s[side + "_w"].float()
    return v + s[side + "_b"].float() if norm == "layer" else v


def _join(s):
    c, y = s["case"], s["y"].float()
    post = _stats(y, c["post"])
    u = _affine((y - post[0][:, None]) * post[1][:, None], s, "post")
    h = (c["scale"] * s["x"].float() + _gate(s)[0] * u).to(s["x"].dtype)
    hf = h.float()
    pre = _stats(hf, c["pre"])
    n = _affine((hf - pre[0][:, None]) * pre[1][:, None], s, "pre")
    return {"h": h, "n": n.to(s["y"].dtype), "stats": torch.stack(post + pre)}


def _back_through_norm(d, hat, rstd, norm):
    """The norm's input gradient, from the gradient of the normalised values."""
    if norm == "none":
        return d
    out = d - hat * (d * hat).mean(1, keepdim=True)
    if norm == "layer":
        out = out - d.mean(1, keepdim=True)
    return out * rstd


def _unjoin(s):
    c, dn, st = s["case"], s["dn"], s["stats"]
    y_hat = (s["y"].float() - st[0][:, None]) * st[1][:, None]
    h_hat = (s["h"].float() - st[2][:, None]) * st[3][:, None]
    d = s["dh"] + _back_through_norm(dn * s["pre_w"].float(), h_hat, st[3][:, None], c["pre"])
    a, slope = _gate(s)
    du = d * a
    dy = _back_through_norm(du * s["post_w"].float(), y_hat, st[1][:, None], c["post"]) if c["post"] != "none" else du
    zero = torch.zeros_like(dn[0])
    dparam = torch.stack([(du * y_hat).sum(0) if c["post"] != "none" else zero,
                          du.sum(0) if c["post"] == "layer" else zero,
                          (dn * h_hat).sum(0), dn.sum(0) if c["pre"] == "layer" else zero])
    out = {"dx": c["scale"] * d, "dy": dy, "dparam": dparam}
    if s["gate"] is not None:
        dgate = d * _affine(y_hat, s, "post") * slope
        out["dgate"] = dgate.sum(0, keepdim=True) if s["gate"].shape[0] == 1 and c["gate"] == "one" else dgate
    return out


def _to_codes(v):
    """Rows of v in blocks of 32: 4-bit codes [rows, blocks, 32] and their scales' exponents.
    The scale is 2^(e - 2), 2^e the largest power of two up to the block's largest magnitude;
    magnitudes round to the nearest of VALUES, ties to the even code, past 6 to 6."""
    n, k = v.shape
    v = torch.nn.functional.pad(v.float(), (0, _up(k, 128) - k)).reshape(n, -1, 32)
    big = v.abs().amax(2)
    e = torch.where(big > 0, torch.frexp(big).exponent - 3, -127).clamp(min=-127)
    a = torch.ldexp(v.abs(), -e[:, :, None])
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    return code + 8 * torch.signbit(v), e


def _pack(code, e):
    """Two codes to a byte, the first in its low half; scales as exponent + 127."""
    code = code.reshape(code.shape[0], -1, 2)
    return (code[:, :, 0] | (code[:, :, 1] << 4)).contiguous(), (e + 127).to(torch.uint8).contiguous()


def _values(code, e):
    table = torch.tensor(VALUES + tuple(-v for v in VALUES), device=code.device)
    return torch.ldexp(table[code.long()], e[:, :, None]).reshape(code.shape[0], -1)


def _quantise(s):
    c = s["case"]
    v = _values(*_to_codes(s["src"].t() if c["down"] else s["src"]))
    return (v[:, : c["rows"]].t() if c["down"] else v[:, : c["cols"]]).contiguous()


def _serve(s):
    c = s["case"]
    x = _values(*_to_codes(s["x"]))
    code = torch.stack([s["codes"] & 15, s["codes"] >> 4], 2).reshape(c["outputs"], -1, 32)
    w = _values(code, s["scales"].int() - 127)
    z = x @ w.t() + s["bias"].float()
    if c["act"] == "silu":
        z = z / (1.0 + (-z).exp())
    elif c["act"] == "tanh":
        z = 2.0 / (1.0 + (-2.0 * z).exp()) - 1.0
    return z.to(s["x"].dtype)


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


def _kernels(s):
    from soklyn_amd import mxfp4, residual
    from soklyn_amd.devblock import distill_error
    c = s["case"]
    if c["kind"] == "distill":
        distill_error(_ctx(), s["logits"], s["index"], s["value"], s["label"] if c["alpha"] < 1.0 else None,
                      temperature=c["temperature"], alpha=c["alpha"], grad=s["grad"], d_prenorm=s["d_prenorm"],
                      d_prenorm_h=s["d_prenorm_h"], loss=s["loss"])
        return {k: s[k] for k in ("loss", "grad", "d_prenorm", "d_prenorm_h") if s[k] is not None}
    if c["kind"] in ("join", "unjoin"):
        if "join" not in s:
            s["join"] = residual.Join(_ctx(), c["cols"], half=c["dtype"] == "f16", half_stream=c["stream"] == "f16",
                                      post_norm=NORMS[c["post"]], pre_norm=NORMS[c["pre"]],
                                      gate_act=ACTS[c["gate_act"]], scale=c["scale"], post_w=s["post_w"],
                                      post_b=s["post_b"], pre_w=s["pre_w"], pre_b=s["pre_b"])
        if c["kind"] == "join":
            s["join"].forward(s["x"], s["y"], s["gate"], h=s["h"], n=s["n"], stats=s["stats"])
            return {k: s[k] for k in ("h", "n", "stats")}
        s["join"].backward(s["h"], s["y"], s["gate"], s["stats"], s["dn"], s["dh"], dx=s["dx"], dy=s["dy"],
                           dgate=s["dgate"], dparam=s["dparam"])
        return {k: s[k] for k in ("dx", "dy", "dparam", "dgate") if s[k] is not None}
    if c["kind"] == "quantise":
        mxfp4.quantise(_ctx(), s["src"], down=c["down"], codes=s["codes"], scales=s["scales"])
        return mxfp4.dequantise(_ctx(), s["codes"], s["scales"], s["values"], down=c["down"])
    if "layer" not in s:
        s["layer"] = mxfp4.Layer(_ctx(), c["inputs"], c["outputs"], c["batch"], s["codes"].to(torch.uint8),
                                 s["scales"], half=c["dtype"] == "f16", act=ACTS[c["act"]], b=s["bias"], out=s["out"])
    return s["layer"].forward(s["x"], c["batch"])


def run(state):
    if own:
        return _kernels(state)
    return {"distill": _distill, "join": _join, "unjoin": _unjoin, "quantise": _quantise,
            "serve": _serve}[state["case"]["kind"]](state)


# ---- 64 bits ----------------------------------------------------------------------------
def _exact_norm(v, norm, w, b):
    if norm == "none":
        return v
    v = v - v.mean(1, keepdim=True) if norm == "layer" else v
    v = v * torch.rsqrt(v.square().mean(1, keepdim=True) + NORM_EPS) * w.double()
    return v + b.double() if norm == "layer" else v


def _exact_stats(v, norm):
    one = torch.ones(v.shape[0], dtype=torch.float64, device=v.device)
    if norm == "none":
        return [0 * one, one]
    mean = v.mean(1) if norm == "layer" else 0 * one
    return [mean, (v.square().mean(1) - mean.square() + NORM_EPS).rsqrt()]


def _exact_values(v):
    """Rows of v as the values that their 4-bit form stands for."""
    n, k = v.shape
    v = torch.nn.functional.pad(v.double(), (0, _up(k, 128) - k)).reshape(n, -1, 32)
    scale = torch.exp2(torch.floor(torch.log2(v.abs().amax(2, keepdim=True).clamp(min=2.0 ** -125))) - 2)
    a = v / scale
    step = torch.where(a.abs() < 2, 0.5, torch.where(a.abs() < 4, 1.0, 2.0))
    return (torch.round(a / step) * step).clamp(-6, 6).mul(scale).reshape(n, -1)


def exact(case, seed):
    c, s = case, prepare(case, seed)
    gate_of = {"identity": lambda v: v, "sigmoid": torch.sigmoid, "tanh": torch.tanh}
    if c["kind"] == "distill":
        z = s["logits"].double().requires_grad_()
        q = torch.zeros_like(z)
        held = s["index"] >= 0
        some = held.any(1)
        w = torch.softmax(torch.where(held, s["value"].double() / c["temperature"], -math.inf)[some], 1)
        q = q.index_put((some.nonzero(), s["index"].clamp(min=0).long()[some]), w, accumulate=True)
        soft = torch.nn.functional.kl_div(torch.log_softmax(z / c["temperature"], 1), q, reduction="none").sum(1)
        hard = torch.nn.functional.cross_entropy(z, s["label"].long(), reduction="none", ignore_index=-1)
        loss = c["alpha"] * c["temperature"] ** 2 * soft + (1 - c["alpha"]) * hard
        grad = torch.autograd.grad(loss.sum(), z)[0] * LOSS_SCALE
        out = {"loss": loss.detach(), "grad": grad, "d_prenorm": grad}
        return dict(out, d_prenorm_h=grad) if s["d_prenorm_h"] is not None else out
    if c["kind"] == "join":
        y = s["y"].double()
        gate = 1.0 if s["gate"] is None else gate_of[c["gate_act"]](s["gate"].double())
        h = c["scale"] * s["x"].double() + gate * _exact_norm(y, c["post"], s["post_w"], s["post_b"])
        kept = h.to(s["x"].dtype).double()   # the norm before the next block reads the stream as stored
        return {"h": h, "n": _exact_norm(kept, c["pre"], s["pre_w"], s["pre_b"]),
                "stats": torch.stack(_exact_stats(y, c["post"]) + _exact_stats(kept, c["pre"]))}
    if c["kind"] == "unjoin":
        keys = ["y", "post_w", "post_b", "pre_w", "pre_b"] + (["gate"] if s["gate"] is not None else [])
        v = {k: s[k].double().requires_grad_() for k in keys}
        gate = gate_of[c["gate_act"]](v["gate"]) if "gate" in v else 1.0
        branch = gate * _exact_norm(v["y"], c["post"], v["post_w"], v["post_b"])
        # the stream that, with this branch added, gives the h at hand
        x = ((s["h"].double() - branch.detach()) / c["scale"]).requires_grad_()
        h = c["scale"] * x + branch
        n = _exact_norm(h, c["pre"], v["pre_w"], v["pre_b"])
        total = (n * s["dn"].double()).sum() + (h * s["dh"].double()).sum()
        got = torch.autograd.grad(total, [x] + [v[k] for k in keys], allow_unused=True)
        got = {k: torch.zeros_like(s["pre_w"].double()) if d is None else d for k, d in zip(["x"] + keys, got)}
        out = {"dx": got["x"], "dy": got["y"],
               "dparam": torch.cat([got[k] for k in ("post_w", "post_b", "pre_w", "pre_b")])}
        return dict(out, dgate=got["gate"]) if "gate" in v else out
    if c["kind"] == "quantise":
        v = _exact_values(s["src"].t() if c["down"] else s["src"])
        return (v[:, : c["rows"]].t() if c["down"] else v[:, : c["cols"]]).contiguous()
    w = torch.tensor(VALUES + tuple(-v for v in VALUES), device="cuda", dtype=torch.float64)
    w = w[torch.stack([s["codes"] % 16, s["codes"] // 16], 2).long()].reshape(c["outputs"], -1, 32)
    w = (w * torch.exp2(s["scales"].double() - 127)[:, :, None]).reshape(c["outputs"], -1)
    z = _exact_values(s["x"]) @ w.t().contiguous() + s["bias"].double()
    return {"identity": lambda v: v, "silu": torch.nn.functional.silu, "tanh": torch.tanh}[c["act"]](z)
