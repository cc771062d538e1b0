"""What gated blocks, the projection into the stream and dropout refuse, without a GPU: their checks come before
anything that looks into the context or touches the device, so a block of zeros stands for one (whose tile size
of 0 is refused for fp16 last of all), and the addresses are never read."""
from __future__ import annotations

import ctypes as C
import os

import pytest
import torch

from soklyn_amd import abi, dropout
from soklyn_amd.gated import Gated
from soklyn_amd.residual import Projection
from tests.test_operator_refusals_cpu import At

INVALID, TRAINING, LIMIT, DIMS, BATCH, HARDWARE, NULL = -1, -2, -3, -4, -5, -6, -8
CTX = C.create_string_buffer(8192)
INF, NAN = float("inf"), float("nan")


@pytest.fixture(scope="module", autouse=True)
def built():
    if not os.path.exists(abi.LIB_PATH):
        pytest.skip("libsoklyn_hip.so not built")


def desc(at, **change):
    d = abi.SklDenseDesc()
    for k, v in dict(dict(dtype=1, inputs=64, outputs=32, max_batch=16, is_training=1, w=at(), b=at(), preact=at(), grad=at(),
                          d_prenorm=at(), d_prenorm_h=at()), **change).items():
        setattr(d, k, v)
    return d


def run(fn, args, **change):
    args.update(change)
    keep = [a for a in args.values() if isinstance(a, abi.SklDenseDesc)]   # alive during the call
    got = abi.status(fn, *(C.byref(a) if isinstance(a, abi.SklDenseDesc) else a for a in args.values()))
    del keep
    return got


def forward(of_gate=None, of_up=None, overlap=None, **change):
    at = At()
    a = dict(ctx=CTX, gate=desc(at, **dict(dict(act=6), **(of_gate or {}))), up=desc(at, **(of_up or {})), x=at(), in_rows=12,
             in_cols=64, batch=8, out=at(), work=None, work_bytes=0)
    if overlap:
        where, what, shift = overlap
        a[where] = {"x": a["x"], "wg": a["gate"].w, "wu": a["up"].w, "bg": a["gate"].b, "a": a["gate"].preact,
                    "u": a["up"].preact, "out": a["out"]}[what] + shift
    return run("skl_gated_forward", a, **change)


BOTH = [(INVALID, dict(dtype=2)), (INVALID, dict(inputs=0)), (INVALID, dict(outputs=0)), (INVALID, dict(max_batch=0)),
        (INVALID, dict(norm=1)), (INVALID, dict(act=5)), (INVALID, dict(act=8))]


@pytest.mark.parametrize("code,change", BOTH + [(NULL, dict(w=None))])
def test_gated_forward_blocks(code, change):
    assert forward(change) == code
    assert forward(None, change) == code


@pytest.mark.parametrize("code,gate,up,change", [
    (NULL, {}, {}, dict(ctx=None)), (NULL, {}, {}, dict(gate=None)), (NULL, {}, {}, dict(up=None)),
    (NULL, {}, {}, dict(x=None)), (NULL, {}, {}, dict(out=None)), (INVALID, dict(dtype=0), {}, {}),
    (INVALID, {}, dict(act=6), {}), (DIMS, dict(outputs=31), {}, {}), (DIMS, {}, dict(inputs=63), {}),
    (DIMS, {}, {}, dict(in_cols=63)), (DIMS, {}, {}, dict(in_rows=7)), (LIMIT, {}, {}, dict(in_rows=17)),
    (LIMIT, {}, dict(max_batch=7), {}), (BATCH, {}, {}, dict(batch=0)), (HARDWARE, {}, {}, dict(work=(1 << 50) + 8)),
    (HARDWARE, {}, {}, {}),   # nothing else is wrong: the context's tile size
    (HARDWARE, dict(b=None, preact=None), dict(b=None, preact=None), {}),
])
def test_gated_forward(code, gate, up, change):
    assert forward(gate, up, **change) == code


@pytest.mark.parametrize("where,what,shift", [("out", "x", 0), ("out", "wg", 64), ("out", "wu", -2), ("out", "bg", 2), ("out", "a", 0),
                                              ("out", "u", 2), ("work", "x", 0), ("work", "out", 0), ("work", "a", 16)])
def test_gated_forward_overlap(where, what, shift):
    assert forward(overlap=(where, what, shift), **(dict(work_bytes=4096) if where == "work" else {})) == INVALID


def ungate(of_gate=None, of_up=None, of_next=None, which="hidden", same=None, **change):
    at = At()
    g, u = desc(at, **dict(dict(act=6), **(of_gate or {}))), desc(at, **(of_up or {}))
    n = desc(at, **dict(dict(inputs=32, outputs=20), **(of_next or {})))
    if same:   # a buffer of the first is one of the second's
        (b1, f1), (b2, f2) = same
        blocks = {"g": g, "u": u, "n": n}
        setattr(blocks[b1], f1, getattr(blocks[b2], f2))
    if which == "hidden":
        return run("skl_gated_hidden_error", dict(ctx=CTX, gate=g, up=u, next=n, batch=8, work=None, work_bytes=0), **change)
    if which == "sum":
        return run("skl_gated_error_from_sum", dict(ctx=CTX, gate=g, up=u, s=at(), batch=8), **change)
    return run("skl_gated_input_grad", dict(ctx=CTX, gate=g, up=u, batch=8, dx=at(), work=None, work_bytes=0), **change)


@pytest.mark.parametrize("which", ["hidden", "sum", "grad"])
@pytest.mark.parametrize("code,change", BOTH)
def test_gated_backward_blocks(which, code, change):
    assert ungate(change, which=which) == code
    assert ungate(None, change, which=which) == code


@pytest.mark.parametrize("which", ["hidden", "sum"])
@pytest.mark.parametrize("code,change", [(TRAINING, dict(is_training=0)), (LIMIT, dict(max_batch=7)), (NULL, dict(preact=None)),
                                         (NULL, dict(d_prenorm=None)), (NULL, dict(d_prenorm_h=None))])
def test_gated_errors_blocks(which, code, change):
    assert ungate(change, which=which) == code
    assert ungate(None, change, which=which) == code


@pytest.mark.parametrize("which,code,change", [
    ("hidden", NULL, dict(ctx=None)), ("hidden", NULL, dict(next=None)), ("hidden", BATCH, dict(batch=0)),
    ("hidden", HARDWARE, dict(work=8)), ("sum", NULL, dict(s=None)), ("sum", BATCH, dict(batch=0)), ("sum", NULL, dict(up=None)),
    ("grad", NULL, dict(dx=None)), ("grad", BATCH, dict(batch=0)), ("grad", LIMIT, dict(batch=17)), ("grad", HARDWARE, dict(work=8)),
    ("hidden", HARDWARE, {}), ("grad", HARDWARE, {}),
])
def test_gated_backward(which, code, change):
    assert ungate(which=which, **change) == code


@pytest.mark.parametrize("code,nxt", [(INVALID, dict(dtype=0)), (INVALID, dict(outputs=0)), (DIMS, dict(inputs=31)),
                                      (DIMS, dict(max_batch=7)), (NULL, dict(w=None)), (NULL, dict(d_prenorm_h=None))])
def test_gated_hidden_error_above(code, nxt):
    assert ungate(of_next=nxt) == code


@pytest.mark.parametrize("which,same", [
    ("hidden", (("g", "d_prenorm"), ("u", "d_prenorm"))), ("hidden", (("g", "d_prenorm"), ("n", "d_prenorm_h"))),
    ("hidden", (("u", "d_prenorm_h"), ("n", "w"))), ("hidden", (("g", "d_prenorm_h"), ("g", "preact"))),
    ("sum", (("u", "d_prenorm"), ("g", "preact"))), ("sum", (("g", "d_prenorm_h"), ("u", "d_prenorm_h"))),
])
def test_gated_backward_overlap(which, same):
    assert ungate(which=which, same=same) == INVALID


@pytest.mark.parametrize("of", ["w", "d_prenorm_h"])
def test_gated_input_grad_overlap(of):
    at = At()
    g, u = desc(at, act=6), desc(at)
    for b in (g, u):
        assert run("skl_gated_input_grad", dict(ctx=CTX, gate=g, up=u, batch=8, dx=getattr(b, of) + 8, work=None,
                                                work_bytes=0)) == INVALID


def project(of_blk=None, same=None, **change):
    at = At()
    b = desc(at, **dict(dict(act=4, mask_coeff=0.5), **(of_blk or {})))
    a = dict(ctx=CTX, blk=b, x=at(), in_rows=12, in_cols=64, batch=8, use_dropout=1, seed=7, stream_dtype=0, scale=1.0,
             stream=at(), h=at(), work=None, work_bytes=0)
    if same:
        where, what, shift = same
        a[where] = (a[what] if what in a else getattr(b, what)) + shift
    return run("skl_dense_forward_residual", a, **change)


@pytest.mark.parametrize("code,blk,change", [(c, b, {}) for c, b in BOTH] + [
    (NULL, {}, dict(ctx=None)), (NULL, {}, dict(blk=None)), (NULL, {}, dict(x=None)), (NULL, {}, dict(h=None)),
    (NULL, dict(w=None), {}), (INVALID, dict(dtype=0), dict(stream_dtype=1)), (INVALID, {}, dict(stream_dtype=2)),
    (INVALID, {}, dict(scale=INF)), (INVALID, {}, dict(scale=NAN)), (INVALID, dict(mask_coeff=1.0), {}),
    (INVALID, dict(mask_coeff=-0.1), {}), (INVALID, dict(mask_coeff=NAN), {}), (HARDWARE, dict(mask_coeff=2.0), dict(use_dropout=0)),
    (DIMS, {}, dict(in_cols=63)), (DIMS, {}, dict(in_rows=7)), (LIMIT, {}, dict(in_rows=17)), (BATCH, {}, dict(batch=0)),
    (HARDWARE, {}, dict(work=8)), (HARDWARE, {}, {}), (HARDWARE, dict(b=None, preact=None), dict(stream=None)),
])
def test_forward_residual(code, blk, change):
    assert project(blk, **change) == code


@pytest.mark.parametrize("where,what,shift", [("h", "x", 0), ("h", "w", 4), ("h", "b", 0), ("h", "preact", 0), ("h", "stream", 4),
                                              ("h", "stream", -4), ("work", "h", 0), ("work", "stream", 16)])
def test_forward_residual_overlap(where, what, shift):
    assert project(same=(where, what, shift), **(dict(work_bytes=4096) if where == "work" else {})) == INVALID


def test_forward_residual_in_place():
    assert project(same=("h", "stream", 0)) == HARDWARE   # the context's tile size alone


def unproject(of_blk=None, same=None, **change):
    at = At()
    b = desc(at, **dict(dict(act=4, mask_coeff=0.5), **(of_blk or {})))
    a = dict(ctx=CTX, blk=b, dh=at(), batch=8, use_dropout=1, seed=7, scale=1.0, dx=at())
    if same:
        where, what, shift = same
        a[where] = (a[what] if what in a else getattr(b, what)) + shift
    return run("skl_dense_residual_error", a, **change)


@pytest.mark.parametrize("code,blk,change", [(c, b, {}) for c, b in BOTH] + [
    (NULL, {}, dict(ctx=None)), (NULL, {}, dict(blk=None)), (NULL, {}, dict(dh=None)), (NULL, dict(preact=None), {}),
    (NULL, dict(d_prenorm=None), {}), (NULL, dict(d_prenorm_h=None), {}), (TRAINING, dict(is_training=0), {}),
    (INVALID, {}, dict(scale=INF)), (INVALID, dict(mask_coeff=1.0), {}), (INVALID, dict(mask_coeff=NAN), {}),
    (BATCH, {}, dict(batch=0)), (LIMIT, {}, dict(batch=17)),
])
def test_residual_error(code, blk, change):
    assert unproject(blk, **change) == code


@pytest.mark.parametrize("where,what,shift", [("dx", "dh", 4), ("dx", "d_prenorm", 0), ("dx", "preact", 0), ("dh", "d_prenorm", 0),
                                              ("dh", "d_prenorm_h", 0)])
def test_residual_error_overlap(where, what, shift):
    assert unproject(same=(where, what, shift)) == INVALID


@pytest.mark.parametrize("code,change", [
    (NULL, dict(ctx=None)), (NULL, dict(x=None)), (NULL, dict(out=None)), (INVALID, dict(dtype=2)), (INVALID, dict(p=1.0)),
    (INVALID, dict(p=-0.5)), (INVALID, dict(p=NAN)), (INVALID, dict(out=(1 << 41) + 2)), (0, dict(rows=0, x=None)), (0, dict(cols=0))])
def test_dropout(code, change):
    a = dict(ctx=CTX, dtype=1, rows=8, cols=64, p=0.5, seed=3, x=1 << 41, out=1 << 42)
    a.update(change)
    assert abi.status("skl_dropout", *a.values()) == code


def test_work_bytes():
    need = abi.load().skl_product_work_bytes
    assert need(0, 4001, 130, 1500, 2) == 0            # fp32 takes operands as they are
    assert need(0, 16, 4096, 1024, 1) == 8 * 16 * 1024 * 4   # few rows over a long k: its slices' sums
    assert need(1, 16, 4096, 8192, 2) == 8 * 16 * 8192 * 4 * 2 and need(1, 65, 4096, 8192, 2) == 0
    assert need(1, 64, 4096, 8192, 2) == 8 * 64 * 8192 * 4 * 2 and need(1, 64, 4096, 1024, 1) == need(0, 33, 4096, 8192, 2) == 0
    assert need(1, 32, 4096, 1024, 1) == 8 * 32 * 1024 * 4 and need(0, 32, 4096, 1024, 1) == 0
    assert need(1, 64, 130, 1500, 2) == 0              # too few tiles for padded copies
    assert need(1, 16384, 2048, 4096, 2) == 0          # whole tiles
    for bad in ((1, 0, 130, 1500, 2), (1, 4001, 0, 1500, 2), (1, 4001, 130, 0, 2), (1, 4001, 130, 1500, 0), (1, 4001, 130, 1500, 3)):
        assert need(*bad) == 0
    # padded copies: 4096 x 256 of the input, twice 256 x 1536 of the weights (the gated forward)
    assert need(1, 4001, 130, 1500, 2) >= 2 * (4096 * 256 + 2 * 256 * 1536)


class NoContext:
    h, device = None, 0


@pytest.mark.parametrize("what", [
    lambda c, t: dropout.apply(c, t(2, 3).double(), t(2, 3), 0.5, 1),
    lambda c, t: dropout.apply(c, t(2, 3), t(3, 2), 0.5, 1),
    lambda c, t: dropout.apply(c, t(4, 3).t(), t(3, 4), 0.5, 1),
    lambda c, t: Gated(c, t(4, 5), t(4, 6), outputs=5),
    lambda c, t: Gated(c, t(4, 5), t(4, 5), t(5, 1), outputs=5),
    lambda c, t: Projection(c, t(4, 5), outputs=6),
    lambda c, t: Projection(c, t(4, 5), outputs=5, half=True),
])
def test_tensors(what):
    def t(*shape):
        return torch.zeros(shape)   # not on the GPU

    with pytest.raises(ValueError):
        what(NoContext(), t)
