"""What the residual, distillation and 4-bit entry points refuse, without a GPU: their checks come
before anything that looks into the context or touches the device, so a block of zeros stands for
one, and the addresses are never read."""
from __future__ import annotations

import ctypes as C
import os

import pytest
import torch

from soklyn_amd import abi, mxfp4
from soklyn_amd.devblock import distill_error
from soklyn_amd.residual import Join

INVALID, TRAINING, LIMIT, DIMS, BATCH, HARDWARE, NULL = -1, -2, -3, -4, -5, -6, -8
CTX = C.create_string_buffer(8192)
INF, NAN = float("inf"), float("nan")


@pytest.fixture(scope="module", autouse=True)
def built():
    if not os.path.exists(abi.LIB_PATH):
        pytest.skip("libsoklyn_hip.so not built")


class At:
    """Addresses far from each other, none of them memory."""

    def __init__(self):
        self.next = 1 << 40

    def __call__(self):
        self.next += 1 << 32
        return self.next


def forward_args(**change):
    at = At()
    a = dict(ctx=CTX, dtype=1, stream_dtype=0, rows=8, cols=64, post=1, pre=2, act=0, gate_rows=1, scale=1.0, x=at(), y=at(),
             gate=at(), post_w=at(), post_b=at(), pre_w=at(), pre_b=at(), h=at(), n=at(), stats=at())
    a.update(change)
    return a


FORWARD = [
    (NULL, dict(ctx=None)), (INVALID, dict(dtype=2)), (INVALID, dict(dtype=0, stream_dtype=1)), (INVALID, dict(stream_dtype=2)),
    (INVALID, dict(cols=0)), (INVALID, dict(cols=8193)), (BATCH, dict(rows=0)), (INVALID, dict(post=3)), (INVALID, dict(pre=3)),
    (INVALID, dict(act=2)), (INVALID, dict(act=5)), (INVALID, dict(scale=INF)), (INVALID, dict(scale=NAN)),
    (DIMS, dict(gate_rows=0)), (DIMS, dict(gate_rows=2)), (DIMS, dict(gate=None)), (INVALID, dict(y=None)),
    (INVALID, dict(y=None, post=0)), (INVALID, dict(y=None, gate=None, gate_rows=0)), (NULL, dict(post_w=None)),
    (NULL, dict(post=2, post_b=None)), (NULL, dict(pre_w=None)), (NULL, dict(pre_b=None)),
    (NULL, dict(x=None, y=None, post=0, gate=None, gate_rows=0)), (NULL, dict(h=None, n=None)),
]


@pytest.mark.parametrize("code,change", FORWARD)
def test_residual_forward(code, change):
    assert abi.status("skl_residual_forward", *forward_args(**change).values()) == code


@pytest.mark.parametrize("out,other,shift", [("h", "x", 2), ("h", "y", 0), ("h", "gate", 0), ("n", "y", 2), ("n", "x", 0),
                                             ("n", "pre_w", -4), ("stats", "x", 8), ("h", "n", 0), ("stats", "h", 4), ("n", "stats", 0)])
def test_residual_forward_overlap(out, other, shift):
    a = forward_args()
    a[out] = a[other] + shift
    assert abi.status("skl_residual_forward", *a.values()) == INVALID


def backward_args(**change):
    at = At()
    need = abi.load().skl_residual_work_bytes(8, 64)
    a = dict(ctx=CTX, dtype=1, stream_dtype=0, rows=8, cols=64, post=1, pre=2, act=0, gate_rows=1, scale=1.0, h=at(), y=at(),
             gate=at(), post_w=at(), post_b=at(), pre_w=at(), stats=at(), dn=at(), dh=at(), dx=at(), dy=at(), dgate=at(),
             dparam=at(), work=at(), work_bytes=need)
    a.update(change)
    return a


@pytest.mark.parametrize("code,change", FORWARD[:20] + [
    (NULL, dict(stats=None)), (NULL, dict(dn=None, dh=None)), (NULL, dict(h=None)), (NULL, dict(pre_w=None)),
    (NULL, dict(y=None, post=0, gate=None, gate_rows=0, dgate=None)), (NULL, dict(gate=None, gate_rows=0)),
    (NULL, dict(work=None)), (NULL, dict(work=None, dparam=None)), (LIMIT, dict(work_bytes=100)), (HARDWARE, dict(work=(1 << 50) + 2)),
])
def test_residual_backward(code, change):
    assert abi.status("skl_residual_backward", *backward_args(**change).values()) == code


@pytest.mark.parametrize("out,other", [("dx", "dn"), ("dy", "dh"), ("dy", "dn"), ("dx", "h"), ("dgate", "gate"), ("dparam", "stats"),
                                       ("work", "y"), ("dx", "dy"), ("work", "dx"), ("dparam", "post_w")])
def test_residual_backward_overlap(out, other):
    a = backward_args()
    a[out] = a[other]
    assert abi.status("skl_residual_backward", *a.values()) == INVALID
    a = backward_args()
    a["dx"] = a["dh"] + 4   # in place is the same buffer, not one next to it
    assert abi.status("skl_residual_backward", *a.values()) == INVALID


def desc(**change):
    at = At()
    d = abi.SklDenseDesc()
    for k, v in dict(dict(dtype=1, inputs=64, outputs=32, max_batch=16, is_training=1, out=at(), grad=at(), d_prenorm=at(),
                          d_prenorm_h=at(), b=at(), preact=at(), predrop=at(), prenorm=at(), centered=at(), norm_rstd=at(),
                          norm_w=at(), norm_b=at()), **change).items():
        setattr(d, k, v)
    return d, at


def distill_status(d=None, **change):
    blk, at = desc(**(d or {}))
    a = dict(ctx=CTX, blk=C.byref(blk), index=at(), value=at(), top=4, label=at(), rows=8, t=2.0, alpha=0.5, loss=at())
    a.update(change)
    return abi.status("skl_dense_distill_error", *a.values())


@pytest.mark.parametrize("code,d,change", [
    (NULL, {}, dict(ctx=None)), (NULL, {}, dict(blk=None)), (INVALID, dict(dtype=2), {}), (INVALID, dict(outputs=0), {}),
    (INVALID, dict(max_batch=0), {}), (INVALID, dict(norm=1), {}), (INVALID, dict(act=6), {}), (TRAINING, dict(is_training=0), {}),
    (BATCH, {}, dict(rows=0)), (LIMIT, {}, dict(rows=17)), (INVALID, {}, dict(top=1025)), (INVALID, dict(outputs=1 << 31), {}),
    (INVALID, {}, dict(t=0.0)), (INVALID, {}, dict(t=-1.0)), (INVALID, {}, dict(t=INF)), (INVALID, {}, dict(t=NAN)),
    (INVALID, {}, dict(t=2.0 ** -61)), (INVALID, {}, dict(t=2.0 ** 61)), (INVALID, {}, dict(alpha=-0.1)), (INVALID, {}, dict(alpha=1.5)), (INVALID, {}, dict(alpha=NAN)), (NULL, {}, dict(index=None)),
    (NULL, {}, dict(value=None)), (NULL, {}, dict(label=None)), (NULL, dict(out=None), {}), (NULL, dict(grad=None), {}),
    (NULL, dict(d_prenorm=None), {}), (NULL, dict(d_prenorm_h=None), {}),
    (INVALID, dict(grad=1 << 50, out=1 << 50), {}), (INVALID, dict(grad=1 << 50, d_prenorm=(1 << 50) + 64), {}),
    (INVALID, dict(out=1 << 50), dict(loss=(1 << 50) + 4)),
])
def test_distill(code, d, change):
    assert distill_status(d, **change) == code


def cast_status(back=False, **change):
    at = At()
    a = dict(ctx=CTX, src=at(), dtype=1, rows=8, cols=64, down=0, codes=at(), scales=at())
    a.update(change)
    if back:
        order = ("ctx", "codes", "scales", "rows", "cols", "down", "src", "dtype")
        return abi.status("skl_mxfp4_dequantise", *[a[k] for k in order])
    return abi.status("skl_mxfp4_quantise", *a.values())


@pytest.mark.parametrize("back", [False, True])
@pytest.mark.parametrize("code,change", [
    (NULL, dict(ctx=None)), (INVALID, dict(dtype=2)), (INVALID, dict(down=2)), (INVALID, dict(cols=0x7fffff81)),
    (INVALID, dict(down=1, rows=0x7fffff81)), (INVALID, dict(rows=1 << 31, cols=1 << 16)), (0, dict(rows=0)), (0, dict(cols=0)), (NULL, dict(src=None)), (NULL, dict(codes=None)),
    (NULL, dict(scales=None)), (HARDWARE, dict(codes=(1 << 50) + 8)), (HARDWARE, dict(scales=(1 << 50) + 2)),
    (INVALID, dict(src=1 << 50, codes=(1 << 50) + 1008)), (INVALID, dict(codes=1 << 50, scales=(1 << 50) + 4)),
])
def test_casts(back, code, change):
    assert cast_status(back, **change) == code


@pytest.mark.parametrize("back", [False, True])
@pytest.mark.parametrize("dtype,rows,cols", [(0, 1, 1 << 30), (1, 1, 1 << 31), (1, 128, (1 << 31) + 5), (0, 129, 1 << 29), (1, 1, (1 << 32) - 1),
                                             (0, 1, (1 << 32) - 64)])
def test_casts_down_more_than_a_launch_takes(back, dtype, rows, cols):
    assert cast_status(back, dtype=dtype, rows=rows, cols=cols, down=1, src=1 << 50, codes=2 << 50, scales=3 << 50) == INVALID


def serve_status(d=None, **change):
    blk, at = desc(**(d or {}))
    a = dict(ctx=CTX, blk=C.byref(blk), x=at(), rows=8, cols=64, batch=8, codes=at(), scales=at(), work=at(),
             size=abi.load().skl_mxfp4_work_bytes(64, 32, 16))
    a.update(change)
    return abi.status("skl_dense_forward_mxfp4", *a.values())


@pytest.mark.parametrize("code,d,change", [
    (NULL, {}, dict(ctx=None)), (NULL, {}, dict(blk=None)), (INVALID, dict(dtype=2), {}), (INVALID, dict(inputs=0), {}),
    (INVALID, dict(inputs=(1 << 24) + 1), dict(cols=(1 << 24) + 1)), (INVALID, dict(outputs=0), {}), (INVALID, dict(norm=4), {}),
    (INVALID, dict(act=8), {}), (NULL, {}, dict(x=None)),
    (DIMS, {}, dict(rows=7)), (LIMIT, {}, dict(rows=17)), (DIMS, {}, dict(cols=65)), (INVALID, dict(act=5), {}),
    (BATCH, {}, dict(batch=0)), (BATCH, dict(norm=3), dict(batch=1)), (NULL, dict(norm=1, prenorm=None), {}),
    (NULL, dict(norm=1, preact=None), {}), (NULL, {}, dict(codes=None)), (NULL, {}, dict(scales=None)), (NULL, dict(out=None), {}),
    (NULL, dict(b=None), {}), (HARDWARE, {}, dict(codes=(1 << 50) + 4)), (HARDWARE, {}, dict(scales=(1 << 50) + 1)),
    (INVALID, dict(out=1 << 50), dict(x=(1 << 50) + 2)), (INVALID, dict(norm=1, centered=1 << 50), dict(x=1 << 50)),
    (INVALID, dict(out=1 << 50), dict(codes=(1 << 50) + 16)),
])
def test_serve(code, d, change):
    assert serve_status(d, **change) == code


@pytest.mark.parametrize("norm", [1, 2, 3])
def test_serve_of_a_workspace_in_the_norms_cache(norm):
    """The product reads its workspace while it writes the pre-norm values."""
    need = abi.load().skl_mxfp4_work_bytes(64, 32, 64)
    at = 1 << 50
    for prenorm in (at, at + 128, at + need - 2, at - 64 * 32 * 2 + 2):
        assert need and serve_status(dict(norm=norm, max_batch=64, prenorm=prenorm), rows=64, batch=64, work=at, size=need) == INVALID


@pytest.mark.parametrize("norm,size", [(1, 2 * 8), (2, 2 * 8), (3, 2 * 32)])
def test_serve_of_an_input_in_the_norms_deviations(norm, size):
    at = 1 << 50
    for x in (at, at + size - 2):
        assert serve_status(dict(norm=norm, norm_rstd=at), x=x) == INVALID


def test_work_sizes():
    lib = abi.load()
    assert lib.skl_residual_work_bytes(0, 64) == lib.skl_residual_work_bytes(64, 0) == 0
    assert lib.skl_residual_work_bytes(1, 64) >= 5 * 64 * 4
    # workspaces do not grow with the rows without end
    assert lib.skl_residual_work_bytes(1 << 31, 8192) <= 256 * 5 * 8192 * 4


@pytest.mark.parametrize("cols", [1, 64, 65, 512, 513, 8192])
def test_work_of_a_join_of_the_most_rows(cols):
    """Up to the last row that 32 bits count, as many planes as for a great many rows."""
    need = abi.load().skl_residual_work_bytes
    for rows in ((1 << 32) - (1 << 24), (1 << 32) - 20480, (1 << 32) - 16, (1 << 32) - 15, (1 << 32) - 1):
        assert need(rows, cols) == need(1 << 31, cols) > 0, rows


def test_work_of_a_layer_covers_its_smaller_batches():
    need = abi.load().skl_mxfp4_work_bytes
    for inputs, outputs in ((64, 32), (4096, 4096), (777, 1531), (300, 20000), (5000, 100)):
        sizes = [need(inputs, outputs, b) for b in (0, 1, 16, 17, 64, 65, 128, 500, 1000, 2048, 4096, 8192, 100000)]
        assert sizes == sorted(sizes) and sizes[0] == 0 and sizes[-1] > 0
    assert need(0, 64, 64) == need(64, 0, 64) == 0


@pytest.mark.parametrize("batch", [(1 << 32) - 256, (1 << 32) - 255, (1 << 32) - 64, (1 << 32) - 1])
def test_work_of_a_layer_of_the_most_rows_or_outputs(batch):
    """Rounding up to whole tiles goes past 32 bits."""
    need = abi.load().skl_mxfp4_work_bytes
    assert need(64, 64, batch) >= need(64, 64, 1 << 31) > 1 << 36
    assert need(64, batch, 64) >= need(64, 1 << 31, 64) > 1 << 32


@pytest.mark.parametrize("inputs,outputs,batch", [(1, 1, (1 << 32) - 1), (1, 1, (1 << 32) - 255), (64, 1, 1 << 29), (4096, 64, 1 << 25),
                                                  (1, (1 << 32) - 1, 1), (1, (1 << 27) + 1, 32), (1, (1 << 32) - 1, 64)])
def test_serve_of_more_than_a_launch_takes(inputs, outputs, batch):
    """Refused whatever the workspace; addresses further from each other than any of the tensors is long."""
    d, _ = desc(dtype=0, inputs=inputs, outputs=outputs, max_batch=batch, **{k: i << 50 for i, k in enumerate((
        "out", "b", "grad", "d_prenorm", "d_prenorm_h", "preact", "predrop", "prenorm", "centered", "norm_rstd", "norm_w", "norm_b"), 1)})
    assert abi.status("skl_dense_forward_mxfp4", CTX, C.byref(d), 13 << 50, batch, inputs, batch, 14 << 50, 15 << 50, 16 << 50,
                      (1 << 64) - 1) == INVALID


class NoContext:
    h, device = CTX, 0

    def synchronize(self):
        raise AssertionError("not reached")


def test_wrappers_refuse_tensors_that_the_calls_do_not_take():
    """Wrong types, shapes, strides and devices (these are on the CPU) never reach an address."""
    ctx, f, h = NoContext(), torch.zeros(4, 8), torch.zeros(4, 8, dtype=torch.float16)
    with pytest.raises(ValueError, match="pre_w"):
        Join(ctx, 8, pre_w=f[:1])
    join = Join(ctx, 8)
    for x, y in ((f, None), (h, None), (f[:, :4], None), (None, f), (torch.zeros(8, 4).t(), None), (None, None)):
        with pytest.raises(ValueError):
            join.forward(x, y, n=torch.zeros(4, 8))
    with pytest.raises(ValueError):
        join.backward(f, f, None, torch.zeros(4, 4), f, f, dgate=f)
    with pytest.raises(ValueError, match="gate"):
        join.forward(f, f, torch.zeros(3, 8), n=f)
    i = torch.zeros(4, 2, dtype=torch.int32)
    with pytest.raises(ValueError):
        distill_error(ctx, f, i, torch.zeros(4, 2), grad=f, d_prenorm=f)
    with pytest.raises(ValueError):
        distill_error(ctx, h, i, torch.zeros(4, 2), grad=f, d_prenorm=f)
    with pytest.raises(ValueError):
        mxfp4.quantise(ctx, f.double())
    with pytest.raises(ValueError):
        mxfp4.quantise(ctx, f)
    with pytest.raises(ValueError):
        mxfp4.dequantise(ctx, torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(4, 4, dtype=torch.uint8), f)
    with pytest.raises(ValueError):
        mxfp4.Layer(ctx, 8, 8, 4, torch.zeros(8, 64, dtype=torch.uint8), torch.zeros(8, 4, dtype=torch.uint8))


def test_shapes_of_codes():
    assert mxfp4.shapes(4, 8) == ((4, 64), (4, 4)) and mxfp4.shapes(129, 8, True) == ((8, 128), (8, 8))
