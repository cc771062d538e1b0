"""Tensors of more than 2^32 elements: the rows at the far end come out as the same rows by
themselves do (bit for bit: they run in the same kernel), or as the formula has them."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from soklyn_amd import abi, mxfp4
from soklyn_amd.devblock import distill_error
from soklyn_amd.residual import Join
from tests.test_gpu_mxfp4 import layer, product_ref

pytestmark = pytest.mark.gpu

FAR = (1 << 32) + 12345


@pytest.fixture(autouse=True)
def memory():
    if torch.cuda.mem_get_info()[0] < 120 << 30:
        pytest.skip("needs 120 GB of free GPU memory")
    yield
    torch.cuda.synchronize()
    torch.cuda.empty_cache()


def far_rows(cols, std=1.0):
    """fp16 zeros of more than 2^32 elements, random in the first and last 4 rows."""
    rows = -(-FAR // cols)
    v = torch.zeros(rows, cols, dtype=torch.float16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(7)
    for at in (slice(0, 4), slice(rows - 4, rows)):
        v[at] = (torch.randn(4, cols, generator=g, device="cuda") * std).half()
    return v


def ends(t):
    return torch.cat([t[:4], t[-4:]])


def test_join(ctx):
    cols = 8192
    y = far_rows(cols)
    rows = y.shape[0]
    w = torch.ones(1, cols, device="cuda").half()
    j = Join(ctx, cols, half=True, half_stream=True, pre_norm=abi.NORM_RMS, pre_w=w)
    h, n, stats = torch.empty_like(y), torch.empty_like(y), torch.empty(4, rows, device="cuda")
    j.forward(None, y, h=h, n=n, stats=stats)
    few = ends(y)
    fh, fn, fs = torch.empty_like(few), torch.empty_like(few), torch.empty(4, 8, device="cuda")
    j.forward(None, few, h=fh, n=fn, stats=fs)
    torch.cuda.synchronize()
    assert torch.equal(ends(h), fh) and torch.equal(ends(n), fn) and torch.equal(ends(stats.t()), fs.t())
    del n, y
    dn = torch.zeros(rows, cols, device="cuda")
    dn[:4], dn[-4:] = fh[:4].float() * 3, fh[4:].float().flip(0)
    dx, fx = torch.empty_like(dn), torch.empty(8, cols, device="cuda")
    dparam, fparam = torch.empty(4, cols, device="cuda"), torch.empty(4, cols, device="cuda")
    j.backward(h, None, None, stats, dn, None, dx=dx, dparam=dparam)
    j.backward(fh, None, None, fs, ends(dn).contiguous(), None, dx=fx, dparam=fparam)
    torch.cuda.synchronize()
    assert torch.equal(ends(dx), fx)
    # the other rows add zeros, in another order: 8 terms, off by 8 u of their magnitudes each way
    mag = (ends(dn).double() * fn.double()).abs().sum(0)
    assert ((dparam[2].double() - fparam[2].double()).abs() <= 16 * 2.0 ** -24 * 2 * mag).all()


def test_distillation(ctx):
    cols, top = 50256, 5
    z = far_rows(cols, 2.5)
    rows = z.shape[0]
    g = torch.Generator(device="cuda").manual_seed(8)
    index = torch.randint(0, cols, (rows, top), generator=g, device="cuda", dtype=torch.int32)
    value = torch.randn(rows, top, generator=g, device="cuda")
    label = torch.randint(0, cols, (rows,), generator=g, device="cuda", dtype=torch.int32)

    def run(z, index, value, label):
        out = dict(grad=torch.empty(z.shape, device="cuda"), d_prenorm=torch.empty(z.shape, device="cuda"),
                   d_prenorm_h=torch.empty_like(z), loss=torch.empty(z.shape[0], device="cuda"))
        distill_error(ctx, z, index, value, label, temperature=2.0, alpha=0.5, **out)
        torch.cuda.synchronize()
        return {k: ends(v) for k, v in out.items()}

    far, few = run(z, index, value, label), run(*(ends(t).contiguous() for t in (z, index, value, label)))
    for k in far:
        assert torch.equal(far[k], few[k]), k


def test_a_join_of_the_most_rows(ctx):
    """2^32 - 1 rows, where a row counter that goes on past the last one starts again at 0: in place, so that a
    row done twice would show."""
    rows = (1 << 32) - 1
    j = Join(ctx, 1, half=True, half_stream=True, pre_norm=abi.NORM_DISABLED, scale=0.5)
    x = torch.ones(rows, 1, dtype=torch.float16, device="cuda")
    j.forward(x, None, h=x)
    torch.cuda.synchronize()
    assert (x == 0.5).all()
    del x
    # (of stats only y's part is read, and there is no y)
    dh, stats = torch.ones(rows, 1, device="cuda"), torch.empty(4, rows, device="cuda")
    dparam = torch.full((4, 1), 7.0, device="cuda")
    j.backward(None, None, None, stats, None, dh, dx=dh, dparam=dparam)
    torch.cuda.synchronize()
    assert (dh == 0.5).all() and (dparam == 0).all()


def test_a_gates_gradient_over_the_most_rows(ctx):
    """A sum of 2^32 - 1 ones, each row's once: those of a thread and of a workgroup are exact, the 1280 planes
    are added in slices of 40 and these 32 to each other, 72 roundings of at most u of the sum."""
    rows = (1 << 32) - 1
    j = Join(ctx, 1, half=True, half_stream=True, pre_norm=abi.NORM_DISABLED)
    gate = torch.full((1, 1), 0.5, dtype=torch.float16, device="cuda")
    y = torch.ones(rows, 1, dtype=torch.float16, device="cuda")
    dh, stats = torch.ones(rows, 1, device="cuda"), torch.zeros(4, rows, device="cuda")
    dgate = torch.zeros(1, 1, device="cuda")
    j.backward(None, y, gate, stats, None, dh, dgate=dgate)
    torch.cuda.synchronize()
    assert abs(dgate.item() - rows) <= 72 * 2.0 ** -24 * rows


def test_distillation_of_the_most_rows(ctx):
    """2^32 - 1 rows of one class, whose probability is 1 and gradient 0, every one of them written."""
    rows = (1 << 32) - 1
    z = torch.ones(rows, 1, dtype=torch.float16, device="cuda")
    label = torch.zeros(rows, dtype=torch.int32, device="cuda")
    out = dict(grad=torch.full((rows, 1), 7.0, device="cuda"), d_prenorm=torch.full((rows, 1), 7.0, device="cuda"),
               d_prenorm_h=torch.full((rows, 1), 7.0, dtype=torch.float16, device="cuda"))
    none = torch.zeros(rows, 0, dtype=torch.int32, device="cuda")
    distill_error(ctx, z, none, none.float(), label, alpha=0.5, **out)
    torch.cuda.synchronize()
    for k, v in out.items():
        assert (v == 0).all(), k


# the threads to a row and rows to a workgroup of each: 16 / 16, 64 / 4, 256 / 1 with a table and without
@pytest.mark.parametrize("rows,n", [((1 << 24) + 4096, 20), ((1 << 22) + 4096, 500), ((1 << 20) + 4096, 2052), ((1 << 20) + 4096, 4100)])
def test_distillation_of_more_rows_than_workgroups(ctx, rows, n):
    """Workgroups that go on to another row: what each of 4096 rows gives by itself, over and over."""
    print(f"distill {rows}x{n}", flush=True)
    base, top = 4096, 7
    g = torch.Generator(device="cuda").manual_seed(n)
    z = (torch.randn(base, n, generator=g, device="cuda") * 2.5).half()
    index = torch.randint(-2, n, (base, top), generator=g, device="cuda", dtype=torch.int32)
    value = torch.randn(base, top, generator=g, device="cuda")
    label = torch.randint(-1, n, (base,), generator=g, device="cuda", dtype=torch.int32)

    def run(z, index, value, label):
        out = dict(grad=torch.empty(z.shape, device="cuda"), d_prenorm=torch.empty(z.shape, device="cuda"),
                   d_prenorm_h=torch.empty_like(z), loss=torch.empty(z.shape[0], device="cuda"))
        distill_error(ctx, z, index, value, label, temperature=2.0, alpha=0.5, **out)
        torch.cuda.synchronize()
        return out

    few = run(z, index, value, label)
    times = rows // base
    far = run(z.repeat(times, 1), index.repeat(times, 1), value.repeat(times, 1), label.repeat(times))
    for k, v in far.items():
        for part in v.view(times, base, -1).split(64):
            assert (part == few[k].view(base, -1)).all(), k


@pytest.mark.parametrize("down", [False, True])
def test_casts(ctx, down):
    v = far_rows(66048)
    codes, scales = mxfp4.quantise(ctx, v, down=down)
    back = torch.empty_like(v)
    mxfp4.dequantise(ctx, codes, scales, back, down=down)
    torch.cuda.synchronize()
    if down:   # the last columns by themselves
        few = v[:, -96:].contiguous()
        fc, fs = mxfp4.quantise(ctx, few, down=True)
        fb = torch.empty_like(few)
        mxfp4.dequantise(ctx, fc, fs, fb, down=True)
        torch.cuda.synchronize()
        assert torch.equal(codes[-96:], fc) and torch.equal(scales[-96:], fs) and torch.equal(back[:, -96:], fb)
    else:
        fc, fs = mxfp4.quantise(ctx, ends(v))
        fb = torch.empty(8, v.shape[1], dtype=v.dtype, device="cuda")
        mxfp4.dequantise(ctx, fc, fs, fb)
        torch.cuda.synchronize()
        assert torch.equal(ends(codes), fc) and torch.equal(ends(scales), fs) and torch.equal(ends(back), fb)
        assert (back[4:-4] == 0).all()


def test_served(ctx):
    K, N = 4096, 80
    x = far_rows(K)
    lay, w, b = layer(ctx, K, N, x.shape[0], True, abi.ACT_IDENTITY, 9)
    out = lay.forward(x, x.shape[0])
    torch.cuda.synchronize()
    z, tol = product_ref(ends(x).cpu().float().numpy(), w, b)
    d = np.abs(ends(out).cpu().double().numpy() - z)
    assert (d <= 1.1 * tol + np.abs(z) * 2.0 ** -11 + 2.0 ** -25).all()
