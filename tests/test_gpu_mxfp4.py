"""skl_mxfp4_quantise / _dequantise, bit for bit against the format's rules on the CPU, and
skl_dense_forward_mxfp4 against the product of those values in 64 bits.

The product's tolerance: the values' products are exact in fp32; each matrix instruction adds 128 of
them to a sum, off by at most 2^-22 of their magnitudes (two half steps for whatever order it adds
in), over K / 128 instructions, and up to 16 sums are joined: (K / 128 + 16) 2^-22 sum |x w|, plus
2^-23 for the bias.  The activations' slope is at most 1.1; their own error is 2^-21 (1 + |z|)
relative (exp and reciprocal, each a few units in the last place, the exponent off by u |z|); fp16
outputs round once more (2^-11, or 2^-25).
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from soklyn_amd import abi, mxfp4

pytestmark = pytest.mark.gpu

GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def pack_ref(v: np.ndarray):
    """Rows of v (fp32 values) as codes and scales, from the rules."""
    n, k = v.shape
    kp = -(-k // 128) * 128
    p = np.zeros((n, kp), np.float64)
    p[:, :k] = v
    p = p.reshape(n, kp // 32, 32)
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        big = np.abs(p).max(2)
        bad = ~np.isfinite(p).all(2)
        e = np.where(big > 0, np.floor(np.log2(np.where(big > 0, big, 1.0))), -200)
        # log2 may round up just under a power of two
        e = np.where(np.ldexp(1.0, e.astype(int)) > big, e - 1, e)
        s = np.where(bad, 255, np.clip(e - 2 + 127, 0, 254)).astype(int)
        a = np.abs(p) * np.ldexp(1.0, 127 - np.where(bad, 127, s))[:, :, None]
        d = np.abs(a[..., None] - GRID)
        code = d.argmin(3)
        # a tie goes to the even code: argmin takes the lower of the two
        nxt = np.minimum(code + 1, 7)
        tie = (np.take_along_axis(d, nxt[..., None], 3)[..., 0] == np.take_along_axis(d, code[..., None], 3)[..., 0])
        code = np.where(tie & (code % 2 == 1) & (nxt > code), nxt, code)
    code = code + 8 * np.signbit(p)
    code = code.reshape(n, kp).astype(np.uint8)
    return code, s.astype(np.uint8)


def values_ref(code, s):
    v = GRID[code & 7] * np.where(code & 8, -1.0, 1.0)
    v = v.reshape(s.shape + (32,)) * np.ldexp(1.0, s.astype(int) - 127)[:, :, None]
    v = np.where(s[:, :, None] == 255, np.nan, v)
    return v.reshape(code.shape)


def numbers(rows, cols, half, seed):
    g = np.random.default_rng(seed)
    v = g.standard_normal((rows, cols)) * np.exp(g.standard_normal((rows, 1)) * 2)
    return v.astype(np.float16).astype(np.float32) if half else v.astype(np.float32)


def up(v, half):
    return torch.from_numpy(v).to(torch.float16 if half else torch.float32).cuda()


def check_codes(ctx, v, half, down, offset=0):
    src = up(v, half)
    if offset:
        b = torch.empty(src.numel() + offset, dtype=src.dtype, device="cuda")[offset:].view(src.shape)
        b.copy_(src)
        src = b
    (cn, cb), (sn, sb) = mxfp4.shapes(*v.shape, down)
    cbuf = torch.full((cn * cb + 128,), 0xA5, dtype=torch.uint8, device="cuda")
    sbuf = torch.full((sn * sb + 128,), 0xA5, dtype=torch.uint8, device="cuda")
    codes, scales = cbuf[64:64 + cn * cb].view(cn, cb), sbuf[64:64 + sn * sb].view(sn, sb)
    mxfp4.quantise(ctx, src, down=down, codes=codes, scales=scales)
    torch.cuda.synchronize()
    for b, n in ((cbuf, cn * cb), (sbuf, sn * sb)):
        assert (b[:64] == 0xA5).all() and (b[64 + n:] == 0xA5).all(), "written outside the output"
    code, s = pack_ref(v.T if down else v)
    got = codes.cpu().numpy()
    got = np.stack([got & 15, got >> 4], 2).reshape(code.shape)
    np.testing.assert_array_equal(scales.cpu().numpy(), s)
    ok = np.repeat(s != 255, 32, 1)
    np.testing.assert_array_equal(got[ok], code[ok])
    want = values_ref(code, s)[:, : v.shape[0] if down else v.shape[1]]
    want = want.T if down else want
    for dt in (torch.float32, torch.float16):
        buf = torch.full((v.size + 128 + offset,), 7.0, dtype=dt, device="cuda")
        out = buf[64 + offset:64 + offset + v.size].view(v.shape)
        mxfp4.dequantise(ctx, codes, scales, out, down=down)
        torch.cuda.synchronize()
        assert (buf[:64 + offset] == 7).all() and (buf[64 + offset + v.size:] == 7).all(), "written outside the output"
        with np.errstate(over="ignore", invalid="ignore"):
            np.testing.assert_array_equal(out.cpu().numpy(), want.astype(np.float32 if dt is torch.float32 else np.float16))


@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("down", [False, True])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 31), (3, 32), (5, 33), (2, 127), (7, 128), (129, 129), (64, 65), (65, 64),
                                       (300, 777), (33, 1000), (1000, 33), (2, 4100)])
def test_codes_scales_and_values(ctx, half, down, rows, cols):
    print(f"quantise {rows}x{cols} half={half} down={down}", flush=True)
    check_codes(ctx, numbers(rows, cols, half, rows + cols), half, down)


@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("down", [False, True])
def test_borders(ctx, half, down):
    """Ties, saturation, zeros of both signs, powers of two and the values next to them."""
    ties = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.5, 7.0, 7.9, 0.0, -0.0, 4.0]
    rows = []
    for e in (-10, -2, 0, 3, 12):
        row = [t * 2.0 ** e for t in ties] + [-t * 2.0 ** e for t in ties]
        rows.append(row + [0.0] * 6)
        up_, dn = np.nextafter(np.float32(1), np.float32(2)), np.nextafter(np.float32(1), np.float32(0))
        rows.append([x * t * 2.0 ** e for t in ties[:7] for x in (up_, dn)] + [4.0 * 2.0 ** e] + [0.0] * 17)
    v = np.array(rows, np.float32)
    v = v.astype(np.float16).astype(np.float32) if half else v
    check_codes(ctx, np.ascontiguousarray(v.T) if down else v, half, down)


def test_smallest_and_largest(ctx):
    g = np.random.default_rng(1)
    f = np.float32
    rows = [g.standard_normal(64).astype(f) * f(2.0 ** e) for e in (-126, -124, -123, -64, -63, 100, 125)]
    rows += [(g.standard_normal(64) * 1e-41).astype(f), np.full(64, 3.4e38, f), np.zeros(64, f), np.full(64, 1e-45, f)]
    for down in (False, True):
        v = np.array(rows, f)
        check_codes(ctx, np.ascontiguousarray(v.T) if down else v, False, down)
    h = np.array([g.standard_normal(64) * 2.0 ** -20, np.full(64, 6e-8), np.full(64, 65504.0)], f).astype(np.float16)
    check_codes(ctx, h.astype(f), True, False)


@pytest.mark.parametrize("down", [False, True])
def test_infinities_and_nan_make_their_block_nan(ctx, down):
    for half in (True, False):
        v = numbers(4, 96, half, 2)
        v[0, 5], v[1, 40], v[2, 95] = np.inf, np.nan, -np.inf
        check_codes(ctx, np.ascontiguousarray(v.T) if down else v, half, down)


@pytest.mark.parametrize("offset", [1, 3, 7])
def test_any_alignment_of_the_values(ctx, offset):
    for half in (True, False):
        check_codes(ctx, numbers(9, 200, half, 3), half, False, offset)
        check_codes(ctx, numbers(200, 9, half, 3), half, True, offset)


ACT_REF = {abi.ACT_IDENTITY: lambda z: z, abi.ACT_SILU: lambda z: z / (1 + np.exp(-z)), abi.ACT_TANH: np.tanh,
           abi.ACT_RELU: lambda z: np.maximum(z, 0), abi.ACT_SIGMOID: lambda z: 1 / (1 + np.exp(-z)),
           abi.ACT_LEAKY: lambda z: np.where(z > 0, z, 0.125 * z)}


def layer(ctx, K, N, max_batch, half, act, seed, **kw):
    g = np.random.default_rng(seed)
    w = (g.standard_normal((K, N)) * np.sqrt(2.0 / K)).astype(np.float32)
    b = (g.standard_normal((1, N)) * 0.1).astype(np.float16).astype(np.float32)
    codes, scales = mxfp4.quantise(ctx, up(w, False), down=True)
    lay = mxfp4.Layer(ctx, K, N, max_batch, codes, scales, half=half, act=act, leaky=0.125, b=up(b, half), **kw)
    return lay, values_ref(*pack_ref(w.T)), b


def product_ref(x, w, b):
    xv = values_ref(*pack_ref(x))
    z = xv @ w.T + b
    K = x.shape[1]
    return z, (K / 128 + 16) * 2.0 ** -22 * (np.abs(xv) @ np.abs(w).T) + 2.0 ** -23 * (np.abs(z) + np.abs(b))


def check_forward(ctx, K, N, M, half, act, seed=1, max_batch=None, offset=0):
    lay, w, b = layer(ctx, K, N, max_batch or M, half, act, seed)
    x = numbers(M, K, half, seed + 1)
    xt = up(x, half)
    if offset:
        t = torch.empty(xt.numel() + offset, dtype=xt.dtype, device="cuda")[offset:].view(xt.shape)
        t.copy_(xt)
        xt = t
    lay.out.fill_(7.0)
    out = lay.forward(xt, M)
    torch.cuda.synchronize()
    got = out.cpu().double().numpy()
    assert (got[M:] == 7.0).all(), "rows behind the batch were written"
    z, tol = product_ref(x, w, b)
    want = ACT_REF[act](z)
    tol = 1.1 * tol + np.abs(want) * 2.0 ** -21 * (1 + np.abs(z)) * (act not in (abi.ACT_IDENTITY, abi.ACT_RELU)) + 1e-30
    if half:
        tol = tol + np.abs(want) * 2.0 ** -11 + 2.0 ** -25
    d = np.abs(got[:M] - want)
    assert (d <= tol).all(), f"{(d / tol).max():.3g} of its tolerance, off by {d.max():.3g}"
    return lay, xt, out


@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("M,K,N", [(1, 1, 1), (1, 4096, 512), (2, 130, 17), (15, 128, 16), (16, 640, 100), (17, 127, 15), (33, 777, 129),
                                   (64, 256, 64), (65, 100, 200), (100, 1531, 301), (128, 512, 128), (129, 384, 257),
                                   (255, 1024, 255), (256, 512, 256), (300, 1000, 511), (512, 640, 512), (777, 333, 300)])
def test_forward_sizes(ctx, half, M, K, N):
    print(f"mxfp4 forward {M}x{K}x{N} half={half}", flush=True)
    check_forward(ctx, K, N, M, half, abi.ACT_SILU, seed=M + K + N)


# batches on either side of each choice of tile, inputs of every remainder that their padding has
@pytest.mark.parametrize("M,N", [(31, 33), (32, 4097), (33, 31), (63, 65), (64, 64 * 256), (65, 64 * 128), (64, 64 * 256 + 1), (127, 9000),
                                 (1024, 1024), (1025, 1024), (3840, 2560), (3841, 2561)])
def test_borders_of_the_tiles(ctx, M, N):
    print(f"mxfp4 forward {M}x{N}, tile {tile_of(M, N)}", flush=True)
    for half, K in ((True, 31), (False, 129), (True, 257)):
        check_forward(ctx, K, N, M, half, abi.ACT_SILU, seed=M + N)


@pytest.mark.parametrize("act", list(ACT_REF))
def test_activations(ctx, act):
    for half in (True, False):
        check_forward(ctx, 256, 80, 24, half, act)
        check_forward(ctx, 512, 512, 600, half, act)


def test_large_grids(ctx):
    """Whole and ragged tiles in numbers that fill the GPU, in both types."""
    check_forward(ctx, 1024, 2048, 2048, True, abi.ACT_SILU)
    check_forward(ctx, 1100, 1999, 2111, True, abi.ACT_TANH)
    check_forward(ctx, 300, 1537, 1500, False, abi.ACT_IDENTITY)


def tile_of(m, n):
    """The tile edge that the product takes (0: the kernel for few rows)."""
    def tiles(t):
        return -(-m // t) * -(-n // t)
    return 0 if m <= 32 else 64 if tiles(64) <= 256 else 256 if tiles(256) >= 160 else 128


# every row and column of tiles of 256: whole and ragged, one k-tile, an odd number of them, the last one half there
@pytest.mark.parametrize("M,K,N,half,act", [
    (3000, 640, 4096, True, abi.ACT_SILU), (3333, 777, 3999, False, abi.ACT_TANH), (33, 300, 40967, True, abi.ACT_IDENTITY),
    (40961, 128, 65, False, abi.ACT_SIGMOID), (2561, 2560, 4099, True, abi.ACT_LEAKY), (4096, 256, 2560, False, abi.ACT_RELU),
    (3500, 1281, 3001, True, abi.ACT_TANH), (2570, 1024, 4010, False, abi.ACT_SILU)])
def test_tiles_of_256(ctx, M, K, N, half, act):
    print(f"mxfp4 forward {M}x{K}x{N} half={half}", flush=True)
    assert tile_of(M, N) == 256
    check_forward(ctx, K, N, M, half, act, seed=M + K + N)


@pytest.mark.parametrize("M,K,N,half,act", [(1500, 400, 1100, True, abi.ACT_SILU), (1025, 900, 1090, False, abi.ACT_TANH),
                                            (129, 128, 17001, True, abi.ACT_IDENTITY)])
def test_tiles_of_128(ctx, M, K, N, half, act):
    assert tile_of(M, N) == 128
    check_forward(ctx, K, N, M, half, act, seed=M + K + N)


def test_the_same_rows_in_every_tile(ctx):
    """Each tile of 256 rows has the same rows, and so the same outputs, bit for bit."""
    M, K, N = 256 * 12, 900, 256 * 14
    assert tile_of(M, N) == 256
    lay, _, _ = layer(ctx, K, N, M, True, abi.ACT_SILU, 12)
    out = lay.forward(up(numbers(256, K, True, 13), True).repeat(12, 1), M)
    torch.cuda.synchronize()
    assert (out.view(12, 256, N) == out[:256]).all()


def test_smaller_batches_of_a_layer(ctx):
    for M in (1, 16, 31, 100):
        check_forward(ctx, 500, 300, M, True, abi.ACT_IDENTITY, max_batch=160)
    lay, w, b = layer(ctx, 640, 384, 512, True, abi.ACT_SILU, 4)
    x = up(numbers(512, 640, True, 5), True)
    whole = lay.forward(x, 512).clone()
    for M in (1, 16, 17, 64, 65, 128, 400):
        out = lay.forward(x, M)
        torch.cuda.synchronize()
        # another kernel may add in another order: one step of fp16 at the outputs' scale
        assert (out[:M].float() - whole[:M].float()).abs().max() <= 2.0 ** -10 * whole.abs().max().float()


@pytest.mark.parametrize("offset", [1, 3])
def test_any_alignment(ctx, offset):
    for M in (8, 200, 600):
        check_forward(ctx, 333, 200, M, True, abi.ACT_IDENTITY, offset=offset)
        check_forward(ctx, 512, 256, M, False, abi.ACT_IDENTITY, offset=offset)


@pytest.mark.parametrize("M", [4, 130, 700])
def test_inputs_that_are_not_finite_stay_in_their_rows(ctx, M):
    lay, _, _ = layer(ctx, 300, 256, M, True, abi.ACT_IDENTITY, 6)
    x = up(numbers(M, 300, True, 7), True)
    clean = lay.forward(x, M).clone()
    x[1, 5], x[3, 299] = float("inf"), float("nan")
    out = lay.forward(x, M)
    torch.cuda.synchronize()
    rows = [r for r in range(M) if r not in (1, 3)]
    assert torch.isnan(out[1]).all() and torch.isnan(out[3]).all()
    assert torch.equal(out[rows], clean[rows])
    x[:] = 0
    out = lay.forward(x, M)
    torch.cuda.synchronize()
    assert torch.equal(out, lay.b.expand(M, 256))


@pytest.mark.parametrize("norm", [abi.NORM_RMS, abi.NORM_LAYER, abi.NORM_BATCH])
@pytest.mark.parametrize("M", [5, 300])
def test_with_a_norm(ctx, norm, M):
    """The pre-norm values are the product's; what the norm makes of them is what the block's own
    forward makes of the same values."""
    lay, w, b = layer(ctx, 384, 200, M, True, abi.ACT_MISH, 8, norm=norm)
    x = numbers(M, 384, True, 9)
    out = lay.forward(up(x, True), M)
    torch.cuda.synchronize()
    z, tol = product_ref(x, w, b * (norm != abi.NORM_BATCH))
    d = np.abs(lay.prenorm.cpu().double().numpy() - z)
    assert (d <= tol + np.abs(z) * 2.0 ** -11 + 2.0 ** -25).all()
    p = lay.prenorm.double()
    dim = 0 if norm == abi.NORM_BATCH else 1
    c = p - p.mean(dim, keepdim=True) if norm != abi.NORM_RMS else p
    y = c / (c.square().mean(dim, keepdim=True) + 1e-6).sqrt()
    want = y * torch.tanh(torch.nn.functional.softplus(y))
    # rstd, the normalised value and the output each round to fp16, and Mish's slope is at most 1.1
    assert ((out.double() - want).abs() <= 6 * 2.0 ** -11 * (1 + y.abs())).all()


def test_captured_and_replayed(ctx):
    side = torch.cuda.Stream()
    cap = abi.Context(0, 16, stream=side.cuda_stream)
    try:
        for M in (8, 600):
            lay, _, _ = layer(cap, 512, 384, M, True, abi.ACT_SILU, 10)
            eager = mxfp4.Layer(ctx, 512, 384, M, lay.codes, lay.scales, half=True, act=abi.ACT_SILU, b=lay.b)
            x = up(numbers(M, 512, True, 11), True)
            codes, scales = mxfp4.quantise(ctx, x)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side, capture_error_mode="thread_local"):
                lay.forward(x, M)
                mxfp4.quantise(cap, x, codes=codes, scales=scales)
            for rep in range(3):
                x.copy_(torch.randn(M, 512, device="cuda") * (rep + 1))
                lay.out.fill_(float("nan"))
                torch.cuda.synchronize()
                graph.replay()
                torch.cuda.synchronize()
                want = eager.forward(x, M)
                wc, ws = mxfp4.quantise(ctx, x)
                torch.cuda.synchronize()
                assert torch.equal(lay.out, want) and torch.equal(wc, codes) and torch.equal(ws, scales)
    finally:
        torch.cuda.synchronize()
        cap.close()
