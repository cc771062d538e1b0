"""The kernels that the products of gated blocks and projections are given, without a GPU."""
from __future__ import annotations

import ctypes as C
import os

import pytest

from soklyn_amd import abi

F32, F16 = 0, 1
GATED, ERROR, PROJECT, GRAD = 0, 1, 2, 3
LEFT, WEIGHTS, LEFT2, WEIGHTS2 = 1, 2, 4, 8


@pytest.fixture(scope="module")
def route():
    if not os.path.exists(abi.LIB_PATH):
        pytest.skip("libsoklyn_hip.so not built")
    f = C.CDLL(abi.LIB_PATH).skl_diag_product_route
    f.restype, f.argtypes = C.c_char_p, [C.c_uint32] * 6
    return lambda *a, off=0: f(*a, off).decode()


# any operand of fp16 off a 4-byte boundary, the second ones too: no loads of dwords to LDS
@pytest.mark.parametrize("kind,operands", [(GATED, (LEFT, WEIGHTS, WEIGHTS2)), (ERROR, (LEFT, WEIGHTS)), (PROJECT, (LEFT, WEIGHTS)),
                                           (GRAD, (LEFT, WEIGHTS, LEFT2, WEIGHTS2))])
@pytest.mark.parametrize("M,N,K", [(1, 264, 4096), (3, 24, 40), (20, 24, 40), (70, 68, 200), (200, 260, 600), (500, 1026, 1024),
                                   (100, 4096, 256)])
def test_one_operand_off_its_boundary(route, kind, operands, M, N, K):
    assert "registers" not in route(kind, F16, M, N, K)
    for off in operands:
        how = route(kind, F16, M, N, K, off=off)
        assert how.endswith((":registers", ":copied")), (off, how)
        assert "registers" not in route(kind, F32, M, N, K, off=off)
        if how.endswith("registers"):   # a tile and waves that the form has (16x16 tiles of a pair on 8 waves, whatever is asked)
            assert how.split(":")[1:3] in (["16", "16"], ["32", "8"], ["64", "4"]), how


# products are one launch, and not priced as the two of a band of 256x256 tiles in front of 128x128 ones: measured
# 1.03 to 1.4 times faster on the kernel named here
@pytest.mark.parametrize("kind,M,N,K,kernel", [
    (GATED, 14592, 1408, 1280, "dma:128"), (GATED, 3328, 5248, 1408, "dma:128"), (PROJECT, 66816, 768, 1408, "dma:128"),
    (PROJECT, 25344, 1408, 640, "dma:128:stored"), (PROJECT, 4352, 8576, 1792, "dma:128:stored"), (GRAD, 69632, 768, 512, "dma:128"),
    (GRAD, 99072, 384, 1920, "dma:128:stored"), (GRAD, 13056, 2816, 1152, "dma:128")])
def test_one_launch(route, kind, M, N, K, kernel):
    assert route(kind, F16, M, N, K) == kernel


# ... but a pair over copies, which is slower on the kernels for operands as stored (0.8 to 0.9 times the speed)
@pytest.mark.parametrize("M,N,K", [(8872, 2856, 1752), (13233, 3320, 776), (12833, 1528, 3800)])
def test_pairs_over_copies(route, M, N, K):
    assert route(GATED, F16, M, N, K) == "dma:256:copied"


# few rows: the stream over the weights where it is measured ahead of the K-splitting kernel, on both sides of its borders
@pytest.mark.parametrize("kind,dtype,M,N,K,rows", [
    (GATED, F16, 1, 64, 3000, True), (GATED, F16, 1, 56, 3000, False), (GATED, F16, 1, 256, 2048, False), (GATED, F16, 16, 512, 2048, True),
    (GATED, F16, 16, 512, 1504, False), (GATED, F16, 16, 1024, 1504, True), (GATED, F16, 1, 4096, 1024, False),
    (GATED, F32, 16, 64, 2000, True), (GATED, F32, 1, 512, 1504, True), (GATED, F32, 1, 256, 1504, True), (GATED, F32, 1, 248, 1504, False), (GATED, F16, 16, 256, 2904, True), (PROJECT, F16, 1, 64, 3000, True),
    (PROJECT, F16, 1, 4096, 2048, False), (PROJECT, F32, 16, 4096, 2048, False), (PROJECT, F32, 17, 4096, 8192, False),
    (GATED, F16, 17, 512, 2048, True), (GATED, F16, 32, 8192, 1504, False), (GATED, F32, 32, 4096, 2048, False),
    (GATED, F32, 32, 256, 3000, True), (GATED, F32, 33, 4096, 8192, False), (PROJECT, F16, 32, 512, 3008, False), (PROJECT, F16, 32, 264, 3480, True), (GATED, F16, 48, 384, 3880, True),
    (PROJECT, F16, 32, 1024, 3008, True), (GATED, F16, 33, 256, 3008, False), (GATED, F16, 64, 512, 3008, True),
    (PROJECT, F16, 64, 4096, 3008, False), (PROJECT, F16, 64, 2048, 4096, True), (PROJECT, F16, 64, 256, 8192, True),
    (GATED, F16, 65, 4096, 8192, False), (ERROR, F16, 1, 4096, 8192, False), (GRAD, F16, 1, 4096, 8192, False)])
def test_few_rows(route, kind, dtype, M, N, K, rows):
    assert (route(kind, dtype, M, N, K) == "rows") == rows


# a pair's tiles: 64x32 once there are enough of them
@pytest.mark.parametrize("M,N,K,off,tile", [(632, 1256, 69, 0, 64), (256, 2432, 448, 0, 64), (200, 480, 2700, 0, 32), (182, 544, 3000, 0, 32),
                                            (300, 416, 1200, 0, 64), (300, 416, 1200, WEIGHTS, 32), (448, 281, 2560, 0, 32)])
def test_tiles_of_a_pair(route, M, N, K, off, tile):
    how = route(GATED, F16, M, N, K, off=off)
    assert how.startswith(f"wave:{tile}:"), how


# 128x128 tiles of an error or projection of odd rows: from 400 on
@pytest.mark.parametrize("kind,M,N,K,dma", [(ERROR, 2752, 2835, 4032, True), (ERROR, 2000, 1531, 1000, False), (PROJECT, 2752, 2835, 4032, True),
                                            (PROJECT, 2000, 1531, 1000, False)])
def test_odd_rows(route, kind, M, N, K, dma):
    assert route(kind, F16, M, N, K).startswith("dma") == dma
