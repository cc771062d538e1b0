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
