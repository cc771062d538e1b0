"""Few rows on both sides of the borders of the stream over the weights: narrow outputs, where a workgroup's columns pass
the last one, short k, and the row counts at which its blocks of rows change; and pairs at the borders of their tiles."""
from __future__ import annotations

import pytest
import torch

from soklyn_amd import abi
from tests.test_gpu_gated import forward_case
from tests.test_gpu_project import project_case

pytestmark = pytest.mark.gpu
F32, F16 = torch.float32, torch.float16
SIZES = [(1, 3000, 64), (1, 3000, 56), (16, 3008, 72), (2, 3000, 136), (15, 4096, 120), (3, 2000, 64), (16, 2000, 516), (4, 1504, 704),
         (7, 1504, 512), (17, 2008, 512), (32, 3000, 256), (24, 3008, 1000), (18, 4000, 264), (33, 3008, 512), (64, 8000, 256),
         (40, 4000, 2000), (63, 4000, 256), (65, 4000, 512)]


@pytest.mark.parametrize("t", [F32, F16], ids=["f32", "f16"])
@pytest.mark.parametrize("m,k,n", SIZES)
def test_gated(ctx, m, k, n, t):
    forward_case(ctx, m, k, n, t, abi.ACT_SILU, n % 3 == 0, m % 2 == 0)


@pytest.mark.parametrize("t,r", [(F32, F32), (F16, F32), (F16, F16)], ids=["f32", "f16_f32", "f16"])
@pytest.mark.parametrize("m,k,n", SIZES)
def test_projection(ctx, m, k, n, t, r):
    project_case(ctx, m, k, n, t, r, act=abi.ACT_SILU, bias=n % 3 == 0, drop=0.25 if m % 2 else 0.0, keep=m % 2 == 0, in_place=n % 16 == 8)


@pytest.mark.parametrize("m,k,n", [(200, 1200, 416), (300, 1200, 416), (300, 1201, 417), (632, 69, 1256), (192, 1500, 480), (500, 100, 500)])
def test_pairs(ctx, m, k, n):
    forward_case(ctx, m, k, n, F16, abi.ACT_TANH, True, True)
