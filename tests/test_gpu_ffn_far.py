"""Activations of gated blocks and projections far from 0, in the forward, the error from a sum and from the layer
above, and the projection's error: each has its limit there and no NaN.  The matrices are identities, so a result is the
activation of one number and every sum is exact; bounds as in ffn_helpers, where z is exact."""
from __future__ import annotations

import pytest
import torch

from soklyn_amd import abi
from soklyn_amd.gated import Gated
from soklyn_amd.residual import Projection
from tests.ffn_helpers import ACTS, LEAKY, U, check, filled, slope

pytestmark = pytest.mark.gpu
F32, F16 = torch.float32, torch.float16
N = 32
# around the ends of e^z (88.72 over, -87.3 and -103.97 under), where Mish's and tanh's forms change, and a type's ends
FAR = [0.0, 0.39, 0.41, 8.0, 17.0, 19.99, 20.0, 20.01, 44.0, 60.0, 88.5, 88.75, 104.0, 1000.0, 65504.0]


def numbers(t):
    """FAR and their negatives, in fp32 some of its largest too, N of them."""
    v = FAR + [-f for f in FAR[1:]] + ([1e30, -1e30, 3e38] if t is F32 else [300.0, -300.0, 2.0])
    assert len(v) == N
    return torch.tensor(v, dtype=t, device="cuda").repeat(3, 1)


def ref(act, z):
    """The activation and its slope in 64 bits, with a bound on what the kernels compute of each (as a share of |z|
    where the value grows with z: half a step of each of 4 roundings)."""
    z = z.double().cpu()
    off = 64 * U * (1 + z.abs().clamp(max=24)) + 4 * U * z.abs()
    return ACTS[act](z, LEAKY), slope(act, z), off


@pytest.mark.parametrize("t", [F32, F16], ids=["f32", "f16"])
@pytest.mark.parametrize("act", list(ACTS))
def test_forward(ctx, act, t):
    z, eye = numbers(t), torch.eye(N, dtype=t, device="cuda")
    m = z.shape[0]
    v, _, off = ref(act, z)
    op = Gated(ctx, eye, eye * 0, None, torch.ones((1, N), dtype=t, device="cuda"), outputs=N, half=t is F16, act=act, leaky=LEAKY)
    out, a, h = (filled((m, N), t) for _ in range(3))
    op.forward(z, out, a=a)
    Projection(ctx, eye, outputs=N, half=t is F16, act=act, leaky=LEAKY).forward(z, None, h)
    torch.cuda.synchronize()
    assert torch.equal(a, z)
    check(out, (v, off), t, "out")
    check(h, (v, off), t, "h")


@pytest.mark.parametrize("t", [F32, F16], ids=["f32", "f16"])
@pytest.mark.parametrize("act", list(ACTS))
def test_errors(ctx, act, t):
    z = numbers(t)
    m, half = z.shape[0], t is F16
    v, d, off = ref(act, z)
    small = (16 + 4 * z.double().cpu().abs().clamp(max=110)) * U * 8   # of a slope, which is at most 1.1
    u = torch.full_like(z, 0.5)
    op = Gated(ctx, None, None, outputs=N, half=half, act=act, leaky=LEAKY)
    for above in (False, True):
        to = {k: filled((m, N), F32) for k in ("dg", "du")} | {k: filled((m, N), F16) if half else None for k in ("dg_h", "du_h")}
        if above:
            op.hidden_error(torch.ones_like(z), torch.eye(N, dtype=t, device="cuda"), z, u, **to)
        else:
            op.error_from_sum(torch.ones((m, N), device="cuda"), z, u, **to)
        torch.cuda.synchronize()
        check(to["dg"], (0.5 * d, small), F32, "dg")
        check(to["du"], (v, off), F32, "du")
    p, p_h = filled((m, N), F32), filled((m, N), F16) if half else None
    Projection(ctx, None, outputs=N, half=half, act=act, leaky=LEAKY).error(torch.ones((m, N), device="cuda"), z, p, d_prenorm_h=p_h)
    torch.cuda.synchronize()
    check(p, (d, 2 * small), F32, "d_prenorm")
