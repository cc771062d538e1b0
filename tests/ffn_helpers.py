"""References in 64 bits, with bounds, for the tests of gated blocks, projections and dropout.

Bounds (u = 2^-24): a sum of K products in fp32 is off by at most (K + 64) u of the sum of their magnitudes;
an activation by its slope (at most 1.1) times that, plus (16 + 4 |z|) u (1 + |z|) of its own (exp to
(2 + 2 |z|) u, a reciprocal and a few products; tanh to 2 units); a stored result by half a step of its type.
"""
from __future__ import annotations

import numpy as np
import torch

from soklyn_amd import abi

U = 2.0 ** -24
ACTS = {abi.ACT_IDENTITY: lambda z, k: z, abi.ACT_SIGMOID: lambda z, k: torch.sigmoid(z),
        abi.ACT_RELU: lambda z, k: torch.relu(z), abi.ACT_LEAKY: lambda z, k: torch.where(z > 0, z, k * z),
        abi.ACT_TANH: lambda z, k: torch.tanh(z), abi.ACT_SILU: lambda z, k: z * torch.sigmoid(z),
        abi.ACT_MISH: lambda z, k: z * torch.tanh(torch.nn.functional.softplus(z, threshold=100.0))}
SMOOTH = [abi.ACT_IDENTITY, abi.ACT_SIGMOID, abi.ACT_TANH, abi.ACT_SILU, abi.ACT_MISH]
LEAKY = 0.1


def half_step(v, dtype):
    """The most by which rounding to dtype moves v."""
    if dtype == torch.float16:
        return (v.abs() * 2.0 ** -11).clamp(min=2.0 ** -25)
    return v.abs() * U + 2.0 ** -150


def act_off(z, dz):
    """The most by which an activation of z, off by dz itself, is off."""
    return 1.1 * dz + (16 + 4 * z.abs()) * U * (1 + z.abs())


def product(x, w, b=None):
    """x w + b in 64 bits and its bound in fp32."""
    x, w = x.double(), w.double()
    z, size = x @ w.contiguous(), x.abs() @ w.abs().contiguous()
    if b is not None:
        z, size = z + b.double(), size + b.double().abs()
    return z, (x.shape[1] + 64) * U * size + 2.0 ** -140


def within(got, want, bound, what=""):
    got = got.double().cpu()
    want, bound = want.cpu(), bound.cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    off = (got - want).abs()
    bad = ~(off <= bound)
    if bad.any():
        i = torch.nonzero(bad)[0].tolist()
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {i}: got {got[tuple(i)]}, want "
                             f"{want[tuple(i)]} +- {bound[tuple(i)]}")


def values(shape, dtype, seed, std=1.0):
    g = np.random.default_rng(seed)
    return torch.from_numpy((g.standard_normal(shape) * std).astype(np.float32)).cuda().to(dtype)


def odd_base(t):
    """The same values one element behind a 256-byte boundary."""
    room = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
    v = room[1:].view(t.shape)
    v.copy_(t)
    return v


def filled(shape, dtype, fill=-7.0):
    return torch.full(shape, fill, dtype=dtype, device="cuda")


def keeps(rows, cols, p, seed):
    """True where dropout keeps an element, by the blocks' hash, in numpy."""
    u32 = np.uint32
    r = np.arange(rows, dtype=np.uint64)[:, None]
    c = np.arange(cols, dtype=np.uint64)[None, :]
    m = np.uint64(0xFFFFFFFF)
    s = ((r * np.uint64(1103515245)) & m) ^ ((np.uint64(seed) + r * np.uint64(7)) & m) ^ ((c * np.uint64(0x4C957F2D)) & m)
    s ^= s >> np.uint64(17)
    s = (s * np.uint64(1103515245) + np.uint64(12345)) & m
    s ^= s >> np.uint64(15)
    return torch.from_numpy(s.astype(u32).astype(np.float32) / np.float32(4294967296.0) >= np.float32(p))


def factors(rows, cols, p, seed):
    scale = 1.0 / float(np.float32(1) - np.float32(p))
    return torch.where(keeps(rows, cols, p, seed), scale, 0.0).double()


def gated_ref(x, wg, wu, bg, bu, act, leaky=LEAKY):
    """{name: (value, bound)} of out, a and u, the bound in front of the rounding to their type."""
    (a, da), (u, du) = product(x, wg, bg), product(x, wu, bu)
    v, dv = ACTS[act](a, leaky), act_off(a, da)
    out = v * u
    return {"out": (out, dv * (u.abs() + du) + v.abs() * du + 4 * U * out.abs()), "a": (a, da), "u": (u, du)}


def slope(act, z, leaky=LEAKY):
    z = z.double().cpu().requires_grad_()
    return torch.autograd.grad(ACTS[act](z, leaky).sum(), z)[0]


def ungate_ref(s, ds, a, u, act, leaky=LEAKY):
    """The gradients dg and du from s (off by ds) and the kept a and u."""
    a, u, s, ds = (t.double().cpu() for t in (a, u, s, ds))
    v, d = ACTS[act](a, leaky), slope(act, a, leaky)
    ev = (16 + 4 * a.abs()) * U * (1 + a.abs())      # of the activation and of its slope
    return {"dg": (s * u * d, u.abs() * (ds * d.abs() + (s.abs() + ds) * 4 * ev) + 4 * U * (s * u * d).abs()),
            "du": (s * v, ds * v.abs() + (s.abs() + ds) * ev + 4 * U * (s * v).abs())}


def check(got, ref, dtype, name):
    want, bound = ref
    within(got, want, bound + half_step(want, dtype) * (1 + 1e-6), name)
