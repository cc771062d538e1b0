"""Gated and Projection look at their weights in every call: a weight or bias whose tensor has become another in place
(through .data, resize_, set_) is refused where its size, type or layout is not the one the call reads.  Without a GPU:
the tensors are on the CPU, which a context of device -1 takes for its own, and the library is not called."""
from __future__ import annotations

import os

import pytest
import torch

from soklyn_amd import abi
from soklyn_amd.gated import Gated
from soklyn_amd.residual import Projection

K, N, ROWS = 6, 6, 3   # square: a transposed weight differs in its strides alone


class Cpu:
    h, device = None, -1


@pytest.fixture(autouse=True)
def built():
    if not os.path.exists(abi.LIB_PATH):
        pytest.skip("libsoklyn_hip.so not built")


def gated():
    op = Gated(Cpu(), *(torch.ones(K, N) for _ in range(2)), *(torch.ones(1, N) for _ in range(2)), outputs=N)
    x, out, dx = torch.ones(ROWS, K), torch.ones(ROWS, N), torch.ones(ROWS, K)
    return op, [lambda: op.forward(x, out), lambda: op.input_grad(out, torch.ones(ROWS, N), dx)]


def projection():
    op = Projection(Cpu(), torch.ones(K, N), torch.ones(1, N), outputs=N)
    return op, [lambda: op.forward(torch.ones(ROWS, K), None, torch.ones(ROWS, N))]


def become(how, w):
    if how == "smaller":
        w.data = torch.ones(1, w.shape[1])[:, :2].contiguous()
    elif how == "larger":
        w.data = torch.ones(w.shape[0] + 1, w.shape[1])
    elif how == "transposed":
        w.data = w.data.t()
    elif how == "strided":
        w.data = torch.ones(w.shape[0], 2 * w.shape[1])[:, ::2]
    elif how == "half":
        w.data = w.data.half()
    elif how == "resize_":
        w.resize_(w.shape[0], 1)
    else:
        w.set_(torch.ones(1))


@pytest.mark.parametrize("how", ["smaller", "larger", "transposed", "strided", "half", "resize_", "set_"])
@pytest.mark.parametrize("make,names", [(gated, ("wg", "wu", "bg", "bu")), (projection, ("w", "b"))], ids=["gated", "projection"])
def test_weights_that_became_others(make, names, how):
    for name in names:
        op, calls = make()
        seen = []
        op._call = tuple(lambda *a: seen.append(a) or 0 for _ in op._call)
        for call in calls:
            call()
        assert len(seen) == len(calls)
        w = getattr(op, name)
        become(how, w)
        for call in calls:
            with pytest.raises(ValueError, match=name):
                call()
        assert len(seen) == len(calls), name


@pytest.mark.parametrize("make,names", [(gated, ("wg", "bu")), (projection, ("w", "b"))], ids=["gated", "projection"])
def test_weights_of_the_same_size_moved(make, names):
    op, calls = make()
    seen = []

    def call(*a):
        d = op._local.d if make is gated else (op._local.desc,)
        seen.append([v for x in d for v in (x.w, x.b)])
        return 0

    op._call = tuple(call for _ in op._call)
    for c in calls:
        c()
    for name in names:
        w = getattr(op, name)
        w.data = torch.zeros(w.shape)
        for c in calls:
            c()
            assert w.data_ptr() in seen[-1]
