"""The workspaces that Python objects hold for their products: what they keep as calls grow.  Without a GPU: memory is
the CPU's and the stream none."""
from __future__ import annotations

import contextlib
import os

import pytest
import torch

from soklyn_amd import abi


class NoContext:
    h, device = None, 0


@pytest.fixture
def taken(monkeypatch):
    """Sizes of the pieces taken so far; `room` bytes at most in one."""
    if not os.path.exists(abi.LIB_PATH):
        pytest.skip("libsoklyn_hip.so not built")
    got, empty = [], torch.empty
    got_room = [1 << 62]

    def cpu_empty(size, **kw):
        assert kw == dict(device="cuda:0", dtype=torch.uint8)
        if size > got_room[0]:
            raise torch.OutOfMemoryError("no room")
        got.append(size)
        return empty(size, dtype=torch.uint8, device="meta")

    monkeypatch.setattr(torch.cuda, "ExternalStream", lambda *a: None)
    monkeypatch.setattr(torch.cuda, "stream", lambda s: contextlib.nullcontext())
    monkeypatch.setattr(torch, "empty", cpu_empty)
    return got, got_room


@pytest.mark.parametrize("step", [1, 1000, 1 << 20])
def test_growing_calls_keep_little(taken, step):
    got, _ = taken
    w, first, last = abi.Workspace(NoContext()), 10 << 20, 0
    for size in range(first, first + 300 * step, step):
        _, have = w.get(size)
        assert have >= size
        last = size
    assert len(got) <= 7 and sum(got) <= 4 * last and got[0] == first


def test_a_larger_piece_than_asked_for_has_to_fit(taken):
    got, room = taken
    w = abi.Workspace(NoContext())
    room[0] = 120
    assert w.get(100)[1] == 100 and w.get(110)[1] == 110 and w.get(50)[1] == 110
    with pytest.raises(torch.OutOfMemoryError):
        w.get(121)
    assert w.get(110)[1] == 110 and got == [100, 110]


def test_sizes_looked_up_are_forgotten(taken):
    w = abi.Workspace(NoContext())
    for m in range(1, 5001):
        assert w.product(0, m, 40, 24, 1) == (None, 0)
    assert len(w._sizes) <= 1024


def test_few_rows_reserve_sums_for_the_forward_alone(taken):
    """The sums over slices of k of few rows are the forward products' (which they alone use); the backward ones take
    their operands as they are."""
    from soklyn_amd.gated import Gated
    got, _ = taken
    ctx = NoContext()
    ctx.device = -1   # its tensors are on the CPU
    rows, inputs, outputs = 8, 256, 1504
    ones = torch.ones
    seen = []
    for k, n, call in ((inputs, outputs, lambda op: op.input_grad(ones(rows, n), ones(rows, n), ones(rows, k))),
                       (outputs, inputs, lambda op: op.hidden_error(ones(rows, 3000), ones(n, 3000), *(ones(rows, n),) * 2,
                                                                    **{v: ones(rows, n) for v in ("dg", "du")}))):
        op = Gated(ctx, ones(k, n), ones(k, n), outputs=n)
        op._call = tuple(lambda *a: seen.append(a[-2:]) or 0 for _ in op._call)
        call(op)
    assert seen == [(None, 0)] * 2 and not got


def test_work_of_backward_products():
    if not os.path.exists(abi.LIB_PATH):
        pytest.skip("libsoklyn_hip.so not built")
    forward, back = abi.load().skl_product_work_bytes, abi.load().skl_product_grad_work_bytes
    for rows in (1, 16, 32, 64, 127):
        assert back(0, rows, 4096, 8192, 2) == back(1, rows, 4096, 8192, 2) == back(1, rows, 4001, 259, 1) == 0
    for sizes in ((1, 4001, 130, 1500, 2), (1, 129, 1001, 259, 1), (1, 128, 4096, 8192, 2), (1, 16384, 2048, 4096, 2),
                  (0, 4001, 130, 1500, 2), (1, 4001, 0, 1500, 2), (1, 4001, 130, 1500, 3)):
        assert back(*sizes) == forward(*sizes)   # copies of ragged operands
