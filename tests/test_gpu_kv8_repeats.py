"""Calls over the 8-bit pool repeat themselves."""

from __future__ import annotations

import pytest
import torch

import kv8_oracle as O
from plastic_infer.kernel.paged_kv8 import kv8_gather, paged_attention_kv8
from test_gpu_kv8_attention import STEP, _rows, _tables

pytestmark = pytest.mark.gpu


def test_calls_repeat_themselves(dev):
    """The same call gives the same bits, whatever ran before and whatever its workspace held."""
    hq, hkv, dim, page = 32, 8, 128, 16
    lens = [512 + 301 * b for b in range(16)]
    tables, pages = _tables(lens, page, 1, 2)
    pool = O.Pool.random(pages, hkv, dim, page, seed=1).to_device(dev)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    t, lens_t = tables.to(dev), i32(lens)
    for dtype in STEP:
        for rows in (1, 5, 80):
            q = _rows(16 * rows, hq, dim, dtype, rows).to(dev)
            cu = i32([rows * b for b in range(17)])
            offs = lens_t - rows
            first = None
            for _ in range(6):
                got = paged_attention_kv8(q, pool, t, lens_t, cu, offs)
                first = got if first is None else first
                assert torch.equal(got, first)
    a, b = (kv8_gather(pool, t, torch.tensor([0] + lens, device=dev).cumsum(0), max(lens))
            for _ in range(2))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("dtype", list(STEP))
@pytest.mark.parametrize("rows", [1, 5, 80])
def test_in_place(dev, rows, dtype):
    """out may be q itself, whichever kernels run; other overlaps are refused."""
    hq, hkv, dim, page = 32, 8, 128, 16
    lens = [300 + 101 * b for b in range(5)]
    tables, pages = _tables(lens, page, 1, 2)
    pool = O.Pool.random(pages, hkv, dim, page, seed=1).to_device(dev)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    q = _rows(5 * rows, hq, dim, dtype, rows).to(dev)
    args = (pool, tables.to(dev), i32(lens), i32([rows * b for b in range(6)]),
            i32([n - rows for n in lens]))
    want = paged_attention_kv8(q, *args)
    room = torch.empty(5 * rows + 1, hq, dim, dtype=dtype, device=dev)
    room[:-1] = q
    with pytest.raises(RuntimeError, match="overlaps"):
        paged_attention_kv8(room[:-1], *args, out=room[1:])
    assert torch.equal(room[:-1], q)
    assert paged_attention_kv8(room[:-1], *args, out=room[:-1]).data_ptr() == room.data_ptr()
    assert torch.equal(room[:-1], want)
