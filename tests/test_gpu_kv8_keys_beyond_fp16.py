"""fp16 q over keys of the 8-bit pool whose values fp16 does not hold, against float64. Bounds: those of
test_gpu_kv8_attention, probabilities rounded once to fp16 at the worst."""

from __future__ import annotations

import pytest
import torch

import kv8_oracle as O
from plastic_infer.kernel.paged_kv8 import paged_attention_kv8, paged_decode_attention_kv8
from test_gpu_kv8_attention import _check, _rows, _tables

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [1, 3, 64])
@pytest.mark.parametrize("k_exp,q_size,scale", [
    (9, 2.0 ** -16, 0.1), (14, 2.0 ** -20, 0.05), (40, 2.0 ** -20, 2.0 ** -30), (-12, 2.0, 0.5),
    (-20, 500.0, 0.7), (-26, 2e4, 1.4), (-60, 2e4, 2.0 ** 34)])
def test_keys_beyond_fp16(dev, k_exp, q_size, scale, rows):
    """In some blocks or in all; scores come to a few units in every case."""
    hq, hkv, dim, page, n = 16, 2, 128, 16, 200
    tables, pages = _tables([n], page, 0, 1)
    q = (_rows(rows, hq, dim, torch.float32, 7).clamp(-3, 3) * q_size).to(torch.float16)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    for every in (1, 3):
        pool = O.Pool.random(pages, hkv, dim, page, seed=5)
        pool.scale["k"][:] = 2.0 ** (k_exp - 5)
        pool.scale["k"][::every] = 2.0 ** k_exp
        args = (q.to(dev), pool.to_device(dev), tables.to(dev), i32([n]))
        if rows == 1:
            got, offs = paged_decode_attention_kv8(*args, scale=scale), None
        else:
            offs = [n - rows]
            got = paged_attention_kv8(*args, i32([0, rows]), i32(offs), scale=scale)
        ref, mag, size = O.attend(q, pool, tables.tolist(), [n], [0, rows], offs, scale)
        assert 1.0 < size.max() < 100.0
        _check(got, ref, mag, size, torch.float16, n, dim, rows=rows == 64)
