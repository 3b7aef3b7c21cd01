"""Rows whose causal limit lies beyond 2^30 tokens. Bounds: those of test_gpu_kv8_attention."""

from __future__ import annotations

import math

import pytest
import torch

import kv8_oracle as O
from plastic_infer.kernel.paged_kv8 import paged_attention_kv8
from test_gpu_kv8_attention import _check, _rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [3, 64])
def test_offsets_beyond_2_to_30(dev, rows, dtype):
    """A context of more than 2^30 tokens, all but the last 90 in one page that every slot names, with
    scores and values of zero; each row sees the last ones up to its own limit. (The sums of the others
    are whole numbers below 2^24 to each lane, and weigh 2^30 e^-36 at most.)"""
    hq, hkv, dim, page, far = 16, 2, 16, 4096, 2 ** 30
    tail, n = 90, 2 ** 30 + 90
    pool = O.Pool.random(2, hkv, dim, page, seed=3)
    pool.codes["k"][0] = 0.0
    pool.codes["v"][0] = 0.0
    pool.codes["k"][1, :, :, 0] = 256.0
    pool.scale["k"][1] = 2.0 ** -6             # 4 in the first element, random up to 6 in the others
    table = torch.zeros(1, far // page + 1, dtype=torch.int32, device=dev)
    table[0, -1] = 1
    q = _rows(rows, hq, dim, dtype, 2) / 16
    q[..., 0] = 40.0                            # a score of 40 and a little
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    off = n - rows - 7
    got = paged_attention_kv8(q.to(dev), pool.to_device(dev), table, i32([n]), i32([0, rows]),
                              i32([off]))
    ref, mag, size = O.attend(q, pool, [[1]], [tail], [0, rows], [off - far], 1 / math.sqrt(dim))
    _check(got, ref, mag, size, dtype, 4096, dim, rows=True)
