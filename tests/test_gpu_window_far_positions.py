"""Windowed attention of rows at positions up to 2^31 and beyond, against float64 (bounds:
reach_oracle.check)."""

from __future__ import annotations

import pytest
import torch

import reach_oracle as O
from plastic_infer.kernel.paged_window import paged_window_attention

pytestmark = pytest.mark.gpu

I32 = torch.int32
TOP = 2 ** 31 - 1


@pytest.mark.parametrize("sinks", [0, 70])
@pytest.mark.parametrize("rows", [1, 2, 40])       # items of one row's, ragged ones, tiles
@pytest.mark.parametrize("dtype", list(O.STEP))
def test_far_positions(dev, dtype, rows, sinks):
    B, n, heads, dim, page, window = 66, 4500, 8, 16, 16, 4096
    order = torch.randperm(n // page + 2, generator=torch.Generator().manual_seed(rows)).tolist()
    k, v = O.pools(len(order), heads, dim, page, dtype, 3)
    bt = O.tables([n], page, order).expand(B, -1).contiguous()     # all of the same pages
    near = [n - rows, 100, n + 200, 4095]
    offs = [(TOP - (b % 64) if b % 3 else 0x7ffff000 - 4096 + 40 * b) if b % 6 else near[b // 6 % 4]
            for b in range(B)]
    cu = [rows * b for b in range(B + 1)]
    q = torch.randn(B * rows, heads, dim, generator=torch.Generator().manual_seed(4)).to(dtype)
    qd, kd, vd, btd = (x.to(dev) for x in (q, k, v, bt))
    cd, od, ld = (torch.tensor(x, dtype=I32, device=dev) for x in (cu, offs, [n] * B))
    got = paged_window_attention(qd, kd, vd, btd, ld, window, sinks, cu_q=cd, q_pos_offsets=od).cpu()
    for b in [x for x in range(B) if x % 6 == 0][:5] + [1, 2, 3, 9, 62, 65]:
        inner = slice(cu[b], cu[b + 1])
        ref = O.windowed(q[inner], k, v, bt[b:b + 1], [n], window, sinks, [0, rows], [offs[b]])
        assert offs[b] < 10 ** 9 or (ref[0] == 0).all() == (sinks == 0)
        O.check(got[inner], *ref, dtype, rows=True)
    far = [b for b in range(B) if offs[b] > 10 ** 9]      # rows that see the sinks alone, or nothing
    if sinks == 0:
        assert all((got[cu[b]:cu[b + 1]] == 0).all() for b in far)
    else:
        assert all((got[cu[b]:cu[b + 1]] != 0).any() for b in far)
