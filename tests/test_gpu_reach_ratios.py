"""Windowed and prefix attention with many q heads to a kv head against float64 (bounds:
reach_oracle.check)."""

from __future__ import annotations

import pytest
import torch

import reach_oracle as O
from plastic_infer.kernel.paged_prefix import paged_prefix_attention
from plastic_infer.kernel.paged_window import paged_window_attention

pytestmark = pytest.mark.gpu

I32 = torch.int32


@pytest.mark.parametrize("rows", [None, [1, 3, 0, 2]])
@pytest.mark.parametrize("dtype", list(O.STEP))
@pytest.mark.parametrize("heads", [128, 129, 160, 256])
def test_ratio(dev, heads, dtype, rows):
    lens, plens, dim, page = [70, 33, 0, 20], [100], 64, 16
    pages = sum(-(-n // page) for n in lens + plens) + 2
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(heads)).tolist()
    k, v = O.pools(pages, 1, dim, page, dtype, heads)
    pt, bt = O.tables(plens, page, order), O.tables(lens, page, order)
    cu = None if rows is None else [sum(rows[:i]) for i in range(len(rows) + 1)]
    n = len(lens) if rows is None else sum(rows)
    q = torch.randn(n, heads, dim, generator=torch.Generator().manual_seed(1)).to(dtype)

    def on(x):
        return None if x is None else torch.tensor(x, dtype=I32, device=dev)

    qd, kd, vd, ptd, btd = (x.to(dev) for x in (q, k, v, pt, bt))
    got = paged_prefix_attention(qd, kd, vd, ptd, on(plens), btd, on(lens), cu_q=on(cu))
    O.check(got, *O.prefixed(q, k, v, pt, plens, bt, lens, None, cu), dtype, rows=True)
    got = paged_window_attention(qd, kd, vd, btd, on(lens), 40, 3, cu_q=on(cu))
    O.check(got, *O.windowed(q, k, v, bt, lens, 40, 3, cu), dtype, rows=True)
