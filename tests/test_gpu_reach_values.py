"""Windowed attention and attention behind shared prefixes where values and probabilities lie far apart:
probabilities far below the pools' least number, infinities before them, values that are not finite in places
that only some rows see, at each width of the kernels (bounds: reach_oracle.check)."""

from __future__ import annotations

import pytest
import torch

import reach_oracle as O
from plastic_infer.kernel.paged_prefix import paged_prefix_attention
from plastic_infer.kernel.paged_window import paged_window_attention

pytestmark = pytest.mark.gpu

I32 = torch.int32
DIMS = [64, 96, 128, 256]


def _ints(dev, x):
    return torch.tensor(x, dtype=I32, device=dev)


def _peaked(n, rows, dim, dtype, gap):
    """One sequence of n tokens whose token 0 scores `gap` above the others, with values of zero: what a row
    gets is the others' share, of large values of one sign."""
    g = torch.Generator().manual_seed(dim + rows)
    page = 16
    k = 0.05 * torch.randn(-(-n // page), 2, dim, page, generator=g)
    v = torch.randn(k.shape, generator=g).abs() * 2.0 ** 11
    k[:, :, 0] = 0
    k[0, :, 0, 0] = gap / 8
    v[0, :, :, 0] = 0
    q = 0.05 * torch.randn(rows, 8, dim, generator=g)
    q[:, :, 0] = 8
    return q.to(dtype), k.to(dtype), v.to(dtype), torch.arange(k.shape[0], dtype=I32)[None]


# exp(-gap) of the largest is 2^-12 to 2^-46; fp16's numbers end at 2^-24
@pytest.mark.parametrize("gap", [8.0, 14.0, 18.0, 22.0, 26.0, 32.0])
@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("rows", [1, 3, 70])
@pytest.mark.parametrize("dtype", list(O.STEP))
def test_small_probabilities_of_large_values(dev, dtype, rows, dim, gap):
    n = 1500
    q, k, v, bt = _peaked(n, rows, dim, dtype, gap)
    dq, dk, dv, dbt = (x.to(dev) for x in (q, k, v, bt))
    cu, offs, lens = [0, rows], [n - rows], [n]
    cut = 400                           # of the prefix; the rest is the sequence's own
    own = bt[:, cut // 16:].contiguous()
    for window, sinks in ((n, 0), (700, 1)):
        got = paged_window_attention(dq, dk, dv, dbt, _ints(dev, lens), window, sinks, _ints(dev, cu),
                                     _ints(dev, offs), 1.0)
        ref = O.windowed(q, k, v, bt, lens, window, sinks, cu, offs, 1.0)
        assert (ref[0] > 0).all()
        O.check(got, *ref, dtype, rows=rows > 1)
    got = paged_prefix_attention(dq, dk, dv, dbt, _ints(dev, [cut]), own.to(dev), _ints(dev, [n - cut]),
                                 None, _ints(dev, cu), _ints(dev, [n - cut - rows]), 1.0)
    ref = O.prefixed(q, k, v, bt, [cut], own, [n - cut], None, cu, [n - cut - rows], 1.0)
    O.check(got, *ref, dtype, rows=rows > 1)


@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("rows", [1, 3, 70])
@pytest.mark.parametrize("dtype", list(O.STEP))
def test_infinite_values_before_small_probabilities(dev, dtype, rows, dim):
    n, gap = 300, 26.0
    q, k, v, bt = _peaked(n, rows, dim, dtype, gap)
    v[2, 0, 3, 7] = float("inf")                     # all rows see it, and both of these
    v[12, 1, 5, 1], v[13, 1, 5, 2] = float("inf"), float("-inf")
    v[n // 16, :, 9, n % 16 - 1] = float("-inf")     # the last row alone
    cu, offs, lens = [0, rows], [n - rows], [n]
    got = paged_window_attention(q.to(dev), k.to(dev), v.to(dev), bt.to(dev), _ints(dev, lens), n, 0,
                                 _ints(dev, cu), _ints(dev, offs), 1.0)
    ref = O.windowed(q, k, v, bt, lens, n, 0, cu, offs, 1.0)
    assert ref[0][:, :4, 3].isposinf().all() and ref[0][:, 4:, 5].isnan().all()
    assert ref[0][-1, :, 9].isneginf().all() and ref[0][:-1, :, 9].isfinite().all()
    O.check(got, *ref, dtype, rows=rows > 1)


@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("rows", [3, 70, 150])
@pytest.mark.parametrize("dtype", list(O.STEP))
def test_odd_values_that_some_rows_see(dev, dtype, rows, dim):
    """A window's edges move over tokens whose values are infinities and NaN."""
    g = torch.Generator().manual_seed(dim)
    n, window, page = 400, 37, 16
    k, v = O.pools(25, 2, dim, page, dtype, dim)
    q = torch.randn(rows, 8, dim, generator=g).to(dtype)
    bt = torch.randperm(25, generator=g).to(I32)[None]
    first = n - rows
    for t, d, x in ((first - window + 1, 0, "inf"), (first - 2, 1, "nan"), (first, 2, "-inf"),
                    (first + 1, dim - 1, "nan"), (n - 1, 3, "inf"), (first - window, slice(None), "nan")):
        v[bt[0, t // page], 1, d, t % page] = float(x)
    cu, offs, lens = [0, rows], [first], [n]
    got = paged_window_attention(q.to(dev), k.to(dev), v.to(dev), bt.to(dev), _ints(dev, lens), window, 0,
                                 _ints(dev, cu), _ints(dev, offs))
    ref = O.windowed(q, k, v, bt, lens, window, 0, cu, offs)
    assert ref[0][:, :4].isfinite().all() and not ref[0][:, 4:].isfinite().all()
    O.check(got, *ref, dtype, rows=True)


# pages of the pool's and not the pool's, ragged rows, more heads to a kv head than an item's rows hold
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [144, 192, 256])
def test_wide_heads_of_many_rows(dev, dtype, dim):
    g = torch.Generator().manual_seed(dim)
    rows, lens, window, sinks, page = [90, 0, 130, 1], [200, 40, 500, 1], 75, 20, 32
    order = torch.randperm(40, generator=g).tolist()
    k, v = O.pools(40, 2, dim, page, dtype, 5)
    q = torch.randn(sum(rows), 6, dim, generator=g).to(dtype)
    bt = O.tables(lens, page, order)
    bt[2, 11] = -1
    cu = [sum(rows[:i]) for i in range(5)]
    args = [x.to(dev) for x in (q, k, v)]
    got = paged_window_attention(*args, bt.to(dev), _ints(dev, lens), window, sinks, _ints(dev, cu))
    O.check(got, *O.windowed(q, k, v, bt, lens, window, sinks, cu), dtype, rows=True)
    pt = O.tables([150], page, order)
    offs = [lens[b] - rows[b] for b in range(4)]
    got = paged_prefix_attention(*args, pt.to(dev), _ints(dev, [150]), bt.to(dev), _ints(dev, lens), None,
                                 _ints(dev, cu), _ints(dev, offs))
    O.check(got, *O.prefixed(q, k, v, pt, [150], bt, lens, None, cu, offs), dtype, rows=True)
