"""Attention over the 8-bit pool against float64 over the pool's own values.

Bound of an element (sums over a row's n keys, p its probabilities, z its largest score's terms
scale |q| . |k|, all in float64):
  half a step of the result's type;
  scores: (D + 8) roundings of fp32 at most, 2^-23 each, of z, and as much again by exp2 and the
    reference point, which a probability takes as a relative error: 2 (D + 8) 2^-23 z;
  probabilities as two bf16 terms: 2^-16 of each (fp32 results: three terms, below 2^-23); calls
    with many rows round them once to q's 16-bit type: half a step of it, 2^-8 or 2^-11 of each;
  the sums over n keys: n roundings of 2^-23 of what is summed, for p v and for p.
All but the first times sum p |v|."""

from __future__ import annotations

import math

import pytest
import torch

import kv8_oracle as O
from plastic_infer.kernel.paged_kv8 import (
    KV8Pools, kv8_append, kv8_attention_workspace_bytes, kv8_gather, paged_attention_kv8,
    paged_decode_attention_kv8)
from plastic_infer.kernel.rotary import rope_params

pytestmark = pytest.mark.gpu

STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
LEAST = {torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -14, torch.float32: 2.0 ** -126}


def _check(got, ref, mag, size, dtype, keys, dim, rows=False):
    assert got.dtype == dtype and got.shape == ref.shape
    rel = 0.0 if dtype == torch.float32 else STEP[dtype] if rows else 2.0 ** -16
    rel = rel + 2.0 ** -22 + 2 * keys * 2.0 ** -23
    rel = rel + 2 * (dim + 8) * 2.0 ** -23 * size
    bound = STEP[dtype] * ref.abs().clamp_min(LEAST[dtype]) + rel * mag
    err = (got.double().cpu() - ref).abs()
    assert (err <= bound).all(), (err / bound).max().item()


def _tables(lens, page, pages_extra, seed):
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lens]
    total = sum(need) + pages_extra
    order = torch.randperm(total, generator=g).tolist()
    t = torch.full((len(lens), max(need + [1])), -1, dtype=torch.int32)
    for b, n in enumerate(need):
        t[b, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.int32)
    return t, total


def _rows(n, hq, dim, dtype, seed):
    return torch.randn(n, hq, dim, generator=torch.Generator().manual_seed(seed)).to(dtype)


DECODE = [  # lens, Hq, Hkv, D, P
    ([1], 4, 1, 128, 16),
    ([0, 3, 64, 65], 8, 2, 128, 16),
    ([200, 17, 1000], 32, 8, 128, 16),
    ([127, 128, 129], 7, 1, 64, 32),
    ([500], 5, 5, 64, 16),
    ([90, 31], 16, 1, 128, 64),
    ([70, 2], 40, 2, 96, 16),
    ([33], 34, 2, 80, 48),
    ([300, 40], 4, 2, 256, 16),
    ([50], 3, 1, 16, 16),
    ([100], 6, 2, 208, 32),
]


@pytest.mark.parametrize("dtype", list(STEP))
@pytest.mark.parametrize("case", DECODE, ids=lambda c: f"{c[0]}h{c[1]}/{c[2]}d{c[3]}p{c[4]}")
def test_decode(dev, case, dtype):
    lens, hq, hkv, dim, page = case
    tables, pages = _tables(lens, page, 2, sum(lens))
    pool = O.Pool.random(pages, hkv, dim, page, seed=dim + hq)
    q = _rows(len(lens), hq, dim, dtype, hq)
    got = paged_decode_attention_kv8(q.to(dev), pool.to_device(dev), tables.to(dev),
                                     torch.tensor(lens, dtype=torch.int32, device=dev))
    cu = list(range(len(lens) + 1))
    ref, mag, size = O.attend(q, pool, tables.tolist(), lens, cu, None, 1 / math.sqrt(dim))
    _check(got, ref, mag, size, dtype, max(lens), dim)
    for b, n in enumerate(lens):
        if n == 0:
            assert (got[b] == 0).all()


ROWS = [  # new rows, lens, offsets (None: no causal limit), Hq, Hkv, D, P
    ([4, 1, 0, 9], [64, 17, 5, 200], "end", 8, 2, 128, 16),
    ([70], [70], "end", 4, 1, 128, 16),
    ([33, 20], [40, 150], "end", 4, 4, 64, 32),
    ([3, 2], [10, 30], None, 6, 2, 96, 16),
    ([5, 5], [90, 20], [-3, 4], 20, 1, 64, 16),
    ([6], [100], [2000], 4, 2, 256, 16),
    ([3, 2, 0, 5, 1], [0, 192, 7, 0, 1], "end", 8, 2, 128, 16),
    ([2, 9], [0, 90], [4, -5], 40, 2, 256, 32),
    ([4, 4], [193, 0], "end", 8, 2, 128, 16),
    ([130, 65], [130, 400], "end", 16, 2, 128, 16),
]


@pytest.mark.parametrize("dtype", list(STEP))
@pytest.mark.parametrize("case", ROWS, ids=lambda c: f"{c[0]}of{c[1]}h{c[3]}/{c[4]}d{c[5]}p{c[6]}")
def test_rows(dev, case, dtype):
    new, lens, offs, hq, hkv, dim, page = case
    tables, pages = _tables(lens, page, 2, sum(lens) + 1)
    pool = O.Pool.random(pages, hkv, dim, page, seed=dim + hq + 1)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    offs = [n - m for n, m in zip(lens, new)] if offs == "end" else offs
    q = _rows(cu[-1] + 3, hq, dim, dtype, hq + 1)       # three rows behind the last sequence
    out = torch.full(q.shape, 5.0, dtype=dtype, device=dev)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    got = paged_attention_kv8(q.to(dev), pool.to_device(dev), tables.to(dev), i32(lens),
                              cu_q=i32(cu), q_pos_offsets=None if offs is None else i32(offs),
                              out=out)
    assert got.data_ptr() == out.data_ptr() and (out[cu[-1]:] == 5.0).all()
    ref, mag, size = O.attend(q[:cu[-1]], pool, tables.tolist(), lens, cu, offs,
                              1 / math.sqrt(dim))
    _check(got[:cu[-1]], ref, mag, size, dtype, max(lens), dim, rows=True)


MANY = [  # as ROWS, and the tables' width in tokens; a kv head's rows 64 a sequence
    ([70, 1, 33], [70, 64, 200], "end", 32, 8, 128, 16, 0),
    ([20, 0, 9], [500, 3, 130], "end", 96, 8, 96, 32, 0),
    ([40, 30], [90, 20], [-3, 4], 40, 2, 64, 16, 0),
    ([50], [45], None, 64, 64, 96, 48, 0),
    ([17], [400], [2000], 128, 1, 128, 64, 0),
    ([65, 40], [65, 300], "end", 128, 16, 64, 16, 600),
    ([9, 12, 1, 30, 0, 17, 8, 9, 10, 6, 5, 11, 7, 9, 9, 13, 8, 9, 12, 7],
     [9, 70, 33, 150, 8, 17, 128, 129, 40, 63, 64, 65, 80, 9, 100, 14, 20, 31, 12, 200], "end",
     128, 32, 128, 16, 2048),
    ([10, 12, 1, 30, 0, 17, 28, 19, 20, 6, 15, 21, 17, 19, 29, 13, 28, 19, 12, 17],
     [10, 70, 33, 150, 8, 17, 128, 129, 40, 63, 64, 65, 80, 19, 100, 14, 30, 31, 12, 200], "end",
     128, 32, 128, 16, 2048),
    ([70], [700], "end", 16, 2, 128, 16, 0),              # cut along the keys
    ([33, 40], [900, 10], "end", 16, 2, 64, 32, 8192),
    ([65, 2, 0], [300, 1000, 40], None, 16, 2, 96, 48, 1200),
    ([40], [600], [-20], 32, 4, 128, 16, 1600),
    ([70, 30], [70, 90], "end", 8, 1, 80, 16, 0),         # padded heads
    ([33, 40], [700, 50], "end", 16, 2, 112, 32, 0),
    ([70], [300], None, 16, 2, 48, 16, 0),
    ([18, 25], [18, 29], "end", 20, 2, 16, 48, 0),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", MANY, ids=lambda c: f"{sum(c[0])}of{max(c[1])}h{c[3]}/{c[4]}d{c[5]}w{c[7]}")
def test_many_rows(dev, case, dtype):
    new, lens, offs, hq, hkv, dim, page, width = case
    tables, pages = _tables(lens, page, 2, sum(lens))
    if width:
        tables = torch.nn.functional.pad(tables, (0, width // page - tables.shape[1]), value=-1)
    pool = O.Pool.random(pages, hkv, dim, page, seed=dim + hq + 2)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    offs = [n - m for n, m in zip(lens, new)] if offs == "end" else offs
    q = _rows(cu[-1] + 3, hq, dim, dtype, hq + 1)       # three rows behind the last sequence
    out = torch.full(q.shape, 5.0, dtype=dtype, device=dev)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    got = paged_attention_kv8(q.to(dev), pool.to_device(dev), tables.to(dev), i32(lens),
                              cu_q=i32(cu), q_pos_offsets=None if offs is None else i32(offs),
                              out=out)
    assert (out[cu[-1]:] == 5.0).all()
    ref, mag, size = O.attend(q[:cu[-1]], pool, tables.tolist(), lens, cu, offs,
                              1 / math.sqrt(dim))
    _check(got[:cu[-1]], ref, mag, size, dtype, max(lens), dim, rows=True)


def test_long_and_many(dev):
    """A long context (cut over all waves), and more sequences than one launch's tables hold:
    against the same values gathered, in fp32 (2^-8 for bf16 results, 2^-13 for what fp32 sums)."""
    dim, hkv, hq, page = 128, 2, 8, 16
    for lens in ([40001], [(7 * b) % 50 for b in range(1500)]):
        tables, pages = _tables(lens, page, 1, 3)
        g = torch.Generator(device=dev).manual_seed(len(lens))
        codes = torch.randn(2, pages, hkv, dim * page, generator=g, device=dev) * 60
        k8, v8 = (c.to(torch.float8_e4m3fn) for c in codes)
        pools = KV8Pools(k8.view(pages, hkv, dim // 16, page, 16), v8.view(pages, hkv, page // 4, dim, 4),
                         *(torch.full((pages, hkv, page // 16), 2.0 ** -6, device=dev) for _ in "kv"))
        q = _rows(len(lens), hq, dim, torch.bfloat16, 4).to(dev)
        lens_t = torch.tensor(lens, dtype=torch.int32, device=dev)
        got = paged_decode_attention_kv8(q, pools, tables.to(dev), lens_t)
        cu = torch.zeros(len(lens) + 1, dtype=torch.int64)
        cu[1:] = torch.tensor(lens).cumsum(0)
        k, v = kv8_gather(pools, tables.to(dev), cu.to(dev), max(lens), dtype=torch.float32)
        for b in range(0, len(lens), max(1, len(lens) // 60)):
            kk, vv = (x[cu[b]:cu[b + 1]].double().cpu() for x in (k, v))
            if lens[b] == 0:
                assert (got[b] == 0).all()
                continue
            s = torch.einsum("hgd,nhd->hgn", q[b].double().cpu().view(hkv, -1, dim), kk)
            p = torch.softmax(s / math.sqrt(dim), -1)
            ref = torch.einsum("hgn,nhd->hgd", p, vv).reshape(hq, dim)
            mag = torch.einsum("hgn,nhd->hgd", p, vv.abs()).reshape(hq, dim)
            assert ((got[b].double().cpu() - ref).abs() <= 2.0 ** -8 * ref.abs() + 2.0 ** -9 * mag).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(1, 4, 128, 0), (8, 96, 128, 0), (8, 96, 64, 0), (8, 96, 96, 0),
                                   (176, 1056, 128, 2048),
                                   (8, 96, 128, 2048), (8, 96, 64, 4096),
                                   (8, 96, 112, 0), (8, 96, 80, 2048), (8, 96, 48, 0)],
                         ids=lambda s: f"h{s[1]}/{s[0]}d{s[2]}w{s[3]}")
def test_what_a_row_may_not_see(dev, shape, dtype):
    """Stale codes behind a context (NaN among them), pages outside the pool, and NaN keys and values
    of tokens that a row's limit hides leave its result alone; where they are seen, they show."""
    (hkv, hq, dim, width), page = shape, 16
    lens, new = [37, 90], [5, 20]
    tables, pages = _tables(lens, page, 1, 7)
    if width:
        tables = torch.nn.functional.pad(tables, (0, width // page - tables.shape[1]), value=-1)
    clean = O.Pool.random(pages, hkv, dim, page, seed=3)
    dirty = O.Pool.random(pages, hkv, dim, page, seed=3)
    for b, n in enumerate(lens):     # past the context
        last = int(tables[b, (n - 1) // page])
        for x in "kv":
            clean.codes[x][last, :, n % page or page:] = 0.0
            dirty.codes[x][last, :, n % page or page:] = math.nan
    cu, offs, g = [0, 5, 25], [32, 70], hq // hkv   # g heads share the first kv head
    q = _rows(25, hq, dim, dtype, 1)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731

    def run(pool, t=tables):
        return paged_attention_kv8(q.to(dev), pool.to_device(dev), t.to(dev), i32(lens),
                                   cu_q=i32(cu), q_pos_offsets=i32(offs)).cpu()

    want = run(clean)
    assert torch.equal(run(dirty), want)
    # sequence 1, position 81: a NaN key, and a NaN value of two elements
    i, o = int(tables[1, 81 // page]), 81 % page
    for x in "kv":
        bad = O.Pool.random(pages, hkv, dim, page, seed=3)
        bad.codes[x][i, 0, o, [3, dim - 2]] = math.nan
        got = run(bad)
        sees = torch.zeros(25, dtype=torch.bool)
        sees[5 + 11:] = True
        assert torch.equal(got[~sees], want[~sees])
        if x == "k":
            assert torch.isnan(got[sees][:, :g]).all() and torch.isfinite(got[:, g:]).all()
        else:
            hit = torch.isnan(got[sees])
            assert hit[:, :g, [3, dim - 2]].all() and hit.sum() == 2 * g * sees.sum()
    # a page that is not there holds no keys
    t = tables.clone()
    t[1, 2] = pages + 9
    got = run(clean, t)
    ref, mag, size = O.attend(q, clean, t.tolist(), lens, cu, offs, 1 / math.sqrt(dim))
    _check(got, ref, mag, size, dtype, 90, dim, rows=True)
    t[0, :] = -1
    assert (run(clean, t)[:5] == 0).all()
    for value in (math.nan, math.inf):
        q[7, 2, 5] = value
        got = run(clean)
        assert torch.isnan(got[7, 2]).all() and torch.isfinite(got[6]).all()
        assert torch.isfinite(got[7, [0, 1, 3]]).all()
        q[7, 2, 5] = 0.0


@pytest.mark.parametrize("dim,width", [(64, 0), (128, 0), (80, 2048)])
def test_values_beyond_fp16(dev, dim, width):
    """Many rows of fp16: values that fp16 does not hold (65504 itself becomes 65536 in the pool) count
    as 65504 where they are seen and leave other rows alone; NaN stays NaN."""
    hkv, hq, page, lens = 4, 48, 16, [90]
    tables, pages = _tables(lens, page, 1, 9)
    if width:
        tables = torch.nn.functional.pad(tables, (0, width // page - tables.shape[1]), value=-1)
    q = _rows(60, hq, dim, torch.float16, 2)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    i, o = int(tables[0, 81 // page]), 81 % page

    def pool(big):
        p = O.Pool.random(pages, hkv, dim, page, seed=4)
        p.codes["v"][i, 0] /= 8      # exact in e4m3, and within fp16 at the scale
        p.codes["v"][i, 0] = O.e4m3(p.codes["v"][i, 0])
        p.scale["v"][i, 0, 0] = 256.0
        p.codes["v"][i, 0, o, 3], p.codes["v"][i, 0, o, dim - 2] = big, -big
        return p

    def run(p):
        return paged_attention_kv8(q.to(dev), p.to_device(dev), tables.to(dev), i32(lens),
                                   cu_q=i32([0, 60]), q_pos_offsets=i32([30])).cpu()

    sees = torch.arange(60) + 30 >= 81
    for big, held in ((256.0, 65504.0 / 256), (448.0, 65504.0 / 256)):
        got = run(pool(big))
        ref, mag, size = O.attend(q, pool(held), tables.tolist(), lens, [0, 60], [30],
                                  1 / math.sqrt(dim))
        assert torch.isfinite(got).all()
        _check(got, ref, mag, size, torch.float16, 90, dim, rows=True)
    bad = pool(256.0)
    bad.codes["v"][i, 0, o, 5] = math.nan
    hit = torch.isnan(run(bad))
    assert hit[sees][:, :hq // hkv, 5].all() and hit.sum() == sees.sum() * (hq // hkv)
    high = pool(256.0)
    high.codes["k"][i, 0, o], high.scale["k"][i, 0, 0] = 256.0, 256.0
    a, b = run(high), run(pool(256.0))
    assert torch.equal(a[(torch.arange(60) + 30) < (81 // page) * page],
                       b[(torch.arange(60) + 30) < (81 // page) * page])


def test_scales_far_apart(dev):
    """Blocks whose scales differ by 2^40, in either pool, and probabilities near one and near zero."""
    dim, page = 64, 16
    pool = O.Pool.random(6, 1, dim, page, seed=11)
    pool.scale["v"][:, 0, 0] = torch.exp2(torch.tensor([-30.0, 10, -8, 0, -20, -8])).double()
    pool.scale["k"][:, 0, 0] = torch.exp2(torch.tensor([-9.0, -40, -7, -7, -8, -11])).double()
    tables = torch.tensor([[0, 1, 2, 3, 4, 5]], dtype=torch.int32)
    for dtype in STEP:
        q = _rows(1, 4, dim, dtype, 2) * 3
        got = paged_decode_attention_kv8(q.to(dev), pool.to_device(dev), tables.to(dev),
                                         torch.tensor([90], dtype=torch.int32, device=dev))
        ref, mag, size = O.attend(q, pool, tables.tolist(), [90], [0, 1], None, 1 / math.sqrt(dim))
        if dtype == torch.float16:
            ref = ref.clamp(-65504, 65504)
            mag = mag.clamp(max=65504.0)
            got = got.clamp(-65504, 65504)
        _check(got, ref, mag, size, dtype, 90, dim)


def test_strides_scale_workspace_streams_and_graphs(dev):
    dim, hkv, hq, page = 128, 2, 8, 16
    lens = [300, 1, 77]
    tables, pages = _tables(lens, page, 1, 5)
    pools = O.Pool.random(pages, hkv, dim, page, seed=2).to_device(dev)
    wide = torch.randn(3, hq + 4, dim, generator=torch.Generator().manual_seed(1)).to(
        torch.bfloat16).to(dev)
    lens_t = torch.tensor(lens, dtype=torch.int32, device=dev)
    t = tables.to(dev)
    want = paged_decode_attention_kv8(wide[:, :hq].contiguous(), pools, t, lens_t, scale=0.05)
    assert torch.equal(paged_decode_attention_kv8(wide[:, :hq], pools, t, lens_t, scale=0.05), want)
    odd = torch.empty(3 * hq * dim + 1, dtype=torch.bfloat16, device=dev)[1:].view(3, hq, dim)
    odd.copy_(wide[:, :hq])
    assert torch.equal(paged_decode_attention_kv8(odd, pools, t, lens_t, scale=0.05), want)
    flip = paged_decode_attention_kv8(-wide[:, :hq], pools, t, lens_t, scale=-0.05)
    assert torch.equal(flip, want)
    row = torch.as_strided(wide, (1, hq, dim), (3, dim, 1))     # one row: its stride says nothing
    assert torch.equal(paged_decode_attention_kv8(row, pools, t[:1], lens_t[:1], scale=0.05),
                       paged_decode_attention_kv8(wide[:1, :hq], pools, t[:1], lens_t[:1], scale=0.05))
    wt = tables.repeat(1, 2).to(dev)[:, ::2]     # a strided table
    st = torch.stack([tables, tables], -1).flatten(1).to(dev)[:, ::2]
    assert wt.shape == st.shape
    assert torch.equal(paged_decode_attention_kv8(wide[:, :hq], pools, st, lens_t, scale=0.05), want)
    # a kept workspace of any content, and a small one
    ws = torch.full((kv8_attention_workspace_bytes(dim),), 0xff, dtype=torch.uint8, device=dev)
    for w in (ws, ws, ws[:100]):
        assert torch.equal(paged_decode_attention_kv8(wide[:, :hq], pools, t, lens_t, scale=0.05,
                                                      workspace=w), want)
    # two captured graphs that share a workspace, replayed in turn between eager calls
    out = torch.empty_like(want)
    two = torch.empty_like(want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        paged_decode_attention_kv8(wide[:, :hq], pools, t, lens_t, out=out, workspace=ws)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for o, s in ((out, 0.05), (two, 0.1)):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            paged_decode_attention_kv8(wide[:, :hq], pools, t, lens_t, scale=s, out=o, workspace=ws)
        graphs.append(graph)
    for i in range(4):
        wide.mul_(-0.9)
        lens_t.sub_(1).clamp_(min=0)
        for graph in graphs:
            graph.replay()
        a = paged_decode_attention_kv8(wide[:, :hq], pools, t, lens_t, scale=0.05)
        b = paged_decode_attention_kv8(wide[:, :hq], pools, t, lens_t, scale=0.1)
        torch.cuda.synchronize()
        assert torch.equal(out, a) and torch.equal(two, b), i


def test_more_sequences_than_a_launch_takes(dev):
    """1100 sequences of 0 to 3 rows, their pages shared by every fourth of them."""
    dim, hkv, hq, page, n = 64, 1, 4, 16, 1100
    new, lens = [b % 4 for b in range(n)], [b % 4 + (5 * b) % 40 for b in range(n)]
    tables = torch.tensor([[(3 * (b // 4) + i) % 50 for i in range(3)] for b in range(n)],
                          dtype=torch.int32)
    pool = O.Pool.random(50, hkv, dim, page, seed=8)
    cu = [0] + torch.tensor(new).cumsum(0).tolist()
    q = _rows(cu[-1], hq, dim, torch.bfloat16, 6)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    offs = [m - k for m, k in zip(lens, new)]
    got = paged_attention_kv8(q.to(dev), pool.to_device(dev), tables.to(dev), i32(lens), cu_q=i32(cu),
                              q_pos_offsets=i32(offs))
    pick = list(range(0, n, 37)) + [1022, 1023, 1024, 1025, n - 1]
    for b in pick:
        r = slice(cu[b], cu[b + 1])
        ref, mag, size = O.attend(q[r], pool, [tables[b].tolist()], [lens[b]], [0, new[b]], [offs[b]],
                                  1 / math.sqrt(dim))
        _check(got[r], ref, mag, size, torch.bfloat16, 43, dim)


def test_pools_beyond_32_bits(dev):
    """Pages whose bytes lie past 2^32: append, gather and all attention kernels as on a small pool."""
    dim, hkv, hq, page = 128, 8, 32, 16
    pages = 2 ** 32 // (dim * hkv * page) + 40
    far, near = (KV8Pools.allocate(n, hkv, dim, page, dev) for n in (pages, 40))
    tables = torch.arange(40, dtype=torch.int32, device=dev).view(2, 20)
    rope = rope_params(dim, device=dev)
    g = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn(500, h, dim, generator=g).to(torch.bfloat16).to(dev) for h in (hq, hkv, hkv))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    cu, lens = i32([0, 220, 500]), i32([220, 280])
    out = []
    for pools, t in ((far, tables + (pages - 40)), (near, tables)):
        r = kv8_append(q, k, v, pools, t, lens, cu, rope)
        out.append([r, *kv8_gather(pools, t, cu.long(), 280),
                    paged_attention_kv8(r, pools, t, lens, cu, i32([0, 0])),
                    paged_attention_kv8(r[:6], pools, t, lens, i32([0, 2, 6]), i32([218, 276])),
                    paged_decode_attention_kv8(r[:2], pools, t, lens)])
    for a, b in zip(*out):
        assert torch.equal(a, b) and a.abs().max() > 0


@pytest.mark.parametrize("rows", [4, 200])
def test_rows_captured_and_on_two_streams(dev, rows):
    """A captured call replayed with other contexts and rows between eager ones, and two calls on
    streams of their own at once, each with its workspace."""
    dim, hkv, hq, page, B = 128, 4, 16, 16, 2
    pool = O.Pool.random(2 * 30, hkv, dim, page, seed=6).to_device(dev)
    t = torch.randperm(60, generator=torch.Generator().manual_seed(1)).int().view(B, 30).to(dev)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    q = _rows(B * rows, hq, dim, torch.bfloat16, 3).to(dev)
    lens, cu, offs = i32([470, 300]), i32([0, rows, 2 * rows]), i32([470 - rows, 300 - rows])
    ws = [torch.empty(kv8_attention_workspace_bytes(dim), dtype=torch.uint8, device=dev)
          for _ in range(2)]

    def call(w=None, out=None):
        return paged_attention_kv8(q, pool, t, lens, cu, offs, out=out, workspace=w)

    out = call(ws[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(ws[0], out)
    for i in range(3):
        q.mul_(-1.1)
        lens.sub_(i32([3, 17]))
        offs.sub_(i32([3, 17]))
        cu[1] -= 1
        out.zero_()
        graph.replay()
        want = call()
        torch.cuda.synchronize()
        assert torch.equal(out, want), i
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s, w in zip(streams, ws):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append([call(w) for _ in range(4)])
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for y in got for x in y)


def test_append_then_attend(dev):
    """A prompt and five decode steps through the cache: rotate, append and attend, against float64
    over the values that the cache then holds."""
    hq, hkv, dim, page = 8, 2, 128, 16
    prompts = [30, 7]
    g = torch.Generator().manual_seed(12)
    rope = rope_params(dim, base=1e6, device=dev)
    pools = KV8Pools.allocate(8, hkv, dim, page, dev)
    tables = torch.tensor([[5, 1, 7, 0], [2, 6, 3, 4]], dtype=torch.int32, device=dev)
    lens = list(prompts)
    cu = torch.tensor([0, 30, 37], dtype=torch.int32, device=dev)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731

    def rows(n):
        return [torch.randn(n, h, dim, generator=g).to(torch.bfloat16).to(dev)
                for h in (hq, hkv, hkv)]

    def reference(q, cu_l, offs):
        pool = O.Pool.from_device(pools)
        return O.attend(q.cpu(), pool, tables.tolist(), lens, cu_l, offs, 1 / math.sqrt(dim))

    q, k, v = rows(37)
    q = kv8_append(q, k, v, pools, tables, i32(lens), cu_new=cu, rope=rope)
    got = paged_attention_kv8(q, pools, tables, i32(lens), cu_q=cu, q_pos_offsets=i32([0, 0]))
    _check(got, *reference(q, cu.tolist(), [0, 0]), torch.bfloat16, 30, dim, rows=True)
    for _ in range(5):
        lens = [n + 1 for n in lens]
        q, k, v = rows(2)
        q = kv8_append(q, k, v, pools, tables, i32(lens), rope=rope)
        got = paged_decode_attention_kv8(q, pools, tables, i32(lens))
        _check(got, *reference(q, [0, 1, 2], None), torch.bfloat16, max(lens), dim)


def test_refusals(dev):
    pools = KV8Pools.allocate(2, 2, 32, 16, dev)
    q = torch.zeros(2, 4, 32, device=dev)
    t = torch.zeros(2, 1, dtype=torch.int32, device=dev)
    n = torch.zeros(2, dtype=torch.int32, device=dev)
    bad = [dict(q=q[:, :3]), dict(q=q[..., :16]), dict(q=q.double()), dict(block_tables=t.long()),
           dict(kv_lens=n.long()), dict(kv_lens=n[:1]), dict(cu_q=n), dict(q=q[:1]),
           dict(q_pos_offsets=n[:1]), dict(q_pos_offsets=n.float()), dict(out=q.half()),
           dict(out=q[:1]), dict(q=q.clone().requires_grad_()),
           dict(pools=KV8Pools(pools.k, pools.v[:1], pools.k_scale, pools.v_scale)),
           dict(pools=KV8Pools.allocate(0, 2, 32, 16, dev)),
           dict(pools=KV8Pools(pools.k.view(torch.uint8), pools.v, pools.k_scale, pools.v_scale))]
    for kw in bad:
        args = dict(q=q, pools=pools, block_tables=t, kv_lens=n) | kw
        with pytest.raises(ValueError):
            paged_attention_kv8(**args)
    assert (paged_attention_kv8(q, pools, t, n) == 0).all()
    assert paged_attention_kv8(q[:0], pools, t[:0], n[:0]).shape == (0, 4, 32)
    assert (paged_decode_attention_kv8(q + 1, pools, t[:, :0], n + 9) == 0).all()
