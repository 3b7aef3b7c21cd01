"""Appends with the rotary positions applied, into float and 8-bit pools, and the 8-bit gather,
against the definitions in float64.

A rotated element is within 2^-22 factor (|a| + |b|) of the exact one before its rounding (the bound
of test_gpu_rotary.py). In the 8-bit pool it is then rounded to e4m3: half a step, 2^-4 of the value or
2^-10 of the scale. Values, scales and everything that is only copied are equal."""

from __future__ import annotations

import math

import pytest
import torch

import kv8_oracle as O
from plastic_infer.kernel.kv_append import kv_append
from plastic_infer.kernel.paged_kv import kv_scatter
from plastic_infer.kernel.paged_kv8 import KV8Pools, kv8_append, kv8_gather
from plastic_infer.kernel.rotary import RopeParams, rope_params, rotary_embed

pytestmark = pytest.mark.gpu

STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def _batch(new, ctx, page, seed, extra=2):
    """(tables, lens, cu, pages) for sequences with `new` rows behind `ctx` tokens."""
    g = torch.Generator().manual_seed(seed)
    lens = [n + c for n, c in zip(new, ctx)]
    need = [max(1, -(-n // page)) for n in lens]
    pages = sum(need) + extra
    order = torch.randperm(pages, generator=g).tolist()
    width = max(need) + 1
    tables = torch.full((len(new), width), -1, dtype=torch.int32)
    for b, n in enumerate(need):
        tables[b, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.int32)
    cu = torch.tensor([0] + list(torch.tensor(new).cumsum(0)), dtype=torch.int32)
    return tables, torch.tensor(lens, dtype=torch.int32), cu, pages


def _positions(new, ctx):
    return torch.cat([torch.arange(c, c + n) for n, c in zip(new, ctx)])


CASES = [  # new rows, context, Hq, Hkv, D, rotated, P
    ([1, 1, 1], [0, 15, 16], 4, 2, 128, 128, 16),
    ([1], [4095], 32, 8, 128, 128, 16),
    ([16, 33, 1, 7], [0, 5, 47, 9], 4, 4, 128, 64, 16),
    ([40, 0, 3], [10, 8, 31], 6, 2, 64, 64, 32),
    ([17, 2], [0, 62], 3, 3, 96, 48, 16),
    ([31], [1], 2, 1, 80, 20, 48),
    ([5, 64], [11, 32], 2, 2, 256, 256, 16),
    ([19], [3], 2, 1, 16, 16, 16),
]
FLOAT_CASES = CASES + [  # head sizes of float pools alone
    ([40, 17], [0, 30], 1, 2, 512, 512, 16),
    ([33, 3], [5, 0], 2, 1, 200, 130, 32),
    ([50, 1], [2, 9], 2, 2, 33, 6, 16),
    ([1, 1], [2, 31], 1, 3, 65, 65 - 1, 16),
]


@pytest.mark.parametrize("dtype", list(STEP))
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("case", FLOAT_CASES, ids=lambda c: f"{c[0]}+{c[1]}d{c[4]}r{c[5]}p{c[6]}")
def test_float_pools(dev, case, interleaved, dtype):
    """The pools of rotary_embed followed by kv_scatter, and nothing else written."""
    new, ctx, hq, hkv, dim, rd, page = case
    tables, lens, cu, pages = _batch(new, ctx, page, dim + page)
    n = sum(new)
    g = torch.Generator().manual_seed(n)
    q, k, v = (torch.randn(n, h, dim, generator=g).to(dtype).to(dev) for h in (hq, hkv, hkv))
    kp, vp = (torch.randn(pages, hkv, dim, page, generator=g).to(dtype).to(dev) for _ in "kv")
    rope = rope_params(dim, rotary_dim=rd, interleaved=interleaved, device=dev)
    pos = _positions(new, ctx)
    wk, wv = kp.clone(), vp.clone()
    qr, kr = rotary_embed(q, k, pos.to(dev), rope)
    rows = torch.cat([tables[b, torch.arange(c, c + m) // page].long() * page
                      + torch.arange(c, c + m) % page for b, (m, c) in enumerate(zip(new, ctx))])
    kv_scatter(kr, v, wk, wv, rows.to(dev))
    got = kv_append(q, k, v, kp, vp, tables.to(dev), lens.to(dev),
                    cu_new=None if set(new) == {1} else cu.to(dev), rope=rope)
    assert torch.equal(got, qr)
    assert torch.equal(kp, wk) and torch.equal(vp, wv)


@pytest.mark.parametrize("page", [7, 24, 1])
def test_float_pools_of_other_page_sizes(dev, page):
    new, ctx = [20, 1, 33], [4, 9, 0]
    tables, lens, cu, pages = _batch(new, ctx, page, page)
    g = torch.Generator().manual_seed(page)
    k, v = (torch.randn(54, 2, 6, generator=g).to(dev) for _ in "kv")
    kp, vp = (torch.randn(pages, 2, 6, page, generator=g).to(dev) for _ in "kv")
    wk, wv = kp.clone(), vp.clone()
    rows = torch.cat([tables[b, torch.arange(c, c + m) // page].long() * page
                      + torch.arange(c, c + m) % page for b, (m, c) in enumerate(zip(new, ctx))])
    kv_scatter(k, v, wk, wv, rows.to(dev))
    assert kv_append(None, k, v, kp, vp, tables.to(dev), lens.to(dev), cu_new=cu.to(dev)) is None
    assert torch.equal(kp, wk) and torch.equal(vp, wv)


def _append8_oracle(pool, tables, new, ctx, k, v, pos, rope, interleaved):
    """The pool after the append, and the bound of each new K value's error before rounding."""
    if rope is None:
        turned, size, c = k.double(), torch.zeros(k.shape, dtype=torch.float64), 1.0
    else:
        turned, size = O.turn(k, pos, rope.turns.cpu(), rope.factor, interleaved)
        c = torch.tensor(math.sqrt(2.0) * rope.factor, dtype=torch.float32)
    fin = lambda x: torch.where(torch.isfinite(x), x, torch.zeros_like(x)).float().abs().amax(-1)  # noqa: E731
    bk, bv = (fin(k) * c).double(), fin(v).double()
    row = 0
    for b, (n, start) in enumerate(zip(new, ctx)):
        if n:
            pool.append("k", turned[row:row + n], bk[row:row + n], tables[b], start)
            pool.append("v", v[row:row + n].double(), bv[row:row + n], tables[b], start)
        row += n
    return turned, size


@pytest.mark.parametrize("dtype", list(STEP))
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{c[0]}+{c[1]}d{c[4]}r{c[5]}p{c[6]}")
def test_8bit_pools(dev, case, interleaved, dtype):
    new, ctx, hq, hkv, dim, rd, page = case
    tables, lens, cu, pages = _batch(new, ctx, page, dim + page + 1)
    n = sum(new)
    g = torch.Generator().manual_seed(n + 1)
    q, k, v = (torch.randn(n, h, dim, generator=g).to(dtype) for h in (hq, hkv, hkv))
    k[:, 0] *= 3e-4          # a head whose scale stays that of earlier tokens
    v[:, -1] *= 40.0         # one whose scale grows
    rope = rope_params(dim, rotary_dim=rd, interleaved=interleaved, device=dev,
                       scaling={"type": "yarn", "factor": 4.0, "original_length": 64}
                       if rd > 20 else None)
    pool = O.Pool.random(pages, hkv, dim, page, seed=n)
    pools = pool.to_device(dev)
    pos = _positions(new, ctx)
    got_q = kv8_append(q.to(dev), k.to(dev), v.to(dev), pools, tables.to(dev), lens.to(dev),
                       cu_new=None if set(new) == {1} else cu.to(dev), rope=rope)
    assert torch.equal(got_q, rotary_embed(q.to(dev), None, pos.to(dev), rope)[0])
    turned, size = _append8_oracle(pool, tables, new, ctx, k, v, pos, rope, interleaved)
    got = O.Pool.from_device(pools)
    for x in "kv":
        assert torch.equal(got.scale[x], pool.scale[x])
    assert torch.equal(got.codes["v"], pool.codes["v"])
    # K: equal but where the rotation's fp32 error crosses the middle of two codes
    gv, pv = got.values("k"), pool.values("k")
    differ = 0
    row = 0
    fresh = torch.zeros(pages, hkv, page, dtype=torch.bool)
    for b, (m, start) in enumerate(zip(new, ctx)):
        for p in range(start, start + m):
            i, o = int(tables[b, p // page]), p % page
            fresh[i, :, o] = True
            s = pool.scale["k"][i, :, o // 16][:, None]
            x = turned[row]
            bound = torch.maximum(x.abs() * 2.0 ** -4, s * 2.0 ** -10) + 2.0 ** -22 * size[row]
            assert ((gv[i, :, o] - x).abs() <= bound * (1 + 2.0 ** -20)).all()
            differ += int((gv[i, :, o] != pv[i, :, o]).sum())
            row += 1
    assert differ <= 1 + n * hkv * dim * 2.0 ** -12
    keep = ~fresh[..., None].expand_as(gv)
    assert torch.equal(gv[keep], pv[keep])
    # the same call again changes nothing
    before = [t.clone() for t in (pools.k.view(torch.uint8), pools.v.view(torch.uint8),
                                  pools.k_scale, pools.v_scale)]
    kv8_append(q.to(dev), k.to(dev), v.to(dev), pools, tables.to(dev), lens.to(dev),
               cu_new=cu.to(dev), rope=rope)
    for a, b in zip(before, (pools.k.view(torch.uint8), pools.v.view(torch.uint8), pools.k_scale,
                             pools.v_scale)):
        assert torch.equal(a, b)


def test_8bit_token_by_token(dev):
    """A context appended one token at a time holds what one append of all of it holds, up to the
    codes that fell below a scale's normal range as it grew."""
    g = torch.Generator().manual_seed(4)
    n, h, d = 37, 2, 64
    size = torch.exp2(torch.randint(-6, 7, (n, 1, 1), generator=g).float())
    k, v = (torch.randn(n, h, d, generator=g) * size for _ in "kv")
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32, device=dev)
    rope = rope_params(d, device=dev)
    one, many = KV8Pools.allocate(3, h, d, 16, dev), KV8Pools.allocate(3, h, d, 16, dev)
    kv8_append(None, k.to(dev), v.to(dev), one, table, torch.tensor([n], dtype=torch.int32, device=dev),
               cu_new=torch.tensor([0, n], dtype=torch.int32, device=dev), rope=rope)
    for t in range(n):
        kv8_append(None, k[t:t + 1].to(dev), v[t:t + 1].to(dev), many, table,
                   torch.tensor([t + 1], dtype=torch.int32, device=dev), rope=rope)
    a, b = O.Pool.from_device(one), O.Pool.from_device(many)
    for x in "kv":
        assert torch.equal(a.scale[x], b.scale[x])
        off = (a.values(x) - b.values(x)).abs()
        # two roundings to steps of 2^-9 of the scale or finer, where the value is below 2^-6 of it
        s = a.scale[x].repeat_interleave(16, -1)[..., None]
        assert (off <= torch.where(a.values(x).abs() <= s * 2.0 ** -6, s * 2.0 ** -9, 0.0 * s)).all()


def test_8bit_special_values(dev):
    """NaN and infinities become NaN and leave the scale to the rest; zeros; the type's extremes."""
    k = torch.zeros(4, 1, 16)
    k[0, 0, 3], k[0, 0, 4], k[0, 0, 5] = math.nan, math.inf, 2.0
    k[1, 0, :] = -3.0
    k[3, 0, 0], k[3, 0, 1], k[3, 0, 2] = 3.0e38, -1e-40, 3.4028234e38   # over 464 * 2^119: NaN
    v = torch.zeros(4, 1, 16)
    v[2, 0, 7] = -448.0
    pools = KV8Pools.allocate(1, 1, 16, 16, dev)
    table = torch.zeros(1, 1, dtype=torch.int32, device=dev)
    cu = torch.tensor([0, 2], dtype=torch.int32, device=dev)
    kv8_append(None, k[:2].to(dev), v[2:].to(dev), pools, table,
               torch.tensor([2], dtype=torch.int32, device=dev), cu_new=cu)
    got = O.Pool.from_device(pools)
    x = got.values("k")[0, 0]
    assert got.scale["k"][0, 0, 0] == 2.0 ** -7 and torch.isnan(x[0, 3:5]).all() and x[0, 5] == 2.0
    assert (x[1] == -3.0).all() and (x[0, :3] == 0).all()
    assert got.scale["v"][0, 0, 0] == 1.0 and got.values("v")[0, 0, 0, 7] == -448.0
    kv8_append(None, k[3:].to(dev), v[:1].to(dev), pools, table,
               torch.tensor([3], dtype=torch.int32, device=dev))
    x = O.Pool.from_device(pools).values("k")[0, 0]
    assert x[2, 0] == 448.0 * 2.0 ** 119 and x[2, 1] == 0 and torch.isnan(x[2, 2])
    assert torch.isnan(x[0, 3:5]).all() and (x[1] == 0).all()
    # a block of zeros: the least scale, and the next token's takes over
    pools = KV8Pools.allocate(1, 1, 16, 16, dev)
    kv8_append(None, k[2:3].to(dev), v[:1].to(dev), pools, table,
               torch.tensor([1], dtype=torch.int32, device=dev))
    assert pools.k_scale.item() == 2.0 ** -100
    kv8_append(None, k[1:2].to(dev), v[:1].to(dev), pools, table,
               torch.tensor([2], dtype=torch.int32, device=dev))
    x = O.Pool.from_device(pools).values("k")[0, 0]
    assert (x[0] == 0).all() and (x[1] == -3.0).all()


@pytest.mark.parametrize("kv8", [False, True])
def test_tokens_without_a_slot(dev, kv8):
    """Page ids outside the pool, positions past the table or before the context, lengths of zero,
    rows behind the last sequence: nothing of theirs is written, q of every sequence is."""
    g = torch.Generator().manual_seed(6)
    k, v, q = (torch.randn(30, 2, 32, generator=g).to(dev) for _ in range(3))
    tables = torch.tensor([[1, 7], [-1, 2], [3, 0], [4, 4]], dtype=torch.int32, device=dev)
    lens = torch.tensor([18, 20, 40, 2], dtype=torch.int32, device=dev)
    cu = torch.tensor([0, 6, 12, 22, 27], dtype=torch.int32, device=dev)   # rows 27..29: no one's
    rope = rope_params(32, device=dev)
    if kv8:
        pools = O.Pool.random(5, 2, 32, 16, seed=1).to_device(dev)
        before = O.Pool.from_device(pools)
        out = kv8_append(q, k, v, pools, tables, lens, cu_new=cu, rope=rope)
        after = O.Pool.from_device(pools)
        # codes: those behind a block's last new token stay, though its scale is a new one
        old, now = ([p.codes[x] for x in "kv"] for p in (before, after))
    else:
        kp, vp = (torch.randn(5, 2, 32, 16, generator=g).to(dev) for _ in "kv")
        old = [t.transpose(2, 3).double().cpu().clone() for t in (kp, vp)]
        out = kv_append(q, k, v, kp, vp, tables, lens, cu_new=cu, rope=rope)
        now = [t.transpose(2, 3).double().cpu() for t in (kp, vp)]
    # sequence 0: positions 12..17, page 1 takes 12..15, page 7 is none; 1: 14, 15 none, 16..19 page
    # 2; 2: 30, 31 page 0, 32.. past the table; 3: -3..-1 before the context, 0, 1 page 4
    want = torch.zeros(5, 16, dtype=torch.bool)
    want[1, 12:], want[2, :4], want[0, 14:], want[4, :2] = True, True, True, True
    for a, b in zip(old, now):
        moved = (a != b).any(dim=(1, 3))
        assert torch.equal(moved, want) if not kv8 else not (moved & ~want)[[3]].any()
        if kv8:   # earlier tokens of a touched block may be rounded to a new scale
            assert (moved | ~want).all() and not moved[3].any() and not moved[2, 4:].any()
            assert not moved[4, 2:].any()
    pos = torch.cat([torch.arange(12, 18), torch.arange(14, 20), torch.arange(30, 40),
                     torch.arange(-3, 2)]).to(dev)
    assert torch.equal(out[:27], rotary_embed(q[:27], None, pos, rope)[0])


@pytest.mark.parametrize("dtype", list(STEP))
@pytest.mark.parametrize("dim,page,lens", [(128, 16, [1, 300, 0, 17]), (64, 32, [33, 64]),
                                           (96, 48, [100]), (256, 16, [5]), (16, 16, [16])])
def test_gather(dev, dtype, dim, page, lens):
    tables, _, cu, pages = _batch(lens, [0] * len(lens), page, dim)
    tables[0, 0] = pages + 3                       # a page outside the pool reads as zeros
    pool = O.Pool.random(pages, 3, dim, page, seed=dim)
    k, v = kv8_gather(pool.to_device(dev), tables.to(dev), cu.to(dev), max(lens), dtype=dtype)
    for x, got in (("k", k), ("v", v)):
        want = torch.cat([pool.context(x, tables[b], n)[0] for b, n in enumerate(lens)])
        assert got.dtype == dtype and torch.equal(got.cpu(), want.to(dtype))
    room = torch.full((sum(lens) + 4, 3, dim), 7.0, dtype=dtype, device=dev)
    kv8_gather(pool.to_device(dev), tables.to(dev), cu.to(dev), max(lens), out=(room, room.clone()))
    assert torch.equal(room[:-4], k) and (room[-4:] == 7.0).all()


def test_strides_streams_and_graphs(dev):
    """Views of one projection, a call on a side stream, and a captured step replayed with other
    inputs: the same pools as eager calls on contiguous copies."""
    g = torch.Generator().manual_seed(9)
    B, hq, hkv, d = 5, 4, 2, 64
    wide = torch.randn(B, hq + 2 * hkv, d, generator=g).to(torch.bfloat16).to(dev)
    q, k, v = wide[:, :hq], wide[:, hq:hq + hkv], wide[:, hq + hkv:]
    tables = torch.arange(B * 3, dtype=torch.int32, device=dev).view(B, 3)
    lens = torch.tensor([1, 16, 17, 30, 47], dtype=torch.int32, device=dev)
    rope = rope_params(d, device=dev)
    pools, same = (KV8Pools.allocate(B * 3, hkv, d, 16, dev) for _ in range(2))
    want = kv8_append(q.contiguous(), k.contiguous(), v.contiguous(), same, tables, lens, rope=rope)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = kv8_append(q, k, v, pools, tables, lens, rope=rope)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = kv8_append(q, k, v, pools, tables, lens, rope=rope)
    for i in range(3):
        wide.mul_(-1.5)
        lens.add_(1).clamp_(max=48)
        graph.replay()
        want = kv8_append(q, k, v, same, tables, lens, rope=rope)
        torch.cuda.synchronize()
        assert torch.equal(got, want), i
        for a, b in ((pools.k, same.k), (pools.v, same.v)):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), i
        assert torch.equal(pools.k_scale, same.k_scale) and torch.equal(pools.v_scale, same.v_scale)


def test_a_negative_factor_turns_the_negative(dev):
    """k rotated times -1.5 is -k rotated times 1.5: the same codes and scales."""
    g = torch.Generator().manual_seed(5)
    k, v = (torch.randn(20, 2, 64, generator=g).to(torch.bfloat16).to(dev) for _ in "kv")
    tables, lens, cu, pages = _batch([17, 3], [0, 14], 16, 3)
    turns = rope_params(64, device=dev).turns
    a, b = (KV8Pools.allocate(pages, 2, 64, 16, dev) for _ in range(2))
    for pools, x, f in ((a, k, -1.5), (b, -k, 1.5)):
        kv8_append(None, x, v, pools, tables.to(dev), lens.to(dev), cu.to(dev), RopeParams(turns, f))
    assert (a.k.float().abs().amax() > 100) and torch.equal(a.k_scale, b.k_scale)
    assert torch.equal(a.k.float(), b.k.float())     # zeros of either sign are equal


def test_rows_behind_the_last_sequence(dev):
    """A padded batch: rows of no sequence go nowhere, whichever pool."""
    g = torch.Generator().manual_seed(4)
    q, k, v = (torch.randn(40, h, 64, generator=g).to(torch.bfloat16).to(dev) for h in (4, 2, 2))
    tables, lens, cu, pages = _batch([17, 3], [0, 14], 16, 3)
    args = (tables.to(dev), lens.to(dev), cu.to(dev), rope_params(64, device=dev))
    a, b = (KV8Pools.allocate(pages, 2, 64, 16, dev) for _ in range(2))
    got, want = kv8_append(q, k, v, a, *args), kv8_append(q[:20], k[:20], v[:20], b, *args)
    assert torch.equal(got[:20], want)
    assert torch.equal(a.k.view(torch.uint8), b.k.view(torch.uint8))
    assert torch.equal(a.v.view(torch.uint8), b.v.view(torch.uint8))
    pools = [torch.zeros(pages, 2, 64, 16, dtype=torch.bfloat16, device=dev) for _ in range(4)]
    got, want = kv_append(q, k, v, *pools[:2], *args), kv_append(q[:20], k[:20], v[:20], *pools[2:], *args)
    assert torch.equal(got[:20], want)
    assert torch.equal(pools[0], pools[2]) and torch.equal(pools[1], pools[3])


def test_refusals(dev):
    x = torch.zeros(2, 2, 32, device=dev)
    i = torch.zeros(2, dtype=torch.int32, device=dev)
    t = torch.zeros(2, 1, dtype=torch.int32, device=dev)
    kp = torch.zeros(2, 2, 32, 16, device=dev)
    pools = KV8Pools.allocate(2, 2, 32, 16, dev)
    rope = rope_params(64, device=dev)
    bad = [dict(k=x[:, :1]), dict(v=x[..., :16]), dict(q=x[:1]), dict(q=x.half()),
           dict(context_lens=i.long()), dict(context_lens=i[:1]), dict(block_tables=t.long()),
           dict(cu_new=i), dict(rope=rope), dict(k=x[:1], v=x[:1], q=None),
           dict(k=x.clone().requires_grad_())]
    for kw in bad:
        args = dict(q=x, k=x, v=x, block_tables=t, context_lens=i) | kw
        with pytest.raises(ValueError):
            kv_append(k_pages=kp, v_pages=kp.clone(), **args)
        with pytest.raises(ValueError):
            kv8_append(pools=pools, **args)
    with pytest.raises(ValueError):
        kv_append(x.half(), x.half(), x.half(), kp, kp, t, i)
    with pytest.raises(ValueError):
        kv8_append(x, x, x, KV8Pools(pools.k, pools.v, pools.k_scale.half(), pools.v_scale), t, i)
    with pytest.raises(ValueError):
        kv8_gather(pools, t, i, 4)
    with pytest.raises(ValueError):
        kv8_gather(pools, t, torch.zeros(3, dtype=torch.int64, device=dev), 4, dtype=torch.int32)
