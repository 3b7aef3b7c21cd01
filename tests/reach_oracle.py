"""Windowed attention and attention behind a shared prefix in float64, row by row, and the bound of what a
kernel's result may be off by."""

from __future__ import annotations

import math

import torch

STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
LEAST = {torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -14, torch.float32: 2.0 ** -126}


def tables(lens, page, order, width=0):
    """Block tables (page ids taken from the list `order`) of sequences of these lengths, -1 elsewhere."""
    need = [-(-n // page) for n in lens]
    t = torch.full((len(lens), max(need + [1, width])), -1, dtype=torch.int32)
    for b, n in enumerate(need):
        t[b, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.int32)
    return t


def pools(pages, heads, dim, page, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    k, v = (torch.randn(pages, heads, dim, page, generator=g).to(dtype) for _ in range(2))
    return k, v


def tokens(k, v, table, n):
    """K and V [n, heads, dim] in fp64 of a table's first n tokens, and which of them are there."""
    P, ids = k.shape[3], table.tolist()
    j = torch.arange(n)
    page = torch.tensor([ids[x] for x in (j // P).tolist()], dtype=torch.int64)
    there = (page >= 0) & (page < k.shape[0])
    page = torch.where(there, page, torch.zeros_like(page))
    return k[page, :, :, j % P].double(), v[page, :, :, j % P].double(), there


def attend(q, k, v, seen, scale=None):
    """q [Hq, D] over k, v [n, Hkv, D] with seen [n]: (result, sum p |v|, the largest score's terms)."""
    Hq, D = q.shape
    k, v = k[seen], v[seen]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    out, mag, size = torch.zeros(Hq, D).double(), torch.zeros(Hq, D).double(), 0.0
    if k.shape[0]:
        G = Hq // k.shape[1]
        k, v = (x.repeat_interleave(G, dim=1) for x in (k, v))
        q = q.double()
        s = torch.einsum("hd,nhd->hn", q, k) * scale
        size = (torch.einsum("hd,nhd->hn", q.abs(), k.abs()).nan_to_num(0, 0, 0).max() *
                abs(scale)).item()
        p = torch.softmax(s, dim=-1)
        out = torch.einsum("hn,nhd->hd", p, v)
        mag = torch.einsum("hn,nhd->hd", p, v.abs())
    return out, mag, size


def windowed(q, k, v, bt, lens, window, sinks, cu=None, offs=None, scale=None):
    """(result, magnitudes, sizes [rows, 1, 1], largest number of keys); rows of no sequence are NaN."""
    out, mag = (torch.full(q.shape, math.nan).double() for _ in range(2))
    size, most = torch.zeros(q.shape[0], 1, 1).double(), 0
    cu = list(range(len(lens) + 1)) if cu is None else cu
    for b, n in enumerate(lens):
        n = min(max(n, 0), bt.shape[1] * k.shape[3])
        kb, vb, there = tokens(k, v, bt[b], n)
        j = torch.arange(n)
        for s, r in enumerate(range(cu[b], min(cu[b + 1], q.shape[0]))):
            p = (n - (cu[b + 1] - cu[b]) if offs is None else offs[b]) + s
            seen = there & (j <= p) & ((p - j < window) | (j < sinks))
            out[r], mag[r], size[r] = attend(q[r], kb, vb, seen, scale)
            most = max(most, int(seen.sum()))
    return out, mag, size, most


def prefixed(q, k, v, pt, plens, bt, lens, cu_seqs=None, cu=None, offs=None, scale=None):
    out, mag = (torch.full(q.shape, math.nan).double() for _ in range(2))
    size, most = torch.zeros(q.shape[0], 1, 1).double(), 0
    cu = list(range(len(lens) + 1)) if cu is None else cu
    cu_seqs = [0, len(lens)] if cu_seqs is None else cu_seqs
    for b, n in enumerate(lens):
        n = min(max(n, 0), bt.shape[1] * k.shape[3])
        kb, vb, there = tokens(k, v, bt[b], n)
        group = [g for g in range(len(plens)) if cu_seqs[g] <= b < cu_seqs[g + 1]]
        shared = 0
        if group:
            shared = min(max(plens[group[0]], 0), pt.shape[1] * k.shape[3])
            kp, vp, tp = tokens(k, v, pt[group[0]], shared)
            kb, vb, there = (torch.cat(x) for x in ((kp, kb), (vp, vb), (tp, there)))
        j = torch.arange(shared + n) - shared
        for s, r in enumerate(range(cu[b], min(cu[b + 1], q.shape[0]))):
            seen = there if offs is None else there & ((j < 0) | (j <= offs[b] + s))
            out[r], mag[r], size[r] = attend(q[r], kb, vb, seen, scale)
            most = max(most, int(seen.sum()))
    return out, mag, size, most


def check(got, ref, mag, size, keys, dtype, rows=False):
    """Bound of an element (sums over a row's keys, p its probabilities, z its largest score's terms
    scale |q| . |k|, all in float64):
      half a step of the result's type;
      scores: (D + 8) roundings of fp32 at most, 2^-23 each, of z, and as much again by exp2 and the
        reference point, which a probability takes as a relative error: 2 (D + 8) 2^-23 z;
      probabilities: two terms of the pool's 16-bit type, 2^-16 of each; calls with many rows round them
        once to it: half a step, 2^-8 or 2^-11 of each (rows);
      the sums over the keys: one rounding of 2^-23 each of what is summed, for p v and for p.
    All but the first times sum p |v|."""
    assert got.dtype == dtype and got.shape == ref.shape
    rel = 0.0 if dtype == torch.float32 else STEP[dtype] if rows else 2.0 ** -16
    rel = rel + 2.0 ** -22 + 2 * keys * 2.0 ** -23 + 2 * (ref.shape[-1] + 8) * 2.0 ** -23 * size
    bound = STEP[dtype] * ref.abs().clamp_min(LEAST[dtype]) + rel * mag
    got = got.double().cpu()
    odd = ~torch.isfinite(ref)
    assert torch.equal(got[odd].isnan(), ref[odd].isnan())
    inf = torch.isinf(ref)
    assert torch.equal(got[inf], ref[inf])
    err = (got - ref).abs()[~odd]
    assert (err <= bound[~odd]).all(), (err / bound[~odd].clamp_min(1e-300)).max().item()
