"""The 8-bit KV pool and the rotary map from their definitions, in float64 on the CPU."""

from __future__ import annotations

import math

import torch

BLOCK = 16


def e4m3(x: torch.Tensor) -> torch.Tensor:
    """x [fp64] as the nearest e4m3 value (ties to even), limited to 448; non-finite: NaN."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(2.0 ** -6, 448.0))) - 3)
    y = (torch.round(x / step) * step).clamp(-448.0, 448.0)
    return torch.where(torch.isfinite(x), y, torch.full_like(x, math.nan))


def scale_for(bound: float) -> float:
    """The smallest power of two, at least 2^-100, of which 448 hold the bound."""
    e = -100
    while e < 119 and 448.0 * 2.0 ** e < bound:
        e += 1
    return 2.0 ** e


def turn(x, positions, turns, factor, interleaved, sign=1.0):
    """(x [N, H, D] rotated, factor (|a| + |b|) of each element's pair), in float64."""
    x = x.double()
    h = turns.numel()
    t = positions.double()[:, None] * turns.double()
    c = (factor * torch.cos(2 * math.pi * (t - t.floor())))[:, None]
    s = (factor * sign * torch.sin(2 * math.pi * (t - t.floor())))[:, None]
    ia = torch.arange(h) * 2 if interleaved else torch.arange(h)
    ib = ia + 1 if interleaved else ia + h
    out, size = x.clone(), x.abs().clone()
    a, b = x[..., ia], x[..., ib]
    out[..., ia], out[..., ib] = a * c - b * s, b * c + a * s
    size[..., ia] = size[..., ib] = factor * (a.abs() + b.abs())
    return out, size


class Pool:
    """Pools as values: codes [N, H, P, D] (fp64, of e4m3's values) and scales [N, H, P / 16]."""

    def __init__(self, pages, heads, dim, page):
        self.shape = (pages, heads, dim, page)
        self.codes = {x: torch.zeros(pages, heads, page, dim, dtype=torch.float64) for x in "kv"}
        self.scale = {x: torch.ones(pages, heads, page // BLOCK, dtype=torch.float64) for x in "kv"}

    @classmethod
    def random(cls, pages, heads, dim, page, seed, spread=1.0):
        """Codes of normal values, scales that differ from block to block."""
        p = cls(pages, heads, dim, page)
        g = torch.Generator().manual_seed(seed)
        for x in "kv":
            p.codes[x] = e4m3(100.0 * torch.randn(p.codes[x].shape, generator=g,
                                                  dtype=torch.float64).clamp(-4, 4))
            e = torch.randint(-8, -5, p.scale[x].shape, generator=g)
            p.scale[x] = torch.exp2(e.double()) * spread
        return p

    def values(self, x):
        return self.codes[x] * self.scale[x].repeat_interleave(BLOCK, -1)[..., None]

    def to_device(self, dev):
        from plastic_infer.kernel.paged_kv8 import KV8Pools

        n, h, d, p = self.shape
        k = self.codes["k"].reshape(n, h, p, d // 16, 16).permute(0, 1, 3, 2, 4)
        v = self.codes["v"].reshape(n, h, p // 4, 4, d).permute(0, 1, 2, 4, 3)
        return KV8Pools(*(t.contiguous().float().to(torch.float8_e4m3fn).to(dev) for t in (k, v)),
                        *(self.scale[x].float().to(dev) for x in "kv"))

    @classmethod
    def from_device(cls, pools):
        p = cls(*pools.shape)
        n, h, d, page = pools.shape
        p.codes["k"] = pools.k.cpu().float().double().permute(0, 1, 3, 2, 4).reshape(n, h, page, d)
        p.codes["v"] = pools.v.cpu().float().double().permute(0, 1, 2, 4, 3).reshape(n, h, page, d)
        p.scale["k"], p.scale["v"] = pools.k_scale.cpu().double(), pools.v_scale.cpu().double()
        return p

    def context(self, x, table, length):
        """Values of a sequence's tokens [length, H, D]; (their page exists [length])."""
        n, h, d, page = self.shape
        out = torch.zeros(length, h, d, dtype=torch.float64)
        there = torch.zeros(length, dtype=torch.bool)
        vals = self.values(x)
        for t in range(0, length, page):
            i, m = int(table[t // page]), min(page, length - t)
            if 0 <= i < n:
                out[t:t + m] = vals[i, :, :m].transpose(0, 1)
                there[t:t + m] = True
        return out, there

    def append(self, x, rows, bounds, table, start):
        """rows [n, H, D] (fp64) at positions start.. of a sequence, bounds [n, H] of their size."""
        n_pages, h, d, page = self.shape
        end = start + rows.shape[0]
        for blk in range(start // BLOCK, -(-end // BLOCK)):
            lo, hi = max(start, blk * BLOCK), min(end, (blk + 1) * BLOCK)
            slot, sub = blk * BLOCK // page, blk % (page // BLOCK)
            if slot >= len(table) or not 0 <= int(table[slot]) < n_pages:
                continue
            i, at = int(table[slot]), sub * BLOCK
            for head in range(h):
                s = scale_for(float(bounds[lo - start:hi - start, head].max()))
                was = float(self.scale[x][i, head, sub])
                if lo > blk * BLOCK:
                    if was < s:
                        old = self.codes[x][i, head, at:at + lo % BLOCK]
                        old.copy_(e4m3(old * (was / s)))
                    s = max(s, was)
                self.scale[x][i, head, sub] = s
                o = at + lo % BLOCK
                self.codes[x][i, head, o:o + hi - lo] = e4m3(rows[lo - start:hi - start, head] / s)


def attend(q, pool, tables, lens, cu, offsets, scale):
    """(out, sum p |v|, score size) of every row, in float64: a row without keys is zeros. Score
    size: the largest scale |q| . |k| that the row sees, for error bounds."""
    _, Hkv, D, P = pool.shape
    rows, Hq, _ = q.shape
    G = Hq // Hkv
    out = torch.zeros(rows, Hq, D, dtype=torch.float64)
    mag, size = torch.zeros_like(out), torch.zeros(rows, Hq, 1, dtype=torch.float64)
    for b, n in enumerate(lens):
        n = max(0, min(int(n), len(tables[b]) * P))
        k, there = pool.context("k", tables[b], n)
        v, _ = pool.context("v", tables[b], n)
        for r in range(cu[b], cu[b + 1]):
            see = there.clone()
            if offsets is not None:
                see &= torch.arange(n) <= int(offsets[b]) + r - cu[b]
            if not see.any():
                continue
            for h in range(Hq):
                kk, vv, x = k[see, h // G], v[see, h // G], q[r, h].double()
                s = scale * (kk @ x)
                p = torch.softmax(s, 0)
                out[r, h] = p @ vv
                mag[r, h] = p @ vv.abs()
                size[r, h] = (abs(scale) * (kk.abs() @ x.abs())).max()
    return out, mag, size
