"""Attention over the 8-bit pool where blocks of a step are not there, behind a context or of pages outside
the pool: nothing that the pool holds elsewhere, scales and codes of page 0 among it, reaches a row."""

from __future__ import annotations

import math

import pytest
import torch

import kv8_oracle as O
from plastic_infer.kernel.paged_kv8 import (
    kv8_gather, paged_attention_kv8, paged_decode_attention_kv8)
from test_gpu_kv8_attention import _rows, _tables

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
BAD = [math.nan, math.inf]


def _pools(lens, hkv, dim, page, bad, seed):
    """(tables, a pool, the same with NaN codes and `bad` scales in every page no table names, and the
    blocks behind the contexts); page 0 is in no table, and a sequence has a page outside the pool."""
    tables, pages = _tables(lens, page, 3, seed)
    tables = torch.where(tables >= 0, tables + 1, tables)     # page 0 in no table
    pages += 1
    used = torch.zeros(pages, dtype=torch.bool)
    used[tables[tables >= 0].long()] = True
    tables[0, 0] = pages + 4                                  # not in the pool
    clean, dirty = (O.Pool.random(pages, hkv, dim, page, seed=seed) for _ in range(2))
    for x in "kv":
        dirty.codes[x][~used] = math.nan
        dirty.scale[x][~used] = bad
        for b, n in enumerate(lens):
            last, at = int(tables[b, (n - 1) // page]), -(-(n % page) // O.BLOCK)
            if n % page:
                dirty.scale[x][last, :, at:] = bad
    assert not used[0]
    return tables, clean, dirty


@pytest.mark.parametrize("bad", BAD)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,page", [(128, 16), (64, 64), (96, 48), (256, 32), (16, 16)])
def test_decode(dev, dim, page, dtype, bad):
    for lens in ([90, 1, 33, 130], [700, 17, 250, 65]):       # tables of few steps, and cut items
        tables, clean, dirty = _pools(lens, 2, dim, page, bad, sum(lens) + dim)
        q = _rows(len(lens), 8, dim, dtype, dim).to(dev)
        lens_t = torch.tensor(lens, dtype=torch.int32, device=dev)
        want, got = (paged_decode_attention_kv8(q, p.to_device(dev), tables.to(dev), lens_t)
                     for p in (clean, dirty))
        assert torch.isfinite(want).all() and torch.equal(got, want)


@pytest.mark.parametrize("bad", BAD)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,dim,page", [(8, 2, 128, 16), (96, 8, 128, 16), (96, 8, 64, 64),
                                             (96, 8, 96, 48), (8, 2, 256, 32)],
                         ids=lambda x: str(x))
@pytest.mark.parametrize("new", [[3, 1, 2, 5], [20, 1, 33, 9]], ids=["few", "more"])
def test_rows(dev, new, hq, hkv, dim, page, dtype, bad):
    lens = [90, 1, 33, 130]
    tables, clean, dirty = _pools(lens, hkv, dim, page, bad, dim + hq)
    cu = [0] + torch.tensor(new).cumsum(0).tolist()
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    q = _rows(cu[-1], hq, dim, dtype, dim).to(dev)
    for width in (0, 2048):                                   # and items cut along their keys
        t = tables
        if width:
            t = torch.nn.functional.pad(t, (0, width // page - t.shape[1]), value=-1)
        for offs in ([n - m for n, m in zip(lens, new)], None):
            want, got = (paged_attention_kv8(q, p.to_device(dev), t.to(dev), i32(lens), i32(cu),
                                             None if offs is None else i32(offs))
                         for p in (clean, dirty))
            assert torch.isfinite(want).all() and torch.equal(got, want)


@pytest.mark.parametrize("bad", BAD)
def test_gather(dev, bad):
    lens = [90, 1, 33, 130]
    tables, clean, dirty = _pools(lens, 2, 64, 16, bad, 4)
    cu = torch.tensor([0] + lens).cumsum(0).to(dev)
    want, got = (kv8_gather(p.to_device(dev), tables.to(dev), cu, 130) for p in (clean, dirty))
    assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("bad", BAD)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,dim", [(8, 2, 128), (96, 8, 128), (96, 8, 64), (8, 2, 256)])
def test_a_k_scale_that_is_none_shows_where_it_is_seen(dev, hq, hkv, dim, dtype, bad):
    """The block of positions 80..95 of one head: rows that see a key of it are NaN (with an infinite scale
    a row may be finite, where its products with them are all negative), others are as they were."""
    n, rows, page, g = 130, 66, 16, hq // hkv
    tables, pages = _tables([n], page, 0, 3)
    clean, dirty = (O.Pool.random(pages, hkv, dim, page, seed=5) for _ in range(2))
    dirty.scale["k"][int(tables[0, 5]), 1] = bad
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    q = _rows(rows, hq, dim, dtype, dim).to(dev)
    want, got = (paged_attention_kv8(q, p.to_device(dev), tables.to(dev), i32([n]), i32([0, rows]),
                                     i32([n - rows])) for p in (clean, dirty))
    sees = torch.arange(rows) + n - rows >= 80
    assert torch.equal(got[~sees], want[~sees])
    assert torch.equal(got[:, :g], want[:, :g]) and torch.equal(got[:, 2 * g:], want[:, 2 * g:])
    assert torch.isnan(got[sees][:, g:2 * g]).all() or bad == math.inf
