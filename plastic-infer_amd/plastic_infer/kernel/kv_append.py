"""New tokens rotated and written into a paged KV pool in one launch.

kv_scatter (paged_kv.py) writes finished K / V rows to given slots; here the slots follow from the
block tables and context lengths, k is rotated on the way and q is returned rotated.
"""

from __future__ import annotations

import torch

from .. import _native as N
from .paged_kv import _check_pool
from .rotary import RopeParams, check_rope, derived, fresh_like, heads_view


def append_call(q: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor,
                pools: tuple[torch.Tensor, torch.Tensor],
                scales: tuple[torch.Tensor, torch.Tensor] | None, shape: tuple[int, int, int, int],
                block_tables: torch.Tensor, context_lens: torch.Tensor,
                cu_new: torch.Tensor | None, rope: RopeParams | None) -> torch.Tensor | None:
    """Checks and launch shared by both pool types; shape: (num_pages, Hkv, D, P)."""
    num_pages, Hkv, D, P = shape
    dev = N.require_device(k, v, *pools, block_tables, context_lens,
                           *(() if q is None else (q,)), *(() if cu_new is None else (cu_new,)),
                           names=("k", "v", "k_pages", "v_pages", "block_tables", "context_lens",
                                  "cu_new" if q is None else "q", "cu_new"))
    if derived(q, k, v):
        raise ValueError("an append has no gradient: call it under torch.no_grad(), on tensors "
                         "without a tangent")
    k, v = heads_view("k", k), heads_view("v", v)
    n = k.shape[0]
    if k.shape != (n, Hkv, D) or v.shape != (n, Hkv, D):
        raise ValueError(f"k and v must be [tokens, {Hkv}, {D}], got {tuple(k.shape)} / "
                         f"{tuple(v.shape)}")
    if v.dtype != k.dtype or (q is not None and q.dtype != k.dtype):
        raise ValueError("q, k and v must share a dtype")
    code = N.dtype_code(k.dtype)
    if block_tables.dtype != torch.int32 or block_tables.dim() != 2:
        raise ValueError("block_tables must be int32 [B, max_pages]")
    B = block_tables.shape[0]
    if context_lens.dtype != torch.int32 or context_lens.shape != (B,):
        raise ValueError("context_lens must be int32 [B]")
    if cu_new is None:
        if n != B:
            raise ValueError("without cu_new there must be exactly one token per sequence")
    elif cu_new.dtype != torch.int32 or cu_new.shape != (B + 1,):
        raise ValueError("cu_new must be int32 [B + 1]")
    if rope is not None:
        check_rope(rope, D, dev)
    out = None
    if q is not None:
        q = heads_view("q", q)
        if q.shape[0] != n or q.shape[2] != D:
            raise ValueError(f"q must be [{n}, heads, {D}], got {tuple(q.shape)}")
        out = fresh_like(q)
    if n == 0 or B == 0:
        return out
    has_q = q is not None and q.shape[1] > 0
    bt, lens = block_tables.contiguous(), context_lens.contiguous()
    cu = None if cu_new is None else cu_new.contiguous()
    N.call_on(dev, "pia_kv_append", out.data_ptr() if has_q else None,
              q.data_ptr() if has_q else None, q.stride(0) if has_q else 0,
              q.stride(1) if has_q else 0, k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(),
              v.stride(0), v.stride(1), pools[0].data_ptr(), pools[1].data_ptr(),
              None if scales is None else scales[0].data_ptr(),
              None if scales is None else scales[1].data_ptr(), bt.data_ptr(), bt.shape[1],
              lens.data_ptr(), N.ptr(cu), n, B, None if rope is None else rope.turns.data_ptr(),
              0 if rope is None else rope.turns.numel(), 1.0 if rope is None else rope.factor,
              1 if rope is not None and rope.interleaved else 0,
              q.shape[1] if has_q else 0, Hkv, D, P, num_pages, code, N.stream_of(dev))
    return out


def kv_append(q: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor,
              v_pages: torch.Tensor, block_tables: torch.Tensor, context_lens: torch.Tensor,
              cu_new: torch.Tensor | None = None,
              rope: RopeParams | None = None) -> torch.Tensor | None:
    """Append each sequence's newest tokens: rows cu_new[b]..cu_new[b+1] of k, v [tokens, Hkv, D]
    (cu_new None: row b) are the last tokens of sequence b, whose context_lens[b] counts them. k,
    rotated at its place in the context by rope (None: as it is), and v go to their slots of
    block_tables[b] in pools [num_pages, Hkv, D, P] of their dtype. Returns q [tokens, Hq, D]
    rotated likewise (None without q). Tokens of pages outside the pool are not written; rows of no
    sequence are read nowhere and hold nothing in the returned q. The pages that take new tokens
    belong to one sequence each."""
    _check_pool(k_pages, v_pages)
    if k.dtype != k_pages.dtype:
        raise ValueError("k and v must have the pools' dtype")
    return append_call(q, k, v, (k_pages, v_pages), None, tuple(k_pages.shape), block_tables,
                       context_lens, cu_new, rope)


__all__ = ["kv_append"]
