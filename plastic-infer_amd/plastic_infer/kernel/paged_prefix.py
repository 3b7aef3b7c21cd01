"""Attention over the paged KV cache for batches that share a long prefix: the prefix's pages are kept
once, and its part of the attention is computed for all rows of a group at once.

paged_kv's calls read every sequence's whole context for itself. Here a context is the group's prefix and
then the sequence's own tokens, in two tables, and the two parts meet by their maxima and sums.
"""

from __future__ import annotations

import functools
import math

import torch

from .. import _native as N
from .paged_window import checked_call, scratch


@functools.lru_cache(maxsize=256)
def _workspace_bytes(rows: int, num_heads: int, head_dim: int, device: int) -> int:
    with torch.cuda.device(device):
        return N.query("pia_prefix_attention_workspace_bytes", rows, num_heads, head_dim)


@functools.lru_cache(maxsize=1024)
def _call_bytes(device: int, *call: int | float) -> int:
    with torch.cuda.device(device):
        return N.query("pia_prefix_attention_call_workspace_bytes", *call)


def prefix_attention_workspace_bytes(rows: int, num_heads: int, head_dim: int,
                                     device: torch.device | None = None) -> int:
    """Bytes of a workspace that does for every call of so many query rows or fewer: room for two pieces
    of all rows in fp32. Calls that share a workspace must be ordered on one stream (a captured graph
    keeps using the one it was captured with)."""
    index = torch.cuda.current_device() if device is None or device.index is None else device.index
    return _workspace_bytes(rows, num_heads, head_dim, index)


def paged_prefix_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                           prefix_tables: torch.Tensor, prefix_lens: torch.Tensor,
                           block_tables: torch.Tensor, kv_lens: torch.Tensor,
                           cu_seqs: torch.Tensor | None = None, cu_q: torch.Tensor | None = None,
                           q_pos_offsets: torch.Tensor | None = None, scale: float | None = None,
                           out: torch.Tensor | None = None,
                           workspace: torch.Tensor | None = None) -> torch.Tensor:
    """paged_attention behind shared prefixes. prefix_tables int32 [groups, max_prefix_pages] and
    prefix_lens int32 [groups] name each group's prefix; group g is the sequences
    cu_seqs[g]..cu_seqs[g+1] (int32 [groups + 1], not decreasing; None: one group of all), and a
    sequence in no group has no prefix. block_tables, kv_lens and q_pos_offsets are about a sequence's
    own tokens behind the prefix: row s of b attends the whole prefix and the own keys j < kv_lens[b]
    and, when q_pos_offsets is given, j <= q_pos_offsets[b] + s. q: [rows, Hq, D], rows of sequence b =
    cu_q[b]..cu_q[b+1] (cu_q None: one row per sequence). A row without a key is zeros; a page id
    outside the pool holds no keys. Rows behind the last sequence are left as they were in `out`, which
    may be q itself and must not overlap it otherwise. Probabilities as in paged_window_attention;
    here many rows of a group are enough.
    workspace: device memory of prefix_attention_workspace_bytes, kept between calls that are ordered
    on one stream; where none (or too little) is given, what the call takes is allocated for it: little
    or nothing for many rows of each sequence over 16-bit pools."""
    dev, q, stride, out = checked_call(
        q, k_pages, v_pages, block_tables, kv_lens, cu_q, q_pos_offsets, out, workspace,
        {"prefix_tables": prefix_tables, "prefix_lens": prefix_lens, "cu_seqs": cu_seqs})
    num_pages, Hkv, D, P = k_pages.shape
    rows, Hq, _ = q.shape
    B = block_tables.shape[0]
    if prefix_tables.dtype != torch.int32 or prefix_tables.dim() != 2:
        raise ValueError("prefix_tables must be int32 [groups, max_prefix_pages]")
    groups = prefix_tables.shape[0]
    if prefix_lens.dtype != torch.int32 or prefix_lens.shape != (groups,):
        raise ValueError("prefix_lens must be int32 [groups]")
    if cu_seqs is None:
        if groups != 1:
            raise ValueError("without cu_seqs there must be exactly one group")
    elif cu_seqs.dtype != torch.int32 or cu_seqs.shape != (groups + 1,):
        raise ValueError("cu_seqs must be int32 [groups + 1]")
    if rows == 0 or B == 0:
        return out
    scale = (1.0 / math.sqrt(D)) if scale is None else float(scale)
    need = _call_bytes(dev.index, groups, prefix_tables.shape[1], block_tables.shape[1],
                       int(cu_q is not None), B, rows, Hq, Hkv, D, P, scale, N.dtype_code(q.dtype))
    ws = scratch(workspace, need, dev)
    pt, plens = prefix_tables.contiguous(), prefix_lens.contiguous()
    bt, lens = block_tables.contiguous(), kv_lens.contiguous()
    gs = None if cu_seqs is None else cu_seqs.contiguous()
    cu = None if cu_q is None else cu_q.contiguous()
    offs = None if q_pos_offsets is None else q_pos_offsets.contiguous()
    N.call_on(dev, "pia_prefix_attention", out.data_ptr(), q.data_ptr(), stride, k_pages.data_ptr(),
              v_pages.data_ptr(), pt.data_ptr(), pt.shape[1], plens.data_ptr(), N.ptr(gs), groups,
              bt.data_ptr(), bt.shape[1], lens.data_ptr(), N.ptr(cu), N.ptr(offs), B, rows, Hq, Hkv,
              D, P, num_pages, scale, N.dtype_code(q.dtype), N.ptr(ws), need, N.stream_of(dev))
    return out


def paged_prefix_decode_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                                  prefix_tables: torch.Tensor, prefix_lens: torch.Tensor,
                                  block_tables: torch.Tensor, context_lens: torch.Tensor,
                                  cu_seqs: torch.Tensor | None = None, scale: float | None = None,
                                  out: torch.Tensor | None = None,
                                  workspace: torch.Tensor | None = None) -> torch.Tensor:
    """paged_decode_attention behind shared prefixes: one query row per sequence, q [B, Hq, D], which
    attends its group's prefix and its context_lens[b] own tokens (the newest among them; 0: the prefix
    alone)."""
    return paged_prefix_attention(q, k_pages, v_pages, prefix_tables, prefix_lens, block_tables,
                                  context_lens, cu_seqs, None, None, scale, out, workspace)


__all__ = ["prefix_attention_workspace_bytes", "paged_prefix_attention",
           "paged_prefix_decode_attention"]
