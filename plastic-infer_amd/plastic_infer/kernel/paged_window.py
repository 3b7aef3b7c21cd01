"""Attention over the paged KV cache with a sliding window: a row sees the last `window` tokens up to its
own position, and the first `sinks` tokens of its context, which stay visible.

paged_kv.paged_attention's rows see their whole context; here a decode step reads sinks + window tokens of
each sequence, however long it is. Pages behind the window may be given up: their entries of the block
table are not read.
"""

from __future__ import annotations

import functools
import math

import torch

from .. import _native as N
from .paged_kv import _check_pool
from .rotary import derived, fresh_like


def checked_call(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                 block_tables: torch.Tensor, kv_lens: torch.Tensor, cu_q: torch.Tensor | None,
                 q_pos_offsets: torch.Tensor | None, out: torch.Tensor | None,
                 workspace: torch.Tensor | None, others: dict[str, torch.Tensor | None]
                 ) -> tuple[torch.device, torch.Tensor, int, torch.Tensor]:
    """The checks that windowed and prefix attention share: (device, q in a layout that the kernels
    read, elements between its rows, out)."""
    tensors = [q, k_pages, v_pages, block_tables, kv_lens]
    names = ["q", "k_pages", "v_pages", "block_tables", "the context lengths"]
    for name, t in (("cu_q", cu_q), ("q_pos_offsets", q_pos_offsets), ("out", out),
                    ("workspace", workspace), *others.items()):
        if t is not None:
            tensors.append(t)
            names.append(name)
    dev = N.require_device(*tensors, names=tuple(names))
    _check_pool(k_pages, v_pages)
    num_pages, Hkv, D, P = k_pages.shape
    if min(num_pages, Hkv, D, P) == 0 or D > 512 or P > 4096:
        raise ValueError(f"the pools need pages and heads, head_dim to 512 and page_size to 4096; got "
                         f"{tuple(k_pages.shape)}")
    if q.dim() != 3 or q.shape[2] != D or q.shape[1] == 0 or q.shape[1] % Hkv:
        raise ValueError(f"q must be [rows, Hq, {D}] with Hq a multiple of {Hkv}, got "
                         f"{tuple(q.shape)}")
    N.dtype_code(q.dtype)
    if q.dtype != k_pages.dtype:
        raise ValueError("q dtype must match the KV pool dtype")
    if derived(q, k_pages, v_pages):
        raise ValueError("attention over the paged cache has no gradient: call it under "
                         "torch.no_grad(), on tensors without a tangent")
    rows, Hq, _ = q.shape
    token, head, elem = q.stride()
    if elem != 1 or head != D or token * q.element_size() % 16 or q.data_ptr() % 16:
        q = q.contiguous()
        if q.data_ptr() % 16:   # a contiguous view that starts between vectors
            q = q.clone()
    stride = q.stride(0) if rows > 1 else Hq * D   # of a single row it says nothing
    if block_tables.dtype != torch.int32 or block_tables.dim() != 2:
        raise ValueError("block_tables must be int32 [B, max_pages]")
    B = block_tables.shape[0]
    if kv_lens.dtype != torch.int32 or kv_lens.shape != (B,):
        raise ValueError("the context lengths must be int32 [B]")
    if cu_q is None:
        if rows != B:
            raise ValueError("without cu_q there must be exactly one query row per sequence")
    elif cu_q.dtype != torch.int32 or cu_q.shape != (B + 1,):
        raise ValueError("cu_q must be int32 [B + 1]")
    if q_pos_offsets is not None and (q_pos_offsets.dtype != torch.int32
                                      or q_pos_offsets.shape != (B,)):
        raise ValueError("q_pos_offsets must be int32 [B]")
    if out is None:
        out = fresh_like(q)
    elif out.shape != (rows, Hq, D) or out.dtype != q.dtype or not out.is_contiguous() \
            or out.data_ptr() % 16:
        raise ValueError("out must be a contiguous, 16-byte aligned tensor of q's shape and dtype")
    return dev, q, stride, out


def scratch(workspace: torch.Tensor | None, need: int, dev: torch.device) -> torch.Tensor | None:
    """The caller's workspace where it is one, or one of the call's own."""
    if need == 0:
        return None
    if workspace is None or workspace.numel() * workspace.element_size() < need \
            or workspace.data_ptr() % 16 or not workspace.is_contiguous():
        return torch.empty(need, dtype=torch.uint8, device=dev)
    return workspace


@functools.lru_cache(maxsize=64)
def _workspace_bytes(head_dim: int, device: int) -> int:
    with torch.cuda.device(device):
        return N.query("pia_window_attention_workspace_bytes", head_dim)


def window_attention_workspace_bytes(head_dim: int, device: torch.device | None = None) -> int:
    """Bytes of the workspace of both calls, whatever the batch. Calls that share a workspace must be
    ordered on one stream (a captured graph keeps using the one it was captured with)."""
    index = torch.cuda.current_device() if device is None or device.index is None else device.index
    return _workspace_bytes(head_dim, index)


def _whole(name: str, x: int, least: int) -> int:
    if isinstance(x, bool) or not isinstance(x, int) or x < least:
        raise ValueError(f"{name} must be a whole number of at least {least}, got {x!r}")
    return min(x, 0x7fffffff)


def paged_window_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                           block_tables: torch.Tensor, kv_lens: torch.Tensor, window: int,
                           sinks: int = 0, cu_q: torch.Tensor | None = None,
                           q_pos_offsets: torch.Tensor | None = None, scale: float | None = None,
                           out: torch.Tensor | None = None,
                           workspace: torch.Tensor | None = None) -> torch.Tensor:
    """paged_attention with a window. q: [rows, Hq, D], rows of sequence b = cu_q[b]..cu_q[b+1] (cu_q
    None: one row per sequence). Row s of b stands at position p = q_pos_offsets[b] + s (None: the rows
    are the context's last) and attends the keys j < kv_lens[b], j <= p with p - j < window or
    j < sinks. A row without a key is zeros; a page id outside the pool holds no keys. Rows behind the
    last sequence are left as they were in `out`, which may be q itself and must not overlap it
    otherwise. Probabilities are held to 2^-16 of each or better; calls of many rows for each sequence, on
    average, over 16-bit pools round them once to the pool's type.
    workspace: device memory of window_attention_workspace_bytes, kept between calls that are ordered
    on one stream; allocated for the call where none (or too little) is given."""
    window, sinks = _whole("window", window, 1), _whole("sinks", sinks, 0)
    dev, q, stride, out = checked_call(q, k_pages, v_pages, block_tables, kv_lens, cu_q,
                                       q_pos_offsets, out, workspace, {})
    num_pages, Hkv, D, P = k_pages.shape
    rows, Hq, _ = q.shape
    B = block_tables.shape[0]
    if rows == 0 or B == 0:
        return out
    need = _workspace_bytes(D, dev.index)
    ws = scratch(workspace, need, dev)
    scale = (1.0 / math.sqrt(D)) if scale is None else float(scale)
    bt, lens = block_tables.contiguous(), kv_lens.contiguous()
    cu = None if cu_q is None else cu_q.contiguous()
    offs = None if q_pos_offsets is None else q_pos_offsets.contiguous()
    N.call_on(dev, "pia_window_attention", out.data_ptr(), q.data_ptr(), stride, k_pages.data_ptr(),
              v_pages.data_ptr(), bt.data_ptr(), bt.shape[1], lens.data_ptr(), N.ptr(cu),
              N.ptr(offs), window, sinks, B, rows, Hq, Hkv, D, P, num_pages, scale,
              N.dtype_code(q.dtype), N.ptr(ws), need, N.stream_of(dev))
    return out


def paged_window_decode_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                                  block_tables: torch.Tensor, context_lens: torch.Tensor,
                                  window: int, sinks: int = 0, scale: float | None = None,
                                  out: torch.Tensor | None = None,
                                  workspace: torch.Tensor | None = None) -> torch.Tensor:
    """paged_decode_attention with a window: one query row per sequence, q [B, Hq, D], at the last of
    its context_lens[b] tokens; it attends the last `window` of them and the first `sinks`."""
    return paged_window_attention(q, k_pages, v_pages, block_tables, context_lens, window, sinks,
                                  None, None, scale, out, workspace)


__all__ = ["window_attention_workspace_bytes", "paged_window_attention",
           "paged_window_decode_attention"]
