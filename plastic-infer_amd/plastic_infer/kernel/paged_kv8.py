"""The paged KV cache in 8 bits: append, gather and attention over e4m3 codes with one power-of-two
scale for every 16 tokens of a page and head.

Half the bytes of a 16-bit pool for a decode step to read. Scales are powers of two, so a code times
its scale is exact in bf16, and the scale of a block can grow as tokens join it without changing the
digits of those already there.
"""

from __future__ import annotations

import functools
import math
from dataclasses import dataclass

import torch

from .. import _native as N
from .kv_append import append_call
from .rotary import RopeParams, derived, fresh_like

BLOCK = 16   # tokens that share a scale


@dataclass(frozen=True)
class KV8Pools:
    """The pools of one device: k float8_e4m3fn [num_pages, Hkv, D / 16, P, 16], v float8_e4m3fn
    [num_pages, Hkv, P / 4, D, 4], scales float32 [num_pages, Hkv, P / 16]. D and P are multiples
    of 16, up to 256 and 4096."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor

    @classmethod
    def allocate(cls, num_pages: int, num_kv_heads: int, head_dim: int, page_size: int = 16,
                 device: torch.device | None = None) -> "KV8Pools":
        """Pools of zeros."""
        _check_shape(head_dim, page_size)
        dev = torch.device("cuda", torch.cuda.current_device()) if device is None else device
        k, v = (torch.zeros(s, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn)
                for s in ((num_pages, num_kv_heads, head_dim // 16, page_size, 16),
                          (num_pages, num_kv_heads, page_size // 4, head_dim, 4)))
        ks, vs = (torch.zeros(num_pages, num_kv_heads, page_size // BLOCK, device=dev)
                  for _ in range(2))
        return cls(k, v, ks, vs)

    @property
    def shape(self) -> tuple[int, int, int, int]:
        """(num_pages, Hkv, D, P)."""
        n, h, c, p, _ = self.k.shape
        return n, h, 16 * c, p

    @property
    def bytes_per_token(self) -> float:
        """K + V bytes of a token, with its part of the scales."""
        _, h, d, _ = self.shape
        return 2 * h * (d + 4 / BLOCK)


def _check_shape(head_dim: int, page_size: int) -> None:
    if not 0 < head_dim <= 256 or head_dim % 16 or not 0 < page_size <= 4096 or page_size % BLOCK:
        raise ValueError(f"8-bit pools take head_dim and page_size in multiples of 16, up to 256 and "
                         f"4096; got {head_dim} and {page_size}")


def _check_pools(p: KV8Pools) -> tuple[int, int, int, int]:
    """(num_pages, Hkv, D, P) of valid pools. Looked at on every call (2 us): tensors can be resized."""
    k, v, ks, vs = p.k, p.v, p.k_scale, p.v_scale
    index = k.get_device()
    if k.dim() == 5 and index >= 0 and v.get_device() == index and ks.get_device() == index \
            and vs.get_device() == index:   # the usual case: nothing to report
        n, h, c, page, e = k.shape
        if n and h and e == 16 and 0 < c <= 16 and 0 < page <= 4096 and page % BLOCK == 0 \
                and v.shape == (n, h, page // 4, 16 * c, 4) \
                and ks.shape == vs.shape == (n, h, page // BLOCK) \
                and k.dtype == v.dtype == torch.float8_e4m3fn \
                and ks.dtype == vs.dtype == torch.float32 and k.is_contiguous() \
                and v.is_contiguous() and ks.is_contiguous() and vs.is_contiguous():
            return n, h, 16 * c, page
    return _checked_shape(p)


def _checked_shape(p: KV8Pools) -> tuple[int, int, int, int]:
    N.require_device(p.k, p.v, p.k_scale, p.v_scale,
                     names=("pools.k", "pools.v", "pools.k_scale", "pools.v_scale"))
    if p.k.dim() != 5 or p.k.shape[4] != 16:
        raise ValueError(f"pools.k must be [num_pages, H, D / 16, P, 16], got {tuple(p.k.shape)}")
    n, h, d, page = p.shape
    _check_shape(d, page)
    if n == 0 or h == 0:
        raise ValueError("8-bit pools need a page and a head")
    if p.v.shape != (n, h, page // 4, d, 4):
        raise ValueError(f"pools.v must be {(n, h, page // 4, d, 4)}, got {tuple(p.v.shape)}")
    if p.k.dtype != torch.float8_e4m3fn or p.v.dtype != torch.float8_e4m3fn:
        raise ValueError("pools.k and pools.v must be float8_e4m3fn")
    want = (n, h, page // BLOCK)
    if p.k_scale.dtype != torch.float32 or p.v_scale.dtype != torch.float32 \
            or p.k_scale.shape != want or p.v_scale.shape != want:
        raise ValueError(f"pools.k_scale and pools.v_scale must be float32 {want}")
    if not (p.k.is_contiguous() and p.v.is_contiguous() and p.k_scale.is_contiguous()
            and p.v_scale.is_contiguous()):
        raise ValueError("KV pools must be contiguous")
    return n, h, d, page


def kv8_append(q: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor, pools: KV8Pools,
               block_tables: torch.Tensor, context_lens: torch.Tensor,
               cu_new: torch.Tensor | None = None,
               rope: RopeParams | None = None) -> torch.Tensor | None:
    """kv_append into 8-bit pools. A block's scale is the smallest power of two that holds its new
    tokens within e4m3's range (rotated k by a bound of the rotation), or the one it has, if that
    is larger and the block holds earlier tokens; those are rounded to a scale that grows. NaN and
    infinite elements become NaN."""
    shape = _check_pools(pools)
    return append_call(q, k, v, (pools.k, pools.v), (pools.k_scale, pools.v_scale), shape,
                       block_tables, context_lens, cu_new, rope)


def kv8_gather(pools: KV8Pools, block_tables: torch.Tensor, cu_seqlens: torch.Tensor,
               max_seq_len: int, out: tuple[torch.Tensor, torch.Tensor] | None = None,
               dtype: torch.dtype = torch.bfloat16) -> tuple[torch.Tensor, torch.Tensor]:
    """kv_gather of 8-bit pools: rows cu_seqlens[b]..cu_seqlens[b+1] of the results hold sequence
    b's tokens in logical order, [total_tokens, Hkv, D] in dtype (or that of the `out` buffers,
    whose first dimension is then the total). bf16 and fp32 hold the pool's values exactly.
    max_seq_len: a bound of every length; 0 gathers nothing. Tokens of a page outside the pool are
    zeros; rows past a sequence's table are left as they are."""
    num_pages, H, D, P = _check_pools(pools)
    dev = N.require_device(pools.k, block_tables, cu_seqlens,
                           names=("pools.k", "block_tables", "cu_seqlens"))
    if block_tables.dtype != torch.int32 or block_tables.dim() != 2:
        raise ValueError("block_tables must be int32 [B, max_pages]")
    bt = block_tables.contiguous()
    cu = (cu_seqlens if cu_seqlens.dtype == torch.int64 else cu_seqlens.to(torch.int64)).contiguous()
    B = bt.shape[0]
    if cu.shape != (B + 1,):
        raise ValueError("cu_seqlens must have B + 1 entries")
    if out is None:
        N.dtype_code(dtype)
        total = int(cu[-1].item())
        k_out = torch.empty(total, H, D, dtype=dtype, device=dev)
        v_out = torch.empty_like(k_out)
    else:
        k_out, v_out = out
        N.require_device(pools.k, k_out, v_out, names=("pools.k", "out[0]", "out[1]"))
        if k_out.dim() != 3 or k_out.shape[1:] != (H, D) or v_out.shape != k_out.shape \
                or v_out.dtype != k_out.dtype \
                or not (k_out.is_contiguous() and v_out.is_contiguous()):
            raise ValueError(f"out buffers must be contiguous [tokens, {H}, {D}] of one dtype")
    code = N.dtype_code(k_out.dtype)
    if B and max_seq_len > 0 and bt.shape[1] > 0:
        N.call_on(dev, "pia_kv8_gather", k_out.data_ptr(), v_out.data_ptr(), pools.k.data_ptr(),
                  pools.v.data_ptr(), pools.k_scale.data_ptr(), pools.v_scale.data_ptr(),
                  bt.data_ptr(), bt.shape[1], cu.data_ptr(), B, k_out.shape[0], H, D, P,
                  num_pages, code, N.stream_of(dev))
    return k_out, v_out


@functools.lru_cache(maxsize=64)
def _workspace_bytes(head_dim: int, device: int) -> int:
    with torch.cuda.device(device):
        return N.query("pia_kv8_attention_workspace_bytes", head_dim)


def kv8_attention_workspace_bytes(head_dim: int, device: torch.device | None = None) -> int:
    """Bytes of the workspace of both attention calls, whatever the batch. Calls that share a
    workspace must be ordered on one stream (a captured graph keeps using the one it was captured
    with)."""
    index = torch.cuda.current_device() if device is None or device.index is None else device.index
    return _workspace_bytes(head_dim, index)


def _attention(q, pools, block_tables, kv_lens, cu_q, q_pos_offsets, scale, out, workspace):
    num_pages, Hkv, D, P = _check_pools(pools)
    tensors, names = [pools.k, q, block_tables, kv_lens], ["pools.k", "q", "block_tables", "kv_lens"]
    for name, t in (("cu_q", cu_q), ("q_pos_offsets", q_pos_offsets), ("out", out),
                    ("workspace", workspace)):
        if t is not None:
            tensors.append(t)
            names.append(name)
    dev = N.require_device(*tensors, names=tuple(names))
    if q.dim() != 3 or q.shape[2] != D or q.shape[1] == 0 or q.shape[1] % Hkv:
        raise ValueError(f"q must be [rows, Hq, {D}] with Hq a multiple of {Hkv}, got "
                         f"{tuple(q.shape)}")
    code = N.dtype_code(q.dtype)
    if derived(q):
        raise ValueError("attention over the 8-bit cache has no gradient: call it under "
                         "torch.no_grad(), on a q without a tangent")
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
    if rows == 0 or B == 0:
        return out
    need = _workspace_bytes(D, dev.index)
    if workspace is None or workspace.numel() * workspace.element_size() < need \
            or workspace.data_ptr() % 16 or not workspace.is_contiguous():
        workspace = torch.empty(need, dtype=torch.uint8, device=dev)
    scale = (1.0 / math.sqrt(D)) if scale is None else float(scale)
    bt, lens = block_tables.contiguous(), kv_lens.contiguous()
    cu = None if cu_q is None else cu_q.contiguous()
    offs = None if q_pos_offsets is None else q_pos_offsets.contiguous()
    N.call_on(dev, "pia_kv8_attention", out.data_ptr(), q.data_ptr(), stride,
              pools.k.data_ptr(), pools.v.data_ptr(), pools.k_scale.data_ptr(),
              pools.v_scale.data_ptr(), bt.data_ptr(), bt.shape[1], lens.data_ptr(), N.ptr(cu),
              N.ptr(offs), B, rows, Hq, Hkv, D, P, num_pages, scale, code, workspace.data_ptr(),
              need, N.stream_of(dev))
    return out


def paged_decode_attention_kv8(q: torch.Tensor, pools: KV8Pools, block_tables: torch.Tensor,
                               context_lens: torch.Tensor, scale: float | None = None,
                               out: torch.Tensor | None = None,
                               workspace: torch.Tensor | None = None) -> torch.Tensor:
    """paged_decode_attention over 8-bit pools: one query row per sequence, q [B, Hq, D] in bf16,
    fp16 or fp32, results in q's dtype. context_lens int32 [B] counts the newest token.
    workspace: device memory of kv8_attention_workspace_bytes, kept between calls that are ordered
    on one stream; allocated for the call where none (or too little) is given."""
    return _attention(q, pools, block_tables, context_lens, None, None, scale, out, workspace)


def paged_attention_kv8(q: torch.Tensor, pools: KV8Pools, block_tables: torch.Tensor,
                        kv_lens: torch.Tensor, cu_q: torch.Tensor | None = None,
                        q_pos_offsets: torch.Tensor | None = None, scale: float | None = None,
                        out: torch.Tensor | None = None,
                        workspace: torch.Tensor | None = None) -> torch.Tensor:
    """paged_attention over 8-bit pools. q: [rows, Hq, D], rows of sequence b = cu_q[b]..cu_q[b+1]
    (cu_q None: one row per sequence). Row s of b attends keys j < kv_lens[b] and, when
    q_pos_offsets is given, j <= q_pos_offsets[b] + s; a row without a key is zeros. Rows behind
    the last sequence are left as they were in `out`, which may be q itself and must not overlap it
    otherwise."""
    return _attention(q, pools, block_tables, kv_lens, cu_q, q_pos_offsets, scale, out, workspace)


__all__ = ["BLOCK", "KV8Pools", "kv8_append", "kv8_gather", "kv8_attention_workspace_bytes",
           "paged_decode_attention_kv8", "paged_attention_kv8"]
