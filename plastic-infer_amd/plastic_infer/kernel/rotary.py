"""Rotary positions of q and k: any part of the head, rotate-half or interleaved pairs, frequencies
scaled for long contexts, with gradients.

A token may have positions on several axes (time, height and width of images and video): each pair
then turns by the position on its own axis.

norm_rope.qk_norm_rope is the decode step's form (whole head, halves, table rows in the model's
dtype). Here the angles come from the positions themselves, in fp64 up to the whole turns, so a
position of a million is as exact as one of ten, and no table is kept.
"""

from __future__ import annotations

import math
from collections.abc import Sequence
from dataclasses import dataclass

import torch
from torch.autograd import forward_ad

from .. import _native as N


@dataclass(frozen=True)
class RopeParams:
    """How heads are rotated: pair i by 2 pi * position * turns[i], cos and sin times factor.
    turns: float64 [pairs] on the device; pairs are (i, i + pairs) of the head's first 2 * pairs
    elements or, interleaved, (2 i, 2 i + 1).
    axes: None (positions [tokens]) or int32 [pairs] on the device: the axis of each pair, a row of
    positions [axes, tokens]. A pair whose axis is no such row is turned as at position 0."""
    turns: torch.Tensor
    factor: float = 1.0
    interleaved: bool = False
    axes: torch.Tensor | None = None

    @property
    def rotary_dim(self) -> int:
        return 2 * self.turns.numel()


def rope_params(head_dim: int, base: float = 10000.0, rotary_dim: int | None = None,
                interleaved: bool = False, scaling: dict | None = None,
                device: torch.device | None = None,
                sections: Sequence[int] | None = None) -> RopeParams:
    """The frequencies base^(-2 i / rotary_dim) of the head's first rotary_dim elements (default:
    all), scaled for contexts longer than trained on:

      {"type": "linear", "factor": f}   positions divided by f
      {"type": "ntk", "factor": f}      base * f^(rotary_dim / (rotary_dim - 2)): the slowest pair
                                        divided by f, the fastest kept
      {"type": "yarn", "factor": f, "original_length": n, "beta_fast": 32, "beta_slow": 1}
                                        pairs that turn more than beta_fast times within n kept,
                                        less than beta_slow divided by f, a ramp between; cos and
                                        sin times 0.1 ln(f) + 1 (Peng et al., 2023)

    sections: how many pairs turn by each axis, in order (their sum is all pairs): (16, 24, 24) for
    time, height and width in a head of 128. Other orders: RopeParams with an `axes` of one's own.
    """
    rd = head_dim if rotary_dim is None else int(rotary_dim)
    if head_dim <= 0 or rd < 0 or rd > head_dim or rd % 2:
        raise ValueError(f"rotary_dim must be even and within head_dim {head_dim}, got {rd}")
    if not 0 < base < math.inf:
        raise ValueError("base must be positive and finite")
    if sections is not None:
        given = tuple(sections)
        sections = [int(x) if x == x // 1 else -1 for x in given]   # no parts of a pair
        if not sections or min(sections) < 0 or sum(sections) != rd // 2:
            raise ValueError(f"sections must be counts that add up to the {rd // 2} pairs, got {given}")
    i = torch.arange(0, rd, 2, dtype=torch.float64)
    factor = 1.0
    kind = None if scaling is None else scaling.get("type")
    if scaling is not None:
        known = {"linear": {"type", "factor"}, "ntk": {"type", "factor"},
                 "yarn": {"type", "factor", "original_length", "beta_fast", "beta_slow"}}
        if kind not in known or set(scaling) - known[kind]:
            raise ValueError(f"unknown rotary scaling {scaling!r}")
        if "factor" not in scaling or (kind == "yarn" and "original_length" not in scaling):
            raise ValueError(f"incomplete rotary scaling {scaling!r}")
        by = float(scaling["factor"])
        if not 1.0 <= by < math.inf:
            raise ValueError("the scaling factor must be at least 1 and finite")
    if kind == "ntk" and rd > 2:
        base = base * by ** (rd / (rd - 2))
    freq = base ** (-i / rd) if rd else i
    if kind == "linear":
        freq = freq / by
    elif kind == "yarn":
        n = int(scaling["original_length"])
        if n <= 0 or base == 1.0:
            raise ValueError("yarn needs a positive original_length and a base other than 1")

        fast, slow = (float(scaling.get(x, d)) for x, d in (("beta_fast", 32), ("beta_slow", 1)))
        if not 0 < slow <= fast < math.inf:
            raise ValueError("yarn's beta_slow must be positive and at most beta_fast")

        def pair_of(turns):   # the pair that turns so often within n positions
            return rd * math.log(n / (turns * 2 * math.pi)) / (2 * math.log(base))

        low = max(math.floor(pair_of(fast)), 0)
        high = min(math.ceil(pair_of(slow)), rd - 1)
        ramp = ((torch.arange(rd // 2, dtype=torch.float64) - low) / max(high - low, 1e-3))
        ramp = ramp.clamp(0.0, 1.0)
        freq = freq / by * ramp + freq * (1.0 - ramp)
        factor = 0.1 * math.log(by) + 1.0
    if device is None:
        device = torch.device("cuda", torch.cuda.current_device())
    axes = None
    if sections is not None:
        axes = torch.repeat_interleave(torch.arange(len(sections), dtype=torch.int32),
                                       torch.tensor(sections)).to(device)
    return RopeParams((freq / (2 * math.pi)).to(device), factor, bool(interleaved), axes)


def derived(*tensors: torch.Tensor | None) -> bool:
    """Whether a derivative in either mode is to be taken of any of them (tangents are looked up only
    inside a dual level)."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return getattr(forward_ad, "_current_level", -1) >= 0 and any(
        t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def check_rope(rope: RopeParams, head_dim: int, dev: torch.device) -> None:
    t = rope.turns
    if not t.is_cuda or t.get_device() != dev.index:
        raise ValueError(f"rope.turns is on {t.device}, expected {dev}")
    if t.dtype != torch.float64 or t.dim() != 1 or not t.is_contiguous():
        raise ValueError("rope.turns must be a contiguous float64 [pairs] tensor")
    if 2 * t.numel() > head_dim:
        raise ValueError(f"rope rotates {2 * t.numel()} elements of a head of {head_dim}")
    if derived(t):
        raise ValueError("rope.turns has no gradient: detach it")
    a = rope.axes
    if a is not None:
        if not a.is_cuda or a.get_device() != dev.index:
            raise ValueError(f"rope.axes is on {a.device}, expected {dev}")
        if a.dtype != torch.int32 or a.shape != t.shape or not a.is_contiguous():
            raise ValueError(f"rope.axes must be a contiguous int32 [{t.numel()}] tensor")


def fresh_like(t: torch.Tensor) -> torch.Tensor:
    """A contiguous tensor of t's shape and type (empty_like takes half the time of empty)."""
    if t.is_contiguous():
        return torch.empty_like(t)
    return torch.empty(t.shape, dtype=t.dtype, device=t.device)


def heads_view(name: str, t: torch.Tensor) -> torch.Tensor:
    """t with contiguous elements inside a head (its tokens and heads may be strided)."""
    if t.dim() != 3:
        raise ValueError(f"{name} must be [tokens, heads, head_dim], got {tuple(t.shape)}")
    return t if t.stride(2) == 1 or t.shape[2] == 1 else t.contiguous()


def _launch(q: torch.Tensor | None, k: torch.Tensor | None, positions: torch.Tensor,
            rope: RopeParams, transposed: bool) -> tuple[torch.Tensor | None, torch.Tensor | None]:
    qo = ko = qp = kp = None
    hq = hkv = qt = qh = kt = kh = 0
    if q is not None:
        q = heads_view("q", q)
        n, hq, D = q.shape
        qt, qh, _ = q.stride()
        qo = fresh_like(q)
        qp = q.data_ptr()
    if k is not None:
        k = heads_view("k", k)
        n, hkv, D = k.shape
        kt, kh, _ = k.stride()
        ko = fresh_like(k)
        kp = k.data_ptr()
    if n and hq + hkv:
        t, turns = (q if q is not None else k), rope.turns
        dev = t.device
        name, axes = "pia_rotary", ()
        if rope.axes is not None:
            name, axes = "pia_rotary_axes", (rope.axes.data_ptr(), positions.shape[0])
        N.call_on(dev, name, N.ptr(qo), N.ptr(ko), qp, kp, qt, qh, kt, kh,
                  positions.data_ptr(), 1 if positions.dtype == torch.int64 else 0, *axes,
                  turns.data_ptr(), turns.numel(), rope.factor, 1 if rope.interleaved else 0,
                  1 if transposed else 0, n, hq, hkv, D, N.dtype_code(t.dtype), N.stream_of(dev))
    return qo, ko


def _rotate(q: torch.Tensor | None, k: torch.Tensor | None, positions: torch.Tensor,
            rope: RopeParams, transposed: bool) -> tuple[torch.Tensor | None, torch.Tensor | None]:
    # a node of the graph is made only for what somebody differentiates
    if derived(q, k):
        return _Rotary.apply(q, k, positions, rope, transposed)
    return _launch(q, k, positions, rope, transposed)


class _Rotary(torch.autograd.Function):
    """The map is linear in q and k: its derivative along a tangent is itself, its gradient the
    transposed map, and so on."""

    @staticmethod
    def forward(ctx, q, k, positions, rope, transposed):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(positions, rope.turns, rope.axes)
        ctx.save_for_forward(positions, rope.turns, rope.axes)
        ctx.form = (rope.factor, rope.interleaved, transposed)
        out = _launch(q, k, positions, rope, transposed)
        ctx.shapes = [None if o is None else o.shape for o in out]
        return out

    @staticmethod
    def jvp(ctx, tq, tk, *_):
        positions, turns, axes = ctx.saved_tensors
        factor, interleaved, transposed = ctx.form
        t = tq if tq is not None else tk
        # of the two one may come without a tangent, and its result needs one
        tq, tk = (x if x is not None or s is None else t.new_zeros(s)
                  for x, s in zip((tq, tk), ctx.shapes))
        return _rotate(tq, tk, positions, RopeParams(turns, factor, interleaved, axes), transposed)

    @staticmethod
    def backward(ctx, gq, gk):
        gq, gk = (g if need else None for g, need in zip((gq, gk), ctx.needs_input_grad))
        if gq is None and gk is None:
            return None, None, None, None, None
        positions, turns, axes = ctx.saved_tensors
        factor, interleaved, transposed = ctx.form
        rope = RopeParams(turns, factor, interleaved, axes)
        return *_rotate(gq, gk, positions, rope, not transposed), None, None, None


def rotary_embed(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor,
                 rope: RopeParams) -> tuple[torch.Tensor, torch.Tensor | None]:
    """(q, k) rotated at their rows' positions. q [tokens, Hq, D], k [tokens, Hkv, D] or None, of one
    dtype (bf16, fp16 or fp32), tokens and heads at any strides; positions int64 or int32
    [tokens], with rope.axes [axes, tokens]. Contiguous results; derivatives of q and k in both modes. (A backward pass is
    captured into a graph only while no eager graph of the same leaves lives: torch's accumulation
    nodes keep the stream that made them, which is then part of the capture.)"""
    if k is None:
        dev = N.require_device(q, positions, names=("q", "positions"))
    else:
        dev = N.require_device(q, k, positions, names=("q", "k", "positions"))
    q = heads_view("q", q)
    n, _, D = q.shape
    if k is not None:
        k = heads_view("k", k)
        if k.shape[0] != n or k.shape[2] != D:
            raise ValueError(f"k must be [{n}, heads, {D}], got {tuple(k.shape)}")
        if k.dtype != q.dtype:
            raise ValueError("q and k must share a dtype")
    N.dtype_code(q.dtype)
    if positions.dtype not in (torch.int64, torch.int32):
        raise ValueError("positions must be int64 or int32")
    if rope.axes is None:
        if positions.shape != (n,):
            raise ValueError(f"positions must be int64 or int32 [{n}]")
    elif positions.dim() != 2 or positions.shape[0] == 0 or positions.shape[1] != n:
        raise ValueError(f"positions must be int64 or int32 [axes, {n}]")
    check_rope(rope, D, dev)
    positions = positions.contiguous()
    return _rotate(q, k, positions, rope, False)


__all__ = ["RopeParams", "rope_params", "rotary_embed"]
