"""Rotary positions with several axes against float64, their gradients against the formula's and
differences, and their refusals.

Bound of an element x c - y s (c, s within an fp32 rounding of their exact values: 2^-24 |factor|, as
much from the angle, whose fp64 error is 2^-53 of its turns): three fp32 roundings of the products and
the sum, 2^-24 each, so 5 * 2^-24 |factor| (|x| + |y|), and half a step of the type."""

from __future__ import annotations

import math

import pytest
import torch

from plastic_infer.kernel.kv_append import kv_append
from plastic_infer.kernel.rotary import RopeParams, rope_params, rotary_embed

pytestmark = pytest.mark.gpu

STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
LEAST = {torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -14, torch.float32: 2.0 ** -126}


def _turned(x, positions, rope, sign=1.0):
    """(exact result, |x| + |y| of each element's pair) in fp64 on the CPU."""
    x, turns, axes = x.detach().double().cpu(), rope.turns.cpu(), rope.axes.cpu().long()
    p = positions.cpu().double()
    there = (axes >= 0) & (axes < p.shape[0])
    pos = torch.where(there[:, None], p[axes.clamp(0, p.shape[0] - 1)], torch.zeros(()).double())
    a = 2 * math.pi * torch.remainder(pos.t() * turns, 1.0)[:, None]
    c, s = rope.factor * torch.cos(a), sign * rope.factor * torch.sin(a)
    n = 2 * turns.numel()
    lo, hi = (slice(0, n, 2), slice(1, n, 2)) if rope.interleaved else \
        (slice(0, n // 2), slice(n // 2, n))
    out, size = x.clone(), torch.zeros_like(x)
    out[..., lo], out[..., hi] = x[..., lo] * c - x[..., hi] * s, x[..., hi] * c + x[..., lo] * s
    size[..., lo] = size[..., hi] = x[..., lo].abs() + x[..., hi].abs()
    return out, size


def _check(got, x, positions, rope, sign=1.0):
    ref, size = _turned(x, positions, rope, sign)
    assert got.dtype == x.dtype and got.shape == x.shape and got.is_contiguous()
    bound = STEP[x.dtype] * ref.abs().clamp_min(LEAST[x.dtype]) + \
        5 * 2.0 ** -24 * abs(rope.factor) * size
    err = (got.detach().double().cpu() - ref).abs()
    assert (err <= bound).all(), (err / bound.clamp_min(1e-300)).max().item()


def _rope(dev, pairs, axes, factor=1.0, interleaved=False):
    turns = 1e4 ** (-torch.arange(pairs, dtype=torch.float64) / max(pairs, 1)) / (2 * math.pi)
    return RopeParams(turns.to(dev), factor, interleaved,
                      torch.tensor(axes, dtype=torch.int32, device=dev))


def _inputs(dev, n, hq, hkv, dim, dtype, num_axes, kind=torch.int64, seed=0):
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(n, hq, dim, generator=g).to(dtype).to(dev)
    k = torch.randn(n, hkv, dim, generator=g).to(dtype).to(dev)
    pos = torch.randint(0, 100000, (num_axes, n), generator=g).to(kind).to(dev)
    return q, k, pos


CASES = [  # tokens, Hq, Hkv, D, axes of the pairs, number of axes
    (1, 4, 1, 128, [0] * 16 + [1] * 24 + [2] * 24, 3),
    (7, 3, 3, 64, [i % 3 for i in range(32)], 3),
    (300, 8, 2, 96, [0, 1] * 12, 2),
    (65, 2, 1, 20, [3, 2, 1, 0, 0], 4),
    (5, 1, 1, 2, [0], 1),
    (9, 2, 2, 8, [1, -1, 2, 0], 2),      # two pairs without an axis of theirs
]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", list(STEP))
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{c[0]}x{c[1]}/{c[2]}d{c[3]}a{c[5]}")
def test_forward(dev, case, dtype, interleaved):
    n, hq, hkv, dim, axes, num_axes = case
    rope = _rope(dev, len(axes), axes, 1.25, interleaved)
    q, k, pos = _inputs(dev, n, hq, hkv, dim, dtype, num_axes)
    qo, ko = rotary_embed(q, k, pos, rope)
    _check(qo, q, pos, rope)
    _check(ko, k, pos, rope)


def test_alike_axes_give_the_bits_of_one_axis(dev):
    q, k, pos = _inputs(dev, 33, 4, 2, 128, torch.bfloat16, 3, torch.int32)
    rope = _rope(dev, 64, [0] * 16 + [1] * 24 + [2] * 24)
    same = pos[1:2].expand(3, -1)
    for a, b in zip(rotary_embed(q, k, same, rope),
                    rotary_embed(q, k, pos[1], RopeParams(rope.turns))):
        assert torch.equal(a, b)


def test_strided_inputs_positions_and_k_alone(dev):
    both = torch.randn(12, 10, 2, 64, device=dev)[:, :, 0]
    q, k = both[:, :8], both[:, 8:]
    rope = _rope(dev, 32, [i % 2 for i in range(32)])
    pos = torch.randint(0, 5000, (12, 2), device=dev).t()
    qo, ko = rotary_embed(q, k, pos, rope)
    _check(qo, q, pos, rope)
    _check(ko, k, pos, rope)
    only, none = rotary_embed(q, None, pos, rope)
    assert none is None and torch.equal(only, qo)
    empty, _ = rotary_embed(q[:0], None, pos[:, :0], rope)
    assert empty.shape == (0, 8, 64)


@pytest.mark.parametrize("dtype", list(STEP))
def test_gradients_are_the_transposed_map(dev, dtype):
    q, k, pos = _inputs(dev, 70, 4, 2, 64, dtype, 3)
    rope = _rope(dev, 32, [i % 3 for i in range(32)], 0.75)
    q.requires_grad_()
    k.requires_grad_()
    gq, gk = torch.randn_like(q), torch.randn_like(k)
    out = rotary_embed(q, k, pos, rope)
    dq, dk = torch.autograd.grad(out, (q, k), (gq, gk))
    _check(dq, gq, pos, rope, sign=-1.0)
    _check(dk, gk, pos, rope, sign=-1.0)


def test_gradients_against_differences(dev):
    # the map is linear: differences of any size have no error but roundings
    q, k, pos = _inputs(dev, 6, 2, 1, 16, torch.float32, 2)
    rope = _rope(dev, 8, [0, 1, 1, 0, 1, 0, 0, 1])
    q.requires_grad_()
    g = torch.randn_like(q)
    (dq,) = torch.autograd.grad(rotary_embed(q, None, pos, rope)[0], q, g)
    for at in ((0, 0, 0), (3, 1, 9), (5, 0, 15)):
        step = torch.zeros_like(q)
        step[at] = 1.0
        with torch.no_grad():
            up, down = (rotary_embed(q + s * step, None, pos, rope)[0].double() for s in (1, -1))
        slope = ((up - down) / 2 * g.double()).sum().item()
        # the pair's two elements, of values below 6 with the step: 60 * 2^-24 from either result by the
        # bound above, a few 2^-24 from the rounding of q + step; together below 2^-16
        assert abs(slope - dq[at].item()) <= 2.0 ** -16 * g.abs().max().item()


def test_second_derivative_and_tangent(dev):
    q, _, pos = _inputs(dev, 5, 2, 1, 8, torch.float32, 2)
    rope = _rope(dev, 4, [0, 1, 0, 1])
    q.requires_grad_()
    g = torch.randn_like(q, requires_grad=True)
    (dq,) = torch.autograd.grad(rotary_embed(q, None, pos, rope)[0], q, g, create_graph=True)
    w = torch.randn_like(dq)
    (dg,) = torch.autograd.grad(dq, g, w)
    _check(dg, w, pos, rope)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(q.detach(), w)
        out, _ = rotary_embed(dual, None, pos, rope)
        _check(torch.autograd.forward_ad.unpack_dual(out).tangent, w, pos, rope)


def test_captured_and_replayed(dev):
    q, k, pos = _inputs(dev, 40, 4, 2, 128, torch.bfloat16, 3)
    rope = rope_params(128, sections=(16, 24, 24), device=dev)
    rotary_embed(q, k, pos, rope)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = rotary_embed(q, k, pos, rope)
    for i in range(3):
        q.normal_()
        pos.add_(i)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, rotary_embed(q, k, pos, rope)):
            assert torch.equal(a, b)


def test_refusals(dev):
    q, k, pos = _inputs(dev, 4, 2, 1, 8, torch.float32, 3)
    rope = _rope(dev, 4, [0, 1, 2, 0])
    with pytest.raises(ValueError, match="axes, 4"):
        rotary_embed(q, k, pos[0], rope)
    with pytest.raises(ValueError, match="axes, 4"):
        rotary_embed(q, k, pos[:, :3], rope)
    with pytest.raises(ValueError, match="axes, 4"):
        rotary_embed(q, k, pos[:0], rope)
    with pytest.raises(ValueError, match="int64 or int32"):
        rotary_embed(q, k, pos.float(), rope)
    with pytest.raises(ValueError, match=r"\[4\]"):
        rotary_embed(q, k, pos, RopeParams(rope.turns))
    with pytest.raises(ValueError, match="rope.axes"):
        rotary_embed(q, k, pos, RopeParams(rope.turns, axes=rope.axes.cpu()))
    with pytest.raises(ValueError, match="rope.axes"):
        rotary_embed(q, k, pos, RopeParams(rope.turns, axes=rope.axes.long()))
    with pytest.raises(ValueError, match="rope.axes"):
        rotary_embed(q, k, pos, RopeParams(rope.turns, axes=rope.axes[:3]))
    pool = torch.zeros(2, 1, 8, 16, device=dev)
    with pytest.raises(ValueError, match="several axes"):
        kv_append(q, k, k, pool, pool.clone(), torch.zeros(4, 1, dtype=torch.int32, device=dev),
                  torch.ones(4, dtype=torch.int32, device=dev), rope=rope)
