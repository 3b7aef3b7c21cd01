"""Rotary positions on the GPU against the map in float64.

Bound of an element a c - b s: the rounding of the result (half a step of the type), and in fp32 those
of c and s (2^-24 of the factor each, their series' 2e-9 besides), of the product b s (2^-24) and of
the sum (2^-24): 3.1 * 2^-24 factor (|a| + |b|), taken as 2^-22."""

from __future__ import annotations

import pytest
import torch

import kv8_oracle as O
from plastic_infer.kernel.rotary import RopeParams, rope_params, rotary_embed

pytestmark = pytest.mark.gpu

STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
LEAST = {torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -14, torch.float32: 2.0 ** -126}


def _check(got, ref, size, dtype):
    assert got.dtype == dtype and got.is_contiguous() and got.shape == ref.shape
    bound = STEP[dtype] * ref.abs().clamp_min(LEAST[dtype]) + 2.0 ** -22 * size
    err = ((got.double().cpu() - ref).abs() / bound.clamp_min(1e-300)).max().item() \
        if ref.numel() else 0.0
    assert err <= 1.0, err


@pytest.mark.parametrize("dtype", list(STEP))
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,hq,hkv,dim,rd", [
    (1, 4, 1, 128, 128), (64, 32, 4, 128, 128), (7, 3, 2, 64, 64), (5, 2, 2, 128, 64),
    (9, 5, 1, 96, 48), (3, 2, 1, 80, 20), (4, 1, 1, 5, 4), (6, 2, 1, 7, 0), (2, 1, 3, 2, 2),
    (4200, 2, 1, 64, 32), (13, 2, 1, 256, 256)])
def test_against_float64(dev, dtype, interleaved, tokens, hq, hkv, dim, rd):
    g = torch.Generator().manual_seed(tokens + dim)
    q = torch.randn(tokens, hq, dim, generator=g).to(dtype)
    k = torch.randn(tokens, hkv, dim, generator=g).to(dtype)
    pos = torch.randint(0, 1 << 20, (tokens,), generator=g)
    rope = rope_params(dim, base=1e6, rotary_dim=rd, interleaved=interleaved,
                       scaling={"type": "yarn", "factor": 4.0, "original_length": 4096}
                       if rd == 64 else None, device=dev)
    qo, ko = rotary_embed(q.to(dev), k.to(dev), pos.to(dev), rope)
    for x, got in ((q, qo), (k, ko)):
        ref, size = O.turn(x, pos, rope.turns.cpu(), rope.factor, interleaved)
        _check(got, ref, size, dtype)
    only, none = rotary_embed(q.to(dev), None, pos.to(torch.int32).to(dev), rope)
    assert none is None and torch.equal(only, qo)


@pytest.mark.parametrize("offset", [0, 1, 8])
def test_strides_and_alignment(dev, offset):
    """Heads and tokens of a wider projection, views that start between vectors, expanded heads,
    transposed elements."""
    g = torch.Generator().manual_seed(3)
    wide = torch.randn(11, 9 * 64 + 8, generator=g).to(torch.bfloat16).to(dev)
    both = wide[:, offset:offset + 9 * 64].unflatten(1, (9, 64))
    pos = torch.arange(11, device=dev) * 977
    rope = rope_params(64, device=dev)
    q, k = rotary_embed(both[:, :6], both[:, 6:8], pos, rope)
    qc, kc = rotary_embed(both[:, :6].contiguous(), both[:, 6:8].contiguous(), pos, rope)
    assert torch.equal(q, qc) and torch.equal(k, kc)
    one = both[:, 8:9].expand(11, 3, 64)
    t = both[:, :2].transpose(1, 2).contiguous().transpose(1, 2)
    q, k = rotary_embed(one, t, pos, rope)
    assert torch.equal(q[:, 0], q[:, 2])
    assert torch.equal(k, rotary_embed(t.contiguous(), None, pos, rope)[0])


def test_negative_and_far_positions(dev):
    pos = torch.tensor([-5, 0, 1, (1 << 31) + 7, 10 ** 12])
    x = torch.randn(5, 1, 8, generator=torch.Generator().manual_seed(1))
    turns = torch.tensor([0.159154943, 0.01, 1e-7, 0.25], dtype=torch.float64)
    got, _ = rotary_embed(x.to(dev), None, pos.to(dev), RopeParams(turns.to(dev)))
    ref, size = O.turn(x, pos, turns, 1.0, False)
    # the product with the position is rounded in fp64: 2^-53 of 1.6e11 turns
    assert ((got.double().cpu() - ref).abs() <= (2.0 ** -22 + 2 * 3.15 * 1.6e11 * 2.0 ** -52) * size
            + 2.0 ** -24 * ref.abs()).all()
    assert torch.equal(got[1].cpu(), x[1])


def test_non_finite_elements_stay_in_their_pairs(dev):
    x = torch.ones(1, 1, 8, device=dev)
    x[0, 0, 1], x[0, 0, 7] = float("inf"), float("nan")
    rope = rope_params(8, rotary_dim=4, device=dev)
    got, _ = rotary_embed(x, None, torch.tensor([3], device=dev), rope)
    bad = ~torch.isfinite(got[0, 0])
    assert bad.tolist() == [False, True, False, True, False, False, False, True]


def test_empty_calls(dev):
    rope = rope_params(16, device=dev)
    none = torch.zeros(0, dtype=torch.int64, device=dev)
    q, k = rotary_embed(torch.zeros(0, 2, 16, device=dev), torch.zeros(0, 1, 16, device=dev), none,
                        rope)
    assert q.shape == (0, 2, 16) and k.shape == (0, 1, 16)
    q, k = rotary_embed(torch.zeros(3, 0, 16, device=dev), torch.ones(3, 1, 16, device=dev),
                        torch.zeros(3, dtype=torch.int64, device=dev), rope)
    assert q.shape == (3, 0, 16) and torch.equal(k, torch.ones_like(k))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
def test_gradients(dev, dtype, interleaved):
    """Against the formula (the transposed map) and, in fp32, against differences: the map is
    linear, so a difference is exact up to the roundings of its two values."""
    g = torch.Generator().manual_seed(8)
    q = torch.randn(6, 3, 32, generator=g).to(dtype)
    k = torch.randn(6, 1, 32, generator=g).to(dtype)
    gq, gk = torch.randn(6, 3, 32, generator=g).to(dtype), torch.randn(6, 1, 32, generator=g).to(dtype)
    pos = torch.arange(6) * 1000
    rope = rope_params(32, rotary_dim=24, interleaved=interleaved, device=dev,
                       scaling={"type": "yarn", "factor": 2.0, "original_length": 128})
    qd, kd = (t.to(dev).requires_grad_() for t in (q, k))
    qo, ko = rotary_embed(qd, kd, pos.to(dev), rope)
    a, b = torch.autograd.grad((qo, ko), (qd, kd), (gq.to(dev), gk.to(dev)))
    for got, grad in ((a, gq), (b, gk)):
        ref, size = O.turn(grad, pos, rope.turns.cpu(), rope.factor, interleaved, sign=-1.0)
        _check(got, ref, size, dtype)
    # one of two outputs, and one of two inputs
    qo, ko = rotary_embed(qd, kd.detach(), pos.to(dev), rope)
    only, = torch.autograd.grad(qo, qd, gq.to(dev))
    assert torch.equal(only, a)
    if dtype == torch.float32:
        step = torch.zeros_like(q)
        step[2, 1, 5] = 1.0
        with torch.no_grad():
            up = rotary_embed((q + step).to(dev), None, pos.to(dev), rope)[0].double()
            down = rotary_embed((q - step).to(dev), None, pos.to(dev), rope)[0].double()
        diff = ((up - down).cpu() / 2 * gq.double()).sum().item()
        assert abs(diff - a[2, 1, 5].item()) < 32 * 2.0 ** -20
        qq = q.to(dev).requires_grad_()
        out, _ = rotary_embed(qq, None, pos.to(dev), rope)
        cot = gq.to(dev).requires_grad_()
        first, = torch.autograd.grad(out, qq, cot, create_graph=True)
        again, = torch.autograd.grad(first, cot, q.to(dev))      # the gradient's own gradient
        assert torch.equal(again, out.detach())


def test_expanded_gradient_and_shared_heads(dev):
    """Gradients that autograd hands over as expanded views, and one leaf used by q and k both."""
    x = torch.randn(4, 2, 16, generator=torch.Generator().manual_seed(5)).to(dev).requires_grad_()
    pos = torch.arange(4, device=dev)
    rope = rope_params(16, device=dev)
    q, k = rotary_embed(x, x, pos, rope)
    (q.sum() + k.sum()).backward()
    one, _ = rotary_embed(x.detach().requires_grad_(), None, pos, rope)
    ref, size = O.turn(torch.ones(4, 2, 16), pos.cpu(), rope.turns.cpu(), 1.0, False, sign=-1.0)
    assert ((x.grad.double().cpu() - 2 * ref).abs() <= 2.0 ** -20 * size + 2.0 ** -23 * ref.abs()).all()


def test_refusals(dev):
    rope = rope_params(16, device=dev)
    q, pos = torch.zeros(2, 1, 16, device=dev), torch.zeros(2, dtype=torch.int64, device=dev)
    for args in ((q[0], None, pos, rope), (q, q[:1], pos, rope), (q, q.half(), pos, rope),
                 (q.double(), None, pos, rope), (q, None, pos[:1], rope),
                 (q, None, pos.float(), rope), (q[..., :8], None, pos, rope),
                 (q, None, pos, RopeParams(rope.turns.float())),
                 (q, None, pos.cpu(), rope)):
        with pytest.raises(ValueError):
            rotary_embed(*args)


def test_captured_forward_and_backward(dev):
    """A captured pass (gradients among it) follows its inputs on every replay, with eager work of
    the same tensors between the replays. No eager graph of the leaf lives while it is captured:
    its accumulation node would bring the stream that made it into the capture."""
    g = torch.Generator().manual_seed(2)
    q = torch.randn(33, 4, 64, generator=g).to(dev).requires_grad_()
    gq = torch.randn(33, 4, 64, generator=g).to(dev)
    pos = torch.arange(33, device=dev)
    rope = rope_params(64, device=dev)

    def step():
        out, _ = rotary_embed(q, None, pos, rope)
        return out.detach(), torch.autograd.grad(out, q, gq)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, grad = step()
    for i in range(4):
        with torch.no_grad():
            q.add_(1.0)
            pos.add_(5)
        graph.replay()
        eager, egrad = step()
        torch.cuda.synchronize()
        assert torch.equal(out, eager) and torch.equal(grad, egrad), i
