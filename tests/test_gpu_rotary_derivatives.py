"""Derivatives of the rotary map in both modes, and calls that record none refusing tensors that carry one.

The map is linear in q and k: a tangent is turned as its tensor is, by the same kernel, so the bits are those
of the call on the tangent alone."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from plastic_infer.kernel import rotary as R
from plastic_infer.kernel.kv_append import kv_append
from plastic_infer.kernel.paged_kv8 import (
    KV8Pools, kv8_append, paged_attention_kv8, paged_decode_attention_kv8)
from plastic_infer.kernel.rotary import RopeParams, rope_params, rotary_embed

pytestmark = pytest.mark.gpu


def _inputs(dev, dtype=torch.float32, seed=1):
    g = torch.Generator().manual_seed(seed)
    q, tq = (torch.randn(5, 3, 32, generator=g).to(dtype).to(dev) for _ in range(2))
    k, tk = (torch.randn(5, 1, 32, generator=g).to(dtype).to(dev) for _ in range(2))
    return q, k, tq, tk, torch.arange(5, device=dev) * 1000


@pytest.mark.parametrize("no_grad", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_forward_mode(dev, dtype, no_grad):
    q, k, tq, tk, pos = _inputs(dev, dtype)
    rope = rope_params(32, rotary_dim=24, device=dev)
    want, wtan = rotary_embed(q, k, pos, rope), rotary_embed(tq, tk, pos, rope)
    tangent = lambda x: forward_ad.unpack_dual(x).tangent  # noqa: E731
    with forward_ad.dual_level(), torch.set_grad_enabled(not no_grad):
        dq, dk = forward_ad.make_dual(q, tq), forward_ad.make_dual(k, tk)
        qo, ko = rotary_embed(dq, dk, pos, rope)
        assert torch.equal(tangent(qo), wtan[0]) and torch.equal(tangent(ko), wtan[1])
        assert torch.equal(forward_ad.unpack_dual(qo).primal, want[0])
        qo, ko = rotary_embed(dq, k, pos, rope)               # one of the two
        assert torch.equal(tangent(qo), wtan[0])
        assert tangent(ko) is None or not tangent(ko).any()
        qo, ko = rotary_embed(q, dk, pos, rope)
        assert torch.equal(tangent(ko), wtan[1])
        assert tangent(qo) is None or not tangent(qo).any()
        qo, none = rotary_embed(dq, None, pos, rope)
        assert none is None and torch.equal(tangent(qo), wtan[0])
        wide = forward_ad.make_dual(q.expand(2, 5, 3, 32)[0].transpose(0, 1).contiguous()
                                    .transpose(0, 1), tq)     # strided
        assert torch.equal(tangent(rotary_embed(wide, None, pos, rope)[0]), wtan[0])
        qo, ko = rotary_embed(q, k, pos, rope)                # inside a level, without a tangent
        assert torch.equal(qo, want[0]) and tangent(qo) is None


def test_forward_over_reverse(dev):
    """The gradient's derivative along a tangent of what it is the gradient of: the cotangent's."""
    q, k, tq, _, pos = _inputs(dev)
    rope = rope_params(32, interleaved=True, device=dev)
    back = R._launch(tq, None, pos, rope, True)[0]
    for graph in (False, True):
        with forward_ad.dual_level():
            leaf = q.clone().requires_grad_()
            out, _ = rotary_embed(leaf, None, pos, rope)
            grad, = torch.autograd.grad(out, leaf, forward_ad.make_dual(q, tq), create_graph=graph)
            assert torch.equal(forward_ad.unpack_dual(grad).tangent, back)


def test_reverse_over_forward(dev):
    q, k, tq, _, pos = _inputs(dev)
    rope = rope_params(32, device=dev)
    tq.requires_grad_()
    with forward_ad.dual_level():
        out, _ = rotary_embed(forward_ad.make_dual(q, tq), None, pos, rope)
        tangent = forward_ad.unpack_dual(out).tangent
        grad, = torch.autograd.grad(tangent, tq, k.expand(5, 3, 32))
    assert torch.equal(grad, R._launch(k.expand(5, 3, 32), None, pos, rope, True)[0])


def test_calls_without_derivatives_refuse_tangents(dev):
    q, k = torch.ones(1, 2, 32, device=dev), torch.ones(1, 1, 32, device=dev)
    pools = KV8Pools.allocate(2, 1, 32, 16, dev)
    kp, vp = (torch.zeros(2, 1, 32, 16, device=dev) for _ in "kv")
    bt = torch.zeros(1, 1, dtype=torch.int32, device=dev)
    n = torch.ones(1, dtype=torch.int32, device=dev)
    with forward_ad.dual_level(), torch.no_grad():
        dual = lambda x: forward_ad.make_dual(x, torch.ones_like(x))  # noqa: E731
        for args in ((dual(q), k, k), (q, dual(k), k), (None, k, dual(k))):
            with pytest.raises(ValueError, match="gradient"):
                kv8_append(*args, pools, bt, n)
            with pytest.raises(ValueError, match="gradient"):
                kv_append(*args, kp, vp, bt, n)
        with pytest.raises(ValueError, match="gradient"):
            paged_decode_attention_kv8(dual(q), pools, bt, n)
        with pytest.raises(ValueError, match="gradient"):
            paged_attention_kv8(dual(q), pools, bt, n)
        assert (pools.k_scale == 0).all() and (kp == 0).all()        # nothing was written
        kv8_append(q, k, k, pools, bt, n)                            # no tangent: as ever
        assert (paged_decode_attention_kv8(q, pools, bt, n) == 1).all()
