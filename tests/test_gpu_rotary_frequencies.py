"""Frequencies that ask for a derivative, which the rotary calls do not have."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from plastic_infer.kernel.kv_append import kv_append
from plastic_infer.kernel.rotary import RopeParams, rope_params, rotary_embed

pytestmark = pytest.mark.gpu


def test_refused(dev):
    q, pos = torch.ones(4, 2, 16, device=dev), torch.arange(4, device=dev)
    turns = rope_params(16, device=dev).turns
    want, _ = rotary_embed(q, None, pos, RopeParams(turns))
    leaf = turns.clone().requires_grad_()
    pools = [torch.zeros(4, 2, 16, 16, device=dev) for _ in "kv"]
    bt, n = (torch.arange(4, dtype=torch.int32, device=dev)[:, None],
             torch.ones(4, dtype=torch.int32, device=dev))
    with pytest.raises(ValueError, match="gradient"):
        rotary_embed(q, None, pos, RopeParams(leaf))
    with pytest.raises(ValueError, match="gradient"):
        kv_append(q, q, q, *pools, bt, n, rope=RopeParams(leaf))
    with torch.no_grad():      # nobody asks for one
        assert torch.equal(rotary_embed(q, None, pos, RopeParams(leaf))[0], want)
    with forward_ad.dual_level():
        with pytest.raises(ValueError, match="gradient"):
            rotary_embed(q, None, pos, RopeParams(forward_ad.make_dual(turns, turns)))
