"""The 8-bit pools' checks, on the CPU: what a call takes is what the tensors are at that call."""

from __future__ import annotations

import pytest
import torch

from plastic_infer.kernel import paged_kv8 as P

CPU = torch.device("cpu")


@pytest.fixture
def pools(monkeypatch):
    monkeypatch.setattr(P.N, "require_device", lambda *tensors, names=None: tensors[0].device)
    p = P.KV8Pools.allocate(6, 2, 32, 32, CPU)
    assert P._check_pools(p) == (6, 2, 32, 32)      # a call before anything changes
    return p


@pytest.mark.parametrize("name", ["k", "v", "k_scale", "v_scale"])
def test_tensors_that_change_are_looked_at_again(pools, name):
    t = getattr(pools, name)
    whole = t.view(torch.uint8).clone().view(t.dtype)
    t.data = whole[:4].clone() if t.dtype == torch.float32 else \
        whole.view(torch.uint8)[:4].clone().view(t.dtype)
    with pytest.raises(ValueError):
        P._check_pools(pools)
    t.data = whole.transpose(0, 1).contiguous().transpose(0, 1) if t.dtype == torch.float32 else \
        whole.view(torch.uint8).transpose(0, 1).contiguous().transpose(0, 1).view(t.dtype)
    assert not t.is_contiguous()
    with pytest.raises(ValueError, match="contiguous"):
        P._check_pools(pools)
    t.data = whole
    assert P._check_pools(pools) == (6, 2, 32, 32)


def test_all_of_them_smaller(pools):
    for name in ("k", "v", "k_scale", "v_scale"):
        t = getattr(pools, name)
        t.data = t.view(torch.uint8)[:5].clone().view(t.dtype)
    assert P._check_pools(pools) == (5, 2, 32, 32)
