"""What a decoder's layer_hook is handed as k over float and over 8-bit pools.

Bound of a rotated bf16 element: test_gpu_rotary.py's. A code of the pool is within half a step of it: 2^-4
of the value, or 2^-10 of the scale."""

from __future__ import annotations

import math

import pytest
import torch

import kv8_oracle as O
from plastic_infer.exec.runner_moe_paged import (
    DecodeBatch, MoeModelConfig, MoePagedDecoder, random_dense_weights, random_expert_banks)
from plastic_infer.kernel.paged_kv8 import KV8Pools
from plastic_infer.moe.offload_cache import OffloadMoeCache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [8, 16])
def test_k_of_the_hook(dev, bits):
    cfg = MoeModelConfig(n_layers=1, n_heads=4, n_kv_heads=2, head_dim=64, hidden_dim=64, vocab_size=8,
                         max_seq_len=64, n_experts=2, n_experts_per_tok=1, moe_intermediate_dim=64,
                         rope_base=10000.0)
    cache = OffloadMoeCache(1, 2, 2, dev)
    cache.set_bank_sources(random_expert_banks(cfg, dev, seed=4, std=0.1))
    lens, page = [23, 1, 40], 16
    tables = torch.arange(9, dtype=torch.int32).view(1, 3, 3)
    pools = kp = vp = None
    if bits == 8:
        pools = KV8Pools.allocate(9, 2, 64, page, dev)
    else:
        kp, vp = (torch.zeros(9, 2, 64, page, dtype=cfg.dtype, device=dev) for _ in "kv")
    dec = MoePagedDecoder(random_dense_weights(cfg, dev, seed=3, std=0.1), cfg, cache, kp, vp,
                          max_batch=3, kv8_pools=pools)
    seen = {}
    dec.layer_hook = lambda l, d: seen.update({x: d[x].cpu() for x in ("k", "k_rotated")})
    lens_t = torch.tensor(lens, dtype=torch.int32)
    dec.step(torch.tensor([3, 1, 7], device=dev),
             DecodeBatch(tables.to(dev), lens_t.to(dev), torch.empty(1, 3, dtype=torch.int64),
                         (lens_t - 1).long().to(dev)))
    turned = seen["k_rotated"]
    if bits == 16:
        assert torch.equal(turned, seen["k"])
    else:
        turns = 10000.0 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64) / (2 * math.pi)
        ref, size = O.turn(seen["k"], lens_t.long() - 1, turns, 1.0, False)
        assert ((turned.double() - ref).abs() <= 2.0 ** -8 * ref.abs().clamp_min(2.0 ** -126)
                + 2.0 ** -22 * size).all()
    for b, n in enumerate(lens):      # what the pool holds of the new token
        i, o = int(tables[0, b, (n - 1) // page]), (n - 1) % page
        if bits == 16:
            assert torch.equal(kp[i, :, :, o].cpu(), turned[b])
            continue
        pool = O.Pool.from_device(pools)
        held, unit = pool.values("k")[i, :, o], pool.scale["k"][i, :, o // O.BLOCK, None]
        # of the exact value, whose rounding to bf16 turned is
        assert ((held - ref[b]).abs() <= (2.0 ** -4 + 2.0 ** -20) * ref[b].abs() + 2.0 ** -10 * unit).all()
