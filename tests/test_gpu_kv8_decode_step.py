"""The MoE decode step over 8-bit pools: what each layer appends, and its attention, against float64
over the tensors that the layer hands out and the values that the pools then hold.

Bounds: a code is within half a step of its value, 2^-4 of it or 2^-10 scales; the attention's are
test_gpu_kv8_attention's."""

from __future__ import annotations

import math

import pytest
import torch

import kv8_oracle as O
from plastic_infer.exec.runner_moe_paged import (
    DecodeBatch, MoeModelConfig, MoePagedDecoder, random_dense_weights, random_expert_banks)
from plastic_infer.kernel.paged_kv8 import KV8Pools
from plastic_infer.moe.offload_cache import OffloadMoeCache
from test_gpu_kv8_attention import _check, _tables

pytestmark = pytest.mark.gpu


def _decoder(dev, cfg, pools, **kw):
    cache = OffloadMoeCache(cfg.n_layers, cfg.n_experts, cfg.n_layers * cfg.n_experts, dev)
    cache.set_bank_sources(random_expert_banks(cfg, dev, seed=4, std=0.1))
    return MoePagedDecoder(random_dense_weights(cfg, dev, seed=3, std=0.1), cfg, cache, None, None,
                           max_batch=8, kv8_pools=pools, **kw)


@pytest.mark.parametrize("qk_norm", [True, False])
def test_steps_over_8_bit_pools(dev, qk_norm):
    cfg = MoeModelConfig(n_layers=2, n_heads=8, n_kv_heads=2, head_dim=128, hidden_dim=256,
                         vocab_size=96, max_seq_len=512, n_experts=16, n_experts_per_tok=4,
                         moe_intermediate_dim=64, rope_base=10000.0, qk_norm=qk_norm)
    lens, steps, page = [0, 15, 130, 63], 3, 16    # before the first step
    L, B = cfg.n_layers, len(lens)
    rows, pages = _tables([n + steps for n in lens] * L, page, 1, 5)
    tables = rows.view(L, B, -1)
    pools = O.Pool.random(pages, cfg.n_kv_heads, cfg.head_dim, page, seed=2).to_device(dev)
    dec = _decoder(dev, cfg, pools)
    turns = 10000.0 ** (-torch.arange(0, 128, 2, dtype=torch.float64) / 128) / (2 * math.pi)
    seen = []

    def hook(l, d):
        pool, pos = O.Pool.from_device(pools), torch.tensor(lens) - 1
        q, k, v, attn = (d[x].cpu() for x in ("q", "k", "v", "attn"))
        cu, t = list(range(B + 1)), tables[l].tolist()
        _check(attn, *O.attend(q, pool, t, lens, cu, None, 128 ** -0.5), torch.bfloat16, max(lens), 128)
        new = {"k": O.turn(k, pos, turns, 1.0, False)[0], "v": v.double()}
        for x in "kv":
            for b in range(B):
                i, o = t[b][int(pos[b]) // page], int(pos[b]) % page
                held = pool.values(x)[i, :, o]
                half = (2.0 ** -4 + 2.0 ** -20) * new[x][b].abs() + 2.0 ** -10 * pool.scale[x][i]
                assert ((held - new[x][b]).abs() <= half).all()
        seen.append(l)

    dec.layer_hook = hook
    for step in range(steps):
        lens = [n + 1 for n in lens]
        lens_t = torch.tensor(lens, dtype=torch.int32)
        batch = DecodeBatch(tables.to(dev), lens_t.to(dev), torch.empty(L, B, dtype=torch.int64),
                            (lens_t - 1).long().to(dev))
        logits = dec.step(torch.tensor([3, 90, 17, step], device=dev), batch)
        assert logits.shape == (B, cfg.vocab_size) and torch.isfinite(logits.float()).all()
    assert seen == [0, 1] * steps


def test_pools_of_the_decoder(dev):
    cfg = MoeModelConfig(n_layers=1, n_heads=4, n_kv_heads=2, head_dim=64, hidden_dim=64, vocab_size=8,
                         max_seq_len=64, n_experts=2, n_experts_per_tok=1, moe_intermediate_dim=64)
    pools = KV8Pools.allocate(4, 2, 64, 16, dev)
    kp = torch.zeros(4, 2, 64, 16, dtype=torch.bfloat16, device=dev)
    for k, kv8 in ((kp, pools), (None, KV8Pools.allocate(4, 2, 32, 16, dev)), (None, None)):
        with pytest.raises(ValueError):
            MoePagedDecoder({}, cfg, None, k, k, max_batch=1, kv8_pools=kv8)
