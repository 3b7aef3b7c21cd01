"""Rotary frequencies against their formulas, and the refusals of the C entry points of rotary
positions, appends and the 8-bit pool (CPU: no compute call is made)."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from plastic_infer import _native as N
from plastic_infer.kernel.paged_kv8 import KV8Pools, kv8_append, paged_decode_attention_kv8
from plastic_infer.kernel.kv_append import kv_append
from plastic_infer.kernel.rotary import RopeParams, rope_params, rotary_embed

CPU = torch.device("cpu")


@pytest.mark.parametrize("rd,base", [(2, 10000.0), (64, 10000.0), (96, 1e6)])
def test_plain_frequencies(rd, base):
    r = rope_params(128, base=base, rotary_dim=rd, device=CPU)
    assert r.turns.dtype == torch.float64 and r.rotary_dim == rd and r.factor == 1.0
    for i in range(rd // 2):
        assert abs(r.turns[i].item() * 2 * math.pi / base ** (-2 * i / rd) - 1) < 1e-14


def test_scaled_frequencies():
    plain = rope_params(64, device=CPU).turns
    lin = rope_params(64, scaling={"type": "linear", "factor": 4.0}, device=CPU)
    assert torch.allclose(lin.turns * 4, plain, rtol=1e-15, atol=0) and lin.factor == 1.0
    ntk = rope_params(64, scaling={"type": "ntk", "factor": 4.0}, device=CPU).turns
    assert ntk[0] == plain[0] and abs(plain[-1] / ntk[-1] - 4) < 1e-12
    yarn = rope_params(64, scaling={"type": "yarn", "factor": 8.0, "original_length": 4096},
                       device=CPU)
    assert abs(yarn.factor - (0.1 * math.log(8.0) + 1)) < 1e-15
    turned = plain * 4096     # turns of each pair within the original length
    for i in range(32):
        ratio = (plain[i] / yarn.turns[i]).item()
        assert 1 - 1e-12 <= ratio <= 8 + 1e-12
        if turned[i] > 64:
            assert ratio == 1.0
        if turned[i] < 0.5:
            assert abs(ratio - 8) < 1e-12


@pytest.mark.parametrize("kw", [dict(rotary_dim=3), dict(rotary_dim=130), dict(base=0.0),
                                dict(scaling={"type": "other", "factor": 2.0}),
                                dict(scaling={"type": "linear", "factor": 0.5}),
                                dict(scaling={"type": "linear", "factor": 2.0, "beta_fast": 1}),
                                dict(scaling={"type": "yarn", "factor": 2.0,
                                              "original_length": 0})])
def test_refused_parameters(kw):
    with pytest.raises(ValueError):
        rope_params(128, device=CPU, **kw)


def test_host_tensors_are_refused():
    rope = RopeParams(torch.zeros(4, dtype=torch.float64))
    x = torch.zeros(2, 2, 16)
    with pytest.raises(ValueError, match="HIP"):
        rotary_embed(x, x, torch.zeros(2, dtype=torch.int64), rope)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="HIP"):
        kv_append(x, x, x, torch.zeros(1, 2, 16, 16), torch.zeros(1, 2, 16, 16), i[:, None], i)
    pools = KV8Pools.allocate(1, 2, 16, 16, device=CPU)
    assert pools.shape == (1, 2, 16, 16) and pools.bytes_per_token == 2 * 2 * (16 + 0.25)
    with pytest.raises(ValueError, match="HIP"):
        kv8_append(x, x, x, pools, i[:, None], i)
    with pytest.raises(ValueError, match="HIP"):
        paged_decode_attention_kv8(x, pools, i[:, None], i)
    for d, p in ((24, 16), (272, 16), (16, 24), (16, 8192), (0, 16)):
        with pytest.raises(ValueError, match="multiples of 16"):
            KV8Pools.allocate(1, 1, d, p, device=CPU)


def _rc(name, *args):
    lib = N.load()
    return getattr(lib, name)(*args), lib.pia_last_error().decode()


def test_rotary_entry_point_refusals():
    def call(pairs=8, tokens=4, hq=2, hkv=1, d=16, dtype=2, ptr=None):
        return _rc("pia_rotary", ptr, ptr, ptr, ptr, 32, 16, 16, 16, ptr, 1, ptr, pairs, 1.0, 0, 0,
                   tokens, hq, hkv, d, dtype, None)
    assert call(dtype=9)[0] == -2
    assert call(pairs=9)[0] == -1 and call(pairs=-1)[0] == -1 and call(d=0)[0] == -1
    assert call(tokens=-1)[0] == -1
    rc, msg = call()
    assert rc == -1 and "null" in msg
    assert call(pairs=2100, d=8192)[0] == -2
    assert call(tokens=0)[0] == 0 and call(hq=0, hkv=0)[0] == 0     # nothing to do


def _append(scales=True, d=16, p=16, tokens=4, seqs=4, pairs=8, dtype=2, cu=None, one=False):
    buf = ctypes.create_string_buffer(64)
    s = ctypes.addressof(buf)
    return _rc("pia_kv_append", None, None, 0, 0, None, 16, 16, None, 16, 16, None, None,
               s if scales else None, s if scales and not one else None, None, 1, None, cu, tokens,
               seqs, None, pairs, 1.0, 0, 2, 1, d, p, 4, dtype, None)


def test_append_entry_point_refusals():
    assert _append(dtype=5)[0] == -2
    assert _append(d=24, pairs=4)[0] == -2 and _append(p=24)[0] == -2
    assert _append(d=1024)[0] == -2
    assert _append(scales=False, d=24, pairs=4)[1].endswith("null pointer")
    assert _append(one=True)[0] == -1
    assert _append(pairs=9)[0] == -1
    assert _append(tokens=5)[0] == -1            # without cu_new one token per sequence
    assert _append(tokens=0, seqs=0)[0] == 0
    rc, msg = _append()
    assert rc == -1 and "null" in msg


def test_kv8_entry_point_refusals():
    def attend(hq=4, hkv=2, d=16, p=16, rows=2, seqs=2, dtype=2, pages=4, ws=0):
        return _rc("pia_kv8_attention", None, None, 64, None, None, None, None, None, 1, None, None,
                   None, seqs, rows, hq, hkv, d, p, pages, 1.0, dtype, None, ws, None)
    assert attend(dtype=7)[0] == -2 and attend(d=8)[0] == -2 and attend(p=8)[0] == -2
    assert attend(hq=3)[0] == -1 and attend(rows=3)[0] == -1 and attend(pages=0)[0] == -1
    assert attend(rows=0, seqs=0)[0] == 0
    assert attend(pages=2 ** 31)[1].endswith("too large") and attend(rows=2 ** 30, seqs=2 ** 30)[0] == -1
    assert "null" in attend()[1]
    assert N.query("pia_kv8_attention_workspace_bytes", 0) == 0
    assert N.query("pia_kv8_attention_workspace_bytes", 300) == 0
    rc, _ = _rc("pia_kv8_gather", None, None, None, None, None, None, None, 1, None, 1, 4, 1, 20,
                16, 4, 2, None)
    assert rc == -2
    rc, msg = _rc("pia_kv8_gather", None, None, None, None, None, None, None, 1, None, 1, 4, 1, 16,
                  16, 4, 2, None)
    assert rc == -1 and "null" in msg
