"""Refusals of the entry points of windowed attention and of attention behind shared prefixes (CPU: no
compute call is made)."""

from __future__ import annotations

import pytest
import torch

from plastic_infer import _native as N
from plastic_infer.kernel import paged_prefix as PP, paged_window as PW

SOME = 1 << 20   # never dereferenced: every call below fails its checks first


def _window(**change):
    a = dict(out=2 * SOME, q=SOME, stride=4 * 64, k=SOME, v=SOME, bt=SOME, bts=4, lens=SOME, cu=None,
             offs=None, window=8, sinks=0, B=2, rows=2, Hq=4, Hkv=2, D=64, P=16, N=10, scale=1.0,
             dtype=2, ws=SOME, wsb=0, stream=None)
    assert set(change) <= set(a)
    N.call("pia_window_attention", *{**a, **change}.values())


def _prefix(**change):
    a = dict(out=2 * SOME, q=SOME, stride=4 * 64, k=SOME, v=SOME, pt=SOME, pts=4, plens=SOME, gs=None,
             groups=1, bt=SOME, bts=4, lens=SOME, cu=None, offs=None, B=2, rows=2, Hq=4, Hkv=2, D=64,
             P=16, N=10, scale=1.0, dtype=2, ws=SOME, wsb=0, stream=None)
    assert set(change) <= set(a)
    N.call("pia_prefix_attention", *{**a, **change}.values())


COMMON = [dict(dtype=3), dict(B=-1), dict(rows=-1), dict(Hq=0), dict(Hkv=0), dict(Hq=5), dict(N=0),
          dict(N=1 << 31), dict(N=1 << 30, Hkv=4), dict(bts=-1), dict(D=0), dict(P=0), dict(D=513),
          dict(P=4097), dict(rows=3), dict(rows=1 << 30, cu=SOME), dict(out=None), dict(q=None),
          dict(k=None), dict(v=None), dict(lens=None), dict(bt=None), dict(out=SOME + 64)]


@pytest.mark.parametrize("bad", COMMON + [dict(window=0), dict(window=-1), dict(sinks=-1)], ids=str)
def test_window(bad):
    with pytest.raises(N.NativeError, match="window_attention"):
        _window(**bad)


@pytest.mark.parametrize("bad", COMMON + [dict(groups=-1), dict(groups=2), dict(pts=-1),
                                          dict(pt=None), dict(plens=None)], ids=str)
def test_prefix(bad):
    with pytest.raises(N.NativeError, match="prefix_attention"):
        _prefix(**bad)


def test_tensors_on_the_host_are_refused():
    q, pool = torch.zeros(1, 2, 64), torch.zeros(2, 1, 64, 16)
    bt, n = torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="HIP"):
        PW.paged_window_decode_attention(q, pool, pool, bt, n, 4)
    with pytest.raises(ValueError, match="HIP"):
        PP.paged_prefix_decode_attention(q, pool, pool, bt, n, bt, n)


@pytest.mark.parametrize("window,sinks", [(0, 0), (-3, 0), (1.0, 0), (True, 0), (4, -1), (4, 0.5)])
def test_windows_are_whole_numbers(window, sinks):
    q, pool = torch.zeros(1, 2, 64), torch.zeros(2, 1, 64, 16)
    bt, n = torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="whole number"):
        PW.paged_window_decode_attention(q, pool, pool, bt, n, window, sinks)


def test_workspaces_that_do_not_do():
    need = N.query("pia_window_attention_workspace_bytes", 64)
    for bad in (dict(ws=None, wsb=need), dict(wsb=need - 1), dict(ws=SOME + 8, wsb=need), dict(wsb=0)):
        with pytest.raises(N.NativeError, match="window_attention: workspace"):
            _window(**bad)
    need = N.query("pia_prefix_attention_workspace_bytes", 2, 4, 64)
    for bad in (dict(ws=None, wsb=need), dict(wsb=need - 1), dict(ws=SOME + 8, wsb=need), dict(wsb=0)):
        with pytest.raises(N.NativeError, match="prefix_attention: workspace"):
            _prefix(**bad)


def test_workspace_bytes():
    def window(dim):
        return N.query("pia_window_attention_workspace_bytes", dim)

    def prefix(rows, heads, dim):
        return N.query("pia_prefix_attention_workspace_bytes", rows, heads, dim)

    assert window(64) > 0 and window(256) >= window(64)
    assert window(33) == window(512) == 0        # the general kernel's
    assert prefix(2, 4, 64) > window(64) and prefix(10 ** 6, 4, 64) > prefix(2, 4, 64)
    assert prefix(2, 4, 33) == prefix(0, 4, 64) == 0
