"""What a call of prefix attention asks of its workspace, on the CPU (no compute call is made)."""

from __future__ import annotations

import itertools

import pytest

from plastic_infer import _native as N

MB = 1 << 20
CALL = dict(groups=1, pts=256, bts=2048, ragged=1, B=8, rows=8192, Hq=32, Hkv=8, D=128, P=16, scale=0.1,
            dtype=2)


def _bytes(**change):
    assert set(change) <= set(CALL)
    return N.query("pia_prefix_attention_call_workspace_bytes", *{**CALL, **change}.values())


def _bound(rows=8192, Hq=32, D=128, **_):
    return N.query("pia_prefix_attention_workspace_bytes", rows, Hq, D)


@pytest.mark.parametrize("rows", [8192, 100_000, 1_000_000])
@pytest.mark.parametrize("dtype", [1, 2])
def test_many_rows_of_a_sequence_take_none(rows, dtype):
    assert _bytes(rows=rows, dtype=dtype) == 0
    assert _bound(rows=rows) > 8 * rows * 32 * 128


@pytest.mark.parametrize("shape", [dict(D=33), dict(D=512), dict(P=5), dict(D=33, ragged=0, B=8192)], ids=str)
def test_the_general_kernel_takes_none(shape):
    assert _bytes(**shape) == 0


@pytest.mark.parametrize("heads", [(8, 8), (32, 8), (128, 1), (8, 1)])
def test_items_that_are_cut_are_few_rows(heads):
    Hq, Hkv = heads
    seen = set()
    for rows, B, D, tokens in itertools.product((64, 100, 300, 1000, 3000, 8192, 70_000), (1, 2, 8),
                                                (16, 64, 96, 128, 256), (10, 4096, 1 << 17)):
        if rows * Hq // Hkv < 64 * B:
            continue                       # few rows of a sequence: pieces of all rows
        need = _bytes(B=B, rows=rows, Hq=Hq, Hkv=Hkv, D=D, pts=tokens // 16 + 1, bts=tokens // 16 + 1)
        assert 0 <= need <= min(_bound(rows=rows, Hq=Hq, D=D), 128 * MB)
        seen.add(need > 0)
    assert seen == {False, True}


@pytest.mark.parametrize("few", [dict(ragged=0, B=8192), dict(B=4096), dict(dtype=0), dict(scale=-0.1),
                                 dict(Hq=129 * 8, rows=256, B=64)], ids=str)
def test_pieces_of_all_rows_take_the_bound(few):
    assert _bytes(**few) == _bound(**{**CALL, **few})
    # without a prefix there are none
    rest = _bytes(**few, groups=0)
    assert rest == _bytes(**few, pts=0) and 0 < rest < 70 * MB


@pytest.mark.parametrize("bad", [dict(B=0), dict(rows=0), dict(rows=-1), dict(Hq=0), dict(Hkv=0), dict(Hq=33),
                                 dict(D=0), dict(P=0), dict(P=-16), dict(pts=-1), dict(bts=-1)], ids=str)
def test_calls_that_are_none(bad):
    assert _bytes(**bad) == 0


def test_too_little_is_refused():
    some = 1 << 20    # never dereferenced: every call below fails its checks
    few = dict(CALL, ragged=0, B=8192)
    need = _bytes(**few)
    for ws, given in ((None, need), (some, need - 1), (some, 0), (some + 8, need)):
        with pytest.raises(N.NativeError, match="prefix_attention: workspace"):
            N.call("pia_prefix_attention", some << 12, some, 32 * 128, some, some, some, 256, some, None,
                   1, some, 2048, some, None, None, 8192, 8192, 32, 8, 128, 16, 10, 0.1, 2, ws, given,
                   None)
