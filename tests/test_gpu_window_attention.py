"""Attention with a sliding window and sinks over the paged pools against float64 (bounds:
reach_oracle.check)."""

from __future__ import annotations

import pytest
import torch

import reach_oracle as O
from plastic_infer.kernel.paged_window import (
    paged_window_attention, paged_window_decode_attention, window_attention_workspace_bytes)

pytestmark = pytest.mark.gpu

I32 = torch.int32


def _case(lens, hq, hkv, dim, page, dtype, rows=None, seed=0, width=0):
    """(q, k, v, tables) on the CPU; rows: of each sequence (None: one each)."""
    g = torch.Generator().manual_seed(1000 + seed)
    pages = sum(-(-n // page) for n in lens) + 3
    order = torch.randperm(pages, generator=g).tolist()
    k, v = O.pools(pages, hkv, dim, page, dtype, seed)
    n = len(lens) if rows is None else sum(rows)
    q = torch.randn(n, hq, dim, generator=g).to(dtype)
    return q, k, v, O.tables(lens, page, order, width)


def _on(dev, *tensors):
    return [t.to(dev) for t in tensors]


def _ints(dev, x):
    return torch.tensor(x, dtype=I32, device=dev)


def _cu(rows):
    return [sum(rows[:i]) for i in range(len(rows) + 1)]


DECODE = [  # lens, window, sinks, Hq, Hkv, D, P
    ([1], 1, 0, 4, 1, 128, 16),
    ([0, 3, 64, 65, 1], 64, 4, 8, 2, 128, 16),
    ([200, 17, 1000, 33], 31, 5, 32, 8, 128, 16),
    ([127, 128, 129, 130], 128, 1, 7, 1, 64, 32),
    ([500, 20], 10 ** 12, 0, 5, 5, 64, 16),
    ([90, 31, 400], 16, 100, 16, 1, 128, 64),       # sinks beyond the context and the window
    ([70, 2, 300], 70, 16, 40, 2, 96, 16),
    ([33, 170], 1, 33, 34, 2, 80, 48),              # more than 16 heads to a kv head
    ([300, 40], 129, 64, 4, 2, 256, 16),
    ([50, 51], 49, 1, 3, 1, 16, 16),
    ([100, 260], 130, 7, 6, 2, 208, 32),
    ([77, 4], 30, 3, 4, 2, 33, 16),                 # an odd head_dim
    ([77, 130], 64, 3, 4, 2, 64, 5),                # odd pages
    ([41, 90], 20, 2, 2, 1, 512, 8),
    ([5000, 1], 2048, 4, 8, 1, 128, 16),
    ([2100, 800, 3], 1000, 0, 4, 4, 64, 128),
]


@pytest.mark.parametrize("dtype", list(O.STEP))
@pytest.mark.parametrize("case", DECODE, ids=lambda c: f"{c[0]}w{c[1]}s{c[2]}h{c[3]}/{c[4]}d{c[5]}p{c[6]}")
def test_decode(dev, case, dtype):
    lens, window, sinks, hq, hkv, dim, page = case
    q, k, v, bt = _case(lens, hq, hkv, dim, page, dtype)
    got = paged_window_decode_attention(*_on(dev, q, k, v, bt), _ints(dev, lens), window, sinks)
    O.check(got, *O.windowed(q, k, v, bt, lens, window, sinks), dtype)


ROWS = [  # rows, contexts (rows among them), offsets (None: the last rows), window, sinks, Hq, Hkv, D, P
    ([1, 3, 0, 6], [40, 300, 20, 6], None, 17, 2, 8, 2, 128, 16),
    ([5, 2], [100, 90], [-3, 200], 30, 4, 4, 1, 64, 16),     # rows before the start and past the end
    ([40, 70], [40, 200], [0, 130], 25, 1, 8, 4, 128, 16),
    ([130], [700], [570], 64, 0, 16, 2, 128, 16),
    ([130], [700], [570], 100, 70, 16, 4, 64, 32),
    ([100, 33, 1, 64], [100, 533, 7, 64], [0, 500, 6, 0], 1, 3, 6, 2, 96, 16),
    ([200], [200], [0], 5000, 4, 5, 1, 128, 16),             # the window holds everything
    ([200, 90], [1200, 100], [1000, 10], 300, 17, 32, 8, 128, 16),
    ([64], [64], [0], 64, 0, 2, 2, 16, 16),
    ([66, 70], [90, 70], [24, 0], 33, 2, 4, 2, 256, 16),
    ([30, 70], [90, 70], [60, 0], 33, 2, 4, 2, 80, 8),
    ([300], [260], [100], 90, 20, 8, 1, 128, 64),            # rows past the cached keys
    ([257], [1300], None, 513, 128, 4, 1, 128, 16),
]


@pytest.mark.parametrize("dtype", list(O.STEP))
@pytest.mark.parametrize("case", ROWS, ids=lambda c: f"{c[0]}of{c[1]}w{c[3]}s{c[4]}h{c[5]}/{c[6]}d{c[7]}p{c[8]}")
def test_rows(dev, case, dtype):
    rows, lens, offs, window, sinks, hq, hkv, dim, page = case
    q, k, v, bt = _case(lens, hq, hkv, dim, page, dtype, rows)
    cu = _cu(rows)
    got = paged_window_attention(*_on(dev, q, k, v, bt), _ints(dev, lens), window, sinks,
                                 _ints(dev, cu), None if offs is None else _ints(dev, offs))
    O.check(got, *O.windowed(q, k, v, bt, lens, window, sinks, cu, offs), dtype, rows=True)


@pytest.mark.parametrize("dtype", list(O.STEP))
@pytest.mark.parametrize("rows", [2, 70])
def test_values_in_unseen_places_do_not_matter(dev, dtype, rows):
    """NaN and infinities behind the window, past the causal limit, past the context and on pages that
    only some rows see: they reach the rows that see them and no others."""
    lens, window, sinks, page = [300], 40, 3, 16
    q, k, v, bt = _case(lens, 8, 2, 128, page, dtype, [rows], seed=7)
    first = 300 - rows - 10           # the last 10 tokens are seen by nobody
    k[bt[0, 18], :, :, 12:] = float("nan")                # past the context
    v[bt[0, 18], :, :, 12:] = float("inf")
    edits = [(5, float("nan")), (100, float("inf")), (295, float("nan")),
             (first + rows - 2, float("inf")),            # the last two rows see it
             (first - window + 1, float("-inf"))]         # the first row alone does
    for t, x in edits:
        v[bt[0, t // page], :, 1:7, t % page] = x
    k[bt[0, 6], 1, 2, 6] = float("nan")                   # token 102, behind every window
    cu, offs = [0, rows], [first]
    got = paged_window_attention(*_on(dev, q, k, v, bt), _ints(dev, lens), window, sinks,
                                 _ints(dev, cu), _ints(dev, offs))
    ref = O.windowed(q, k, v, bt, lens, window, sinks, cu, offs)
    assert ref[0].isinf().any() and ref[0].isfinite().any()
    O.check(got, *ref, dtype, rows=True)


@pytest.mark.parametrize("dtype", list(O.STEP))
def test_nan_and_infinite_keys_and_values_that_are_seen(dev, dtype):
    lens = [50, 200, 90]
    q, k, v, bt = _case(lens, 4, 2, 64, 16, dtype, seed=3)
    k[bt[0, 2], 0, 5, 1] = float("nan")       # token 33 of the first: its heads 0 and 1 are NaN
    v[bt[1, 12], 1, 9, 2] = float("inf")      # token 194 of the second
    v[bt[2, 5], :, 3, 9] = float("inf")       # tokens 89 and 88 of the third: NaN
    v[bt[2, 5], :, 3, 8] = float("-inf")
    got = paged_window_decode_attention(*_on(dev, q, k, v, bt), _ints(dev, lens), 32, 1)
    ref = O.windowed(q, k, v, bt, lens, 32, 1)
    assert ref[0].isnan().any() and ref[0].isinf().any()
    O.check(got, *ref, dtype)


def test_pages_given_up_and_pages_that_are_not_there(dev):
    lens, window, sinks, page = [400, 130], 60, 16, 16
    q, k, v, bt = _case(lens, 8, 2, 128, page, torch.bfloat16, seed=5)
    whole = paged_window_decode_attention(*_on(dev, q, k, v, bt), _ints(dev, lens), window, sinks)
    gone = bt.clone()
    gone[0, 1:21] = torch.tensor([-1, 10 ** 6] * 10, dtype=I32)    # tokens 16 .. 335 of 400
    got = paged_window_decode_attention(*_on(dev, q, k, v, gone), _ints(dev, lens), window, sinks)
    assert torch.equal(got, whole)
    gone[0, 22] = -5                    # a page that is seen: its tokens are no keys
    gone[1] = k.shape[0]                # every page of the second: zeros
    got = paged_window_decode_attention(*_on(dev, q, k, v, gone), _ints(dev, lens), window, sinks)
    O.check(got, *O.windowed(q, k, v, gone, lens, window, sinks), torch.bfloat16)
    assert (got[1] == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [[1, 1], [3, 2], [90, 50]])
def test_rows_of_no_sequence_and_out_in_place(dev, dtype, rows):
    lens = [100, 260]
    q, k, v, bt = _case(lens, 8, 2, 64, 16, dtype, [4, *rows, 5], seed=9)
    cu = [4, 4 + rows[0], 4 + sum(rows)]
    args = _on(dev, k, v, bt)
    buf = q.to(dev)
    out = paged_window_attention(buf, *args, _ints(dev, lens), 50, 2, _ints(dev, cu), out=buf)
    assert out.data_ptr() == buf.data_ptr()
    assert torch.equal(out[:4].cpu(), q[:4]) and torch.equal(out[cu[2]:].cpu(), q[cu[2]:])
    ref, mag, size, keys = O.windowed(q, k, v, bt, lens, 50, 2, cu)
    inner = slice(4, cu[2])
    O.check(out[inner], ref[inner], mag[inner], size[inner], keys, dtype, rows=True)


def test_strided_and_misaligned_q_and_scale(dev):
    lens = [100, 30]
    q, k, v, bt = _case(lens, 4, 2, 64, 16, torch.float16, seed=2)
    args = _on(dev, k, v, bt)
    base = torch.zeros(2, 3, 4, 64, dtype=torch.float16, device=dev)
    base[:, 1] = q.to(dev)
    odd = torch.zeros(q.numel() + 1, dtype=torch.float16, device=dev)
    odd[1:] = q.to(dev).flatten()
    for scale in (0.3, -0.2, 0.0):
        ref = O.windowed(q, k, v, bt, lens, 20, 1, scale=scale)
        for x in (base[:, 1], odd[1:].view(q.shape),
                  q.to(dev).transpose(1, 2).contiguous().transpose(1, 2)):
            got = paged_window_decode_attention(x, *args, _ints(dev, lens), 20, 1, scale)
            O.check(got, *ref, torch.float16)
        # the same as rows, where the kernel for many rows would not take every scale
        many = q.repeat_interleave(40, 0)
        cu = [0, 40, 80]
        ref = O.windowed(many, k, v, bt, lens, 20, 1, cu, [60, 0], scale)
        got = paged_window_attention(many.to(dev), *args, _ints(dev, lens), 20, 1, _ints(dev, cu),
                                     _ints(dev, [60, 0]), scale)
        O.check(got, *ref, torch.float16, rows=True)


def test_a_whole_window_is_plain_attention(dev):
    from plastic_infer.kernel.paged_kv import paged_attention

    rows, lens = [80, 33], [300, 40]
    q, k, v, bt = _case(lens, 8, 2, 128, 16, torch.bfloat16, rows)
    cu, offs = _ints(dev, _cu(rows)), _ints(dev, [220, 7])
    args = _on(dev, q, k, v, bt) + [_ints(dev, lens)]
    got = paged_window_attention(*args, 10 ** 6, 0, cu, offs)
    want = paged_attention(*args, cu, offs)
    ref = O.windowed(q, k, v, bt, lens, 10 ** 6, 0, _cu(rows), [220, 7])
    O.check(got, *ref, torch.bfloat16, rows=True)
    O.check(want, *ref, torch.bfloat16, rows=True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [None, [3, 1, 5, 2], [90, 30, 200, 7]])
def test_captured_replayed_and_repeated(dev, dtype, rows):
    lens = [400, 90, 1500, 7]
    q, k, v, bt = _case(lens, 8, 2, 128, 16, dtype, rows)
    q, k, v, bt = _on(dev, q, k, v, bt)
    lens_t = _ints(dev, lens)
    cu = None if rows is None else _ints(dev, _cu(rows))
    ws = torch.full((max(1, window_attention_workspace_bytes(128)),), 0x7f, dtype=torch.uint8,
                    device=dev)

    def call():
        return paged_window_attention(q, k, v, bt, lens_t, 300, 4, cu, workspace=ws)

    first = call()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    with torch.cuda.graph(other):
        out2 = call()       # two graphs that share a workspace, replayed in turn
    for i in range(4):
        if i:
            q.normal_()
            lens_t.sub_(1)
        ws.fill_(0xff if i % 2 else 0)
        graph.replay()
        other.replay()
        torch.cuda.synchronize()
        want = call()
        assert torch.equal(out, want) and torch.equal(out2, want)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):       # another stream, a workspace of its own
            apart = paged_window_attention(q, k, v, bt, lens_t, 300, 4, cu)
        side.synchronize()
        assert torch.equal(apart, want)
        if i == 0:
            assert torch.equal(want, first)


def test_more_sequences_than_a_launch_holds(dev):
    n = 2100
    lens = [(7 * i) % 90 for i in range(n)]
    g = torch.Generator().manual_seed(0)
    k, v = O.pools(40, 1, 64, 16, torch.bfloat16, 0)
    bt = torch.randint(0, 40, (n, 6), generator=g, dtype=I32)
    q = torch.randn(n, 2, 64, generator=g).to(torch.bfloat16)
    got = paged_window_decode_attention(*_on(dev, q, k, v, bt), _ints(dev, lens), 20, 1)
    O.check(got, *O.windowed(q, k, v, bt, lens, 20, 1), torch.bfloat16)
    two = q.repeat_interleave(2, 0)
    cu = [2 * i for i in range(n + 1)]
    got = paged_window_attention(*_on(dev, two, k, v, bt), _ints(dev, lens), 20, 1, _ints(dev, cu))
    O.check(got, *O.windowed(two, k, v, bt, lens, 20, 1, cu), torch.bfloat16, rows=True)


@pytest.mark.parametrize("rows", [None, [2], [80]])
def test_pool_beyond_32_bits(dev, rows):
    # 2^31 elements lie 4 GB into a pool: pages beyond that, and a context of which little is read
    pages, page = 2 ** 31 // (2 * 128 * 64) + 40, 64
    k = torch.zeros(pages, 2, 128, page, dtype=torch.bfloat16, device=dev)
    v = torch.zeros_like(k)
    g = torch.Generator().manual_seed(1)
    few = torch.randn(30, 2, 128, page, generator=g).to(torch.bfloat16)
    k[-30:], v[-30:] = few.to(dev), few.flip(0).to(dev)
    length, window = 30 * page - 5, 200
    bt = torch.arange(pages - 30, pages, dtype=I32)[None]
    n = 1 if rows is None else rows[0]
    q = torch.randn(n, 8, 128, generator=g).to(torch.bfloat16)
    cu = None if rows is None else [0, n]
    got = paged_window_attention(q.to(dev), k, v, bt.to(dev), _ints(dev, [length]), window, 3,
                                 None if cu is None else _ints(dev, cu))
    small = (bt - (pages - 30)).contiguous()
    O.check(got, *O.windowed(q, few, few.flip(0), small, [length], window, 3, cu), torch.bfloat16,
            rows=rows is not None)


def test_empty_calls(dev):
    q, k, v, bt = _case([5], 2, 1, 64, 16, torch.float32)
    q, k, v, bt = _on(dev, q, k, v, bt)
    none = torch.zeros(0, dtype=I32, device=dev)
    assert paged_window_decode_attention(q[:0], k, v, bt[:0], none, 4).shape == (0, 2, 64)
    got = paged_window_decode_attention(q, k, v, bt[:, :0], _ints(dev, [5]), 4)
    assert (got == 0).all()


def test_refusals(dev):
    q, k, v, bt = _case([40, 50], 4, 2, 64, 16, torch.bfloat16)
    q, k, v, bt = _on(dev, q, k, v, bt)
    lens = _ints(dev, [40, 50])

    def call(window=8, sinks=1, q=q, k=k, v=v, bt=bt, lens=lens, **more):
        return paged_window_attention(q, k, v, bt, lens, window, sinks, **more)

    for bad in (dict(window=0), dict(window=-1), dict(window=2.0), dict(window=True),
                dict(sinks=-1), dict(sinks=1.5), dict(q=q[:, :3]), dict(q=q[:1]),
                dict(q=q.float()), dict(q=q[..., :32]), dict(lens=lens.long()), dict(lens=lens[:1]),
                dict(bt=bt.long()), dict(bt=bt[0]), dict(v=v[:2]), dict(v=v.half()),
                dict(k=k.transpose(0, 1)), dict(cu_q=lens), dict(cu_q=_ints(dev, [0, 1, 2]).long()),
                dict(q_pos_offsets=lens[:1]), dict(out=q[:1]), dict(out=q.float()),
                dict(lens=lens.cpu()), dict(q=q.cpu())):
        with pytest.raises(ValueError):
            call(**bad)
    with pytest.raises(ValueError, match="gradient"):
        call(q=q.float().requires_grad_(), k=k.float(), v=v.float())
    from plastic_infer._native import NativeError
    buf = torch.zeros(3, 4, 64, dtype=torch.bfloat16, device=dev)
    with pytest.raises(NativeError, match="overlaps"):
        call(q=buf[:2], out=buf[1:])
    call()      # and nothing of that is left behind
    torch.cuda.synchronize()
