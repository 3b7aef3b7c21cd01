"""Attention behind shared prefixes over the paged pools against float64 (bounds: reach_oracle.check)."""

from __future__ import annotations

import pytest
import torch

import reach_oracle as O
from plastic_infer.kernel.kv_append import kv_append
from plastic_infer.kernel.paged_prefix import (
    paged_prefix_attention, paged_prefix_decode_attention, prefix_attention_workspace_bytes)
from plastic_infer.kernel.paged_window import paged_window_decode_attention
from plastic_infer.kernel.rotary import rope_params, rotary_embed

pytestmark = pytest.mark.gpu

I32 = torch.int32


def _case(plens, lens, hq, hkv, dim, page, dtype, rows=None, seed=0):
    """(q, k, v, prefix tables, tables) on the CPU."""
    g = torch.Generator().manual_seed(2000 + seed)
    pages = sum(-(-n // page) for n in [*plens, *lens]) + 3
    order = torch.randperm(pages, generator=g).tolist()
    k, v = O.pools(pages, hkv, dim, page, dtype, seed)
    n = len(lens) if rows is None else sum(rows)
    q = torch.randn(n, hq, dim, generator=g).to(dtype)
    return q, k, v, O.tables(plens, page, order), O.tables(lens, page, order)


def _on(dev, *tensors):
    return [t.to(dev) for t in tensors]


def _ints(dev, x):
    return torch.tensor(x, dtype=I32, device=dev)


def _cu(rows):
    return [sum(rows[:i]) for i in range(len(rows) + 1)]


def _run(dev, q, k, v, pt, plens, bt, lens, cu_seqs=None, cu=None, offs=None, **more):
    q, k, v, pt, bt = _on(dev, q, k, v, pt, bt)
    opt = [None if x is None else _ints(dev, x) for x in (cu_seqs, cu, offs)]
    return paged_prefix_attention(q, k, v, pt, _ints(dev, plens), bt, _ints(dev, lens), *opt, **more)


DECODE = [  # prefixes, own lengths, cu_seqs, Hq, Hkv, D, P
    ([1], [0], None, 4, 1, 128, 16),
    ([300], [5, 0, 64, 1], None, 8, 2, 128, 16),
    ([1000], [17] * 9 + [200] * 40, None, 8, 2, 128, 16),
    ([0], [3, 0], None, 4, 2, 64, 16),                        # no prefix, and a row without a key
    ([70, 0, 130, 9], [3, 20, 0, 8, 100, 2], [0, 2, 3, 3, 5], 7, 1, 64, 32),   # an empty group, a loner
    ([40, 500], [30] * 12, [2, 7, 11], 6, 2, 96, 16),         # sequences before and behind the groups
    ([257], [10] * 20, None, 16, 1, 128, 64),
    ([90], [33, 2], None, 34, 2, 80, 48),
    ([300], [40] * 10, None, 4, 2, 256, 16),
    ([100], [20, 60], None, 6, 2, 208, 32),
    ([77], [4, 30], None, 4, 2, 33, 16),
    ([77, 20], [130, 3, 2], [0, 1, 3], 4, 2, 64, 5),
    ([41], [9, 2], None, 2, 1, 512, 8),
    ([3000], [100] * 33, None, 4, 4, 64, 128),
    ([2500], list(range(0, 130, 2)), None, 5, 1, 128, 16),
]


@pytest.mark.parametrize("dtype", list(O.STEP))
@pytest.mark.parametrize("case", DECODE, ids=lambda c: f"{c[0]}+{len(c[1])}x{max(c[1])}h{c[3]}/{c[4]}d{c[5]}p{c[6]}")
def test_decode(dev, case, dtype):
    plens, lens, cu_seqs, hq, hkv, dim, page = case
    q, k, v, pt, bt = _case(plens, lens, hq, hkv, dim, page, dtype)
    got = _run(dev, q, k, v, pt, plens, bt, lens, cu_seqs)
    # rows of a group are many together, and the prefix's probabilities may be rounded once
    O.check(got, *O.prefixed(q, k, v, pt, plens, bt, lens, cu_seqs), dtype, rows=True)


MANY = [  # prefixes, own lengths, cu_seqs, Hq, Hkv, D, P: both parts side by side over 16-bit pools
    ([700, 130], [i % 70 for i in range(60)], [3, 30, 58], 6, 2, 96, 16),     # loners at both ends
    ([300], [500] * 24, None, 8, 2, 80, 32),
    ([1500, 0, 64], [i * 7 % 300 for i in range(90)], [0, 40, 50, 90], 4, 1, 64, 16),
    ([400, 90], [20 + i for i in range(48)], [0, 24, 48], 12, 3, 48, 48),
    ([5000], [33] * 70, None, 32, 8, 128, 16),
    ([200], [2500] * 20, None, 4, 1, 128, 16),        # own tokens beyond what goes side by side
]


@pytest.mark.parametrize("dtype", list(O.STEP))
@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("case", MANY, ids=lambda c: f"{c[0]}+{len(c[1])}x{max(c[1])}h{c[3]}/{c[4]}d{c[5]}p{c[6]}")
def test_many_sequences(dev, case, dtype, ragged):
    plens, lens, cu_seqs, hq, hkv, dim, page = case
    rows = [1 + i % 3 for i in range(len(lens))] if ragged else None
    cu = _cu(rows) if ragged else None
    q, k, v, pt, bt = _case(plens, lens, hq, hkv, dim, page, dtype, rows, seed=len(lens))
    got = _run(dev, q, k, v, pt, plens, bt, lens, cu_seqs, cu)
    O.check(got, *O.prefixed(q, k, v, pt, plens, bt, lens, cu_seqs, cu), dtype, rows=True)


ROWS = [  # prefixes, rows, contexts, offsets, cu_seqs, Hq, Hkv, D, P
    ([100], [1, 3, 0, 6], [40, 30, 20, 6], [39, 27, 20, 0], None, 8, 2, 128, 16),
    ([60], [5, 2], [10, 9], [-8, 20], None, 4, 1, 64, 16),     # rows that see no own key yet
    ([300], [40, 70], [40, 200], [0, 130], None, 8, 4, 128, 16),
    ([64, 1000], [130, 65, 200], [130, 70, 333], [0, 5, 133], [0, 1, 3], 16, 2, 128, 16),
    ([500, 20], [100, 33, 1, 64], [100, 533, 7, 0], None, [0, 2, 3], 6, 2, 96, 32),
    ([65], [66, 70], [90, 70], [24, 0], None, 4, 2, 256, 16),
    ([30], [30, 70], [90, 70], [60, 0], None, 4, 2, 80, 8),
    ([0], [100], [100], [0], None, 8, 2, 64, 16),
    ([700], [200, 90], [200, 100], [0, 10], None, 32, 8, 128, 16),
    ([900], [4] * 30, [4] * 30, [0] * 30, None, 8, 2, 128, 16),
    ([129], [257], [0], None, None, 4, 1, 128, 64),
]


@pytest.mark.parametrize("dtype", list(O.STEP))
@pytest.mark.parametrize("case", ROWS, ids=lambda c: f"{c[0]}+{len(c[1])}x{max(c[1])}h{c[5]}/{c[6]}d{c[7]}p{c[8]}")
def test_rows(dev, case, dtype):
    plens, rows, lens, offs, cu_seqs, hq, hkv, dim, page = case
    q, k, v, pt, bt = _case(plens, lens, hq, hkv, dim, page, dtype, rows)
    got = _run(dev, q, k, v, pt, plens, bt, lens, cu_seqs, _cu(rows), offs)
    O.check(got, *O.prefixed(q, k, v, pt, plens, bt, lens, cu_seqs, _cu(rows), offs), dtype, rows=True)


@pytest.mark.parametrize("dtype", list(O.STEP))
@pytest.mark.parametrize("rows", [None, [2, 3, 1], [70, 20, 90]])
def test_values_in_unseen_places_do_not_matter(dev, dtype, rows):
    plens, lens = [75], [90, 23, 95]
    q, k, v, pt, bt = _case(plens, lens, 8, 2, 128, 16, dtype, rows, seed=4)
    cu = None if rows is None else _cu(rows)
    offs = None if rows is None else [n - r for n, r in zip(lens, rows)]
    for table, n in ((pt[0], 75), (bt[0], 90), (bt[1], 23), (bt[2], 95)):
        k[table[n // 16], :, :, n % 16:] = float("nan")        # past the prefix, past the contexts
        v[table[n // 16], :, :, n % 16:] = float("inf")
    v[bt[0, 5], :, 1:7, 9] = float("-inf")                     # the last token: only the last row's
    v[pt[0, 2], :, 40, 3] = float("inf")                       # in the prefix: everybody's
    got = _run(dev, q, k, v, pt, plens, bt, lens, None, cu, offs)
    ref = O.prefixed(q, k, v, pt, plens, bt, lens, None, cu, offs)
    assert ref[0].isinf().any() and ref[0].isfinite().any()
    O.check(got, *ref, dtype, rows=True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_nan_keys_reach_whoever_sees_them(dev, dtype):
    plens, lens = [200, 90], [30, 40, 50, 60]
    q, k, v, pt, bt = _case(plens, lens, 4, 2, 64, 16, dtype, seed=3)
    k[pt[1, 2], 0, 5, 1] = float("nan")       # the second group's heads 0 and 1
    k[bt[0, 1], 1, 5, 1] = float("nan")       # the first sequence's heads 2 and 3
    got = _run(dev, q, k, v, pt, plens, bt, lens, [0, 2, 4])
    ref = O.prefixed(q, k, v, pt, plens, bt, lens, [0, 2, 4])
    assert 0 < ref[0].isnan().sum() < ref[0].numel()
    O.check(got, *ref, dtype, rows=True)


@pytest.mark.parametrize("rows", [None, [80, 70]])
def test_pages_that_are_not_there(dev, rows):
    plens, lens = [200], [90, 33]
    q, k, v, pt, bt = _case(plens, lens, 8, 2, 128, 16, torch.float16, rows)
    cu = None if rows is None else _cu(rows)
    pt[0, 3], pt[0, 7], bt[0, 0], bt[1] = -1, 10 ** 6, k.shape[0], -7
    got = _run(dev, q, k, v, pt, plens, bt, lens, None, cu)
    O.check(got, *O.prefixed(q, k, v, pt, plens, bt, lens, None, cu), torch.float16, rows=True)
    pt[:], bt[:] = -1, -1
    assert (_run(dev, q, k, v, pt, plens, bt, lens, None, cu) == 0).all()


def test_lengths_beyond_the_tables(dev):
    plens, lens = [70], [20, 30]
    q, k, v, pt, bt = _case(plens, lens, 8, 2, 128, 16, torch.bfloat16)
    got = _run(dev, q, k, v, pt, [10 ** 9], bt, [10 ** 9, -4])
    O.check(got, *O.prefixed(q, k, v, pt, [10 ** 9], bt, [10 ** 9, -4]), torch.bfloat16, rows=True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [[1, 1], [3, 2], [90, 50]])
def test_rows_of_no_sequence_and_out_in_place(dev, dtype, rows):
    plens, lens = [130], [100, 60]
    q, k, v, pt, bt = _case(plens, lens, 8, 2, 64, 16, dtype, [4, *rows, 5], seed=9)
    cu = [4, 4 + rows[0], 4 + sum(rows)]
    qd, kd, vd, ptd, btd = _on(dev, q, k, v, pt, bt)
    out = paged_prefix_attention(qd, kd, vd, ptd, _ints(dev, plens), btd, _ints(dev, lens), None,
                                 _ints(dev, cu), out=qd)
    assert out.data_ptr() == qd.data_ptr()
    assert torch.equal(out[:4].cpu(), q[:4]) and torch.equal(out[cu[2]:].cpu(), q[cu[2]:])
    ref, mag, size, keys = O.prefixed(q, k, v, pt, plens, bt, lens, None, cu)
    inner = slice(4, cu[2])
    O.check(out[inner], ref[inner], mag[inner], size[inner], keys, dtype, rows=True)


@pytest.mark.parametrize("scale", [0.3, -0.2, 0.0])
def test_strided_q_and_scale(dev, scale):
    plens, lens = [150], [30] * 20
    q, k, v, pt, bt = _case(plens, lens, 8, 2, 64, 16, torch.float16, seed=2)
    ref = O.prefixed(q, k, v, pt, plens, bt, lens, scale=scale)
    base = torch.zeros(20, 3, 8, 64, dtype=torch.float16, device=dev)
    base[:, 1] = q.to(dev)
    args = _on(dev, k, v, pt) + [_ints(dev, plens), bt.to(dev), _ints(dev, lens)]
    for x in (base[:, 1], q.to(dev).transpose(1, 2).contiguous().transpose(1, 2)):
        got = paged_prefix_decode_attention(x, *args, scale=scale)
        O.check(got, *ref, torch.float16, rows=True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [None, [2] * 24, [90] * 6 + [5] * 18])
def test_captured_replayed_and_repeated(dev, dtype, rows):
    plens, lens = [600, 200], [100 + 3 * i for i in range(24)]
    q, k, v, pt, bt = _on(dev, *_case(plens, lens, 8, 2, 128, 16, dtype, rows))
    plens_t, lens_t, gs = _ints(dev, plens), _ints(dev, lens), _ints(dev, [0, 17, 24])
    cu = None if rows is None else _ints(dev, _cu(rows))
    ws = torch.full((max(1, prefix_attention_workspace_bytes(q.shape[0], 8, 128)),), 0x7f,
                    dtype=torch.uint8, device=dev)

    def call(ws=ws):
        return paged_prefix_attention(q, k, v, pt, plens_t, bt, lens_t, gs, cu, workspace=ws)

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
            lens_t.sub_(7)
            plens_t.sub_(31)
        ws.fill_(0xff if i % 2 else 0)
        graph.replay()
        other.replay()
        torch.cuda.synchronize()
        want = call()
        assert torch.equal(out, want) and torch.equal(out2, want)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):       # another stream, a workspace of its own
            apart = call(None)
        side.synchronize()
        assert torch.equal(apart, want)
        if i == 0:
            assert torch.equal(want, first)


def test_more_sequences_than_a_launch_holds(dev):
    n = 2100
    plens, cu_seqs = [50, 90, 20], [0, 700, 701, 2050]
    lens = [(7 * i) % 40 for i in range(n)]
    g = torch.Generator().manual_seed(0)
    k, v = O.pools(40, 1, 64, 16, torch.bfloat16, 0)
    bt = torch.randint(0, 40, (n, 3), generator=g, dtype=I32)
    pt = torch.randint(0, 40, (3, 6), generator=g, dtype=I32)
    q = torch.randn(n, 2, 64, generator=g).to(torch.bfloat16)
    got = _run(dev, q, k, v, pt, plens, bt, lens, cu_seqs)
    O.check(got, *O.prefixed(q, k, v, pt, plens, bt, lens, cu_seqs), torch.bfloat16, rows=True)


def test_more_groups_than_a_launch_holds(dev):
    n = 1500
    plens = [(11 * i) % 70 for i in range(n)]
    g = torch.Generator().manual_seed(0)
    k, v = O.pools(40, 1, 64, 16, torch.bfloat16, 0)
    bt = torch.randint(0, 40, (2 * n, 1), generator=g, dtype=I32)
    pt = torch.randint(0, 40, (n, 5), generator=g, dtype=I32)
    lens = [i % 17 for i in range(2 * n)]
    q = torch.randn(2 * n, 8, 64, generator=g).to(torch.bfloat16)
    cu_seqs = [2 * i for i in range(n + 1)]
    got = _run(dev, q, k, v, pt, plens, bt, lens, cu_seqs)
    O.check(got, *O.prefixed(q, k, v, pt, plens, bt, lens, cu_seqs), torch.bfloat16, rows=True)


@pytest.mark.parametrize("rows", [None, [80] * 40])
def test_pool_beyond_32_bits(dev, rows):
    pages, page = 2 ** 31 // (2 * 128 * 64) + 40, 64
    k = torch.zeros(pages, 2, 128, page, dtype=torch.bfloat16, device=dev)
    v = torch.zeros_like(k)
    g = torch.Generator().manual_seed(1)
    few = torch.randn(30, 2, 128, page, generator=g).to(torch.bfloat16)
    k[-30:], v[-30:] = few.to(dev), few.flip(0).to(dev)
    lens, plens = [1 + i for i in range(40)], [15 * page - 5]
    pt = torch.arange(15, dtype=I32)[None]
    bt = (15 + torch.arange(40, dtype=I32) % 15)[:, None]
    n = 40 if rows is None else sum(rows)
    q = torch.randn(n, 8, 128, generator=g).to(torch.bfloat16)
    cu = None if rows is None else _cu(rows)
    args = [x.to(dev) for x in (pt + pages - 30, bt + pages - 30)]
    got = paged_prefix_attention(q.to(dev), k, v, args[0], _ints(dev, plens), args[1],
                                 _ints(dev, lens), None, None if cu is None else _ints(dev, cu))
    if rows is not None:     # the oracle is slow: some of the rows
        keep = [0, 79, 80, 1700, n - 1]
        one = [i // 80 for i in keep]
        ref = O.prefixed(q[keep], few, few.flip(0), pt, plens, bt[one], [lens[i] for i in one])
        got = got[keep]
    else:
        ref = O.prefixed(q, few, few.flip(0), pt, plens, bt, lens)
    O.check(got, *ref, torch.bfloat16, rows=True)


def test_a_run_of_them_together(dev):
    """Image prompts: positions with three axes, appended behind a shared prefix, a step over prefix and
    own tokens, and one over the same tokens as one sequence with a window."""
    dtype, hq, hkv, dim, page, dt = torch.bfloat16, 8, 2, 64, 16, torch.bfloat16
    shared, own, B = 100, [20, 37, 5], 3
    g = torch.Generator().manual_seed(5)
    rope = rope_params(dim, sections=(8, 12, 12), device=dev)
    k_pages = torch.zeros(30, hkv, dim, page, dtype=dtype, device=dev)
    v_pages = torch.zeros_like(k_pages)
    order = torch.randperm(30, generator=g).tolist()
    # one sequence's table is the prefix's whole pages and then its own: 112 tokens shared
    shared = 112
    pt, bt = O.tables([shared], page, order), O.tables(own, page, order)

    def made(n, t0):
        x = torch.randn(n, hq + 2 * hkv, dim, generator=g).to(dt).to(dev)
        q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
        t = torch.arange(t0, t0 + n)
        pos = torch.stack([t // 8, t % 8 // 4, t % 4]).to(dev)
        q, k = rotary_embed(q, k, pos, rope)
        return q, k, v.contiguous()

    with torch.no_grad():
        _, k, v = made(shared, 0)
        kv_append(None, k, v, k_pages, v_pages, pt.to(dev), _ints(dev, [shared]),
                  cu_new=_ints(dev, [0, shared]))
        parts = [made(n, shared) for n in own]
        q, k, v = (torch.cat([p[i] for p in parts]) for i in range(3))
        cu = _cu(own)
        kv_append(None, k, v, k_pages, v_pages, bt.to(dev), _ints(dev, own), cu_new=_ints(dev, cu))
        args = (k_pages, v_pages, pt.to(dev), _ints(dev, [shared]), bt.to(dev), _ints(dev, own))
        rows = paged_prefix_attention(q, *args, None, _ints(dev, cu), _ints(dev, [0] * B))
        last = torch.tensor([c - 1 for c in cu[1:]], device=dev)
        step = paged_prefix_decode_attention(q[last], *args)
        whole = torch.cat([pt.expand(B, -1), bt], dim=1)
        window = paged_window_decode_attention(q[last], k_pages, v_pages, whole.to(dev),
                                               _ints(dev, [shared + n for n in own]), 50, 2)
    kc, vc, qc = k_pages.cpu(), v_pages.cpu(), q.cpu()
    O.check(rows, *O.prefixed(qc, kc, vc, pt, [shared], bt, own, None, cu, [0] * B), dtype, rows=True)
    O.check(step, *O.prefixed(qc[last.cpu()], kc, vc, pt, [shared], bt, own), dtype, rows=True)
    O.check(window, *O.windowed(qc[last.cpu()], kc, vc, whole, [shared + n for n in own], 50, 2), dtype)


def test_empty_calls(dev):
    q, k, v, pt, bt = _on(dev, *_case([30], [5], 2, 1, 64, 16, torch.float32))
    none, lens, plens = torch.zeros(0, dtype=I32, device=dev), _ints(dev, [5]), _ints(dev, [30])
    assert paged_prefix_decode_attention(q[:0], k, v, pt, plens, bt[:0], none).shape == (0, 2, 64)
    got = paged_prefix_decode_attention(q, k, v, pt[:, :0], plens, bt[:, :0], lens)
    assert (got == 0).all()
    # no groups at all
    got = paged_prefix_decode_attention(q, k, v, pt[:0], none, bt, lens, cu_seqs=_ints(dev, [0]))
    ref = O.windowed(q.cpu(), k.cpu(), v.cpu(), bt.cpu(), [5], 10, 0)
    O.check(got, *ref, torch.float32)


def test_refusals(dev):
    q, k, v, pt, bt = _on(dev, *_case([30], [40, 50], 4, 2, 64, 16, torch.bfloat16))
    lens, plens = _ints(dev, [40, 50]), _ints(dev, [30])

    def call(q=q, k=k, v=v, pt=pt, plens=plens, bt=bt, lens=lens, **more):
        return paged_prefix_attention(q, k, v, pt, plens, bt, lens, **more)

    for bad in (dict(pt=pt.long()), dict(pt=pt[0]), dict(pt=pt.expand(2, -1)),
                dict(plens=plens.long()), dict(plens=lens), dict(pt=pt.cpu()),
                dict(cu_seqs=_ints(dev, [0, 1, 2])), dict(cu_seqs=_ints(dev, [0, 2]).long()),
                dict(q=q[:, :3]), dict(q=q[:1]), dict(q=q.float()), dict(lens=lens[:1]),
                dict(bt=bt.long()), dict(v=v[:2]), dict(cu_q=lens), dict(q_pos_offsets=lens[:1]),
                dict(out=q[:1])):
        with pytest.raises(ValueError):
            call(**bad)
    with pytest.raises(ValueError, match="gradient"):
        call(q=q.float(), k=k.float().requires_grad_(), v=v.float())
    call()
    torch.cuda.synchronize()
