"""Prefix attention takes the workspace that it uses and no more, with the same results."""

from __future__ import annotations

import pytest
import torch

import reach_oracle as O
from plastic_infer.kernel import paged_prefix as PP

pytestmark = pytest.mark.gpu

I32 = torch.int32


def _case(dev, prefix, lens, rows, hq, hkv, dim, dtype, seed=0):
    page = 16
    pages = sum(-(-n // page) for n in [prefix, *lens]) + 2
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    k, v = O.pools(pages, hkv, dim, page, dtype, seed)
    pt, bt = O.tables([prefix], page, order), O.tables(lens, page, order)
    q = torch.randn(sum(rows), hq, dim, generator=torch.Generator().manual_seed(seed + 1)).to(dtype)
    cu = [sum(rows[:i]) for i in range(len(rows) + 1)]
    ints = [torch.tensor(x, dtype=I32, device=dev) for x in ([prefix], lens, cu)]
    args = [x.to(dev) for x in (q, k, v, pt)] + [ints[0], bt.to(dev), ints[1]]
    return args, ints[2], lambda: O.prefixed(q, k, v, pt, [prefix], bt, lens, None, cu)


def _call_bytes(dev, args, B, rows):
    q, k, pt, bt = args[0], args[1], args[3], args[5]
    return PP._call_bytes(dev.index, 1, pt.shape[1], bt.shape[1], 1, B, rows, q.shape[1], k.shape[1],
                          k.shape[2], 16, 1.0 / q.shape[2] ** 0.5, 2 if q.dtype == torch.bfloat16 else 1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_many_rows_allocate_their_output(dev, dtype):
    rows = [1024] * 8
    args, cu, _ = _case(dev, 64, [16] * 8, rows, 32, 8, 128, dtype)
    assert _call_bytes(dev, args, 8, sum(rows)) == 0
    bound = PP.prefix_attention_workspace_bytes(sum(rows), 32, 128)
    ws = torch.empty(bound, dtype=torch.uint8, device=dev)
    want = PP.paged_prefix_attention(*args, cu_q=cu, workspace=ws)
    del ws
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    got = PP.paged_prefix_attention(*args, cu_q=cu)
    out = got.numel() * got.element_size()
    assert torch.cuda.max_memory_allocated() - before <= out + (1 << 20) < bound
    assert torch.equal(got, want)


def test_a_workspace_that_is_not_one_is_replaced_by_what_the_call_takes(dev):
    rows = [2, 1]
    args, cu, ref = _case(dev, 300, [40] * 2, rows, 8, 2, 128, torch.bfloat16)
    need = _call_bytes(dev, args, 2, 3)
    for ws in (torch.empty(need + 16, dtype=torch.uint8, device=dev)[8:],       # between vectors
               torch.empty(2 * need, dtype=torch.uint8, device=dev)[::2],       # with holes
               torch.empty(need - 1, dtype=torch.uint8, device=dev)):           # too little
        ws.fill_(0x7f)
        O.check(PP.paged_prefix_attention(*args, cu_q=cu, workspace=ws), *ref(), torch.bfloat16, rows=True)
        assert (ws == 0x7f).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,prefix,dim", [([100], 3000, 128), ([70, 33], 2000, 64), ([65], 4000, 256),
                                             ([2, 1, 3], 500, 128)])
def test_the_workspace_of_a_call_is_enough(dev, rows, prefix, dim, dtype):
    args, cu, ref = _case(dev, prefix, [40] * len(rows), rows, 8, 2, dim, dtype, seed=dim)
    need = _call_bytes(dev, args, len(rows), sum(rows))
    assert 0 < need <= PP.prefix_attention_workspace_bytes(sum(rows), 8, dim)
    room = torch.full((need + 4096,), 0x7f, dtype=torch.uint8, device=dev)
    got = PP.paged_prefix_attention(*args, cu_q=cu, workspace=room[:need])
    assert (room[need:] == 0x7f).all() and not (room[:need] == 0x7f).all()
    O.check(got, *ref(), dtype, rows=True)
    ws = torch.full((PP.prefix_attention_workspace_bytes(sum(rows), 8, dim),), 0x7f, dtype=torch.uint8,
                    device=dev)
    for other in (ws, None):
        assert torch.equal(got, PP.paged_prefix_attention(*args, cu_q=cu, workspace=other))
