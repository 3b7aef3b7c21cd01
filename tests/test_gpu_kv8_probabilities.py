"""How many bits each attention kernel of the 8-bit pool keeps of its probabilities, also of those far
below a row's largest.

Bounds: those of test_gpu_kv8_attention, with probabilities as two bf16 terms (2^-16 of each) wherever a
call does not round them once, as calls of many 16-bit rows do. Those of fp16 rows may also lose of each
probability what comes to 2^-25 of the output together, half of fp16's least number."""

from __future__ import annotations

import math

import pytest
import torch

import kv8_oracle as O
from plastic_infer.kernel.paged_kv8 import paged_attention_kv8, paged_decode_attention_kv8
from test_gpu_kv8_attention import LEAST, MANY, ROWS, STEP, _check, _rows, _tables

pytestmark = pytest.mark.gpu


def _rounds_once(dtype, rows, seqs, hq, hkv, dim):
    """Whether a call takes the kernel for many rows (the C library's rule)."""
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    return dtype != torch.float32 and dim <= 128 and rows * (hq // hkv) >= 64 * seqs \
        and rows * hq >= 2 * cus


@pytest.mark.parametrize("dtype", list(STEP))
@pytest.mark.parametrize("case", [(*c, 0) for c in ROWS] + MANY,
                         ids=lambda c: f"{sum(c[0])}of{max(c[1])}h{c[3]}/{c[4]}d{c[5]}w{c[7]}")
def test_terms_of_the_probabilities(dev, case, dtype):
    new, lens, offs, hq, hkv, dim, page, width = case
    cu = [0] + torch.tensor(new).cumsum(0).tolist()
    if _rounds_once(dtype, cu[-1], len(new), hq, hkv, dim):
        return
    tables, pages = _tables(lens, page, 2, sum(lens) + 1)
    if width:
        tables = torch.nn.functional.pad(tables, (0, width // page - tables.shape[1]), value=-1)
    pool = O.Pool.random(pages, hkv, dim, page, seed=dim + hq + 3)
    offs = [n - m for n, m in zip(lens, new)] if offs == "end" else offs
    q = _rows(cu[-1], hq, dim, dtype, hq + 1)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    got = paged_attention_kv8(q.to(dev), pool.to_device(dev), tables.to(dev), i32(lens), i32(cu),
                              None if offs is None else i32(offs))
    ref, mag, size = O.attend(q, pool, tables.tolist(), lens, cu, offs, 1 / math.sqrt(dim))
    _check(got, ref, mag, size, dtype, max(lens), dim)


SINK = [  # rows, Hq, Hkv, D, the table's width in tokens
    (1, 16, 2, 64, 0), (3, 16, 2, 64, 0), (2, 16, 2, 256, 0),
    (64, 16, 2, 64, 0), (64, 16, 2, 128, 0), (70, 16, 2, 96, 0),
    (64, 48, 48, 80, 0),
    (64, 16, 2, 128, 8192), (64, 16, 2, 64, 8192),     # cut along the keys
    (43, 1056, 176, 128, 2048),                        # items of 256 rows
]


@pytest.mark.parametrize("dtype", list(STEP))
@pytest.mark.parametrize("case", SINK, ids=lambda c: f"{c[0]}h{c[1]}/{c[2]}d{c[3]}w{c[4]}")
@pytest.mark.parametrize("mass,v_exp", [(2.0 ** -6, 7), (2.0 ** -10, 7), (2.0 ** -16, 7), (2.0 ** -16, -7),
                                        (2.0 ** -16, -4), (2.0 ** -30, 7), (2.0 ** -30, -3),
                                        (2.0 ** -30, -4)])
def test_a_key_that_takes_nearly_all(dev, mass, v_exp, case, dtype):
    """One key takes all but `mass` of each row's probability and has a V of zeros; what is left is
    spread over up to 1000 alike keys, whose V (codes to 400, scale 2^v_exp) make the result."""
    rows, hq, hkv, dim, width = case
    page, n = 16, 1001
    tables, pages = _tables([n], page, 0, 1)
    pool = O.Pool.random(pages, hkv, dim, page, seed=5)
    pool.scale["k"][:] = 2.0 ** -7
    pool.scale["v"][:] = 2.0 ** v_exp
    pool.codes["k"] = O.e4m3(pool.codes["k"] / 64)       # scores near zero
    first = int(tables[0, 0])
    pool.codes["v"][first, :, 0] = 0.0
    pool.codes["k"][first, :, 0] = 0.0
    pool.codes["k"][first, :, 0, 0] = 256.0              # 2 at the scale
    q = _rows(rows, hq, dim, dtype, 7) / 8
    # the key's score: that of a thousand keys of about zero, over their mass
    q[..., 0] = math.log(1000.0 / mass) * math.sqrt(dim) / 2.0
    if width:
        tables = torch.nn.functional.pad(tables, (0, width // page - tables.shape[1]), value=-1)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    args = (q.to(dev), pool.to_device(dev), tables.to(dev), i32([n]))
    once = _rounds_once(dtype, rows, 1, hq, hkv, dim)
    lost = 2.0 ** -25 if once and dtype == torch.float16 else 0.0
    for offs in (None, [n - rows]) if rows > 1 else (None,):
        if rows == 1:
            got = paged_decode_attention_kv8(*args)
        else:
            got = paged_attention_kv8(*args, i32([0, rows]), None if offs is None else i32(offs))
        some, heads = slice(max(0, rows - 2), rows), slice(0, min(hq, 4 * (hq // hkv)))
        part = O.Pool(pages, heads.stop * hkv // hq, dim, page)
        for x in "kv":
            part.codes[x], part.scale[x] = (t[x][:, :part.shape[1]] for t in (pool.codes, pool.scale))
        ref, mag, size = O.attend(q[some, heads], part, tables.tolist(), [n], [0, q[some].shape[0]],
                                  None if offs is None else [offs[0] + some.start], 1 / math.sqrt(dim))
        err = (got[some, heads].double().cpu() - ref).abs()
        rel = STEP[dtype] if once else 0.0 if dtype == torch.float32 else 2.0 ** -16
        rel = rel + 2.0 ** -22 + 2 * n * 2.0 ** -23 + 2 * (dim + 8) * 2.0 ** -23 * size
        bound = STEP[dtype] * ref.abs().clamp_min(LEAST[dtype]) + rel * mag + lost
        assert (err <= bound).all(), (err / bound).max().item()
        assert torch.isfinite(got).all()
