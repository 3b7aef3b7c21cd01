"""Calls of the rotary, KV append and 8-bit KV cache operators, with their plain forms.

Each case is one call that a serving or training program makes:

  rotary   rotary positions of q and k (forward, or forward and gradients)
  append   the new tokens of a batch rotated and written into a float pool's pages
  append8  the same into the 8-bit pool, and the contexts read back from it
  gather8  contexts read back from the 8-bit pool in logical order
  decode8  attention of one new token per sequence over the 8-bit pool
  rows8    causal attention of several rows per sequence over the 8-bit pool

The 8-bit pool: K codes [pages, kv heads, D / 16, P, 16], V codes [pages, kv heads, P / 4, D, 4],
both float8_e4m3fn, and one fp32 scale, a power of two, for every 16 tokens of a page and head.

Sizes are those of the package's benchmark and configurations (32 q / 8 kv heads of 128 over
contexts to 8192, 32 / 4 heads, 16-token pages) and generic ones around them.
"""

import math
import pathlib
import sys

import torch

own = False

_PKG = str(pathlib.Path(__file__).resolve().parent.parent / "plastic-infer_amd")

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
ELEM = {"bf16": 2, "fp16": 2, "fp32": 4}
BLOCK = 16           # tokens that share a scale
LARGEST = 448.0      # of float8_e4m3fn
LEAST_SCALE = 2.0 ** -100


def listed():
    return [
        # q and k of one decode step, a batch of 64 interactive requests
        dict(_rotary(64, 32, 4), name="rotary_step_bf16"),
        # a training step's 8192 tokens: forward and both gradients, context stretched four times
        dict(_rotary(8192, 32, 8, grad=True, scaling="yarn"), name="rotary_train_bf16"),
        # one decode step of a full batch: every sequence's token rotated and appended
        dict(_append("append8", 256, 1, 1, 0, 47, 32, 8), name="append8_step_b256_bf16"),
        # ragged prompts into a 16-bit pool, interleaved pairs in half of each head
        dict(_append("append", 8, 141, 1100, 0, 0, 16, 8, interleaved=True, part=2),
             name="append_prompts_bf16"),
        # chunks of prompts behind what is cached, blocks cut at both ends
        dict(_append("append8", 8, 500, 2001, 0, 333, 32, 8, dtype="fp16"),
             name="append8_prompts_fp16"),
        # two short chats read back
        dict(_gather(2, 200, 301, 8), name="gather8_2seq_bf16"),
        # long contexts read back to be handed on
        dict(_gather(16, 512, 8192, 8), name="gather8_16seq_bf16"),
        # one interactive request: latency of a single-sequence step
        dict(_attend("decode8", 1, 1, 1, 3001, 3001, 32, 8, dtype="fp16"), name="decode8_b1_fp16"),
        # a full serving batch at mixed contexts, grouped-query 4
        dict(_attend("decode8", 256, 1, 1, 512, 8192, 32, 8), name="decode8_b256_bf16"),
        # two very long documents on a small model's head size
        dict(_attend("decode8", 2, 1, 1, 100001, 131072, 32, 8, head_dim=64),
             name="decode8_long_hd64_bf16"),
        # a few proposed tokens per request checked at once
        dict(_attend("rows8", 16, 1, 6, 700, 4000, 32, 4, dtype="fp16"), name="rows8_few_fp16"),
        # chunked prefill of long prompts: 1024-token chunks behind 4096 tokens of context
        dict(_attend("rows8", 8, 1024, 1024, 4096, 4096, 32, 8), name="rows8_chunk_bf16"),
    ]


def _rotary(tokens, heads, kv_heads, head_dim=128, part=1, interleaved=False, scaling="none",
            grad=False, packed=False, dtype="bf16"):
    return {"op": "rotary", "tokens": tokens, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "part": part, "interleaved": interleaved, "scaling": scaling,
            "grad": grad, "packed": packed, "dtype": dtype}


def _append(op, seqs, rows_lo, rows_hi, ctx_lo, ctx_hi, heads, kv_heads, head_dim=128, page=16,
            part=1, interleaved=False, dtype="bf16"):
    return {"op": op, "seqs": seqs, "rows_lo": rows_lo, "rows_hi": rows_hi, "ctx_lo": ctx_lo,
            "ctx_hi": ctx_hi, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "page": page, "part": part, "interleaved": interleaved, "dtype": dtype}


def _gather(seqs, lo, hi, kv_heads, head_dim=128, page=16, dtype="bf16"):
    return {"op": "gather8", "seqs": seqs, "rows_lo": 0, "rows_hi": 0, "ctx_lo": lo, "ctx_hi": hi,
            "heads": kv_heads, "kv_heads": kv_heads, "head_dim": head_dim, "page": page,
            "dtype": dtype}


def _attend(op, seqs, rows_lo, rows_hi, ctx_lo, ctx_hi, heads, kv_heads, head_dim=128, page=16,
            dtype="bf16"):
    return {"op": op, "seqs": seqs, "rows_lo": rows_lo, "rows_hi": rows_hi, "ctx_lo": ctx_lo,
            "ctx_hi": ctx_hi, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "page": page, "dtype": dtype}


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choices(("rotary", "append", "append8", "gather8", "decode8", "rows8"),
                     (3, 2, 3, 2, 5, 4))[0]
    dtype = rng.choices(("bf16", "fp16", "fp32"), (4, 2, 1))[0]
    heads, kv_heads = rng.choice(((32, 8), (16, 8), (32, 4), (8, 8), (28, 4), (40, 8)))
    head_dim = rng.choices((128, 64, 96), (5, 2, 1))[0]
    page = rng.choices((16, 32), (4, 1))[0]
    part, interleaved = rng.choice((1, 1, 2)), rng.random() < 0.4
    if op == "rotary":
        return _rotary(_log_int(rng, 1, 6000), heads, kv_heads, head_dim, part, interleaved,
                       rng.choice(("none", "linear", "yarn")), rng.random() < 0.5,
                       rng.random() < 0.5, dtype)
    if op in ("append", "append8"):
        if rng.random() < 0.5:  # a decode step
            return _append(op, _log_int(rng, 1, 256), 1, 1, 0, 47, heads, kv_heads, head_dim, page,
                           part, interleaved, dtype)
        hi = _log_int(rng, 9, 2000)
        return _append(op, _log_int(rng, 1, 6), max(1, hi // 6), hi, 0, rng.choice((0, 100, 333)),
                       heads, kv_heads, head_dim, page, part, interleaved, dtype)
    if op == "gather8":
        hi = _log_int(rng, 16, 6000)
        return _gather(_log_int(rng, 1, 12), max(1, hi // 8), hi, kv_heads, head_dim, page, dtype)
    if op == "decode8":
        hi = _log_int(rng, 64, 60000)
        seqs = max(1, min(_log_int(rng, 1, 256), int(6e8 / (2 * kv_heads * head_dim * hi))))
        if dtype == "fp32":
            seqs = max(1, seqs // 2)
        return _attend(op, seqs, 1, 1, rng.choice((1, max(1, hi // 16), hi)), hi, heads, kv_heads,
                       head_dim, page, dtype)
    few = rng.random() < 0.5
    hi = _log_int(rng, 2, 8) if few else _log_int(rng, 16, 1000 if dtype != "fp32" else 200)
    return _attend(op, _log_int(rng, 1, 24 if few else 6), max(1, hi // 5), hi, 0,
                   rng.choice((0, _log_int(rng, 16, 4000))), heads, kv_heads, head_dim, page, dtype)


def _spread(n, lo, hi, g):
    """n whole numbers, evenly spaced over lo..hi, in a random order: their sum is the case's."""
    steps = torch.linspace(lo, hi, n, dtype=torch.float64).round().long() if n > 1 else \
        torch.tensor([hi])
    return steps[torch.randperm(n, generator=g)]


def _rope(case):
    """(turns per position of each pair [fp64], factor of cos and sin) of a case."""
    rd = case["head_dim"] // case["part"]
    i = torch.arange(0, rd, 2, dtype=torch.float64)
    freq = 1e6 ** (-i / rd)
    kind, factor = case.get("scaling", "none"), 1.0
    if kind == "linear":
        freq = freq / 4.0
    elif kind == "yarn":
        length, by = 8192, 4.0
        at = [rd * math.log(length / (b * 2 * math.pi)) / (2 * math.log(1e6)) for b in (32, 1)]
        low, high = max(math.floor(at[0]), 0), min(math.ceil(at[1]), rd - 1)
        ramp = (torch.arange(rd // 2, dtype=torch.float64) - low) / max(high - low, 1e-3)
        ramp = ramp.clamp(0, 1)
        freq = freq / by * ramp + freq * (1 - ramp)
        factor = 0.1 * math.log(by) + 1.0
    return (freq / (2 * math.pi)).cuda(), factor


def _quantise(x):
    """Codes and scales of x [..., BLOCK, D] in blocks of tokens: (fp8 [..., BLOCK, D], [...])."""
    scale = _scale_of(x.abs().amax(dim=(-1, -2)).float())
    return (x.float() / scale[..., None, None]).to(torch.float8_e4m3fn), scale


def _scale_of(bound):
    """The smallest power of two that holds `bound` (fp32, finite, >= 0) in the codes' range."""
    m, e = torch.frexp(bound)      # bound = m 2^e, 0.5 <= m < 1; 448 = 0.875 * 2^9
    e = e - 9 + (m > 0.875).to(e.dtype)
    scale = torch.ldexp(torch.ones_like(bound), e.clamp(-100, 119))
    return torch.where(bound > 0, scale, torch.full_like(bound, LEAST_SCALE))


def prepare(case, seed):
    g = torch.Generator().manual_seed(seed)
    gc = torch.Generator(device="cuda").manual_seed(seed)
    dt, D, Hq, Hkv = DTYPES[case["dtype"]], case["head_dim"], case["heads"], case["kv_heads"]
    state = {"case": case}

    def rows(n, h):
        return torch.randn(n, h, D, generator=gc, device="cuda").to(dt)

    if case["op"] == "rotary":
        n = case["tokens"]
        state["turns"], state["factor"] = _rope(case)
        state["positions"] = torch.randint(0, 32768, (n,), generator=gc, device="cuda")
        if case["packed"]:   # views of one projection's output
            both = rows(n, Hq + 2 * Hkv)
            state["q"], state["k"] = both[:, :Hq], both[:, Hq:Hq + Hkv]
        else:
            state["q"], state["k"] = rows(n, Hq), rows(n, Hkv)
        if case["grad"]:
            state["q"], state["k"] = (state[x].detach().requires_grad_() for x in "qk")
            state["gq"], state["gk"] = rows(n, Hq), rows(n, Hkv)
        return state

    B, P = case["seqs"], case["page"]
    new = _spread(B, case["rows_lo"], case["rows_hi"], g)
    lens = _spread(B, case["ctx_lo"], case["ctx_hi"], g)
    if case["op"] in ("append", "append8", "rows8"):
        lens = lens + new      # the context counts the new tokens
    width = int(-(-lens.max() // P))
    pages = int((-(-lens // P)).sum()) + 3      # pages in a random order, a few of other requests
    order = torch.randperm(pages, generator=g).to(torch.int32)
    bt, at = torch.zeros(B, width, dtype=torch.int32), 0
    for b, n in enumerate((-(-lens // P)).tolist()):
        bt[b, :n] = order[at:at + n]
        at += n
    state["block_tables"], state["lens"] = bt.cuda(), lens.to(torch.int32).cuda()
    state["total"], state["longest"] = int(lens.sum()), int(lens.max())
    state["most"] = int(new.max())
    cu = torch.zeros(B + 1, dtype=torch.int64)
    cu[1:] = torch.cumsum(new, 0)
    state["cu"] = cu.to(torch.int32).cuda()
    state["cu_lens"] = torch.cat([torch.zeros(1, dtype=torch.int64), torch.cumsum(lens, 0)]).cuda()
    state["offsets"] = (lens - new).to(torch.int32).cuda()
    n = int(cu[-1])
    if case["op"] == "append":
        shape = (pages, Hkv, D, P)
        state["k_pages"] = torch.randn(shape, generator=gc, device="cuda").to(dt)
        state["v_pages"] = torch.randn(shape, generator=gc, device="cuda").to(dt)
    else:
        # keys and values of every token in the pool, some heads larger than others
        size = torch.linspace(0.25, 3.0, Hkv, device="cuda")[:, None, None, None]
        x = torch.randn(pages, Hkv, P // BLOCK, BLOCK, D, generator=gc, device="cuda")
        codes, state["k_scale"] = _quantise(x * size)
        state["k8"] = codes.view(torch.uint8).reshape(pages, Hkv, P, D // 16, 16).permute(
            0, 1, 3, 2, 4).contiguous().view(torch.float8_e4m3fn)
        x = torch.randn(pages, Hkv, P // BLOCK, BLOCK, D, generator=gc, device="cuda")
        codes, state["v_scale"] = _quantise(x * size)
        state["v8"] = codes.view(torch.uint8).reshape(pages, Hkv, P // 4, 4, D).permute(
            0, 1, 2, 4, 3).contiguous().view(torch.float8_e4m3fn)
    if case["op"] in ("append", "append8"):
        state["turns"], state["factor"] = _rope(case)
        state["q"], state["k"], state["v"] = rows(n, Hq), rows(n, Hkv), rows(n, Hkv)
    elif case["op"] in ("decode8", "rows8"):
        state["q"] = rows(B if case["op"] == "decode8" else n, Hq)
    return state


def _back(case):
    """The type that contexts are read back in: bf16 holds the pool's values as they are."""
    return DTYPES["bf16" if case["op"] == "append8" and case["dtype"] == "fp32" else case["dtype"]]


def run(state):
    return (_own_run if own else _plain_run)(state)


# ---- the framework's calls --------------------------------------------------------------------

def _own_run(state):
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    from plastic_infer.kernel.kv_append import kv_append
    from plastic_infer.kernel.paged_kv8 import (
        KV8Pools, kv8_append, kv8_gather, paged_attention_kv8, paged_decode_attention_kv8)
    from plastic_infer.kernel.rotary import RopeParams, rotary_embed

    case = state["case"]
    rope = None
    if "turns" in state:
        rope = RopeParams(state["turns"], state["factor"], case["interleaved"])
    if case["op"] == "rotary":
        q, k = rotary_embed(state["q"], state["k"], state["positions"], rope)
        if not case["grad"]:
            return q, k
        return q, k, *torch.autograd.grad((q, k), (state["q"], state["k"]),
                                          (state["gq"], state["gk"]))
    bt, lens = state["block_tables"], state["lens"]
    cu = None if case["rows_hi"] == 1 else state["cu"]
    if case["op"] == "append":
        q = kv_append(state["q"], state["k"], state["v"], state["k_pages"], state["v_pages"], bt,
                      lens, cu_new=cu, rope=rope)
        return q, state["k_pages"], state["v_pages"]
    pools = KV8Pools(state["k8"], state["v8"], state["k_scale"], state["v_scale"])
    dt = _back(case)
    if case["op"] in ("append8", "gather8"):
        out = ()
        if case["op"] == "append8":
            out = (kv8_append(state["q"], state["k"], state["v"], pools, bt, lens, cu_new=cu,
                              rope=rope),)
        shape = (state["total"], case["kv_heads"], case["head_dim"])
        room = (torch.empty(shape, dtype=dt, device="cuda"), torch.empty(shape, dtype=dt,
                                                                         device="cuda"))
        return *out, *kv8_gather(pools, bt, state["cu_lens"], state["longest"], out=room)
    if case["op"] == "decode8":
        return paged_decode_attention_kv8(state["q"], pools, bt, lens)
    return paged_attention_kv8(state["q"], pools, bt, lens, cu_q=state["cu"],
                               q_pos_offsets=state["offsets"])


# ---- the plain forms --------------------------------------------------------------------------

def _plain_rotate(x, positions, turns, factor, interleaved, back=False):
    """x [N, H, D] in fp32 rotated at its rows' positions (back: the transposed map)."""
    x = x.float()
    rd = 2 * turns.numel()
    t = positions.double()[:, None] * turns[None, :]
    angle = 2 * math.pi * (t - t.round())
    c = (factor * torch.cos(angle)).float()[:, None, :]
    s = (factor * torch.sin(angle)).float()[:, None, :]
    if back:
        s = -s
    a, b = (x[..., 0:rd:2], x[..., 1:rd:2]) if interleaved else (x[..., :rd // 2],
                                                                x[..., rd // 2:rd])
    pair = (a * c - b * s, b * c + a * s)
    turned = torch.stack(pair, dim=-1).flatten(-2) if interleaved else torch.cat(pair, dim=-1)
    return torch.cat([turned, x[..., rd:]], dim=-1)


def _plain_values(state, table=None):
    """K and V of the pool's pages (those of a table) in fp32, [..., P, Hkv, D]."""
    k, v, ks, vs = state["k8"], state["v8"], state["k_scale"], state["v_scale"]
    if table is not None:
        at = table.long()
        k, v = (x.view(torch.uint8)[at].view(torch.float8_e4m3fn) for x in (k, v))
        ks, vs = ks[at], vs[at]
    P = k.shape[-2]
    spread = lambda s: s.repeat_interleave(BLOCK, dim=-1)[..., None]  # noqa: E731
    k = k.float().transpose(-3, -2).flatten(-2) * spread(ks)             # [..., Hkv, P, D]
    v = v.float().transpose(-2, -1).flatten(-3, -2) * spread(vs)
    assert k.shape[-2] == P
    return k.transpose(-3, -2), v.transpose(-3, -2)


def _plain_contexts(state):
    """(K, V) of every sequence in fp32, [B, longest context in whole pages, Hkv, D]."""
    return tuple(x.flatten(1, 2) for x in _plain_values(state, state["block_tables"]))


def _places(state):
    """Where each new row goes: (its position, its page, its offset in the page)."""
    cu, lens = state["cu"].long(), state["lens"].long()
    i = torch.arange(state["k"].shape[0], device="cuda")
    b = torch.searchsorted(cu, i, right=True) - 1
    pos = lens[b] - (cu[b + 1] - i)
    P = state["case"]["page"]
    return pos, state["block_tables"][b, pos // P].long(), pos % P


def _plain_run(state):
    case = state["case"]
    dt = DTYPES[case["dtype"]]
    if "turns" in state:
        form = (state["turns"], state["factor"], case["interleaved"])
    if case["op"] == "rotary":
        pos = state["positions"]
        with torch.no_grad():
            out = [_plain_rotate(state[x], pos, *form).to(dt) for x in "qk"]
            if case["grad"]:
                out += [_plain_rotate(state[x], pos, *form, back=True).to(dt) for x in ("gq", "gk")]
        return tuple(out)
    if case["op"] in ("append", "append8"):
        pos, page, off = _places(state)
        q, k = (_plain_rotate(state[x], pos, *form) for x in "qk")
        if case["op"] == "append":
            state["k_pages"][page, :, :, off] = k.to(dt)
            state["v_pages"][page, :, :, off] = state["v"]
            return q.to(dt), state["k_pages"], state["v_pages"]
        turned = torch.tensor(math.sqrt(2.0) * form[1], dtype=torch.float32, device="cuda")
        _plain_append8(state, "k", k, state["k"].float().abs().amax(-1) * turned, page, off)
        _plain_append8(state, "v", state["v"].float(), state["v"].float().abs().amax(-1), page, off)
        return q.to(dt), *_plain_packed(state, _back(case))
    if case["op"] == "gather8":
        return _plain_packed(state, dt)
    k, v = _plain_contexts(state)
    cu = state["cu"].long()
    B, T, Hkv, D = k.shape
    G = case["heads"] // Hkv
    if case["op"] == "decode8":
        q, last = state["q"].float()[:, None], state["lens"].long()[:, None] - 1
    else:       # rows padded to the longest run; a row sees the keys up to its own position
        R = state["most"]
        r = torch.arange(R, device="cuda")
        at = (cu[:-1, None] + r).clamp(max=state["q"].shape[0] - 1)
        q = state["q"].float()[at]
        last = torch.minimum(state["offsets"].long()[:, None] + r,
                             state["lens"].long()[:, None] - 1)
    R = q.shape[1]
    q = q.view(B, R, Hkv, G, D).permute(0, 2, 1, 3, 4).reshape(B * Hkv, R * G, D)
    k = k.permute(0, 2, 3, 1).reshape(B * Hkv, D, T)
    v = v.transpose(1, 2).reshape(B * Hkv, T, D)
    s = torch.matmul(q, k).view(B, Hkv, R, G, T) * (1.0 / math.sqrt(D))
    seen = torch.arange(T, device="cuda") <= last[..., None]               # [B, R, T]
    s = s.masked_fill(~seen[:, None, :, None, :], -math.inf)
    e = torch.exp(s - s.amax(-1, keepdim=True))
    p = (e / e.sum(-1, keepdim=True)).view(B * Hkv, R * G, T)
    o = torch.matmul(p, v).view(B, Hkv, R, G, D).permute(0, 2, 1, 3, 4).reshape(B, R, Hkv * G, D)
    if case["op"] == "decode8":
        return o[:, 0].to(dt)
    i = torch.arange(state["q"].shape[0], device="cuda")
    b = torch.searchsorted(cu, i, right=True) - 1
    return o[b, i - cu[b]].to(dt)


def _plain_packed(state, dt):
    """The contexts' K and V, one after the other, [total, Hkv, D]."""
    T = state["block_tables"].shape[1] * state["case"]["page"]
    keep = torch.arange(T, device="cuda") < state["lens"][:, None]
    return tuple(x[keep].to(dt) for x in _plain_contexts(state))


def _plain_append8(state, name, x, bound, page, off):
    """x [N, Hkv, D] into the pool's codes: each block takes the scale that holds its new tokens'
    bounds and, where it holds earlier ones, its old scale, which those are rounded to."""
    codes, scale = state[name + "8"], state[name + "_scale"]
    N, Hkv, nb = scale.shape
    block = page * nb + off // BLOCK
    most = torch.zeros(N * nb, Hkv, device="cuda")
    most.scatter_reduce_(0, block[:, None].expand(-1, Hkv), bound, "amax")
    first = torch.full((N * nb,), BLOCK, device="cuda")
    first.scatter_reduce_(0, block, off % BLOCK, "amin")
    most = most.view(N, nb, Hkv).transpose(1, 2)
    first = first.view(N, 1, nb)
    fresh = _scale_of(most)
    now = torch.where(first == BLOCK, scale, torch.where(first == 0, fresh,
                                                         torch.maximum(scale, fresh)))
    # tokens ahead of the first new one in a block
    old = torch.arange(BLOCK, device="cuda") < first[..., None]             # [N, 1, nb, BLOCK]
    ratio = torch.where(old, (scale / now)[..., None], torch.ones((), device="cuda")).flatten(2)
    ratio = ratio[:, :, None, :, None] if name == "k" else ratio.view(N, Hkv, -1, 1, 4)
    codes.copy_((codes.float() * ratio).to(torch.float8_e4m3fn))
    scale.copy_(now)
    head = torch.arange(Hkv, device="cuda")
    new = x / now[page[:, None], head, (off // BLOCK)[:, None]][..., None]
    new = new.to(torch.float8_e4m3fn).view(torch.uint8)
    at = codes.view(torch.uint8)
    if name == "k":
        at[page, :, :, off] = new.view(*new.shape[:2], -1, 16)
    else:
        at[page, :, off // 4, :, off % 4] = new


# ---- amounts ----------------------------------------------------------------------------------

def _lengths(case):
    """(new rows, context) of the case's sequences, paired in order: the sums are the case's."""
    B = case["seqs"]

    def spaced(lo, hi):
        return [round(lo + (hi - lo) * i / (B - 1)) for i in range(B)] if B > 1 else [hi]

    new, ctx = spaced(case["rows_lo"], case["rows_hi"]), spaced(case["ctx_lo"], case["ctx_hi"])
    return new, ctx


def work(case):
    D, Hq, Hkv, e = case["head_dim"], case["heads"], case["kv_heads"], ELEM[case["dtype"]]
    if case["op"] == "rotary":
        n = case["tokens"] * (Hq + Hkv) * D
        passes = 2 if case["grad"] else 1
        return {"bytes": passes * (2 * n * e + 8 * case["tokens"]), "flops": 3 * n * passes}
    new, ctx = _lengths(case)
    n, total = sum(new), sum(ctx)
    kv = Hkv * D * 2
    if case["op"] == "append":
        return {"bytes": n * (2 * Hq * D + 2 * kv) * e, "flops": 3 * n * (Hq + Hkv) * D}
    if case["op"] == "append8":      # and the contexts read back
        return {"bytes": n * (2 * Hq * D * e + kv * (e + 1)) + (total + n) * kv * (1 + e),
                "flops": 3 * n * (Hq + Hkv) * D}
    if case["op"] == "gather8":
        return {"bytes": total * kv * (1 + e), "flops": total * kv}
    if case["op"] == "decode8":
        return {"bytes": total * (kv + Hkv / 2) + 2 * case["seqs"] * Hq * D * e,
                "flops": 4 * total * Hq * D}
    seen = sum(r * c + r * (r + 1) / 2 for r, c in zip(new, ctx))
    return {"bytes": (total + n) * (kv + Hkv / 2) + 2 * n * Hq * D * e, "flops": 4 * seen * Hq * D}


# ---- the definition in 64 bits ------------------------------------------------------------------

def _exact_rotate(x, positions, turns, factor, interleaved, sign=1.0):
    """Pairs as complex numbers times factor e^(2 pi i turns position)."""
    x = x.detach().double()
    half = turns.numel()
    t = positions.double()[:, None, None] * turns
    w = torch.polar(torch.full_like(t, factor), sign * 2 * math.pi * torch.remainder(t, 1.0))
    out = x.clone()
    if interleaved:
        z = torch.complex(x[..., 0:2 * half:2].contiguous(), x[..., 1:2 * half:2].contiguous()) * w
        out[..., 0:2 * half:2], out[..., 1:2 * half:2] = z.real, z.imag
    else:
        z = torch.complex(x[..., :half].contiguous(), x[..., half:2 * half].contiguous()) * w
        out[..., :half], out[..., half:2 * half] = z.real, z.imag
    return out


def _exact_round(x):
    """x [fp64] to the nearest value with 3 stored bits from 2^-6 on, in steps of 2^-9 below."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def _exact_pool(state):
    """The pool as values: [(codes [N, Hkv, P, D] in fp64, scale [N, Hkv, P / BLOCK])] of K, V."""
    k = state["k8"].double()
    v = state["v8"].double()
    N, H, _, P, _ = k.shape
    return [(torch.cat([k[:, :, c] for c in range(k.shape[2])], dim=-1), state["k_scale"].double()),
            (torch.stack([v[:, :, t // 4, :, t % 4] for t in range(P)], dim=2),
             state["v_scale"].double())]


def exact(case, seed):
    state = prepare(case, seed)
    if "turns" in state:
        form = (state["turns"], state["factor"], case["interleaved"])
    if case["op"] == "rotary":
        pos = state["positions"]
        out = [_exact_rotate(state[x], pos, *form) for x in "qk"]
        if case["grad"]:
            out += [_exact_rotate(state[x], pos, *form, sign=-1.0) for x in ("gq", "gk")]
        return tuple(out)
    bt, lens, P = state["block_tables"].tolist(), state["lens"].tolist(), case["page"]
    cu = state["cu"].tolist()
    Hkv, D, G = case["kv_heads"], case["head_dim"], case["heads"] // case["kv_heads"]
    if case["op"] in ("append", "append8"):
        if sum(lens) > 60000:
            return None
        pos = torch.cat([torch.arange(n - (cu[b + 1] - cu[b]), n) for b, n in enumerate(lens)])
        pos = pos.cuda()
        q, k = (_exact_rotate(state[x], pos, *form) for x in "qk")
        v = state["v"].double()
    if case["op"] == "append":
        pools = [state["k_pages"].double(), state["v_pages"].double()]
        for b, n in enumerate(lens):
            at = pos[cu[b]:cu[b + 1]]
            page = state["block_tables"][b].long()[at // P]
            for pool, x in zip(pools, (k, v)):
                pool[page, :, :, at % P] = x[cu[b]:cu[b + 1]]
        return q, *pools
    if case["op"] == "append8":
        gathered = []
        for (codes, scale), x, given, c in zip(_exact_pool(state), (k, v), ("k", "v"),
                                               (float(torch.tensor(math.sqrt(2.0) * form[1],
                                                                   dtype=torch.float32)), 1.0)):
            flat = (codes * scale.repeat_interleave(BLOCK, -1)[..., None])
            # fp32: the scale is a matter of the bound as it is computed
            bound = (state[given].float().abs().amax(-1) * torch.tensor(c, dtype=torch.float32,
                                                                        device="cuda")).double()
            out = []
            for b, n in enumerate(lens):
                pages = state["block_tables"][b].long()[:-(-n // P)]
                seq = flat[pages].transpose(1, 2).reshape(-1, Hkv, D)           # [tokens, Hkv, D]
                sc = scale[pages].transpose(1, 2).reshape(-1, Hkv)              # [blocks, Hkv]
                start = n - (cu[b + 1] - cu[b])
                b0, b1 = start // BLOCK, -(-n // BLOCK)
                lim = torch.zeros(b1 * BLOCK, Hkv, dtype=torch.float64, device="cuda")
                lim[start:n] = bound[cu[b]:cu[b + 1]]
                lim = lim.view(b1, BLOCK, Hkv).amax(1)[b0:]
                fit = torch.exp2(torch.ceil(torch.log2(lim / LARGEST)).clamp(min=-100))
                if start % BLOCK:
                    fit[0] = torch.maximum(fit[0], sc[b0])
                unit = fit.repeat_interleave(BLOCK, 0)[..., None]
                seq = seq[:b1 * BLOCK].clone()
                seq[start:n] = x[cu[b]:cu[b + 1]]
                seq[b0 * BLOCK:] = _exact_round(seq[b0 * BLOCK:] / unit) * unit
                out.append(seq[:n])
            gathered.append(torch.cat(out))
        return q, *gathered
    if case["op"] == "rows8" and sum((cu[b + 1] - cu[b]) * n for b, n in enumerate(lens)) > 1e8:
        return None
    out, ks, vs = [], [], []
    for b, n in enumerate(lens):
        pages = state["block_tables"][b].long()[:-(-n // P)]
        part = {y: state[y].view(torch.uint8)[pages].view(torch.float8_e4m3fn)
                for y in ("k8", "v8")}
        part |= {y: state[y][pages] for y in ("k_scale", "v_scale")}
        k, v = ((c * f.repeat_interleave(BLOCK, -1)[..., None]).transpose(0, 1)
                .reshape(Hkv, -1, D)[:, :n] for c, f in _exact_pool(part))
        if case["op"] == "gather8":
            ks.append(k.transpose(0, 1))
            vs.append(v.transpose(0, 1))
            continue
        rows = [b, b + 1] if case["op"] == "decode8" else cu[b:b + 2]
        q = state["q"][rows[0]:rows[1]].double()
        r = q.shape[0]
        q = q.view(r, Hkv, G, D).permute(1, 2, 0, 3).reshape(Hkv, G * r, D)
        s = (q @ k.transpose(1, 2)).view(Hkv, G, r, n) / math.sqrt(D)
        late = torch.arange(n, device="cuda") > torch.arange(n - r, n, device="cuda")[:, None]
        p = torch.softmax(s.masked_fill(late, -math.inf), dim=-1).view(Hkv, G * r, n)
        out.append((p @ v).view(Hkv, G, r, D).permute(2, 0, 1, 3).reshape(r, Hkv * G, D))
    if case["op"] == "gather8":
        return torch.cat(ks), torch.cat(vs)
    return torch.cat(out)
