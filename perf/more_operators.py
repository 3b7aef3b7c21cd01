"""Calls of attention with a sliding window and sinks, of attention behind a shared prefix and of
rotary positions with several axes, with their plain forms.

Each case is one call that a serving or training program makes:

  window   one new token per sequence, which sees the last `window` tokens and the first `sinks`
  wrows    several rows per sequence, each with a window that ends at it
  prefix   one new token per sequence, groups of sequences behind a prefix that is kept once
  prows    several rows per sequence behind their group's prefix, causal among their own tokens
  axes     rotary positions of q and k from (time, height, width) (forward, or forward and gradients)

K and V lie in the paged pools [pages, kv heads, head_dim, page] of the package.

Sizes are those of the package's benchmark and configurations (32 q / 8 kv heads of 128 over contexts
to 8192, 32 / 4 heads, 16-token pages, chunks of 1024 rows) and generic ones around them.
"""

import math
import pathlib
import sys

import torch

own = False

_PKG = str(pathlib.Path(__file__).resolve().parent.parent / "plastic-infer_amd")

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
ELEM = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # one interactive request of a model whose layers see 1024 tokens back
        dict(_window("window", 1, 1, 1, 3001, 3001, 1024, 4, 32, 8, dtype="fp16"),
             name="window_b1_fp16"),
        # a full serving batch at mixed contexts, most of them beyond the window
        dict(_window("window", 128, 1, 1, 512, 8192, 4096, 4, 32, 8), name="window_b128_bf16"),
        # fp32 pools in larger pages, a short window and a page of sinks
        dict(_window("window", 24, 1, 1, 100, 2500, 500, 16, 16, 4, page=32, dtype="fp32"),
             name="window_b24_fp32"),
        # a few proposed tokens per request checked at once, small heads
        dict(_window("wrows", 16, 1, 6, 700, 4000, 1000, 1, 32, 4, head_dim=64, dtype="fp16"),
             name="window_few_fp16"),
        # chunked prefill: 1024-token chunks behind 4096 tokens, a window of 2048
        dict(_window("wrows", 8, 1024, 1024, 4096, 4096, 2048, 4, 32, 8),
             name="window_chunk_bf16"),
        # chats that start from one instruction text
        dict(_prefix("prefix", 1, 64, 64, 8192, 8192, 1, 1, 60, 700, 32, 8), name="prefix_b64_bf16"),
        # a full batch of questions on one long document
        dict(_prefix("prefix", 1, 256, 256, 32768, 32768, 1, 1, 33, 300, 32, 8),
             name="prefix_b256_long_bf16"),
        # a few tools' instruction texts, a few requests on each, small heads
        dict(_prefix("prefix", 4, 3, 9, 700, 2900, 1, 1, 0, 400, 32, 4, head_dim=64, dtype="fp16"),
             name="prefix_groups_fp16"),
        # samples of one prompt, drawn on in fp32
        dict(_prefix("prefix", 1, 24, 24, 2000, 2000, 1, 1, 1, 200, 16, 4, dtype="fp32"),
             name="prefix_b24_fp32"),
        # new prompts of many requests behind one instruction text
        dict(_prefix("prows", 1, 12, 12, 4096, 4096, 100, 450, 0, 0, 32, 8), name="prefix_rows_bf16"),
        # q and k of one decode step behind images
        dict(_axes(64, 32, 4, 3), name="axes_step_bf16"),
        # a training step's 8192 tokens of text and video: forward and both gradients
        dict(_axes(8192, 32, 8, 3, grad=True), name="axes_train_bf16"),
    ]


def _window(op, seqs, rows_lo, rows_hi, ctx_lo, ctx_hi, window, sinks, heads, kv_heads,
            head_dim=128, page=16, dtype="bf16"):
    return {"op": op, "seqs": seqs, "rows_lo": rows_lo, "rows_hi": rows_hi, "ctx_lo": ctx_lo,
            "ctx_hi": ctx_hi, "window": window, "sinks": sinks, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "dtype": dtype}


def _prefix(op, groups, size_lo, size_hi, prefix_lo, prefix_hi, rows_lo, rows_hi, ctx_lo, ctx_hi,
            heads, kv_heads, head_dim=128, page=16, dtype="bf16"):
    return {"op": op, "groups": groups, "size_lo": size_lo, "size_hi": size_hi,
            "prefix_lo": prefix_lo, "prefix_hi": prefix_hi, "rows_lo": rows_lo, "rows_hi": rows_hi,
            "ctx_lo": ctx_lo, "ctx_hi": ctx_hi, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "page": page, "dtype": dtype}


def _axes(tokens, heads, kv_heads, axes, head_dim=128, part=1, interleaved=False, grad=False,
          dtype="bf16"):
    return {"op": "axes", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "axes": axes,
            "head_dim": head_dim, "part": part, "interleaved": interleaved, "grad": grad,
            "dtype": dtype}


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choices(("window", "wrows", "prefix", "prows", "axes"), (4, 4, 4, 3, 3))[0]
    dtype = rng.choices(("bf16", "fp16", "fp32"), (4, 2, 1))[0]
    heads, kv_heads = rng.choice(((32, 8), (16, 8), (32, 4), (8, 8), (28, 4), (40, 8), (16, 2)))
    head_dim = rng.choices((128, 64, 96, 256), (5, 2, 1, 1))[0]
    page = rng.choices((16, 32, 64), (4, 1, 1))[0]
    kind = {"head_dim": head_dim, "page": page, "dtype": dtype}
    slow = dtype == "fp32" or head_dim == 256
    if op == "axes":
        return _axes(_log_int(rng, 1, 6000), heads, kv_heads, rng.choice((2, 3, 3, 4)), head_dim,
                     rng.choice((1, 1, 2)), rng.random() < 0.4, rng.random() < 0.5, dtype)
    if op == "window":
        hi = _log_int(rng, 30, 20000)
        window = _log_int(rng, 1, 6000)
        reach = min(hi, window + 100) * 2 * kv_heads * head_dim
        seqs = max(1, min(_log_int(rng, 1, 200), int(5e8 / reach), int(4e6 / hi)))
        return _window(op, seqs, 1, 1, rng.choice((1, max(1, hi // 9), hi)), hi, window,
                       rng.choice((0, 1, 4, _log_int(rng, 5, 200))), heads, kv_heads, **kind)
    if op == "wrows":
        few = rng.random() < 0.4
        rows = _log_int(rng, 2, 8) if few else _log_int(rng, 16, 150 if slow else 900)
        return _window(op, _log_int(rng, 1, 24 if few else 6), max(1, rows // 5), rows, 0,
                       rng.choice((0, _log_int(rng, 16, 4000))), _log_int(rng, 4, 3000),
                       rng.choice((0, 1, 4, _log_int(rng, 5, 200))), heads, kv_heads, **kind)
    groups = rng.choice((1, 1, 2, 5))
    hi = _log_int(rng, 20, 10000 if groups == 1 else 3000)
    lo = hi if groups == 1 else max(1, hi // 4)
    if op == "prefix":
        size = _log_int(rng, 1, 150 if groups == 1 else 16)
        if slow:
            size = max(1, size // 3)
        return _prefix(op, groups, max(1, size // 2), size, lo, hi, 1, 1, 0, _log_int(rng, 1, 900),
                       heads, kv_heads, **kind)
    rows = _log_int(rng, 2, 60 if slow else 300)
    return _prefix(op, groups, 1, _log_int(rng, 1, 9 if groups == 1 else 3), lo // 2 + 1, hi // 2 + 1,
                   max(1, rows // 4), rows, 0, rng.choice((0, 0, _log_int(rng, 1, 500))), heads,
                   kv_heads, **kind)


def _spaced(n, lo, hi):
    return [round(lo + (hi - lo) * i / (n - 1)) for i in range(n)] if n > 1 else [hi]


def _mixed(values, g):
    return torch.tensor(values)[torch.randperm(len(values), generator=g)]


def _tables(lens, page, pages, g):
    """Block tables of sequences of these lengths over `pages`, which lie in a random order."""
    need = -(-lens // page)
    bt, at = torch.zeros(len(lens), max(1, int(need.max())), dtype=torch.int32), 0
    for b, n in enumerate(need.tolist()):
        bt[b, :n] = pages[at:at + n]
        at += n
    return bt, pages[at:]


def prepare(case, seed):
    g = torch.Generator().manual_seed(seed)
    gc = torch.Generator(device="cuda").manual_seed(seed)
    dt, D, Hq, Hkv = DTYPES[case["dtype"]], case["head_dim"], case["heads"], case["kv_heads"]
    state = {"case": case}

    def rows(n, h):
        return torch.randn(n, h, D, generator=gc, device="cuda").to(dt)

    if case["op"] == "axes":
        n, A = case["tokens"], case["axes"]
        pairs = D // case["part"] // 2
        i = torch.arange(pairs, dtype=torch.float64)
        state["turns"] = (1e6 ** (-i / pairs) / (2 * math.pi)).cuda()
        # a quarter of the pairs turn by time, the others by the axes of an image, in blocks
        edge = [0, pairs // 4] + [pairs // 4 + (pairs - pairs // 4) * j // (A - 1)
                                  for j in range(1, A)]
        axis = torch.zeros(pairs, dtype=torch.int32)
        for a in range(A):
            axis[edge[a]:edge[a + 1]] = a
        state["axis"] = axis.cuda()
        # text, then frames of 24 x 32 patches: time goes by frame, height and width inside it
        t = torch.arange(n)
        text = t < n // 3
        frame, inside = (t - n // 3) // 768, (t - n // 3) % 768
        pos = torch.stack([n // 3 + frame] + [n // 3 + (inside // 32, inside % 32, inside % 7)[j]
                                              for j in range(A - 1)])
        state["positions"] = (torch.where(text, t, pos) +
                              torch.randint(0, 20000, (1,), generator=g)).cuda()
        state["q"], state["k"] = rows(n, Hq), rows(n, Hkv)
        if case["grad"]:
            state["q"].requires_grad_()
            state["k"].requires_grad_()
            state["gq"], state["gk"] = rows(n, Hq), rows(n, Hkv)
        return state

    P = case["page"]
    if case["op"] in ("prefix", "prows"):
        sizes = _mixed(_spaced(case["groups"], case["size_lo"], case["size_hi"]), g)
        shared = _mixed(_spaced(case["groups"], case["prefix_lo"], case["prefix_hi"]), g)
        B = int(sizes.sum())
    else:
        B = case["seqs"]
    new = _mixed(_spaced(B, case["rows_lo"], case["rows_hi"]), g)
    lens = _mixed(_spaced(B, case["ctx_lo"], case["ctx_hi"]), g)
    if case["op"] in ("wrows", "prows"):
        lens = lens + new      # the context counts the new tokens
    state["offsets"] = (lens - new).to(torch.int32).cuda()
    total = int((-(-lens // P)).sum()) + 3      # a few pages are other requests'
    if case["op"] in ("prefix", "prows"):
        total += int((-(-shared // P)).sum())
    free = torch.randperm(total, generator=g).to(torch.int32)
    if case["op"] in ("prefix", "prows"):
        bt, free = _tables(shared, P, free, g)
        state["prefix_tables"], state["prefix_lens"] = bt.cuda(), shared.to(torch.int32).cuda()
        cu = torch.cat([torch.zeros(1, dtype=torch.int64), torch.cumsum(sizes, 0)])
        state["cu_seqs"], state["largest"] = cu.to(torch.int32).cuda(), int(sizes.max())
    bt, _ = _tables(lens, P, free, g)
    state["block_tables"], state["lens"] = bt.cuda(), lens.to(torch.int32).cuda()
    cu = torch.cat([torch.zeros(1, dtype=torch.int64), torch.cumsum(new, 0)])
    state["cu"], state["most"] = cu.to(torch.int32).cuda(), int(new.max())
    if case["op"] == "prows":
        cg = cu[state["cu_seqs"].cpu().long()]
        state["largest"] = int((cg[1:] - cg[:-1]).max())   # rows of a group
    # some heads' keys are larger than others'
    size = torch.linspace(0.25, 2.5, Hkv, device="cuda")[:, None, None]
    for name in ("k_pages", "v_pages"):
        x = torch.randn(total, Hkv, D, P, generator=gc, device="cuda")
        state[name] = (x * size if name == "k_pages" else x).to(dt)
    state["q"] = rows(int(cu[-1]), Hq)
    return state


def run(state):
    return (_own_run if own else _plain_run)(state)


# ---- the framework's calls --------------------------------------------------------------------

def _own_run(state):
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    case = state["case"]
    if case["op"] == "axes":
        from plastic_infer.kernel.rotary import RopeParams, rotary_embed
        rope = RopeParams(state["turns"], 1.0, case["interleaved"], state["axis"])
        q, k = rotary_embed(state["q"], state["k"], state["positions"], rope)
        if not case["grad"]:
            return q, k
        return q, k, *torch.autograd.grad((q, k), (state["q"], state["k"]),
                                          (state["gq"], state["gk"]))
    pool = state["k_pages"], state["v_pages"]
    if case["op"] in ("window", "wrows"):
        from plastic_infer.kernel.paged_window import (
            paged_window_attention, paged_window_decode_attention)
        args = state["block_tables"], state["lens"], case["window"], case["sinks"]
        if case["op"] == "window":
            return paged_window_decode_attention(state["q"], *pool, *args)
        return paged_window_attention(state["q"], *pool, *args, cu_q=state["cu"],
                                      q_pos_offsets=state["offsets"])
    from plastic_infer.kernel.paged_prefix import (
        paged_prefix_attention, paged_prefix_decode_attention)
    args = (state["prefix_tables"], state["prefix_lens"], state["block_tables"], state["lens"])
    cu_seqs = state["cu_seqs"] if case["groups"] > 1 else None
    if case["op"] == "prefix":
        return paged_prefix_decode_attention(state["q"], *pool, *args, cu_seqs=cu_seqs)
    return paged_prefix_attention(state["q"], *pool, *args, cu_seqs=cu_seqs, cu_q=state["cu"],
                                  q_pos_offsets=state["offsets"])


# ---- the plain forms --------------------------------------------------------------------------

def _plain_rotate(state, x, back=False):
    """x [N, H, D] in fp32, every pair turned by its own axis's position (back: the transposed map)."""
    x = x.float()
    rd = 2 * state["turns"].numel()
    t = state["positions"][state["axis"].long()].t().double() * state["turns"]    # [N, pairs]
    angle = 2 * math.pi * (t - t.round())
    c, s = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    if back:
        s = -s
    inter = state["case"]["interleaved"]
    a, b = (x[..., 0:rd:2], x[..., 1:rd:2]) if inter else (x[..., :rd // 2], x[..., rd // 2:rd])
    pair = (a * c - b * s, b * c + a * s)
    turned = torch.stack(pair, dim=-1).flatten(-2) if inter else torch.cat(pair, dim=-1)
    return torch.cat([turned, x[..., rd:]], dim=-1)


def _plain_kv(state, table):
    """K [B, Hkv, D, tokens] and V [B, Hkv, tokens, D] of a table's pages, in fp32."""
    k, v = (state[x][table.long()].float() for x in ("k_pages", "v_pages"))     # [B, n, Hkv, D, P]
    return (k.permute(0, 2, 3, 1, 4).flatten(3).contiguous(),
            v.permute(0, 2, 1, 4, 3).flatten(2, 3).contiguous())


def _plain_q(q, Hkv):
    """q [B, R, Hq, D] as [B, Hkv, R * G, D] in fp32."""
    B, R, Hq, D = q.shape
    return q.float().view(B, R, Hkv, Hq // Hkv, D).transpose(1, 2).reshape(B, Hkv, -1, D)


def _plain_part(q, k, v, seen):
    """(outputs, largest scores, sums) of q [B, Hkv, R * G, D] over the keys with seen [B, R, T]."""
    B, Hkv, RG, D = q.shape
    R, T = seen.shape[1:]
    s = (torch.matmul(q, k) * (1.0 / math.sqrt(D))).view(B, Hkv, R, RG // R, T)
    s = s.masked_fill(~seen[:, None, :, None], -math.inf).view(B, Hkv, RG, T)
    m = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m))
    return torch.matmul(e, v), m, e.sum(-1, keepdim=True)


def _plain_out(o, R):
    """[B, Hkv, R * G, D] back as [B, R, Hq, D]."""
    B, Hkv, RG, D = o.shape
    return o.view(B, Hkv, R, RG // R, D).transpose(1, 2).reshape(B, R, -1, D)


def _plain_run(state):
    case = state["case"]
    dt = DTYPES[case["dtype"]]
    if case["op"] == "axes":
        with torch.no_grad():
            out = [_plain_rotate(state, state[x]).to(dt) for x in "qk"]
            if case["grad"]:
                out += [_plain_rotate(state, state[x], back=True).to(dt) for x in ("gq", "gk")]
        return tuple(out)
    Hkv, P, dev = case["kv_heads"], case["page"], state["q"].device
    cu, lens, bt = state["cu"].long(), state["lens"].long(), state["block_tables"]
    if case["op"] == "window":     # the tokens in reach, gathered one by one
        W, S = case["window"], case["sinks"]
        first = torch.arange(S, device=dev).expand(len(lens), S)
        last = lens[:, None] - W + torch.arange(W, device=dev)
        token = torch.cat([first, last], dim=1)
        seen = torch.cat([first < lens[:, None], last >= S], dim=1)
        token = torch.where(seen, token, torch.zeros_like(token))
        page = torch.gather(bt.long(), 1, token // P)
        k, v = (state[x][page, :, :, token % P].float() for x in ("k_pages", "v_pages"))
        k, v = k.permute(0, 2, 3, 1).contiguous(), v.transpose(1, 2).contiguous()
        o, _, l = _plain_part(_plain_q(state["q"][:, None], Hkv), k, v, seen[:, None])
        return _plain_out(o / torch.where(l == 0, 1.0, l), 1)[:, 0].to(dt)
    # rows padded to the longest run of a sequence
    R = state["most"]
    r = torch.arange(R, device=dev)
    at = (cu[:-1, None] + r).clamp(max=state["q"].shape[0] - 1)
    place = state["offsets"].long()[:, None] + r                                 # [B, R]
    if case["op"] == "prefix":
        place = lens[:, None] - 1
    k, v = _plain_kv(state, bt)
    j = torch.arange(k.shape[-1], device=dev)
    seen = (j <= place[..., None]) & (j < lens[:, None, None])
    if case["op"] == "wrows":
        seen &= (j > place[..., None] - case["window"]) | (j < case["sinks"])
    o, m, l = _plain_part(_plain_q(state["q"][at], Hkv), k, v, seen)
    i = torch.arange(state["q"].shape[0], device=dev)
    b = torch.searchsorted(cu, i, right=True) - 1
    o, m, l = (_plain_out(x, R)[b, i - cu[b]] for x in (o, m, l))                # [rows, Hq, .]
    if case["op"] in ("prefix", "prows"):
        # rows of a group together, padded to the largest group's
        cg = cu[state["cu_seqs"].long()]
        R = state["largest"]
        at = (cg[:-1, None] + torch.arange(R, device=dev)).clamp(max=state["q"].shape[0] - 1)
        k, v = _plain_kv(state, state["prefix_tables"])
        seen = torch.arange(k.shape[-1], device=dev) < state["prefix_lens"][:, None, None]
        parts = _plain_part(_plain_q(state["q"][at], Hkv), k, v, seen.expand(-1, R, -1))
        grp = torch.searchsorted(cg, i, right=True) - 1
        po, pm, pl = (_plain_out(x, R)[grp, i - cg[grp]] for x in parts)
        top = torch.maximum(m, pm)
        f, pf = torch.exp(m - top), torch.exp(pm - top)
        o, l = o * f + po * pf, l * f + pl * pf
    return (o / torch.where(l == 0, 1.0, l)).to(dt)


# ---- amounts ----------------------------------------------------------------------------------

def _reach(new, ctx, window, sinks):
    """(keys that some of the last `new` rows of `ctx` tokens see, keys summed over the rows)."""
    start = max(0, ctx - new - window + 1)
    keys = ctx - start + min(start, sinks)
    rows = sum(min(p + 1, window) + min(sinks, max(0, p + 1 - window))
               for p in range(ctx - new, ctx))
    return keys, rows


def work(case):
    D, Hq, Hkv, e = case["head_dim"], case["heads"], case["kv_heads"], ELEM[case["dtype"]]
    if case["op"] == "axes":
        n = case["tokens"] * (Hq + Hkv) * D
        passes = 2 if case["grad"] else 1
        return {"bytes": passes * (2 * n * e + 8 * case["axes"] * case["tokens"]),
                "flops": 3 * n * passes}
    kv = 2 * Hkv * D * e
    if case["op"] in ("window", "wrows"):
        new = _spaced(case["seqs"], case["rows_lo"], case["rows_hi"])
        ctx = _spaced(case["seqs"], case["ctx_lo"], case["ctx_hi"])
        more = 1 if case["op"] == "wrows" else 0
        parts = [_reach(n, c + more * n, case["window"], case["sinks"]) for n, c in zip(new, ctx)]
        return {"bytes": sum(k for k, _ in parts) * kv + 2 * sum(new) * Hq * D * e,
                "flops": 4 * sum(r for _, r in parts) * Hq * D}
    sizes = _spaced(case["groups"], case["size_lo"], case["size_hi"])
    shared = _spaced(case["groups"], case["prefix_lo"], case["prefix_hi"])
    B = sum(sizes)
    new = _spaced(B, case["rows_lo"], case["rows_hi"])
    ctx = _spaced(B, case["ctx_lo"], case["ctx_hi"])
    n = sum(new)
    if case["op"] == "prefix":
        keys = seen = sum(ctx)
    else:
        keys = sum(ctx) + n
        seen = sum(r * c + r * (r + 1) / 2 for r, c in zip(new, ctx))
    return {"bytes": (sum(shared) + keys) * kv + 2 * n * Hq * D * e,
            "flops": 4 * (seen + n / B * sum(s * p for s, p in zip(sizes, shared))) * Hq * D}


# ---- the definition in 64 bits ------------------------------------------------------------------

def _exact_rotate(state, x, sign):
    """Pairs as complex numbers times e^(2 pi i turns position)."""
    x = x.detach().double()
    half = state["turns"].numel()
    t = torch.stack([state["positions"][int(a)].double() * f
                     for a, f in zip(state["axis"].tolist(), state["turns"])], dim=-1)[:, None]
    w = torch.polar(torch.ones_like(t), sign * 2 * math.pi * torch.remainder(t, 1.0))
    lo, hi = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if state["case"]["interleaved"] else \
        (slice(0, half), slice(half, 2 * half))
    z = torch.complex(x[..., lo].contiguous(), x[..., hi].contiguous()) * w
    out = x.clone()
    out[..., lo], out[..., hi] = z.real, z.imag
    return out


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "axes":
        out = [_exact_rotate(state, state[x], 1.0) for x in "qk"]
        if case["grad"]:
            out += [_exact_rotate(state, state[x], -1.0) for x in ("gq", "gk")]
        return tuple(out)
    lens, cu, offs = (state[x].tolist() for x in ("lens", "cu", "offsets"))
    Hkv, D, P = case["kv_heads"], case["head_dim"], case["page"]
    G = case["heads"] // Hkv
    shared = state["prefix_lens"].tolist() if "prefix_lens" in state else [0]
    edges = state["cu_seqs"].tolist() if "prefix_lens" in state else [0, len(lens)]
    cost = sum((cu[b + 1] - cu[b]) * (n + shared[sum(b >= x for x in edges[1:])])
               for b, n in enumerate(lens))
    if cost > 1e8:
        return None

    def tokens(name, table, n):   # [Hkv, n, D]
        pages = state[name][table[:-(-n // P)].long()].double()
        return pages.permute(1, 0, 3, 2).reshape(Hkv, -1, D)[:, :n]

    out, group, kept = [], 0, None
    for b, n in enumerate(lens):
        while b >= edges[group + 1]:
            group, kept = group + 1, None
        q = state["q"][cu[b]:cu[b + 1]].double()
        rows = q.shape[0]
        q = q.view(rows, Hkv, G, D).permute(1, 2, 0, 3).reshape(Hkv, G * rows, D)
        k, v = (tokens(x, state["block_tables"][b], n) for x in ("k_pages", "v_pages"))
        first = n - 1 if case["op"] in ("window", "prefix") else offs[b]
        at = first + torch.arange(rows, device="cuda")[:, None]
        j = torch.arange(n, device="cuda")
        hidden = j > at
        if case["op"] in ("window", "wrows"):
            hidden = hidden | ((j <= at - case["window"]) & (j >= case["sinks"]))
        if shared[group]:
            if kept is None:
                kept = [tokens(x, state["prefix_tables"][group], shared[group])
                        for x in ("k_pages", "v_pages")]
            k, v = torch.cat([kept[0], k], dim=1), torch.cat([kept[1], v], dim=1)
            hidden = torch.cat([torch.zeros(rows, shared[group], dtype=torch.bool, device="cuda"),
                                hidden], dim=1)
        s = (q @ k.transpose(1, 2)).view(Hkv, G, rows, -1) / math.sqrt(D)
        p = torch.softmax(s.masked_fill(hidden, -math.inf), dim=-1).view(Hkv, G * rows, -1)
        out.append((p @ v).view(Hkv, G, rows, D).permute(2, 0, 1, 3).reshape(rows, Hkv * G, D))
    return torch.cat(out)
