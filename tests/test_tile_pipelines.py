"""The tiled attention kernels' pipelines: no LDS buffer is read by one wave and written by another between
the same two barriers. The kernels' own text is followed, from the first tile's staging over six steps of
the loop (CPU; a race of waves shows in results hardly ever)."""

from __future__ import annotations

import pathlib
import re

import pytest

CSRC = pathlib.Path(__file__).resolve().parents[1] / "plastic-infer_amd" / "csrc"
START = "// K is staged two tiles ahead of the outputs"
# calls that touch a buffer: which argument names it
TOUCH = {"stage_k": ("write K", 1), "stage_v": ("write V", 1), "kread": ("read K", 0),
         "vread": ("read V", 0)}


def _closing(text, at):
    """The place behind the bracket that closes the one at `at`."""
    pair = {"(": ")", "{": "}"}[text[at]]
    depth = 0
    for i in range(at, len(text)):
        depth += (text[i] == text[at]) - (text[i] == pair)
        if depth == 0:
            return i + 1
    raise AssertionError("no closing bracket")


def _split(args):
    parts, depth = [""], 0
    for c in args:
        depth += (c in "([{") - (c in ")]}")
        if c == "," and depth == 0:
            parts.append("")
        else:
            parts[-1] += c
    return [p.strip() for p in parts]


def _lambdas(text):
    """name -> (parameters, body, where it begins and ends)"""
    out = {}
    for m in re.finditer(r"auto (\w+) = \[&\]\(", text):
        end = _closing(text, m.end() - 1)
        brace = text.index("{", end)
        assert re.fullmatch(r"\s*(RT_INLINE|-> [\w&: ]+?)?\s*", text[end:brace]), m.group(1)
        close = _closing(text, brace)
        params = [re.findall(r"[A-Za-z_]\w*", p)[-1] for p in _split(text[m.end():end - 1]) if p]
        out[m.group(1)] = (params, text[brace + 1:close - 1], m.start(), close)
    return out


def _value(expr, env):
    try:
        return eval(expr, {"__builtins__": {}}, env)
    except (NameError, SyntaxError, TypeError):
        return None


def _events(text, env, known):
    out = []
    for m in re.finditer(r"\b(\w+)\(", text):
        name = m.group(1)
        if name != "__syncthreads" and name not in TOUCH and name not in known:
            continue
        args = _split(text[m.end():_closing(text, m.end() - 1) - 1])
        if name == "__syncthreads":
            out.append("barrier")
        elif name in TOUCH:
            what, i = TOUCH[name]
            buf = _value(args[i], env)
            assert buf in (0, 1), (name, args, env)
            out.append(f"{what}{buf}")
        else:
            params, body, _, _ = known[name]
            out += _events(body, {p: _value(a, env) for p, a in zip(params, args)}, known)
    return out


def _pipeline(source):
    source = re.sub(r"//[^\n]*", lambda m: m.group(0) if START in m.group(0) else "", source)
    known = _lambdas(source)
    begin = source.index(START)
    prologue = source[begin:known["step"][2]]
    for _, _, a, b in sorted(known.values(), key=lambda x: x[2]):   # what it defines is not yet called
        if begin <= a and b <= known["step"][2]:
            prologue = prologue.replace(source[a:b], "")
    kept = {n: known[n] for n in ("stage", "stage_next", "scores", "turn", "step") if n in known}
    events = _events(prologue, {}, kept)
    for i in range(6):
        events += _events("step(sc, sn, it, buf)", {"buf": i & 1}, kept)
    return events


def _conflicts(events):
    """Buffers that are read and written between two barriers."""
    bad, epoch = [], set()
    for e in [*events, "barrier"]:
        if e != "barrier":
            epoch.add(e)
            continue
        bad += [e[5:] for e in epoch if e.startswith("read") and "write" + e[4:] in epoch]
        epoch = set()
    return bad


@pytest.mark.parametrize("kernel", ["reach_tiles.hip", "kv8_prefill.hip"])
def test_no_buffer_is_read_and_written_between_two_barriers(kernel):
    events = _pipeline((CSRC / kernel).read_text())
    # the test follows what it should: both buffers of K and V are written and read
    assert {f"{w} {x}{b}" for w in ("read", "write") for x in "KV" for b in (0, 1)} <= set(events)
    assert events.count("barrier") >= 7
    assert not _conflicts(events), events


def test_a_missing_barrier_is_found():
    events = _pipeline((CSRC / "reach_tiles.hip").read_text())
    at = [i for i, e in enumerate(events) if e == "barrier"]
    found = [bool(_conflicts(events[:i] + events[i + 1:])) for i in at[:-1]]
    assert sum(found) >= 6, events
