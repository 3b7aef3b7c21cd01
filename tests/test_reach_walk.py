"""The tiles and blocks that the streaming kernel of windowed attention walks, from the kernels' own header
compiled for the host (CPU): every token that a row of an item sees is in one step of it, and no block is read
from behind the table, whatever the positions."""

from __future__ import annotations

import pathlib
import subprocess

import pytest

CSRC = pathlib.Path(__file__).resolve().parents[1] / "plastic-infer_amd" / "csrc"

STUB = r"""
#pragma once
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <vector>
#define __device__
#define __forceinline__ inline
#define __builtin_amdgcn_exp2f exp2f
using std::max;
using std::min;
struct float2 { float x, y; };
typedef void* hipStream_t;
"""

MAIN = r"""
#include "reach.h"
using namespace pia::reach;

// The walk of the ranges form: every item of a sequence takes steps_of() steps.
static int walk(int len, int off, int rows, int G, int window, int sinks, int step, int P) {
  Args a{};
  const int32_t lens[1] = {len}, offs[1] = {off}, cu[2] = {0, rows};
  a.lens = lens; a.offs = offs; a.cu = cu;
  a.rows = rows; a.B = 1; a.G = G; a.Hq = G; a.Hkv = 1; a.P = P;
  a.window = window; a.sinks = sinks;
  a.bt_stride = (int64_t(len) + P - 1) / P;
  const Seq s = sequence(a, 0);
  const int steps = steps_of(a, s, step), nh = head_tiles(a, s, step);
  for (int i = 0; i < items_of(s.n, G); ++i) {
    const int p0 = 16 * i / G, p1 = min((16 * i + 15) / G, s.n - 1);
    const int lo = lowest(a, s, p0), end = limit(s, p1);
    const int t0 = a.window ? max(nh, lo / step) : 0;
    std::vector<int64_t> tiles;
    for (int t = 0; t < steps; ++t) {
      const int tile = tile_of(nh, t0, t, step);
      if (int64_t(tile) * step > FAR) { printf("tile %d of step %d\n", tile, t); return 1; }
      tiles.push_back(tile);
      for (int m = 0; m < step / 16; ++m) {
        const int kb = tile * (step / 16) + m;
        const int64_t from = int64_t(kb) * 16;     // the block's tokens, in 64 bits
        if (from < 0 || from > FAR + step) { printf("block %d of step %d\n", kb, t); return 1; }
        const bool seen = from < end && (!window || from < sinks || from + 16 > lo);
        if (block_seen(a, lo, end, kb) != seen) { printf("block %d seen %d\n", kb, !seen); return 1; }
        if (seen && (kb / (P / 16) < 0 || kb / (P / 16) >= a.bt_stride)) {
          printf("entry %d of %lld\n", kb / (P / 16), (long long)a.bt_stride);
          return 1;
        }
      }
    }
    // tiles with a token that some row sees, by the definition: each once
    for (int p = p0; p <= p1; ++p) {
      const int64_t pos = int64_t(off) + p;
      for (int64_t j : {pos - window, pos - window + 1, pos - 1, pos, int64_t(0), int64_t(sinks) - 1,
                        int64_t(len) - 1, int64_t(sinks), pos - window / 2, int64_t(len) / 2}) {
        if (j < 0 || j >= s.len || j > pos || (window && pos - j >= window && j >= sinks)) continue;
        if (std::count(tiles.begin(), tiles.end(), j / step) != 1) {
          printf("token %lld of position %lld\n", (long long)j, (long long)pos);
          return 1;
        }
      }
    }
  }
  return 0;
}

int main() {
  const int top = 0x7fffffff;
  for (int step : {16, 32, 64})
    for (int P : {16, 48, 4096})
      for (int G : {1, 3, 4, 16, 33})
        for (int rows : {1, 2, 17, 40})
          for (int window : {1, 64, 100, 4095, 4096, 9000, 1 << 30, top})
            for (int sinks : {0, 1, 70, 5000, top})
              for (int len : {1, 63, 4096, 4500, 20000})
                for (int64_t off : {int64_t(-5), int64_t(0), int64_t(len - rows), int64_t(len + 50),
                                    int64_t(FAR) - 3000, int64_t(FAR), int64_t(top) - 64,
                                    int64_t(top) - 1, int64_t(top)})
                  if (walk(len, int(off), rows, G, window, sinks, step, P)) {
                    printf("len %d off %lld rows %d G %d window %d sinks %d step %d page %d\n", len,
                           (long long)off, rows, G, window, sinks, step, P);
                    return 1;
                  }
  return 0;
}
"""


def _run(tmp_path, header):
    (tmp_path / "pia_internal.h").write_text(STUB)
    (tmp_path / "reach.h").write_text(header)
    (tmp_path / "walk.cpp").write_text(MAIN)
    exe = tmp_path / "walk"
    subprocess.run(["g++", "-O1", "-std=c++17", "-fwrapv", "-o", exe, tmp_path / "walk.cpp"], check=True)
    return subprocess.run([exe], capture_output=True, text=True, timeout=120)


def test_walk(tmp_path):
    run = _run(tmp_path, (CSRC / "reach.h").read_text())
    assert run.returncode == 0, run.stdout


@pytest.mark.parametrize("right,wrong", [
    ("min(t0 + t - nh, FAR / step)", "t0 + t - nh"),                  # tiles beyond 32 bits
    ("(span + step - 2) / step + 1", "(span + step - 2) / step"),     # a step too few
    ("kb * 16 < end &&", "")])                                        # blocks behind the table
def test_mistakes_are_found(tmp_path, right, wrong):
    header = (CSRC / "reach.h").read_text()
    assert header.count(right) == 1
    run = _run(tmp_path, header.replace(right, wrong))
    assert run.returncode == 1, run.stdout
    print(run.stdout)
