// Attention over the paged float pools in which a row sees a part of the context, or more than its own:
//
//   window  the row at position p sees tokens j <= p of its sequence with p - j < window or j < sinks
//   prefix  a row sees all tokens of its group's prefix and then those of its own sequence
//
// Both are two stretches of keys: the first `head` tokens of one table (the sinks in the sequence's own, or
// the prefix's), which every row sees whole but where a causal limit cuts the sinks, and tokens lo .. lim - 1
// of the sequence's table, with limits that move with the row. The kernels differ in how they share the
// work; what a row sees they all take from here.
#pragma once

#include "pia_internal.h"

namespace pia {
namespace reach {

struct Args {
  void* out;
  const void* q;
  int64_t q_stride;  // elements between rows
  const void *kp, *vp;
  const int32_t* bt;
  int64_t bt_stride;
  const int32_t *lens, *cu, *offs;
  int64_t rows, num_pages, first_row;  // first_row: of a launch that takes a part of the rows
  float scale_log2;
  int B, Hq, Hkv, G, D, P;
  int window, sinks;  // window 0: every token up to the row's limit
  const int32_t* pt;  // prefix tables, null: none
  int64_t pt_stride;
  const int32_t *plens, *gs;  // gs null: one group of all sequences
  int groups;
};

// tokens of a table that are there
__device__ __forceinline__ int held(int len, int64_t stride, int P) {
  return int(min(int64_t(max(len, 0)), min(stride * P, int64_t(0x7ffffff0))));
}

// The group of sequence b (-1: none)
__device__ __forceinline__ int group_of(const Args& a, int b) {
  if (!a.pt || a.groups <= 0) return -1;
  if (!a.gs) return 0;
  int lo = 0, hi = a.groups - 1;  // the last that begins at or before b
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a.gs[mid] <= b) lo = mid; else hi = mid - 1;
  }
  return a.gs[lo] <= b && b < a.gs[lo + 1] ? lo : -1;
}

// A sequence: its rows and tokens, the position of its first row (window) or the causal offset
struct Seq {
  int64_t row0;
  int n, len;
  int off;
  bool causal;
};
__device__ __forceinline__ Seq sequence(const Args& a, int b) {
  Seq s;
  s.row0 = a.cu ? a.cu[b] : b;
  const int64_t n = a.cu ? int64_t(a.cu[b + 1]) - s.row0 : 1;
  s.n = s.row0 < 0 ? 0 : int(max(int64_t(0), min(n, a.rows - s.row0)));
  s.len = held(a.lens[b], a.bt_stride, a.P);
  s.causal = a.offs || a.window;
  s.off = a.offs ? a.offs[b] : a.window ? s.len - s.n : 0;
  return s;
}
// Row pos of a sequence sees tokens lo .. lim - 1, and (window) the first `sinks` of those below lim
__device__ __forceinline__ int limit(const Seq& s, int pos) {
  return s.causal ? int(max(int64_t(0), min(int64_t(s.len), int64_t(s.off) + pos + 1))) : s.len;
}
__device__ __forceinline__ int lowest(const Args& a, const Seq& s, int pos) {
  if (!a.window) return 0;
  return int(max(int64_t(0), min(int64_t(0x7ffffff0), int64_t(s.off) + pos + 1 - a.window)));
}

}  // namespace reach

// Any head_dim to 512, page size and group: one wave for each row and head (reach_general.hip)
int launch_reach_general(const reach::Args& a, int dtype, hipStream_t s);

}  // namespace pia
