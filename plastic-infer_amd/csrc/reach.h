// Attention over the paged float pools in which a row sees a part of the context, or more than its own:
//
//   window  the row at position p sees tokens j <= p of its sequence with p - j < window or j < sinks
//   prefix  a row sees all tokens of its group's prefix and then those of its own sequence
//
// The kernels differ in how they share the work; what a row sees they all take from here.
#pragma once

#include "pia_internal.h"

namespace pia {
namespace reach {

constexpr int FAR = 0x7ffff000;  // beyond every token, with room for a few tiles behind it

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
  // of the kernels that share work
  int first, count;  // the sequences (by_group: groups) of a launch
  int by_group;      // a "sequence" is a group: all its rows, over its prefix
  int whole;         // no item is cut
  int splits;        // workgroups of an item; 0: none are an item's
  unsigned long long* counters;  // of an item's workgroups, and the launch's token in them
  unsigned long long token;
  float* parts;      // pieces of items, by wave
  int64_t* pref;
  // Pieces of rows: unnormalised outputs [n, rows * Hq, D] and (reference point in log2 units, sum)
  // [n, rows * Hq]. dst: where results go instead of out; src: src_cuts pieces of the prefix and behind
  // them one of the rest.
  float* dst;
  float2* dst_ml;
  const float* src;
  const float2* src_ml;
  int src_cuts;
};

// tokens of a table that are there
__device__ __forceinline__ int held(int len, int64_t stride, int P) {
  return int(min(int64_t(max(len, 0)), min(stride * P, int64_t(FAR))));
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

// A sequence: its rows and tokens, and the position of its first row where rows are limited by theirs
struct Seq {
  int64_t row0;
  int n, len, off;
  bool causal;
};
// the first row of sequence b <= B
__device__ __forceinline__ int64_t row_of(const Args& a, int b) { return a.cu ? a.cu[b] : b; }
__device__ __forceinline__ int edge_of(const Args& a, int g) {  // the first sequence of group g
  return a.gs ? min(max(a.gs[g], 0), a.B) : g == 0 ? 0 : a.B;
}
__device__ __forceinline__ Seq sequence(const Args& a, int b) {
  Seq s;
  s.row0 = row_of(a, b);
  const int64_t n = row_of(a, b + 1) - s.row0;
  s.n = s.row0 < 0 ? 0 : int(max(int64_t(0), min(n, a.rows - s.row0)));
  s.len = held(a.lens[b], a.bt_stride, a.P);
  s.causal = a.offs || a.window;
  s.off = a.offs ? a.offs[b] : a.window ? s.len - s.n : 0;
  return s;
}
__device__ __forceinline__ Seq group(const Args& a, int g) {
  Seq s;
  s.row0 = row_of(a, edge_of(a, g));
  const int64_t n = row_of(a, edge_of(a, g + 1)) - s.row0;
  s.n = s.row0 < 0 ? 0 : int(max(int64_t(0), min(n, a.rows - s.row0)));
  s.len = held(a.plens[g], a.pt_stride, a.P);
  s.off = 0;
  s.causal = false;
  return s;
}
// Row pos of a sequence sees tokens lowest .. limit - 1 and (window) the first `sinks` of those below limit
__device__ __forceinline__ int limit(const Seq& s, int pos) {
  return s.causal ? int(max(int64_t(0), min(int64_t(s.len), int64_t(s.off) + pos + 1))) : s.len;
}
__device__ __forceinline__ int lowest(const Args& a, const Seq& s, int pos) {
  if (!a.window) return 0;
  return int(max(int64_t(0), min(int64_t(FAR), int64_t(s.off) + pos + 1 - a.window)));
}

// Items of 16 (position, head) rows, whose tokens go by steps: a tile of `step` tokens each.
__device__ __forceinline__ int items_of(int n, int G) { return int((int64_t(n) * G + 15) >> 4); }
// Tiles of the sinks that some row sees
__device__ __forceinline__ int head_tiles(const Args& a, const Seq& s, int step) {
  if (!a.window) return 0;
  return (min(a.sinks, limit(s, s.n - 1)) + step - 1) / step;
}
// Steps of each item of a sequence: as many as any of them needs
__device__ __forceinline__ int steps_of(const Args& a, const Seq& s, int step) {
  const int total = (limit(s, s.n - 1) + step - 1) / step;
  if (!a.window) return total;
  const int nh = head_tiles(a, s, step);
  if (s.n == 1) return nh + max(0, total - max(nh, lowest(a, s, 0) / step));
  // an item's rows are of 15 / G + 2 positions at most; that many tokens and the window's lie in so many tiles
  const int64_t span = int64_t(a.window) + min(s.n, 15 / a.G + 2) - 1;
  return int(min(int64_t(total), nh + (span + step - 2) / step + 1));
}
// The tile of an item's step t: nh tiles of the sinks, then those from t0 on. Items have steps past their own
// tokens, and where positions come near 2^31 past all that 32 bits count: those are the tile at FAR, where no
// token is.
__device__ __forceinline__ int tile_of(int nh, int t0, int t, int step) {
  return t < nh ? t : min(t0 + t - nh, FAR / step);
}
// Whether some row of an item sees a token of block kb (16 tokens), where they see the sinks' and lo .. end - 1
__device__ __forceinline__ bool block_seen(const Args& a, int lo, int end, int kb) {
  return kb * 16 < end && (!a.window || kb * 16 < a.sinks || kb * 16 + 16 > lo);
}

// The prefix's pieces of a row of sequence b, if it has any
__device__ __forceinline__ bool has_prefix(const Args& a, int b) {
  const int g = group_of(a, b);
  return g >= 0 && held(a.plens[g], a.pt_stride, a.P) > 0;
}
// the weight of a piece whose reference is m against the joined one
__device__ __forceinline__ float weight(float m, float joined) {
  return m == joined ? (m == -INFINITY ? 0.f : 1.f) : __builtin_amdgcn_exp2f(m - joined);
}

// How the tiled kernel takes a call: 256 rows at a time or 128, and the pieces of an item
struct TilePlan {
  bool wide;
  int cuts;
};

}  // namespace reach

// Any head_dim to 512, page size and group: one wave for each row and head (reach_general.hip)
int launch_reach_general(const reach::Args& a, int dtype, hipStream_t s);

// Items of 16 rows over a contiguous range of their steps for each resident wave (reach_stream.h), for the
// sequences or (by_group) for the groups. tokens: a bound of the tokens that an item walks.
int launch_reach_stream_f32(const reach::Args& a, int64_t tokens, hipStream_t s);
int launch_reach_stream_f16(const reach::Args& a, int64_t tokens, hipStream_t s);
int launch_reach_stream_bf16(const reach::Args& a, int64_t tokens, hipStream_t s);
// Tiles in LDS for 128 or 256 rows at a time (reach_tiles.hip), 16-bit pools: whether a call's shape is taken,
// into how many pieces (at most `most`) it would cut each item of such a call, and its launch. Pieces
// go to dst; those of sequences are joined there, those of groups are not.
bool reach_tiles_shape(const reach::Args& a, int dtype);
reach::TilePlan reach_tiles_plan(const reach::Args& a, int64_t tokens, int64_t most);
int launch_reach_tiles(const reach::Args& a, int dtype, reach::TilePlan plan, hipStream_t s);
// a number that no other launch has, in the upper 48 bits
unsigned long long reach_token();
// bytes of the streaming kernel's pieces by wave, and of the numbers before them
int64_t reach_stream_parts_bytes(int D);
int64_t reach_stream_pref_bytes();

}  // namespace pia
