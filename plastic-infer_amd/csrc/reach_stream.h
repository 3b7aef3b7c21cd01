// The streaming kernel of windowed attention and of attention behind a shared prefix: few rows for each
// key, any dtype, head_dim to 256 in multiples of 16, pages in multiples of 16 tokens.
//
// Bound by HBM where there is enough to read: K and V of the keys that some row sees, once (128 sequences, window
// of 4096 on 512 .. 8192 tokens, 32 / 8 heads of 128, bf16: 283 us with the joining, 6.0 TB/s, 1.01 times the bytes);
// small calls by their chain of dependent loads (lengths, page ids, K, V) and the launch: one sequence in a window
// of 1024 13.3 us, of 64 8.7. Their waves wait for memory for half of their cycles (24 fp32 sequences in a window of
// 500: 45 %, with 17 % in products; 16 sequences of 1 .. 6 rows: 57 % and 2 %). An item is 16 (position, head) rows of a sequence (or of a group, over its
// prefix) and kv head; it walks the tiles that some of its rows see by steps of STEP tokens. The next step's K and
// V are on their way while a step is computed. Two forms:
//
//   ranges (many items)  all steps of all items, in order, are cut into one contiguous range for every resident
//     wave, whatever the batch looks like, and loads run on across items. An item that lies in one range is finished
//     there; pieces of the others (at most two a wave) go to the workspace, and a second kernel joins them.
//     Items of a few steps (WHOLE, by what the host knows) are not cut, and have no second kernel.
//   items (ITEM, no more items than resident workgroups)  a workgroup has a run of an item's steps, its four waves
//     a quarter each, joined in LDS. Where an item has several workgroups, each leaves its piece behind the caches
//     of its XCD and counts itself; the last to arrive joins all pieces. (One sequence, window of 1024: 17.0 us as
//     ranges, 13.2 so.) The counter holds a number of the launch, so the workspace needs no clearing.
//
// Pieces are joined in their order in both: results do not depend on timing.
//
// Both products run on the matrix cores, whose operands come from memory in place. The pool's rows are
// [d][token], so that a lane's load is some neighbouring tokens of one element. kd = lane / 16, n16 = lane % 16:
//   S^T = K . q^T  a unit is UB bytes of a row (TU tokens); lane l loads unit(n16) of the rows d = 4 i + kd: whole
//                  128-byte lines of each page at once. The elements of its rows are the k slots (16 bits: eight
//                  rows i by v_perm; fp32: one row), each token of the unit a product of its own, q the other
//                  operand from LDS. Lane l then has in s[c][v] row n16's score of token c of unit(4 kd + v).
//   O^T = V^T . P^T  lane l loads 16 bytes of the rows d = 16 nb + n16: 8 (4) tokens, and unit() is so chosen that they
//                  are the tokens of the lane's scores. A row's outputs sit in its own lanes, elements 16 nb + 4 kd + j.
//
// Precision: products of 16-bit values are exact in fp32, in which scores, sums and outputs are held. The
// probabilities over 16-bit pools are two terms of the pool's type (2^-17 of each), the first rounded toward zero
// and neither ever 0 for a positive value: an infinite V then gives that infinity and not infinity - infinity.
// fp16's numbers end at 2^-38 of the reference, so a step with smaller ones than 2^-24 of it multiplies what
// the two terms leave, too (the rest): without that, thousands of them before V much larger than the likely
// tokens' were off by the least number each.
// Over fp32 pools all products are fp32's, a step's summed on their own first.
//
// A row's result may depend on what it sees only. Scores of other tokens are -inf. V of tokens that no row
// of the item sees are zeros. Where rows differ in what they see (not ALIKE) and such a tile holds a V that is
// not finite, it is summed on the vector ALU, row by row.
#pragma once

#include <algorithm>

#include "attn_tiles.h"
#include "attn_tiles_f32.h"
#include "reach.h"

namespace pia {
namespace reach_stream {

using reach::Args;
using reach::Seq;
using reach::head_tiles;
using reach::items_of;
using reach::steps_of;
using tile::f32x4_t;

constexpr int MAX_SEQS = 1024;  // sequences per launch (their tables in LDS)
constexpr int WG_WAVES = 4;
// Two waves per SIMD. Ranges and runs are made for as many, also where LDS holds one workgroup on a CU: fp32 at
// head_dim over 128 (89 to 99 KB) and items of rows that see different tokens there (89 KB) take them in two rounds.
constexpr int WGS_PER_CU = 2;
// Steps of items that are not cut where items outnumber the resident workgroups (32 / 8 heads of 128, us; not cut
// for cut): 512 sequences, window of 128 (5 steps) 67.5 for 72, 128 sequences 27.7 for 31.5; a window of 192 (6) 87
// for 90 and 39.8 for 34.6.
constexpr int WHOLE = 5;
constexpr int MAX_SPLITS = 64;  // workgroups of an item
// Steps of a wave above which even ranges for all waves are better than items of workgroups' own. A window's
// items are alike (64 sequences, 2048: 84 us for 102 in ranges; 16 sequences, 8192: 89 for 99); contexts need not
// be, and the longest would be waited for.
constexpr int ITEM_STEPS = 8, ITEM_STEPS_WINDOW = 16;
constexpr int JOIN_MANY = 128, JOIN_FEW = 512;  // threads of the joining workgroups

// log2: how far a row's maximum may run ahead of its reference, and what probabilities are scaled by. fp16's
// numbers, to 2^15, then go down to 2^-38 of the reference (8 and 7 in place of 1 and 14: a window of 1024 before
// one sequence with wide scores 14.7 us for 13.7, its steps nearly all with a rest).
template <int DT>
constexpr float RESCALE = DT == PIA_DTYPE_F16 ? 1.0f : 8.0f;
template <int DT>
constexpr float SHIFT = DT == PIA_DTYPE_F16 ? 14.0f : 0.0f;

template <int DT, int DP>
struct Form {
  static constexpr bool F32 = DT == PIA_DTYPE_F32;
  static constexpr int E = F32 ? 4 : 2;
  static constexpr int UB = DP > 128 ? 4 : 8;  // registers
  static constexpr int TU = UB / E, STEP = 16 * TU, MB = STEP / 16;
  static constexpr int NI = DP / 4, NB = DP / 16;
  static constexpr int NU = F32 ? MB : STEP / 32;  // 16-byte V loads of a row
  static constexpr int QS = NI + 16 / E;           // stride of a lane's q elements in LDS
  using T = typename Elem<DT>::T;
};

// 64-bit quotient of numbers that nearly always have 32 bits (the long division is 150 instructions)
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
  if (((a | b) >> 32) == 0) return int64_t(uint32_t(a) / uint32_t(b));
  return a / b;
}
// Ranges of the waves: total steps over n waves, one more for the first total % n of them. The first
// step of wave w, and the wave that has step x.
__device__ __forceinline__ int64_t first_of(int64_t w, int64_t n, int64_t total) {
  const int64_t q = quotient(total, n);
  return q * w + min(w, total - q * n);
}
__device__ __forceinline__ int64_t wave_of(int64_t x, int64_t n, int64_t total) {
  const int64_t q = quotient(total, n), more = total - q * n, edge = (q + 1) * more;
  return x < edge ? quotient(x, q + 1) : more + quotient(x - edge, q);
}
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

template <int DP>
constexpr int64_t part_floats = 16 * (DP + 2);  // 16 rows' outputs, references and sums

__device__ __forceinline__ Seq seq_at(const Args& a, int b) {
  return a.by_group ? reach::group(a, a.first + b) : reach::sequence(a, a.first + b);
}
// Eight probabilities as two 16-bit operands. fill ~0: neither is 0 for a positive one, but the least number;
// 0: they may be.
template <int DT>
__device__ __forceinline__ void split2(const float (&p)[8], uint4 (&t)[2], uint32_t fill) {
  typedef unsigned short u16x2_t __attribute__((ext_vector_type(2)));
  uint32_t w[2][4];
#pragma unroll
  for (int f = 0; f < 4; ++f) {
    float a = p[2 * f], b = p[2 * f + 1];
    const uint32_t low =
        fill & (min(__float_as_uint(a), 1u) | (min(__float_as_uint(b), 1u) << 16));  // 1 where positive
    auto filled = [&](uint32_t x) {
      return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2_t, x),
                                                                    __builtin_bit_cast(u16x2_t, low)));
    };
    if constexpr (DT == PIA_DTYPE_F16) {
      const auto h = __builtin_amdgcn_cvt_pkrtz(a, b);
      a -= float(h[0]);
      b -= float(h[1]);
      w[0][f] = filled(__builtin_bit_cast(uint32_t, h));
    } else {  // truncated to 0 below 2^-126 alone
      w[0][f] = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
      a -= bf16_hi(__float_as_uint(a));
      b -= bf16_hi(__float_as_uint(b));
    }
    w[1][f] = filled(tile::pack16x2<DT>(a, b));
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) t[k] = make_uint4(w[k][0], w[k][1], w[k][2], w[k][3]);
}

// fp16, of probabilities below 2^-10, in 2^38ths (2^-25 at most, so 2^13 of them): what rounding to two terms
// took or, if `least`, minus the least numbers that split2 put in.
constexpr float REST_BELOW = 0x1p-10f, REST = 0x1p38f, PUT = 0x1p14f;
__device__ __forceinline__ uint4 rest2(const float (&p)[8], bool least) {
  uint32_t w[4];
#pragma unroll
  for (int f = 0; f < 4; ++f) {
    float y[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float x = p[2 * f + e];
      asm volatile("" : "+v"(x));  // so that nothing of this is kept for split2, which costs registers
      const float hi = float(__builtin_amdgcn_cvt_pkrtz(x, x)[0]);
      const float lo = float(static_cast<_Float16>(x - hi));
      y[e] = least ? (hi == 0.f ? -PUT : 0.f) + (lo == 0.f ? -PUT : 0.f) : (x - hi - lo) * REST;
      y[e] = x > 0.f && x < REST_BELOW ? y[e] : 0.f;
    }
    w[f] = tile::pack16x2<PIA_DTYPE_F16>(y[0], y[1]);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// sum of eight fp16 numbers' squares onto c: finite if they all are
__device__ __forceinline__ float squares(const uint4& x, float c) {
  typedef _Float16 h2 __attribute__((ext_vector_type(2)));
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    c = __builtin_amdgcn_fdot2(__builtin_bit_cast(h2, w[i]), __builtin_bit_cast(h2, w[i]), c, false);
  return c;
}
// zeros for those that are not finite
__device__ __forceinline__ uint4 finite_of(const uint4& x) {
  auto of = [](uint32_t w) {
    return w & (((w & 0x7c00u) == 0x7c00u ? 0u : 0xffffu) |
                ((w & 0x7c000000u) == 0x7c000000u ? 0u : 0xffff0000u));
  };
  return make_uint4(of(x.x), of(x.y), of(x.z), of(x.w));
}

// UB bytes of a row
template <int UB>
struct Unit {
  uint32_t w[UB / 4];
};
template <int UB, bool NT>
__device__ __forceinline__ Unit<UB> load_unit(const void* p) {
  typedef uint32_t vec __attribute__((ext_vector_type(UB / 4)));
  vec v;
  if constexpr (NT) v = __builtin_nontemporal_load(static_cast<const vec*>(p));
  else v = *static_cast<const vec*>(p);
  return __builtin_bit_cast(Unit<UB>, v);
}

// Stores and loads of what workgroups on other XCDs read or wrote in this launch: through the XCD's L2 (SC1, what
// relaxed atomics of agent scope are), 16 bytes at a time. at: bytes from the descriptor's base.
constexpr int FAR_AUX = 16;
__device__ __forceinline__ auto far_memory(float* p, int64_t floats) {
  return __builtin_amdgcn_make_buffer_rsrc(p, 0, int(floats * 4), 0x00020000);
}
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
template <class R>
__device__ __forceinline__ void put_far(R r, int at, const float4& v) {
  __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_t, v), r, at, 0, FAR_AUX);
}
template <class R>
__device__ __forceinline__ void put_far(R r, int at, const float2& v) {
  __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2_t, v), r, at, 0, FAR_AUX);
}
template <class R>
__device__ __forceinline__ float4 get_far4(R r, int at) {
  return __builtin_bit_cast(float4, __builtin_amdgcn_raw_buffer_load_b128(r, at, 0, FAR_AUX));
}
template <class R>
__device__ __forceinline__ float2 get_far2(R r, int at) {
  return __builtin_bit_cast(float2, __builtin_amdgcn_raw_buffer_load_b64(r, at, 0, FAR_AUX));
}
// Counts a workgroup in at its item's counter, which holds (token of the launch, arrivals); true for the last
// of n. What it held before (another launch's, or anything) is replaced by whoever comes first. The last one
// leaves it at no arrivals, for a graph that replays the launch with its token. 48 random bits of a token: what
// an unused workspace holds is taken for it once in 2^48.
__device__ __forceinline__ bool arrive(unsigned long long* counter, unsigned long long token, int n) {
  unsigned long long seen =
      __hip_atomic_load(counter, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  for (;;) {
    const bool ours = (seen >> 16) == (token >> 16);
    const unsigned long long to = ours ? seen + 1 : token + 1;
    if (!ours) {
      if (__hip_atomic_compare_exchange_strong(counter, &seen, to, __ATOMIC_RELAXED, __ATOMIC_RELAXED,
                                               __HIP_MEMORY_SCOPE_AGENT))
        return n == 1;
      continue;  // another one of this launch put the token there
    }
    const unsigned long long before =
        __hip_atomic_fetch_add(counter, 1ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (int(before & 0xffffu) + 1 < n) return false;
    __hip_atomic_store(counter, token, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return true;
  }
}

// A row's four outputs o (of sum l), normalised
template <int DT>
__device__ __forceinline__ void store4(typename Elem<DT>::T* out, const float (&o)[4], float l) {
  using T = typename Elem<DT>::T;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  struct alignas(4 * sizeof(T)) Pack {
    T v[4];
  } pk;
#pragma unroll
  for (int j = 0; j < 4; ++j) Elem<DT>::store(pk.v, j, l == 0.f ? 0.f : o[j] * inv);
  *reinterpret_cast<Pack*>(out) = pk;
}

// ALIKE: all rows of an item see the same tokens. FULL: head_dim is DP. ITEM: a workgroup takes one of a.splits
// runs of an item's steps, and the last of an item's workgroups joins them.
template <int DT, int DP, bool ALIKE, bool FULL, bool ITEM>
__global__ __launch_bounds__(64 * WG_WAVES, WGS_PER_CU) void reach_stream_kernel(Args a) {
  using F = Form<DT, DP>;
  using T = typename F::T;
  constexpr int TU = F::TU, STEP = F::STEP, MB = F::MB, NI = F::NI, NB = F::NB, NU = F::NU;
  constexpr int NW = WG_WAVES, NTH = 64 * NW;
  constexpr bool F32 = F::F32;
  __shared__ int64_t pref[ITEM ? 1 : MAX_SEQS + 1];
  __shared__ int4 seqs[ITEM ? 1 : MAX_SEQS];  // first row (below 2^30), rows, tokens, offset
  __shared__ int64_t wsum[NW];
  __shared__ __align__(16) T qs[ITEM ? 1 : NW][64 * F::QS];
  __shared__ float ps[ALIKE ? 1 : NW][ALIKE ? 1 : 16 * (STEP + 1)];
  // ITEM: items of the sequences before each; the waves' pieces
  __shared__ int item_pref[ITEM ? MAX_SEQS + 1 : 1];
  constexpr int RS = DP + 4;
  __shared__ __align__(16) float red[ITEM ? NW * 16 * RS : 4];
  __shared__ float red_m[ITEM ? NW * 16 : 1], red_l[ITEM ? NW * 16 : 1];
  __shared__ int is_last;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int kd = lane >> 4, n16 = lane & 15;
  const int D = FULL ? DP : a.D;

  // where a wave is: step t of item i of kv head h of sequence b; tiles nh .. of the item begin at t0
  struct Cursor {
    int b, h, i, t, items, steps, nh, t0, end;
  };
  int64_t total = 0;
  Seq mine{};  // ITEM: the sequence
  Cursor cur{};
  int split = 0, item = 0;  // ITEM: which of the item's runs, and the item's number
  if constexpr (ITEM) {
    int j;
    const unsigned id = blockIdx.x / unsigned(a.splits);
    split = int(blockIdx.x - id * unsigned(a.splits));
    if (a.cu || a.by_group) {
      if (threadIdx.x == 0) item_pref[0] = 0;
      int carry = 0;
      for (int c0 = 0; c0 < a.count; c0 += NTH) {
        const int b = c0 + threadIdx.x;
        int incl = b < a.count ? items_of(seq_at(a, b).n, a.G) : 0;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
          const int y = __shfl_up(incl, o, 64);
          if (lane >= o) incl += y;
        }
        if (lane == 63) wsum[wave] = incl;
        __syncthreads();
        int base = carry;
        for (int w = 0; w < wave; ++w) base += int(wsum[w]);
        if (b < a.count) item_pref[b + 1] = base + incl;
#pragma unroll
        for (int w = 0; w < NW; ++w) carry += int(wsum[w]);
        __syncthreads();
      }
      if (!xcd_item(id, carry, a.Hkv, cur.h, j)) return;
      int lo = 0, hi = a.count - 1;  // the last sequence with item_pref[b] <= j
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (item_pref[mid] <= j) lo = mid; else hi = mid - 1;
      }
      cur.b = uniform(lo);
      cur.h = uniform(cur.h);
      cur.i = uniform(item_pref[cur.b + 1] - 1 - j);  // the last rows first
      item = uniform(j * a.Hkv + cur.h);
    } else {
      const unsigned ips = unsigned(a.G + 15) >> 4, k = id / ips;
      cur.i = int(id - k * ips);
      cur.b = int(k / unsigned(a.Hkv));
      cur.h = int(k - unsigned(cur.b) * unsigned(a.Hkv));
      if (cur.b >= a.count) return;
      item = int(id);
    }
    mine = seq_at(a, cur.b);
  }
  if constexpr (!ITEM) {
  // steps of the sequences before each
  if (threadIdx.x == 0) pref[0] = 0;
  int64_t carry = 0;
  for (int c0 = 0; c0 < a.count; c0 += NTH) {
    const int b = c0 + threadIdx.x;
    int64_t incl = 0;
    if (b < a.count) {
      const Seq s = seq_at(a, b);
      seqs[b] = make_int4(int(s.row0), s.n, s.len, s.off);
      if (s.n > 0) incl = int64_t(items_of(s.n, a.G)) * a.Hkv * steps_of(a, s, STEP);
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int64_t y = __shfl_up(incl, o, 64);
      if (lane >= o) incl += y;
    }
    if (lane == 63) wsum[wave] = incl;
    __syncthreads();
    int64_t base = carry;
    for (int w = 0; w < wave; ++w) base += wsum[w];
    if (b < a.count) pref[b + 1] = base + incl;
#pragma unroll
    for (int w = 0; w < WG_WAVES; ++w) carry += wsum[w];
    __syncthreads();
  }
  if (blockIdx.x == 0 && (a.src || !a.whole))  // for the kernel that joins the pieces
    for (int b = threadIdx.x; b <= a.count; b += NTH) a.pref[b] = pref[b];
  total = carry;
  }
  // what a lane has of row `row` and q head `head`, elements 16 nb + 4 kd + j
  auto finish = [&](f32x4_t (&o)[NB], float m, float l, int64_t row, int head) {
    const int64_t at = row * a.Hq + head;
    if (a.dst) {
      float* p = a.dst + at * D + 4 * kd;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
        if (FULL || 16 * nb < D)
          *reinterpret_cast<float4*>(p + 16 * nb) =
              make_float4(o[nb][0], o[nb][1], o[nb][2], o[nb][3]);
      if (kd == 0) a.dst_ml[at] = make_float2(m, l);
      return;
    }
    T* out = static_cast<T*>(a.out) + at * D + 4 * kd;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
      if (FULL || 16 * nb < D) {
        const float x[4] = {o[nb][0], o[nb][1], o[nb][2], o[nb][3]};
        store4<DT>(out + 16 * nb, x, l);
      }
  };
  f32x4_t acc[NB];
  if (!ITEM && a.whole && !a.src) {  // nothing will be joined: rows of sequences without steps, 16 at a time
    for (int b = blockIdx.x; b < a.count; b += gridDim.x) {
      if (pref[b + 1] != pref[b]) continue;
      const int4 s = seqs[b];
      const int64_t n = int64_t(s.y) * a.Hq;
      for (int64_t r = wave * 16 + n16; r < n; r += 16 * WG_WAVES) {
        const int64_t pos = r / a.Hq;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) acc[nb] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        finish(acc, -INFINITY, 0.f, s.x + pos, int(r - pos * a.Hq));
      }
    }
  }
  const int64_t nw = ITEM ? 1 : min(int64_t(gridDim.x) * WG_WAVES, total);
  const int64_t w = int64_t(wave) * gridDim.x + blockIdx.x;  // few steps: over all compute units
  if (!ITEM && w >= nw) return;
  auto seq_with = [&](int64_t x) {  // the last sequence that starts at or before x (and is not empty)
    int lo = 0, hi = a.count - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (pref[mid] <= x) lo = mid; else hi = mid - 1;
    }
    return lo;
  };
  auto get = [&](int b) {
    if constexpr (ITEM) return mine;
    const int4 x = seqs[b];
    Seq s;
    s.row0 = uniform(x.x);
    s.n = uniform(x.y);
    s.len = uniform(x.z);
    s.off = uniform(x.w);
    s.causal = !a.by_group && (a.offs || a.window);
    return s;
  };
  int64_t x0 = 0, x1 = 0;
  if constexpr (!ITEM) {
  x0 = first_of(w, nw, total);
  x1 = first_of(w + 1, nw, total);
  }
  if (!ITEM && a.whole) {  // the items that begin in the range
    auto item_from = [&](int64_t x) {
      if (x >= total) return total;
      const int b = seq_with(x), steps = steps_of(a, get(b), STEP);
      const int t = int(uint32_t(x - pref[b]) % uint32_t(steps));
      return t ? x + steps - t : x;
    };
    x0 = item_from(x0);
    x1 = item_from(x1);
    if (x0 >= x1) return;
  }
  int count = uniform(int(min(x1 - x0, int64_t(0x7fffffff))));

  auto open = [&](Cursor& c) {
    const Seq s = get(c.b);
    c.t0 = a.window ? max(c.nh, reach::lowest(a, s, 16 * c.i / a.G) / STEP) : 0;
    c.end = reach::limit(s, min((16 * c.i + 15) / a.G, s.n - 1));
  };
  auto enter = [&](Cursor& c) {
    const Seq s = get(c.b);
    c.items = items_of(s.n, a.G);
    c.steps = steps_of(a, s, STEP);
    c.nh = head_tiles(a, s, STEP);
  };
  auto advance = [&](Cursor& c) {
    if (++c.t < c.steps || ITEM) return;
    c.t = 0;
    if (++c.i == c.items) {
      c.i = 0;
      if (++c.h == a.Hkv) {
        c.h = 0;
        do ++c.b;
        while (c.b < a.count && uniform(int(pref[c.b + 1] == pref[c.b])));
        if (c.b >= a.count) return;
        enter(c);
      }
    }
    open(c);
  };
  auto tile_of = [&](const Cursor& c) { return reach::tile_of(c.nh, c.t0, c.t, STEP); };
  int pieces = 0;  // ITEM: waves that have steps
  if constexpr (ITEM) {
    cur.nh = head_tiles(a, mine, STEP);
    open(cur);
    const int tiles = (cur.end + STEP - 1) / STEP;
    const int all = min(cur.nh, tiles) + max(0, tiles - max(cur.t0, cur.nh));
    const int from = int(int64_t(all) * split / a.splits),
              steps = int(int64_t(all) * (split + 1) / a.splits) - from;
    pieces = min(steps, NW);
    const int q = steps / NW, r = steps - q * NW;
    cur.t = from + wave * q + min(wave, r);
    count = q + (wave < r ? 1 : 0);
    cur.steps = cur.t + count;
  } else {
    cur.b = uniform(seq_with(x0));
    enter(cur);
    const int64_t at = x0 - pref[cur.b], seg = quotient(at, cur.steps);
    cur.t = uniform(int(at - seg * cur.steps));
    cur.h = uniform(int(quotient(seg, cur.items)));
    cur.i = uniform(int(seg - int64_t(cur.h) * cur.items));
    open(cur);
  }

  // Pages: lane m < MB has that of block m of a step (-1 where no row sees any of it) and the block's place
  // in it. The ids are as loaded: what is made of them is made where they are used, a step later.
  const int PB = a.P / 16;
  const uint32_t np = uint32_t(a.num_pages);
  const int32_t* table = a.by_group ? a.pt : a.bt;
  const int64_t stride = a.by_group ? a.pt_stride : a.bt_stride;
  struct Where {
    int id, sub, h;
  };
  auto where = [&](const Cursor& c, bool real) {
    const int kb = tile_of(c) * MB + lane, slot = PB == 1 ? kb : kb / PB;
    Where r{-1, kb - slot * PB, c.h};
    if (real && lane < MB && reach::block_seen(a, reach::lowest(a, get(c.b), 16 * c.i / a.G), c.end, kb))
      r.id = table[int64_t(a.first + c.b) * stride + slot];
    return r;
  };
  // The element that a lane's block begins at, in the pool. Lanes of a block that is not there read another
  // of the step (the last; page 0 where there is none): what they get is not used.
  const int64_t tile_elems = int64_t(D) * a.P;
  auto blocks_there = [&](const Where& r) {
    return int(__ballot(lane < MB && uint32_t(r.id) < np)) & ((1 << MB) - 1);
  };
  auto base_of = [&](const Where& r, int there, int block) {
    const int other = there ? 31 - __builtin_clz(there) : 0;
    const int from = (there >> block) & 1 ? block : other;
    const int id = there ? __shfl(r.id, from, 64) : 0, sub = there ? __shfl(r.sub, from, 64) : 0;
    return (int64_t(id) * a.Hkv + r.h) * tile_elems + sub * 16;
  };
  // unit of a lane's K: see Form; its block and tokens in it
  const int unit = F::UB == 8 ? 8 * ((n16 >> 1) & 1) + 2 * (n16 >> 2) + (n16 & 1) : n16;
  const int k_block = unit * TU / 16, k_tok = unit * TU % 16;
  const int64_t row4 = 4 * int64_t(a.P), row16 = 16 * int64_t(a.P);
  Unit<F::UB> kr[NI];
  uint4 vr[NU][NB];
  if constexpr (!FULL) {
#pragma unroll
    for (int i = 0; i < NI; ++i) kr[i] = Unit<F::UB>{};
#pragma unroll
    for (int u = 0; u < NU; ++u)
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) vr[u][nb] = make_uint4(0u, 0u, 0u, 0u);
  }
  auto load_k = [&](const Where& r) {
    const int there = blocks_there(r);
    const T* p = static_cast<const T*>(a.kp) + base_of(r, there, k_block) + k_tok + kd * a.P;
#pragma unroll
    for (int i = 0; i < NI; ++i)
      if (FULL || 4 * i < D) kr[i] = load_unit<F::UB, ALIKE>(p + i * row4);
  };
  auto load_v = [&](const Where& r) {
    const int there = blocks_there(r);
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      const int block = F32 ? u : 2 * u + (kd >> 1), tok = F32 ? 4 * kd : 8 * (kd & 1);
      const T* p = static_cast<const T*>(a.vp) + base_of(r, there, block) + tok + n16 * a.P;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
        if (FULL || 16 * nb < D) vr[u][nb] = tile32::load16<ALIKE>(p + nb * row16);
    }
  };

  // q of an item: vectors of 16 bytes by lanes, element (r, d) to [(d % 4) 16 + r][d / 4]
  T* q_lds = &qs[ITEM ? 0 : wave][0];
  auto stage_q = [&](const Seq& s, int rows_left) {
    constexpr int VE = 16 / F::E, PER = DP / VE, N = ITEM ? NTH : 64;
    const int me = ITEM ? int(threadIdx.x) : lane;
#pragma unroll
    for (int y = 0; y < (16 * PER + N - 1) / N; ++y) {
      const int v = y * N + me, rr = v / PER, d = v % PER * VE;
      if (16 * PER % N != 0 && v >= 16 * PER) break;
      const int fr = 16 * cur.i + rr, fp = fr / a.G;
      const bool ok = rr < rows_left && (FULL || d < D);
      const T* p = static_cast<const T*>(a.q) + (s.row0 + (ok ? fp : 0)) * a.q_stride +
                   int64_t(cur.h * a.G + (ok ? fr - fp * a.G : 0)) * D + (ok ? d : 0);
      uint4 z = *reinterpret_cast<const uint4*>(p);
      z.x = ok ? z.x : 0u;
      z.y = ok ? z.y : 0u;
      z.z = ok ? z.z : 0u;
      z.w = ok ? z.w : 0u;
      if constexpr (F32) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          q_lds[(e * 16 + rr) * F::QS + d / 4] = __uint_as_float(tile32::word(z, e));
      } else {
        // d, d + 4 are neighbours of one lane
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t lo16 = tile32::word(z, e >> 1), hi16 = tile32::word(z, 2 + (e >> 1));
          *reinterpret_cast<uint32_t*>(&q_lds[(e * 16 + rr) * F::QS + d / 4]) =
              __builtin_amdgcn_perm(hi16, lo16, (e & 1) ? 0x07060302u : 0x05040100u);
        }
      }
    }
  };

  Cursor nxt = cur;
  if (count > 1) advance(nxt);
  Cursor far = nxt;
  Where w_cur = where(cur, count > 0), w_nxt = where(nxt, count > 1);
  load_k(w_cur);
  load_v(w_cur);

  // the item's rows: lane l's are of row l % 16, which sees tokens below `hs` of the sinks' tiles and
  // lo .. lim - 1; what all rows see, and any
  int lim = 0, lo = 0, hs = 0, lim_all = 0, lo_all = 0, hs_all = 0, lim_any = 0, lo_any = 0, hs_any = 0;
  int64_t row = 0;
  int head = 0;
  bool live = false;
  float m = -INFINITY, l = 0.f;
  bool opened = false;
  int begun = 0;  // step of the range at which the item began
  if constexpr (ITEM) {
    stage_q(mine, mine.n * a.G - 16 * cur.i);
    __syncthreads();
  }
  for (int x = 0; x < count; ++x) {
    if (x + 2 < count) advance(far);
    const Where w_far = where(far, x + 2 < count);
    if (!opened) {
      opened = true;
      begun = x;
      const Seq s = get(cur.b);
      const int rows_left = s.n * a.G - 16 * cur.i;
      const int r = 16 * cur.i + n16, pos = r / a.G;
      live = n16 < rows_left;
      row = s.row0 + (live ? pos : 0);
      head = cur.h * a.G + (live ? r - pos * a.G : 0);
      const int p0 = 16 * cur.i / a.G, p1 = min((16 * cur.i + 15) / a.G, s.n - 1);
      lim_all = reach::limit(s, p0);
      lim_any = reach::limit(s, p1);
      lo_any = reach::lowest(a, s, p0);
      lo_all = reach::lowest(a, s, p1);
      hs_all = a.window ? min(a.sinks, lim_all) : 0;
      hs_any = a.window ? min(a.sinks, lim_any) : 0;
      lim = ALIKE ? lim_all : reach::limit(s, min(pos, s.n - 1));
      lo = ALIKE ? lo_all : reach::lowest(a, s, min(pos, s.n - 1));
      hs = a.window ? min(a.sinks, lim) : 0;
      if constexpr (!ITEM) {
        __builtin_amdgcn_wave_barrier();
        stage_q(s, rows_left);
        __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
        __builtin_amdgcn_wave_barrier();
      }
      m = -INFINITY;
      l = 0.f;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) acc[nb] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }

    // scores
    f32x4_t s[TU];
    {
      const uint4* qv = reinterpret_cast<const uint4*>(q_lds + lane * F::QS);
      constexpr int CH = F32 ? 4 / TU : 1;  // chains of products of a sum
      f32x4_t t[CH][TU];
#pragma unroll
      for (int k = 0; k < CH; ++k)
#pragma unroll
        for (int c = 0; c < TU; ++c) t[k][c] = f32x4_t{0.f, 0.f, 0.f, 0.f};
      if constexpr (F32) {
#pragma unroll
        for (int i4 = 0; i4 < NI / 4; ++i4) {
          const uint4 y = qv[i4];
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int c = 0; c < TU; ++c)
              t[j % CH][c] = tile32::mfma_f32(__uint_as_float(kr[4 * i4 + j].w[c]),
                                              tile32::comp(y, j), t[j % CH][c]);
        }
      } else {
#pragma unroll
        for (int I = 0; I < NI / 8; ++I) {
          const uint4 y = qv[I];
#pragma unroll
          for (int c = 0; c < TU; ++c) {
            uint32_t k4[4];
#pragma unroll
            for (int f = 0; f < 4; ++f)
              k4[f] = __builtin_amdgcn_perm(kr[8 * I + 2 * f + 1].w[c >> 1], kr[8 * I + 2 * f].w[c >> 1],
                                            (c & 1) ? 0x07060302u : 0x05040100u);
            t[0][c] = tile::mfma16<DT>(make_uint4(k4[0], k4[1], k4[2], k4[3]), y, t[0][c]);
          }
        }
      }
#pragma unroll
      for (int c = 0; c < TU; ++c) {
        s[c] = t[0][c];
#pragma unroll
        for (int k = 1; k < CH; ++k) s[c] += t[k][c];
        s[c] *= a.scale_log2;
      }
    }
    load_k(w_nxt);

    // A lane's scores are of the tokens of its V vectors: those of vector u are tokens at(u) .. + NV - 1 of the
    // step, and token c of unit(4 kd + v) is number place(v, c) of vector v * TU / NV
    constexpr int NV = 16 / F::E;
    auto at = [&](int u) { return (F32 ? 16 : 32) * u + NV * kd; };
    auto place = [](int v, int c) { return (v * TU + c) % NV; };
    const int there = blocks_there(w_cur);
    const int base = tile_of(cur) * STEP;
    const bool in_head = cur.t < cur.nh;
    const bool full = there == (1 << MB) - 1 &&
                      ((base >= lo_all && base + STEP <= lim_all) ||
                       (in_head && base + STEP <= hs_all));
    // NV tokens from token t of the step on, as bits: those of [from, to) and those below `below`
    auto bits = [&](int t, int from, int to, int below) {
      auto first = [](int n) { return (1u << min(max(n, 0), NV)) - 1u; };
      t += base;
      const uint32_t x = (first(to - t) & ~first(from - t)) | (in_head ? first(below - t) : 0u);
      return (there >> ((t - base) >> 4)) & 1 ? x : 0u;
    };
    if (!full) {
#pragma unroll
      for (int u = 0; u < NU; ++u) {
        const uint32_t see = bits(at(u), lo, lim, hs);
#pragma unroll
        for (int v = u * NV / TU; v < (u + 1) * NV / TU; ++v)
#pragma unroll
          for (int c = 0; c < TU; ++c)
            s[c][v] = (see >> place(v, c)) & 1u ? s[c][v] : -INFINITY;
      }
    }
    // softmax, base 2
    float mx = -INFINITY;
#pragma unroll
    for (int c = 0; c < TU; ++c)
#pragma unroll
      for (int v = 0; v < 4; ++v) mx = __builtin_elementwise_maximum(mx, s[c][v]);
    mx = tile::maximum_col4(mx);
    const float mref = mx - m > RESCALE<DT> || mx != mx ? mx : m;
    if (__ballot(m != mref)) {
      const float alpha = reach::weight(m, mref);
      l *= alpha;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) acc[nb] *= alpha;
    }
    m = mref;
    const float nm = mref == -INFINITY ? 0.f : SHIFT<DT> - mref;
#pragma unroll
    for (int c = 0; c < TU; ++c)
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        s[c][v] = __builtin_amdgcn_exp2f(s[c][v] + nm);
        l += s[c][v];
      }
    bool by_row = false;
    if (!full) {
      // V of tokens that no row sees: zeros
      uint32_t odd = 0;
#pragma unroll
      for (int u = 0; u < NU; ++u) {
        const uint32_t any = bits(at(u), lo_any, lim_any, hs_any);
        const uint32_t some = ALIKE ? 0u : any & ~bits(at(u), lo_all, lim_all, hs_all);
        auto words = [](uint32_t x, int w) {
          return F32 ? ((x >> w) & 1u ? 0xffffffffu : 0u)
                     : ((x >> (2 * w)) & 1u ? 0xffffu : 0u) | ((x >> (2 * w)) & 2u ? 0xffff0000u : 0u);
        };
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const uint32_t keep = words(any, w), part = words(some, w);
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) {
            uint32_t& y = w == 0 ? vr[u][nb].x : w == 1 ? vr[u][nb].y : w == 2 ? vr[u][nb].z : vr[u][nb].w;
            y &= keep;
            if constexpr (!ALIKE) {  // an exponent of all ones among what some rows do not see
              const uint32_t z = y & part;
              if constexpr (F32) {
                odd |= (z & 0x7f800000u) == 0x7f800000u ? 1u : 0u;
              } else {
                constexpr uint32_t X = DT == PIA_DTYPE_F16 ? 0x7c00u : 0x7f80u;
                odd |= ((z & X) == X ? 1u : 0u) | ((z & (X << 16)) == X << 16 ? 1u : 0u);
              }
            }
          }
        }
      }
      if constexpr (!ALIKE) by_row = __ballot(odd) != 0;
    }
    if (ALIKE || !by_row) {
      if constexpr (F32) {
#pragma unroll
        for (int n0 = 0; n0 < NB; n0 += 2) {
          f32x4_t t[2] = {f32x4_t{0.f, 0.f, 0.f, 0.f}, f32x4_t{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
          for (int u = 0; u < NU; ++u)
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
              for (int n = 0; n < 2; ++n)
                t[n] = tile32::mfma_f32(tile32::comp(vr[u][n0 + n], j),
                                        F::UB == 8 ? s[j & 1][2 * u + (j >> 1)] : s[0][j], t[n]);
#pragma unroll
          for (int n = 0; n < 2; ++n) acc[n0 + n] += t[n];
        }
      } else {
        // fp16: whether there are positive ones that need more than two terms, and whether V is finite
        bool rest = false, finite = true;
        if constexpr (DT == PIA_DTYPE_F16) {
          uint32_t least = ~0u;  // of the positive ones, less one
#pragma unroll
          for (int c = 0; c < TU; ++c)
#pragma unroll
            for (int v = 0; v < 4; ++v) least = min(least, __float_as_uint(s[c][v]) - 1u);
          rest = __ballot(least < __float_as_uint(REST_BELOW) - 1u) != 0;
          if (__builtin_expect(rest, 0)) {
            float z[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int u = 0; u < NU; ++u)
#pragma unroll
              for (int nb = 0; nb < NB; ++nb) z[nb & 3] = squares(vr[u][nb], z[nb & 3]);
            finite = __ballot(!((z[0] + z[1]) + (z[2] + z[3]) < INFINITY)) == 0;
          }
        }
        const uint32_t fill = rest && finite ? 0u : ~0u;
        auto probabilities = [&](int u, float (&p)[8]) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            p[e] = F::UB == 8 ? s[e & 3][2 * u + (e >> 2)] : s[e & 1][e >> 1];
        };
#pragma unroll
        for (int u = 0; u < NU; ++u) {
          float p[8];
          probabilities(u, p);
          uint4 t[2];
          split2<DT>(p, t, fill);
#pragma unroll
          for (int k = 1; k >= 0; --k)
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) acc[nb] = tile::mfma16<DT>(vr[u][nb], t[k], acc[nb]);
        }
        if (__builtin_expect(rest, 0)) {
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) acc[nb] *= REST;
          if (!finite) {  // infinities have entered already
#pragma unroll
            for (int u = 0; u < NU; ++u)
#pragma unroll
              for (int nb = 0; nb < NB; ++nb) vr[u][nb] = finite_of(vr[u][nb]);
          }
#pragma unroll 1
          for (int put = 0; put < (finite ? 1 : 2); ++put)
#pragma unroll
            for (int u = 0; u < NU; ++u) {
              float p[8];
              probabilities(u, p);
              const uint4 z = rest2(p, put != 0);
#pragma unroll
              for (int nb = 0; nb < NB; ++nb) acc[nb] = tile::mfma16<DT>(vr[u][nb], z, acc[nb]);
            }
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) acc[nb] *= 1.f / REST;
        }
      }
    } else if constexpr (!ALIKE) {
      // row by row: each row's probabilities from LDS, V from memory, tokens that the row sees only
      float* pw = &ps[wave][0];
#pragma unroll
      for (int c = 0; c < TU; ++c)
#pragma unroll
        for (int v = 0; v < 4; ++v)
          pw[n16 * (STEP + 1) + at(v * TU / NV) + place(v, c)] = s[c][v];
      __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
      __builtin_amdgcn_wave_barrier();
#pragma unroll 1
      for (int o = 0; o < STEP; ++o) {
        const int tok = base + o, block = o >> 4;
        if (!((there >> block) & 1)) continue;
        const int id = __builtin_amdgcn_readlane(w_cur.id, block),
                  sub = __builtin_amdgcn_readlane(w_cur.sub, block);
        const bool sees = (tok >= lo && tok < lim) || (in_head && tok < hs);
        int k4 = 4 * kd, P = a.P;  // hidden, or the rows' offsets are kept for all tokens and spilled
        asm volatile("" : "+v"(k4), "+s"(P));
        const T* p = static_cast<const T*>(a.vp) +
                     (int64_t(id) * a.Hkv + w_cur.h) * tile_elems + sub * 16 + (o & 15) + int64_t(k4) * P;
        const float pr = pw[n16 * (STEP + 1) + o];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          if (!FULL && 16 * nb >= D) continue;
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float y = Elem<DT>::load(p, int64_t(16 * nb + j) * P);
            acc[nb][j] = sees ? fmaf(pr, y, acc[nb][j]) : acc[nb][j];
          }
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
    load_v(w_nxt);

    // end of the item or of the range
    if (cur.t + 1 == cur.steps || x + 1 == count) {
      const float lsum = tile32::sum_col4(l), mr = m == -INFINITY ? m : m - SHIFT<DT>;
      if constexpr (ITEM) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
          *reinterpret_cast<float4*>(red + (wave * 16 + n16) * RS + 16 * nb + 4 * kd) =
              make_float4(acc[nb][0], acc[nb][1], acc[nb][2], acc[nb][3]);
        if (kd == 0) {
          red_m[wave * 16 + n16] = mr;
          red_l[wave * 16 + n16] = lsum;
        }
      } else if (cur.t + 1 == cur.steps && cur.t == x - begun) {
        if (live) finish(acc, mr, lsum, row, head);
      } else {
        float* part = a.parts + (w * 2 + (begun == 0 ? 0 : 1)) * part_floats<DP>;
        if (live) {
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
            *reinterpret_cast<float4*>(part + n16 * DP + 16 * nb + 4 * kd) =
                make_float4(acc[nb][0], acc[nb][1], acc[nb][2], acc[nb][3]);
          if (kd == 0) {
            part[16 * DP + n16] = mr;
            part[16 * DP + 16 + n16] = lsum;
          }
        }
      }
      opened = false;
    }
    cur = nxt;
    nxt = far;
    w_cur = w_nxt;
    w_nxt = w_far;
  }
  if constexpr (ITEM) {  // the waves' pieces joined in order, the splits', then the prefix's
    __syncthreads();
    const int rows = min(16, mine.n * a.G - 16 * cur.i), per_row = D / 4;
    const bool prefix = a.src && reach::has_prefix(a, a.first + cur.b);
    const int64_t R = a.rows * a.Hq;
    const auto far = far_memory(a.parts + int64_t(item) * a.splits * part_floats<DP>,
                                a.splits * part_floats<DP>);
    struct Sum {
      float m, l;
      float4 o;
      __device__ __forceinline__ void add(float m1, float l1, const float4& x) {
        const float to = __builtin_elementwise_maximum(m, m1);
        const float f0 = reach::weight(m, to), f = reach::weight(m1, to);
        l = l * f0 + l1 * f;
        o = make_float4(fmaf(x.x, f, o.x * f0), fmaf(x.y, f, o.y * f0), fmaf(x.z, f, o.z * f0),
                        fmaf(x.w, f, o.w * f0));
        m = to;
      }
    };
    auto of_waves = [&](int r, int d) {
      Sum x{-INFINITY, 0.f, make_float4(0.f, 0.f, 0.f, 0.f)};
      for (int p = 0; p < pieces; ++p)
        x.add(red_m[p * 16 + r], red_l[p * 16 + r],
              *reinterpret_cast<const float4*>(red + (p * 16 + r) * RS + d));
      return x;
    };
    if (a.splits > 1) {
      // The piece to memory, then the arrival: see arrive(). The last workgroup reads them.
      for (int u = threadIdx.x; u < rows * per_row; u += NTH) {
        const int r = u / per_row, d = 4 * (u - r * per_row);
        const Sum x = of_waves(r, d);
        const int p = split * int(part_floats<DP>);
        put_far(far, 4 * (p + r * DP + d), x.o);
        if (d == 0) put_far(far, 4 * (p + 16 * DP + 2 * r), make_float2(x.m, x.l));
      }
      __builtin_amdgcn_s_waitcnt(0);  // this wave's stores have completed
      __syncthreads();                // and all waves'
      if (threadIdx.x == 0) is_last = arrive(a.counters + item, a.token, a.splits) ? 1 : 0;
      __syncthreads();
      if (!is_last) return;
    }
    for (int u = threadIdx.x; u < rows * per_row; u += NTH) {
      const int r = u / per_row, d = 4 * (u - r * per_row);
      const int rr = 16 * cur.i + r, pos = rr / a.G;
      const int64_t at = (mine.row0 + pos) * a.Hq + cur.h * a.G + rr - pos * a.G;
      constexpr int N = 8;  // pieces on their way at once
      Sum x{-INFINITY, 0.f, make_float4(0.f, 0.f, 0.f, 0.f)};
      if (a.splits > 1) {
        for (int p0 = 0; p0 < a.splits; p0 += 2 * N) {
          float2 pm[2 * N];
          float4 po[2 * N];
#pragma unroll
          for (int k = 0; k < 2 * N; ++k) {
            const int p = min(p0 + k, a.splits - 1) * int(part_floats<DP>);
            pm[k] = get_far2(far, 4 * (p + 16 * DP + 2 * r));
            po[k] = get_far4(far, 4 * (p + r * DP + d));
          }
#pragma unroll
          for (int k = 0; k < 2 * N; ++k)
            if (p0 + k < a.splits) x.add(pm[k].x, pm[k].y, po[k]);
        }
      } else {
        x = of_waves(r, d);
      }
      if (prefix) {
        for (int p0 = 0; p0 < a.src_cuts; p0 += N) {
          float2 pm[N];
          float4 po[N];
#pragma unroll
          for (int k = 0; k < N; ++k) {
            const int64_t c = min(p0 + k, a.src_cuts - 1) * R + at;
            pm[k] = a.src_ml[c];
            po[k] = *reinterpret_cast<const float4*>(a.src + c * D + d);
          }
#pragma unroll
          for (int k = 0; k < N; ++k)
            if (p0 + k < a.src_cuts) x.add(pm[k].x, pm[k].y, po[k]);
        }
      }
      if (a.dst && !a.src) {
        *reinterpret_cast<float4*>(a.dst + at * D + d) = x.o;
        if (d == 0) a.dst_ml[at] = make_float2(x.m, x.l);
      } else {
        const float y[4] = {x.o.x, x.o.y, x.o.z, x.o.w};
        store4<DT>(static_cast<T*>(a.out) + at * D + d, y, x.l);
      }
    }
  }
}

// The items that were cut: their pieces joined, in the order of the waves. Behind a prefix all items, which
// are pieces of rows where they were not cut (the one behind the prefix's), joined with the prefix's. A
// workgroup has rows_per_wg rows of an item, all of them or, where there are few items with many pieces,
// one. Items without keys are zeros.
template <int DT, int DP>
__global__ __launch_bounds__(JOIN_FEW) void reach_stream_join_kernel(Args a, int64_t waves,
                                                                     int rows_per_wg) {
  using T = typename Elem<DT>::T;
  constexpr int STEP = Form<DT, DP>::STEP;
  const int64_t id = blockIdx.x / unsigned(a.Hkv);
  const int h = int(blockIdx.x - unsigned(id) * unsigned(a.Hkv));
  int b, i;
  if (a.cu || a.by_group) {
    // items of sequence b are numbered from (its first row) G / 16 + b on
    auto base = [&](int k) {
      const int64_t r = reach::row_of(a, a.by_group ? reach::edge_of(a, a.first + k) : a.first + k);
      return (r * a.G >> 4) + k;
    };
    const int64_t from = base(0);
    const int lane = threadIdx.x & 63;
    int lo = 0, n = a.count;  // the last of n that begins at or before id, 64 of them at once
    while (n > 1) {
      const int step = (n + 63) >> 6, at = lane * step;
      const uint64_t in = __ballot(at < n && base(lo + at) - from <= id);
      const int last = in ? 63 - __builtin_clzll(in) : 0;
      lo += last * step;
      n = min(step, n - last * step);
    }
    b = lo;
    i = int(id + from - base(b));
  } else {
    const int items = (a.G + 15) >> 4;
    b = int(uint32_t(id) / uint32_t(items));
    i = int(id - int64_t(b) * items);
  }
  if (b >= a.count) return;
  const Seq s = seq_at(a, b);
  if (i < 0 || i >= items_of(s.n, a.G)) return;
  const int r0 = blockIdx.y * rows_per_wg;
  const int rows = min(min(16, s.n * a.G - 16 * i) - r0, rows_per_wg);
  if (rows <= 0) return;
  const int steps = steps_of(a, s, STEP);
  const int64_t total = a.pref[a.count], nw = min(waves, total), R = a.rows * a.Hq;
  const int64_t from = a.pref[b] + (int64_t(h) * items_of(s.n, a.G) + i) * steps, to = from + steps;
  int64_t w0 = 0, w1 = 0;
  bool cut = false;
  if (steps > 0 && !a.whole) {
    w0 = wave_of(from, nw, total);
    w1 = wave_of(to - 1, nw, total);
    cut = w0 != w1;
  }
  if (steps > 0 && !cut && !a.src) return;  // finished by its wave
  const float* first =
      a.parts + (w0 * 2 + (cut && first_of(w0, nw, total) >= from ? 0 : 1)) * part_floats<DP>;
  // pieces of rows: the prefix's, and the item's own where it was not cut
  const int own = steps > 0 && !cut ? 1 : 0;
  const int c0 = a.src && reach::has_prefix(a, a.first + b) ? 0 : a.src_cuts,
            c1 = a.src ? a.src_cuts + own : 0;
  // S lanes in a row have four elements u of the item (row r, elements d .. d + 3) and every S-th piece
  // each, eight of them on their way at once; they meet by exchanges, in a fixed order.
  const int per_row = a.D / 4, U = rows * per_row, np = int(w1 - w0) + 1;
  const int threads = blockDim.x;
  int S = 1;
  while (S < 64 && 2 * S * U <= threads && 16 * S < np && cut) S *= 2;
  const int sp = threadIdx.x & (S - 1);
  for (int u0 = 0; u0 < U; u0 += threads / S) {
    const int u = u0 + int(threadIdx.x) / S, rl = u / per_row, r = r0 + rl, d = 4 * (u - rl * per_row);
    if (u >= U) return;  // in whole groups of S lanes
    float M = -INFINITY, L = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](float m, float l, float4 x) {
      const float to = __builtin_elementwise_maximum(M, m);
      const float f0 = reach::weight(M, to), f = reach::weight(m, to);
      L = L * f0 + l * f;
      o = make_float4(fmaf(x.x, f, o.x * f0), fmaf(x.y, f, o.y * f0), fmaf(x.z, f, o.z * f0),
                      fmaf(x.w, f, o.w * f0));
      M = to;
    };
    if (cut) {
      constexpr int N = 8;
      for (int p0 = sp; p0 < np; p0 += N * S) {
        float pm[N], pl[N];
        float4 po[N];
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const int pi = min(p0 + j * S, np - 1);  // past the end: the last one again, without weight
          const float* p = pi == 0 ? first : a.parts + (w0 + pi) * 2 * part_floats<DP>;
          pm[j] = p[16 * DP + r];
          pl[j] = p[16 * DP + 16 + r];
          po[j] = *reinterpret_cast<const float4*>(p + r * DP + d);
        }
#pragma unroll
        for (int j = 0; j < N; ++j)
          if (p0 + j * S < np) add(pm[j], pl[j], po[j]);
      }
    }
    if (S > 1) {
      float m = M;
      for (int k = 1; k < S; k *= 2) m = __builtin_elementwise_maximum(m, __shfl_xor(m, k, 64));
      const float f = reach::weight(M, m);
      L *= f;
      o = make_float4(o.x * f, o.y * f, o.z * f, o.w * f);
      M = m;
      for (int k = 1; k < S; k *= 2) {
        L += __shfl_xor(L, k, 64);
        o.x += __shfl_xor(o.x, k, 64);
        o.y += __shfl_xor(o.y, k, 64);
        o.z += __shfl_xor(o.z, k, 64);
        o.w += __shfl_xor(o.w, k, 64);
      }
    }
    if (sp) continue;
    const int rr = 16 * i + r, pos = rr / a.G;
    const int64_t at = (s.row0 + pos) * a.Hq + h * a.G + rr - pos * a.G;
    if (c0 < c1) {
      constexpr int N = 8;  // on their way at once
      for (int p0 = c0; p0 < c1; p0 += N) {
        float2 pm[N];
        float4 po[N];
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const int64_t c = min(p0 + j, c1 - 1) * R + at;
          pm[j] = a.src_ml[c];
          po[j] = *reinterpret_cast<const float4*>(a.src + c * a.D + d);
        }
#pragma unroll
        for (int j = 0; j < N; ++j)
          if (p0 + j < c1) add(pm[j].x, pm[j].y, po[j]);
      }
    }
    if (a.dst && !a.src) {
      *reinterpret_cast<float4*>(a.dst + at * a.D + d) = o;
      if (d == 0) a.dst_ml[at] = make_float2(M, L);
      continue;
    }
    const float x[4] = {o.x, o.y, o.z, o.w};
    store4<DT>(static_cast<T*>(a.out) + at * a.D + d, x, L);
  }
}

inline int64_t resident_waves() { return int64_t(device_cus()) * WGS_PER_CU * WG_WAVES; }
constexpr int64_t PREF_BYTES = (MAX_SEQS + 1) * 8 + 248;  // whole 256 bytes

// Into how many runs of steps, a workgroup's each, every item is cut (0: all items' steps over the resident
// waves instead). items: at most so many; likely: about so many. A second step of a wave takes as long as the
// arrival and reading of another workgroup's piece (3 us), so up to two of each wave are not cut (one sequence,
// window of 128: 9.2 us, cut 11.3). Of more, each wave gets one where a workgroup for each compute unit is enough
// for that, else as many as that leaves it (4 sequences, window of 4096: 22 us, with two workgroups on each 32; 24
// fp32 sequences, 500: 24 and 28): further ones share a unit's bandwidth and leave more pieces. One more where
// that would leave a third of the units idle (16 sequences of 1 .. 6 rows: 19 us, without 22); two on each where a
// wave's run would be too long.
inline int item_splits(int64_t items, int64_t likely, int64_t steps, bool window) {
  const int64_t cus = device_cus(), slots = cus * WGS_PER_CU;
  if (items > slots) return 0;
  if (steps <= 2 * WG_WAVES) return 1;
  const int64_t one = cus / likely;
  for (const int64_t cut : {3 * one * likely < 2 * cus ? one + 1 : one, slots / items}) {
    const int64_t n =
        std::max<int64_t>(1, std::min({ceil_div(steps, WG_WAVES), cut, int64_t(MAX_SPLITS),
                                       2 * WG_WAVES * slots / items}));  // the workspace's pieces
    if (ceil_div(steps, n * WG_WAVES) <= (window ? ITEM_STEPS_WINDOW : ITEM_STEPS)) return int(n);
  }
  return 0;
}

template <int DT, int DP>
void launch_shape(const Args& a, int64_t items, bool alike, hipStream_t s) {
  const bool full = a.D == DP;
#define PIA_RS(A, F, I)                                                                           \
  hipLaunchKernelGGL(                                                                             \
      (reach_stream_kernel<DT, DP, A, F, I>),                                                     \
      dim3(unsigned(I ? ceil_div(items, 8) * 8 * a.splits : device_cus() * WGS_PER_CU)),          \
      dim3(64 * WG_WAVES), 0, s, a)
#define PIA_RS_I(I)                                              \
  if (alike) {                                                   \
    if (full) PIA_RS(true, true, I); else PIA_RS(true, false, I); \
  } else {                                                       \
    if (full) PIA_RS(false, true, I); else PIA_RS(false, false, I); \
  }
  if (a.splits) {
    PIA_RS_I(true)
  } else {
    PIA_RS_I(false)
  }
#undef PIA_RS_I
#undef PIA_RS
  if (a.splits || (a.whole && !a.src)) return;
  // few items: many pieces each, which many threads share, on every compute unit; many: two or three
  const bool few = items * 4 <= resident_waves();
  const int rows = a.cu || a.by_group ? 16 : std::min(a.G, 16);
  const int parts =
      few ? int(std::max<int64_t>(1, std::min<int64_t>(rows, device_cus() / items))) : 1;
  const int rows_per_wg = (rows + parts - 1) / parts;
  hipLaunchKernelGGL((reach_stream_join_kernel<DT, DP>),
                     dim3(unsigned(items), unsigned((rows + rows_per_wg - 1) / rows_per_wg)),
                     dim3(few ? JOIN_FEW : JOIN_MANY), 0, s, a, resident_waves(), rows_per_wg);
}

template <int DT>
int launch_dtype(Args a, int64_t tokens, hipStream_t s) {
  const int n = a.by_group ? a.groups : a.B;
  const int step = a.D > 128 ? Form<DT, 256>::STEP : Form<DT, 128>::STEP;
  // As many as the tables have room for (lengths are on the device): short contexts under wide tables are cut as
  // long ones (64 sequences of 300 tokens behind a prefix of 8192: 52 us, with tables of 4096 tokens 63, of
  // 32768 69). A window's tiles may begin and end within one.
  const int64_t steps = std::min(ceil_div(tokens, step) + (a.window ? 2 : 0),
                                 ceil_div((a.by_group ? a.pt_stride : a.bt_stride) * a.P, step));
  a.whole = steps <= WHOLE;
  const bool alike = a.by_group || !a.cu || (!a.offs && !a.window);
  // more sequences than a launch's tables hold: by parts, one after the other on the stream
  for (int b0 = 0; b0 < n; b0 += MAX_SEQS) {
    a.first = b0;
    a.count = std::min(n - b0, MAX_SEQS);
    const int64_t items = (a.cu || a.by_group ? (a.rows * a.G >> 4) + a.count + 1
                                              : int64_t(a.count) * ((a.G + 15) / 16)) * a.Hkv;
    if (items > 0x1fffffff) return fail(PIA_EINVAL, "attention: too many rows");
    // of the bound above, half an item of each sequence is not there
    const int64_t likely =
        std::max<int64_t>(1, items - (a.cu || a.by_group ? (a.count / 2 + 1) * int64_t(a.Hkv) : 0));
    a.splits = item_splits(items, likely, steps, a.window != 0);
    a.counters = reinterpret_cast<unsigned long long*>(a.pref);
    a.token = a.splits > 1 ? reach_token() : 0;
    if (a.D <= 64) launch_shape<DT, 64>(a, items, alike, s);
    else if (a.D <= 128) launch_shape<DT, 128>(a, items, alike, s);
    else launch_shape<DT, 256>(a, items, alike, s);
    const int rc = check_launch("reach_stream");
    if (rc) return rc;
  }
  return 0;
}

}  // namespace reach_stream
}  // namespace pia
