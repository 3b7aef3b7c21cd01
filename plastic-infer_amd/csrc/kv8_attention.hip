// Attention over the 8-bit paged KV pool: one query row per sequence (decode) or several with a
// causal limit for each, any q type, head_dim to 256.
//
// Bound by HBM for decode: a context token of a kv head is 2 D bytes and a few scales, against
// 4 G D operations. What the vector ALU does for a byte has to stay small, so both products run on
// the matrix cores, with operands that come from memory in place:
//
//   S^T = K . q^T  A is K: lane l holds token l % 16's elements of chunk l / 16 (kv8.h), widened to
//                  16 bits, where an e4m3 code is exact; B is q. Lane l then has the scores of row
//                  l % 16 for tokens 4 (l / 16) + j of each block.
//   O += P . V     those scores' exponentials are the A operand as they are; B is V, whose words
//                  hold an element's tokens 4 (l / 16) .. + 3. Two blocks make 32 tokens.
//
// Precision: the codes are exact in bf16 (and fp16), their scales are applied to scores and
// probabilities in fp32. q is exact: one bf16 or fp16 term, or three bf16 terms of an fp32 value.
// The probabilities times V's scale are the sum of two bf16 terms (2^-17 of each; three for fp32
// results: 2^-25), so a result is as good as its type. Scores, sums and outputs are fp32.
//
// Work: an item is 16 (position, head) rows of a sequence and kv head; its keys go by steps of
// 16 MB tokens. All steps of all items, in order, are cut into one contiguous range for every
// resident wave, whatever the batch looks like. The next step's K and V are on their way while a
// step is computed, across items too. An item that lies in one range is finished there; pieces of
// the others (at most two a wave) go to the workspace, and a second kernel joins them in order, so
// results do not depend on timing. Items of three steps at most (by the table's width) are not cut: a
// wave takes those that begin in its range, and there is no second kernel. In us, cut and whole: one
// sequence of 64 keys 10.4 and 8.4 (the call from Python 13.5 and 10.5), of 192 10.6 and 11.4 (13.5 and
// 11.3), of 256 10.6 and 13.1; 256 sequences of 192 24.3 and 22.4. A short context under a wide table is
// cut all the same: the host does not know the keys.
//
// Measured (both kernels): 256 sequences of 512 to 8192 keys, 32 heads of 128 over 8, bf16: 372-382 us,
// 6.0-6.2 TB/s, the first kernel alone at the 6.4 that reads reach. Two of 100000 and 131072 keys,
// head_dim 64: 53 us, 4.5 TB/s. One of 3001 keys: 13 us, two launches and what each has to look up
// before its first load. 16 sequences of 1 to 6 rows, 8 heads to a kv head, 700 to 4000 keys: 30 us;
// their pieces are as many bytes as the keys.
#include <algorithm>

#include "attn_tiles.h"
#include "attn_tiles_f32.h"
#include "kv8.h"

namespace pia {
namespace {

using tile::f32x4_t;

constexpr int KA_MAX_SEQS = 1024;  // sequences per launch (their tables in LDS)
constexpr int KA_WG_WAVES = 4;
constexpr int KA_WGS_PER_CU = 2;   // two waves per SIMD
constexpr int KA_RSRC_WORD3 = 0x00020000;
constexpr int KA_WHOLE = 3;  // steps of a table whose items are not cut
constexpr float KA_RESCALE = 8.0f;  // log2: how far a row's maximum may run ahead of its reference
constexpr int KA_JOIN_MANY = 128, KA_JOIN_FEW = 512;  // threads of the joining workgroups

struct AttnArgs {
  void* out;
  const void* q;
  int64_t q_stride;
  const uint8_t *kp, *vp;
  const float *ks, *vs;
  const int32_t* bt;
  int64_t bt_stride;
  const int32_t *lens, *cu, *offs;
  int64_t rows, num_pages;
  float* parts;
  int64_t* pref;
  float scale_log2;
  int B, Hq, Hkv, G, D, P, whole;  // whole: no item is cut
};

// A sequence's part of a call: its rows, the keys that some row of it may see (kv_len) and their steps.
struct Seq {
  int64_t row0;
  int n, kv_len, off, items, steps;
};
__device__ __forceinline__ Seq sequence(const AttnArgs& a, int b, int tokens) {
  Seq s;
  s.row0 = a.cu ? a.cu[b] : b;
  const int64_t n = a.cu ? int64_t(a.cu[b + 1]) - s.row0 : 1;
  s.n = s.row0 < 0 ? 0 : int(max(int64_t(0), min(n, a.rows - s.row0)));
  s.kv_len = int(min(int64_t(max(a.lens[b], 0)), min(a.bt_stride * a.P, int64_t(0x7ffffff0))));
  s.off = a.offs ? a.offs[b] : 0;
  if (a.offs) s.kv_len = kv8::seen(s.kv_len, s.off, s.n - 1);
  s.items = int((int64_t(s.n) * a.G + 15) >> 4);
  s.steps = (s.kv_len + tokens - 1) / tokens;
  return s;
}

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

template <int DP>
constexpr int64_t part_floats = 16 * (DP + 2);  // 16 rows' outputs, maxima and sums

template <int QT>
struct Q;  // terms of q and of the probabilities, and the 16-bit type of K and q
template <> struct Q<PIA_DTYPE_BF16> { static constexpr int NQ = 1, NP = 2, KT = PIA_DTYPE_BF16; };
template <> struct Q<PIA_DTYPE_F16> { static constexpr int NQ = 1, NP = 2, KT = PIA_DTYPE_F16; };
template <> struct Q<PIA_DTYPE_F32> { static constexpr int NQ = 3, NP = 3, KT = PIA_DTYPE_BF16; };

// eight consecutive q elements (which are there to be read) as NQ operands, zeros where not ok
template <int QT>
__device__ __forceinline__ void load_q(const typename Elem<QT>::T* p, bool ok,
                                       uint4 (&t)[Q<QT>::NQ]) {
  if constexpr (QT == PIA_DTYPE_F32) {
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[i] = p[i];
      x[i] = ok ? x[i] : 0.f;
    }
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        w[i] = tile::pack_bf16x2(x[2 * i], x[2 * i + 1]);
        x[2 * i] -= bf16_lo(w[i]);
        x[2 * i + 1] -= bf16_hi(w[i]);
      }
      t[k] = make_uint4(w[0], w[1], w[2], w[3]);
    }
  } else {
    t[0] = *reinterpret_cast<const uint4*>(p);
    t[0].x = ok ? t[0].x : 0u;
    t[0].y = ok ? t[0].y : 0u;
    t[0].z = ok ? t[0].z : 0u;
    t[0].w = ok ? t[0].w : 0u;
  }
}

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ float lane_value(float x, int lane) {
  return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), lane));
}
// ONCE: one position and one item per sequence and kv head, so K and V are read once by the call, and
// all rows of an item see the same keys.
template <int QT, int DP, bool ONCE>
__global__ __launch_bounds__(64 * KA_WG_WAVES, KA_WGS_PER_CU) void kv8_attention_kernel(AttnArgs a) {
  using T = typename Elem<QT>::T;
  constexpr int NQ = Q<QT>::NQ, NP = Q<QT>::NP, KT16 = Q<QT>::KT;
  constexpr int MB = DP > 128 ? 2 : 4;  // blocks of a step (registers)
  constexpr int STEP = 16 * MB, ND = DP / 64, AUX = ONCE ? 2 : 0;
  __shared__ int64_t pref[KA_MAX_SEQS + 1];
  __shared__ int4 seq_of[KA_MAX_SEQS];  // first row (below 2^31), rows, keys, offset
  __shared__ int64_t wsum[KA_WG_WAVES];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  constexpr int NTH = 64 * KA_WG_WAVES;

  // steps of the sequences before each
  if (threadIdx.x == 0) pref[0] = 0;
  int64_t carry = 0;
  for (int c0 = 0; c0 < a.B; c0 += NTH) {
    const int b = c0 + threadIdx.x;
    int64_t incl = 0;
    if (b < a.B) {
      const Seq s = sequence(a, b, STEP);
      seq_of[b] = make_int4(int(s.row0), s.n, s.kv_len, s.off);
      incl = int64_t(s.items) * a.Hkv * s.steps;
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
    if (b < a.B) pref[b + 1] = base + incl;
#pragma unroll
    for (int w = 0; w < KA_WG_WAVES; ++w) carry += wsum[w];
    __syncthreads();
  }
  if (blockIdx.x == 0)  // for the kernel that joins the pieces
    for (int b = threadIdx.x; b <= a.B; b += NTH) a.pref[b] = pref[b];
  const int64_t total = carry;
  if (a.whole) {  // nothing will be joined: rows of sequences without keys are zeros
    for (int b = blockIdx.x; b < a.B; b += gridDim.x) {
      const int4 s = seq_of[b];
      if (s.z > 0) continue;
      uint4* o = reinterpret_cast<uint4*>(static_cast<T*>(a.out) + int64_t(s.x) * a.Hq * a.D);
      const int64_t n = int64_t(s.y) * a.Hq * a.D * int(sizeof(T)) / 16;
      for (int64_t i = threadIdx.x; i < n; i += NTH) o[i] = make_uint4(0u, 0u, 0u, 0u);
    }
  }
  const int64_t nw = min(int64_t(gridDim.x) * KA_WG_WAVES, total);
  const int64_t w = int64_t(wave) * gridDim.x + blockIdx.x;  // few steps: over all compute units
  if (w >= nw) return;
  auto seq_at = [&](int64_t x) {  // the last sequence that starts at or before x (and is not empty)
    int lo = 0, hi = a.B - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (pref[mid] <= x) lo = mid; else hi = mid - 1;
    }
    return lo;
  };
  int64_t x0 = first_of(w, nw, total), x1 = first_of(w + 1, nw, total);
  if (a.whole) {  // the items that begin in the range
    auto item_from = [&](int64_t x) {
      if (x >= total) return total;
      const int b = seq_at(x), steps = (seq_of[b].z + STEP - 1) / STEP;
      const int t = int(uint32_t(x - pref[b]) % uint32_t(steps));
      return t ? x + steps - t : x;
    };
    x0 = item_from(x0);
    x1 = item_from(x1);
    if (x0 >= x1) return;
  }
  const int count = uniform(int(min(x1 - x0, int64_t(0x7fffffff))));

  // where a wave is: step t of item i of kv head h of sequence b
  struct Cursor {
    int b, h, i, t, items, steps, kv_len;
  };
  auto enter = [&](Cursor& c) {
    const int4 s = seq_of[c.b];
    c.kv_len = uniform(s.z);
    c.steps = (c.kv_len + STEP - 1) / STEP;
    c.items = uniform(int((int64_t(s.y) * a.G + 15) >> 4));
  };
  auto advance = [&](Cursor& c) {
    if (++c.t < c.steps) return;
    c.t = 0;
    if (++c.i < c.items) return;
    c.i = 0;
    if (++c.h < a.Hkv) return;
    c.h = 0;
    do ++c.b;
    while (c.b < a.B && uniform(int(pref[c.b + 1] == pref[c.b])));
    if (c.b < a.B) enter(c);
  };
  Cursor cur;
  {
    cur.b = uniform(seq_at(x0));
    enter(cur);
    const int64_t at = x0 - pref[cur.b], seg = quotient(at, cur.steps);
    cur.t = uniform(int(at - seg * cur.steps));
    cur.h = uniform(int(quotient(seg, cur.items)));
    cur.i = uniform(int(seg - int64_t(cur.h) * cur.items));
  }

  // Pages: lane m < MB has that of block m of a step (-1 where there is none) and the block's place in
  // it. The ids are as loaded: what is made of them is made where they are used, a step later, so that
  // no step waits for them (and with them for the K and V on their way).
  const int PB = a.P / 16, g = lane >> 4, n16 = lane & 15;
  const uint32_t np = a.num_pages > 0x7fffffff ? 0x7fffffffu : uint32_t(a.num_pages);
  struct Where {
    int id, sub, h;
  };
  auto where = [&](const Cursor& c, bool real) {
    const int kb = c.t * MB + lane, slot = PB == 1 ? kb : kb / PB;
    Where r{-1, kb - slot * PB, c.h};
    if (real && lane < MB && kb * 16 < c.kv_len) r.id = a.bt[int64_t(c.b) * a.bt_stride + slot];
    return r;
  };
  const int64_t tile_bytes = int64_t(a.D) * a.P;
  uint32_t k_off[ND], v_off[ND];
#pragma unroll
  for (int i = 0; i < ND; ++i) {
    k_off[i] = uint32_t(((g + 4 * i) * a.P + n16) * 16);
    v_off[i] = uint32_t(g * 4 * a.D + 256 * i + 16 * n16);
  }
  // Buffer descriptors: a block that is not there gets an empty one, whose loads return zeros
  // without reading, so loading has no branch; chunks of K past head_dim lie past its end.
  uint4 kr[MB][ND], vr[MB][ND];
  auto load_k = [&](const Where& r) {
#pragma unroll
    for (int m = 0; m < MB; ++m) {
      const int id = __builtin_amdgcn_readlane(r.id, m), sub = __builtin_amdgcn_readlane(r.sub, m);
      const bool ok = uint32_t(id) < np;
      const int64_t head = int64_t(id) * a.Hkv + r.h;
      const auto rs = __builtin_amdgcn_make_buffer_rsrc(
          const_cast<uint8_t*>(a.kp + (ok ? head : 0) * tile_bytes + sub * 256), 0,
          ok ? int(tile_bytes) - sub * 256 : 0, KA_RSRC_WORD3);
#pragma unroll
      for (int i = 0; i < ND; ++i)
        kr[m][i] = __builtin_bit_cast(uint4,
                                      __builtin_amdgcn_raw_buffer_load_b128(rs, k_off[i], 0, AUX));
    }
  };
  auto load_v = [&](const Where& r) {
#pragma unroll
    for (int m = 0; m < MB; ++m) {
      const int id = __builtin_amdgcn_readlane(r.id, m), sub = __builtin_amdgcn_readlane(r.sub, m);
      const bool ok = uint32_t(id) < np;
      const int64_t head = int64_t(id) * a.Hkv + r.h;
      const auto rs = __builtin_amdgcn_make_buffer_rsrc(
          const_cast<uint8_t*>(a.vp + (ok ? head : 0) * tile_bytes + int64_t(sub) * 16 * a.D), 0,
          ok ? 16 * a.D : 0, KA_RSRC_WORD3);
#pragma unroll
      for (int i = 0; i < ND; ++i)
        vr[m][i] = __builtin_bit_cast(uint4,
                                      __builtin_amdgcn_raw_buffer_load_b128(rs, v_off[i], 0, AUX));
    }
  };
  float sk = 1.f, sv = 1.f;  // lane m < MB: block m's scales
  auto load_scales = [&](const Where& r) {
    const int64_t at = uint32_t(r.id) < np ? (int64_t(r.id) * a.Hkv + r.h) * PB + r.sub : 0;
    sk = a.ks[at];
    sv = a.vs[at];
  };

  Cursor nxt = cur;
  if (count > 1) advance(nxt);
  Cursor far = nxt;
  Where w_cur = where(cur, true), w_nxt = where(nxt, count > 1);
  load_k(w_cur);
  load_scales(w_cur);
  load_v(w_cur);

  // the item's rows: lane l's q operands and limit are those of row l % 16
  uint4 qr[ND][2][NQ];
  int lim = 0, lim_min = 0, rows_left = 0;
  int64_t row0 = 0;
  float m = -INFINITY, l = 0.f;
  f32x4_t acc[4 * ND];
  bool opened = false;
  int begun = 0;  // step of the range at which the item began

  for (int x = 0; x < count; ++x) {
    if (x + 2 < count) advance(far);
    const Where w_far = where(far, x + 2 < count);
    if (!opened) {
      opened = true;
      begun = x;
      const int4 s = seq_of[cur.b];
      const int off = uniform(s.w);
      row0 = uniform(s.x);
      rows_left = uniform(s.y) * a.G - 16 * cur.i;
      const int r = 16 * cur.i + n16, pos = r / a.G;
      const bool ok = n16 < rows_left;
      const T* qp = static_cast<const T*>(a.q) + (row0 + (ok ? pos : 0)) * a.q_stride +
                    int64_t(cur.h * a.G + (ok ? r - pos * a.G : 0)) * a.D;
#pragma unroll
      for (int i = 0; i < ND; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int d = 16 * (g + 4 * i) + 8 * e;
          load_q<QT>(qp + (d < a.D ? d : 0), ok && d < a.D, qr[i][e]);
        }
      // q is waited for here, once an item: left to its use, the wait would be there in every step, and
      // with it one for the step's K and V
#pragma unroll
      for (int i = 0; i < ND; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int n = 0; n < NQ; ++n)
            asm volatile("" : "+v"(qr[i][e][n].x), "+v"(qr[i][e][n].y), "+v"(qr[i][e][n].z),
                              "+v"(qr[i][e][n].w));
      lim = lim_min = cur.kv_len;
      if (!ONCE && a.offs) {
        lim = kv8::seen(lim, off, pos);
        lim_min = kv8::seen(lim_min, off, (16 * cur.i) / a.G);
      }
      m = -INFINITY;
      l = 0.f;
#pragma unroll
      for (int nb = 0; nb < 4 * ND; ++nb) acc[nb] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }

    // scores
    f32x4_t s[MB];
#pragma unroll
    for (int b = 0; b < MB; ++b) {
      s[b] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < ND; ++i) {
        const uint4 k = kr[b][i];
        const uint4 lo = kv8::widen8<KT16>(k.x, k.y), hi = kv8::widen8<KT16>(k.z, k.w);
#pragma unroll
        for (int n = NQ - 1; n >= 0; --n) {
          s[b] = tile::mfma16<KT16>(lo, qr[i][0][n], s[b]);
          s[b] = tile::mfma16<KT16>(hi, qr[i][1][n], s[b]);
        }
      }
    }
    load_k(w_nxt);

    // softmax, base 2
    const int there = int(__ballot(lane < MB && uint32_t(w_cur.id) < np)) & ((1 << MB) - 1);
    const int base = cur.t * STEP;
    const bool full = there == (1 << MB) - 1 && base + STEP <= lim_min;
    float mx = -INFINITY;
#pragma unroll
    for (int b = 0; b < MB; ++b) {
      const float f = a.scale_log2 * lane_value(sk, b);
#pragma unroll
      for (int j = 0; j < 4; ++j) s[b][j] *= f;
    }
    if (!full) {
      const int rel = lim - (base + 4 * g);
#pragma unroll
      for (int b = 0; b < MB; ++b)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (!(16 * b + j < rel && ((there >> b) & 1))) s[b][j] = -INFINITY;
    }
#pragma unroll
    for (int b = 0; b < MB; ++b)
#pragma unroll
      for (int j = 0; j < 4; ++j) mx = __builtin_elementwise_maximum(mx, s[b][j]);
    mx = tile::maximum_col4(mx);
    const float mref = mx - m > KA_RESCALE || mx != mx ? mx : m;
    const float alpha = m == mref ? 1.f : __builtin_amdgcn_exp2f(m - mref);
    const bool moved = m != mref;
    m = mref;
    const float nm = mref == -INFINITY ? 0.f : -mref;
    float ls = 0.f;
    f32x4_t p[MB];
#pragma unroll
    for (int b = 0; b < MB; ++b)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        p[b][j] = __builtin_amdgcn_exp2f(s[b][j] + nm);
        ls += p[b][j];
      }
    l = l * alpha + ls;
    if (__ballot(moved)) {
      float aj[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) aj[j] = __shfl(alpha, 4 * g + j, 64);
#pragma unroll
      for (int nb = 0; nb < 4 * ND; ++nb)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[nb][j] *= aj[j];
    }
    // probabilities times V's scales, as the sum of NP bf16 terms: operand c is blocks 2 c, 2 c + 1
    uint4 pt[MB / 2][NP];
#pragma unroll
    for (int c = 0; c < MB / 2; ++c) {
      uint32_t t[NP][4];
#pragma unroll
      for (int b2 = 0; b2 < 2; ++b2) {
        // a block that is not there has no scale: what load_scales has for it is any block's, NaN perhaps
        const float f = (there >> (2 * c + b2)) & 1 ? lane_value(sv, 2 * c + b2) : 0.f;
#pragma unroll
        for (int j2 = 0; j2 < 2; ++j2) {
          float u = p[2 * c + b2][2 * j2] * f, v = p[2 * c + b2][2 * j2 + 1] * f;
#pragma unroll
          for (int k = 0; k < NP; ++k) {
            const uint32_t wd = tile::pack_bf16x2(u, v);
            t[k][2 * b2 + j2] = wd;
            u -= bf16_lo(wd);
            v -= bf16_hi(wd);
          }
        }
      }
#pragma unroll
      for (int k = 0; k < NP; ++k) pt[c][k] = make_uint4(t[k][0], t[k][1], t[k][2], t[k][3]);
    }
    // the next scales into the registers of these, whose last use this was: a copy of them, made for
    // the step to come, would wait for them, and so for every load before
    load_scales(w_nxt);
    // V of tokens past the context is whatever the page held: zeros
    if (base + STEP > cur.kv_len) {
#pragma unroll
      for (int b = 0; b < MB; ++b) {
        const int nv = cur.kv_len - (base + 16 * b + 4 * g);
        const uint32_t keep = nv >= 4 ? 0xffffffffu : nv <= 0 ? 0u : (1u << (8 * nv)) - 1u;
#pragma unroll
        for (int i = 0; i < ND; ++i) {
          vr[b][i].x &= keep;
          vr[b][i].y &= keep;
          vr[b][i].z &= keep;
          vr[b][i].w &= keep;
        }
      }
    }
    // Zero times NaN is NaN, so a NaN of V would reach rows that may not see its token. Where rows
    // differ in what they see, NaN codes are taken out, and put into the rows that see them by a
    // product of their places.
    if (!ONCE && a.offs && !full) {
      uint32_t any = 0;
#pragma unroll
      for (int b = 0; b < MB; ++b)
#pragma unroll
        for (int i = 0; i < ND; ++i)
          any |= kv8::nan_codes(vr[b][i].x) | kv8::nan_codes(vr[b][i].y) |
                 kv8::nan_codes(vr[b][i].z) | kv8::nan_codes(vr[b][i].w);
      if (__ballot(any != 0)) {
        const int rel = lim - (base + 4 * g);
#pragma unroll 1
        for (int nb = 0; nb < 4 * ND; ++nb) {
          f32x4_t hit = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int c = 0; c < MB / 2; ++c) {
            uint32_t see[4], at[2];
#pragma unroll
            for (int b2 = 0; b2 < 2; ++b2) {
              const int b = 2 * c + b2;
              const bool here = (there >> b) & 1;
#pragma unroll
              for (int j2 = 0; j2 < 2; ++j2)
                see[2 * b2 + j2] = (here && 16 * b + 2 * j2 < rel ? 0x3f80u : 0u) |
                                   (here && 16 * b + 2 * j2 + 1 < rel ? 0x3f800000u : 0u);
              uint32_t wd = 0;
#pragma unroll
              for (int i = 0; i < ND; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  if (nb == 4 * i + e) {
                    uint32_t* q4 = reinterpret_cast<uint32_t*>(&vr[b][i]);
                    wd = kv8::nan_codes(q4[e]);
                    q4[e] &= ~(wd * 0xffu);
                  }
              at[b2] = wd * 0x38u;  // the code of 1
            }
            hit = tile::mfma16<PIA_DTYPE_BF16>(make_uint4(see[0], see[1], see[2], see[3]),
                                               kv8::widen8<PIA_DTYPE_BF16>(at[0], at[1]), hit);
          }
#pragma unroll
          for (int k = 0; k < 4 * ND; ++k)
            if (nb == k)
#pragma unroll
              for (int j = 0; j < 4; ++j)
                if (hit[j] > 0.f) acc[k][j] = __builtin_nanf("");
        }
      }
    }
#pragma unroll
    for (int c = 0; c < MB / 2; ++c)
#pragma unroll
      for (int i = 0; i < ND; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint4 v = kv8::widen8<PIA_DTYPE_BF16>(tile32::word(vr[2 * c][i], e),
                                                 tile32::word(vr[2 * c + 1][i], e));
#pragma unroll
          for (int k = NP - 1; k >= 0; --k)
            acc[4 * i + e] = tile::mfma16<PIA_DTYPE_BF16>(pt[c][k], v, acc[4 * i + e]);
        }
    load_v(w_nxt);

    // end of the item or of the range
    if (cur.t + 1 == cur.steps || x + 1 == count) {
      const float lsum = tile32::sum_col4(l);
      const bool whole = cur.t + 1 == cur.steps && cur.t == x - begun;
      if (whole) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float lj = __shfl(lsum, 4 * g + j, 64);
          const int r = 16 * cur.i + 4 * g + j, pos = r / a.G;
          if (4 * g + j >= rows_left) continue;
          T* o = static_cast<T*>(a.out) +
                 ((row0 + pos) * a.Hq + cur.h * a.G + r - pos * a.G) * a.D;
          const float inv = lj == 0.f ? 0.f : 1.f / lj;
#pragma unroll
          for (int i = 0; i < ND; ++i) {
            const int d = 64 * i + 4 * n16;
            if (d < a.D) {
              struct alignas(4 * sizeof(T)) Pack {
                T v[4];
              } pk;
#pragma unroll
              for (int e = 0; e < 4; ++e)
                Elem<QT>::store(pk.v, e, lj == 0.f ? 0.f : acc[4 * i + e][j] * inv);
              *reinterpret_cast<Pack*>(o + d) = pk;
            }
          }
        }
      } else {
        float* part = a.parts + (w * 2 + (begun == 0 ? 0 : 1)) * part_floats<DP>;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (4 * g + j < rows_left)
#pragma unroll
            for (int i = 0; i < ND; ++i)
              *reinterpret_cast<float4*>(part + (4 * g + j) * DP + 64 * i + 4 * n16) =
                  make_float4(acc[4 * i][j], acc[4 * i + 1][j], acc[4 * i + 2][j],
                              acc[4 * i + 3][j]);
        if (g == 0) {
          part[16 * DP + n16] = m;
          part[16 * DP + 16 + n16] = lsum;
        }
      }
      opened = false;
    }
    cur = nxt;
    nxt = far;
    w_cur = w_nxt;
    w_nxt = w_far;
  }
}

// The items that were cut: their pieces joined, in the order of the waves. A workgroup has rows_per_wg
// rows of an item, all of them or, where there are few items with many pieces, one.
// Items without keys are zeros.
// the weight of a piece whose maximum is m against the joined one
__device__ __forceinline__ float weight(float m, float joined) {
  return m == joined ? (m == -INFINITY ? 0.f : 1.f) : __builtin_amdgcn_exp2f(m - joined);
}

template <int QT, int DP>
__global__ __launch_bounds__(KA_JOIN_FEW) void kv8_attention_join_kernel(AttnArgs a,
                                                                         int64_t waves,
                                                                         int rows_per_wg) {
  using T = typename Elem<QT>::T;
  constexpr int STEP = 16 * (DP > 128 ? 2 : 4);
  int64_t id = blockIdx.x / unsigned(a.Hkv);
  const int h = int(blockIdx.x - unsigned(id) * unsigned(a.Hkv));
  int b, i;
  if (a.cu) {
    // items of sequence b are numbered from cu[b] G / 16 + b on
    b = kv8::last_at(a.B, id, [&](int k) { return (int64_t(a.cu[k]) * a.G >> 4) + k; });
    i = int(id - ((int64_t(a.cu[b]) * a.G >> 4) + b));
  } else {
    const int items = (a.G + 15) >> 4;
    b = int(uint32_t(id) / uint32_t(items));
    i = int(id - int64_t(b) * items);
  }
  const Seq s = sequence(a, b, STEP);
  if (i < 0 || i >= s.items) return;
  const int r0 = blockIdx.y * rows_per_wg;
  const int rows = min(min(16, s.n * a.G - 16 * i) - r0, rows_per_wg);
  if (rows <= 0) return;
  const int64_t total = a.pref[a.B], nw = min(waves, total);
  const int64_t from = a.pref[b] + (int64_t(h) * s.items + i) * s.steps, to = from + s.steps;
  int64_t w0 = 0, w1 = 0;
  if (s.steps > 0) {
    w0 = wave_of(from, nw, total);
    w1 = wave_of(to - 1, nw, total);
    if (w0 == w1) return;  // finished by its wave
  }
  const float* first = a.parts + (w0 * 2 + (s.steps > 0 && first_of(w0, nw, total) >= from ? 0 : 1)) *
                                     part_floats<DP>;
  // S lanes in a row have four elements u of the item (row r, elements d .. d + 3) and every S-th piece
  // each, eight of them on their way at once; they meet by exchanges, in a fixed order. A lane has up to
  // 16 pieces where there are threads for that: with four, the single rows of one sequence of 3000 keys
  // take a microsecond more, and items of 16 rows with 18 pieces two.
  const int per_row = a.D / 4, U = rows * per_row, np = int(w1 - w0) + 1;
  const int threads = blockDim.x;
  int S = 1;
  while (S < 64 && 2 * S * U <= threads && 16 * S < np && s.steps > 0) S *= 2;
  const int sp = threadIdx.x & (S - 1);
  for (int u0 = 0; u0 < U; u0 += threads / S) {
    const int u = u0 + int(threadIdx.x) / S, rl = u / per_row, r = r0 + rl, d = 4 * (u - rl * per_row);
    if (u >= U) return;  // in whole groups of S lanes
    float M = -INFINITY, L = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    if (s.steps > 0) {
      constexpr int N = 8;
      for (int p0 = sp; p0 < np; p0 += N * S) {
        float pm[N], pl[N];
        float4 po[N];
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const int pi = min(p0 + j * S, np - 1);  // past the end: the last one again, without weight
          const float* p = pi == 0 ? first : a.parts + (w0 + pi) * 2 * part_floats<DP>;
          pm[j] = p0 + j * S < np ? p[16 * DP + r] : -INFINITY;
          pl[j] = p[16 * DP + 16 + r];
          po[j] = *reinterpret_cast<const float4*>(p + r * DP + d);
        }
        float m = M;
#pragma unroll
        for (int j = 0; j < N; ++j) m = __builtin_elementwise_maximum(m, pm[j]);
        const float f0 = weight(M, m);
        L *= f0;
        o = make_float4(o.x * f0, o.y * f0, o.z * f0, o.w * f0);
#pragma unroll
        for (int j = 0; j < N; ++j) {
          if (p0 + j * S >= np) continue;
          const float f = weight(pm[j], m);
          L += pl[j] * f;
          o = make_float4(fmaf(po[j].x, f, o.x), fmaf(po[j].y, f, o.y), fmaf(po[j].z, f, o.z),
                          fmaf(po[j].w, f, o.w));
        }
        M = m;
      }
    }
    if (S > 1) {
      float m = M;
      for (int k = 1; k < S; k *= 2) m = __builtin_elementwise_maximum(m, __shfl_xor(m, k, 64));
      const float f = weight(M, m);
      L *= f;
      o = make_float4(o.x * f, o.y * f, o.z * f, o.w * f);
      for (int k = 1; k < S; k *= 2) {
        L += __shfl_xor(L, k, 64);
        o.x += __shfl_xor(o.x, k, 64);
        o.y += __shfl_xor(o.y, k, 64);
        o.z += __shfl_xor(o.z, k, 64);
        o.w += __shfl_xor(o.w, k, 64);
      }
    }
    if (sp) continue;
    const float inv = L == 0.f ? 0.f : 1.f / L;
    const int rr = 16 * i + r, pos = rr / a.G;
    T* out = static_cast<T*>(a.out) + ((s.row0 + pos) * a.Hq + h * a.G + rr - pos * a.G) * a.D + d;
    struct alignas(4 * sizeof(T)) Pack {
      T v[4];
    } pk;
    Elem<QT>::store(pk.v, 0, L == 0.f ? 0.f : o.x * inv);
    Elem<QT>::store(pk.v, 1, L == 0.f ? 0.f : o.y * inv);
    Elem<QT>::store(pk.v, 2, L == 0.f ? 0.f : o.z * inv);
    Elem<QT>::store(pk.v, 3, L == 0.f ? 0.f : o.w * inv);
    *reinterpret_cast<Pack*>(out) = pk;
  }
}

int padded(int D) { return D <= 64 ? 64 : D <= 128 ? 128 : 256; }
int64_t resident_waves() { return int64_t(device_cus()) * KA_WGS_PER_CU * KA_WG_WAVES; }
constexpr int64_t KA_PREF_BYTES = (KA_MAX_SEQS + 1) * 8 + 248;  // whole 256 bytes

template <int QT, int DP>
void launch(const AttnArgs& a, int64_t items, bool once, hipStream_t s) {
  const unsigned wgs = unsigned(device_cus() * KA_WGS_PER_CU);
  if (once)
    hipLaunchKernelGGL((kv8_attention_kernel<QT, DP, true>), dim3(wgs), dim3(64 * KA_WG_WAVES), 0, s, a);
  else
    hipLaunchKernelGGL((kv8_attention_kernel<QT, DP, false>), dim3(wgs), dim3(64 * KA_WG_WAVES), 0, s, a);
  if (a.whole) return;
  // few items: many pieces each, which many threads share, on every compute unit; many: two or three
  const bool few = items * 4 <= resident_waves();
  const int rows = a.cu ? 16 : std::min(a.G, 16);
  const int parts = few ? int(std::max<int64_t>(1, std::min<int64_t>(rows, device_cus() / items))) : 1;
  const int rows_per_wg = (rows + parts - 1) / parts;
  hipLaunchKernelGGL((kv8_attention_join_kernel<QT, DP>),
                     dim3(unsigned(items), unsigned((rows + rows_per_wg - 1) / rows_per_wg)),
                     dim3(few ? KA_JOIN_FEW : KA_JOIN_MANY), 0, s, a, resident_waves(),
                     rows_per_wg);
}

// Whether `out` (bytes) holds any byte of n rows of `row` bytes, `stride` bytes apart from q on
bool holds_rows(uintptr_t out, int64_t bytes, uintptr_t q, int64_t n, int64_t row, int64_t stride) {
  if (stride <= 0) n = 1;
  // the first row that ends behind out's beginning
  const int64_t to = int64_t(out) - int64_t(q) - row;
  const int64_t r = to < 0 || n == 1 ? 0 : to / stride + 1;
  const int64_t from = int64_t(q) + r * stride;
  return r < n && from < int64_t(out) + bytes && from + row > int64_t(out);
}

}  // namespace
}  // namespace pia

using namespace pia;

extern "C" int64_t pia_kv8_attention_workspace_bytes(int head_dim) {
  if (head_dim <= 0 || head_dim > 256) return 0;
  const int DP = padded(head_dim);
  return KA_PREF_BYTES + resident_waves() * 2 * 16 * (DP + 2) * int64_t(sizeof(float));
}

extern "C" int pia_kv8_attention(void* out, const void* q, int64_t q_stride, const void* k_pages,
                                 const void* v_pages, const float* k_scales, const float* v_scales,
                                 const int32_t* block_tables, int64_t bt_stride,
                                 const int32_t* kv_lens, const int32_t* cu_q,
                                 const int32_t* q_pos_offsets, int num_seqs, int64_t total_q_rows,
                                 int num_heads, int num_kv_heads, int head_dim, int page_size,
                                 int64_t num_pages, float scale, int dtype, void* workspace,
                                 int64_t workspace_bytes, void* stream) {
  if (dtype != PIA_DTYPE_F32 && dtype != PIA_DTYPE_F16 && dtype != PIA_DTYPE_BF16)
    return fail(PIA_EUNSUPPORTED, "kv8_attention: dtype must be bf16, fp16 or fp32");
  if (num_seqs < 0 || total_q_rows < 0 || num_heads <= 0 || num_kv_heads <= 0 || num_pages <= 0 ||
      bt_stride < 0)
    return fail(PIA_EINVAL, "kv8_attention: invalid size");
  if (num_heads % num_kv_heads)
    return fail(PIA_EINVAL, "kv8_attention: num_heads % num_kv_heads != 0");
  if (!kv8::pool_shape(head_dim, page_size))
    return fail(PIA_EUNSUPPORTED,
                "kv8_attention: head_dim and page_size in multiples of 16, up to 256 and 4096");
  if (!cu_q && total_q_rows != num_seqs)
    return fail(PIA_EINVAL, "kv8_attention: without cu_q one row per sequence");
  if (num_seqs == 0 || total_q_rows == 0) return 0;
  if (num_pages > 0x7fffffff || num_pages * num_kv_heads > 0x7fffffff || total_q_rows > 0x3fffffff ||
      total_q_rows * num_heads > 0x7ffffff0)
    return fail(PIA_EINVAL, "kv8_attention: pool or rows too large");
  if (!out || !q || !k_pages || !v_pages || !k_scales || !v_scales || !kv_lens ||
      (bt_stride && !block_tables) || !workspace)
    return fail(PIA_EINVAL, "kv8_attention: null pointer");
  const int elem = dtype == PIA_DTYPE_F32 ? 4 : 2;
  if (!aligned(q, 16) || !aligned(out, 16) || (q_stride * elem) % 16 || !aligned(k_pages, 16) ||
      !aligned(v_pages, 16) || !aligned(workspace, 16))
    return fail(PIA_EINVAL, "kv8_attention: q rows, out, pools and workspace must be 16-byte aligned");
  // every row is read before it is written, by whoever writes it, but not before others are
  const int64_t row = int64_t(num_heads) * head_dim * elem;
  if (!(out == q && q_stride * elem == row) &&
      holds_rows(uintptr_t(out), total_q_rows * row, uintptr_t(q), total_q_rows, row, q_stride * elem))
    return fail(PIA_EINVAL, "kv8_attention: out overlaps q");
  if (workspace_bytes < pia_kv8_attention_workspace_bytes(head_dim))
    return fail(PIA_EINVAL, "kv8_attention: workspace too small");
  const int G = num_heads / num_kv_heads, DP = padded(head_dim);
  hipStream_t s = as_stream(stream);
  AttnArgs a{out, q, q_stride, static_cast<const uint8_t*>(k_pages),
             static_cast<const uint8_t*>(v_pages), k_scales, v_scales, block_tables, bt_stride,
             kv_lens, cu_q, q_pos_offsets, total_q_rows, num_pages,
             reinterpret_cast<float*>(static_cast<char*>(workspace) + KA_PREF_BYTES),
             static_cast<int64_t*>(workspace), scale * 1.4426950408889634f, num_seqs, num_heads,
             num_kv_heads, G, head_dim, page_size,
             ceil_div(bt_stride * page_size, DP > 128 ? 32 : 64) <= KA_WHOLE};
  if (kv8_prefill_path(dtype, num_heads, num_kv_heads, head_dim, num_seqs, total_q_rows, cu_q,
                       scale))
    return launch_kv8_prefill(dtype, out, q, q_stride, a.kp, a.vp, a.ks, a.vs, block_tables,
                              bt_stride, kv_lens, cu_q, q_pos_offsets, num_seqs, total_q_rows,
                              num_heads, num_kv_heads, head_dim, page_size, num_pages,
                              a.scale_log2, a.parts, resident_waves() * 2 * 16, s);
  const bool once = !cu_q && G <= 16;
  // more sequences than a launch's tables hold: by parts, one after the other on the stream
  for (int b0 = 0; b0 < num_seqs; b0 += KA_MAX_SEQS) {
    AttnArgs c = a;
    c.B = std::min(num_seqs - b0, KA_MAX_SEQS);
    c.bt += int64_t(b0) * bt_stride;
    c.lens += b0;
    if (c.offs) c.offs += b0;
    int64_t items;
    if (cu_q) {
      c.cu += b0;
      items = (total_q_rows * G >> 4) + c.B;
    } else {
      c.q = static_cast<const char*>(q) + int64_t(b0) * q_stride * elem;
      c.out = static_cast<char*>(out) + int64_t(b0) * num_heads * head_dim * elem;
      c.rows = c.B;
      items = int64_t(c.B) * ((G + 15) / 16);
    }
    items *= num_kv_heads;
    if (items > 0x7fffffff) return fail(PIA_EINVAL, "kv8_attention: too many rows");
#define PIA_K8(QT)                                        \
  switch (DP) {                                           \
    case 64: launch<QT, 64>(c, items, once, s); break;    \
    case 128: launch<QT, 128>(c, items, once, s); break;  \
    default: launch<QT, 256>(c, items, once, s); break;   \
  }
    if (dtype == PIA_DTYPE_F32) {
      PIA_K8(PIA_DTYPE_F32)
    } else if (dtype == PIA_DTYPE_F16) {
      PIA_K8(PIA_DTYPE_F16)
    } else {
      PIA_K8(PIA_DTYPE_BF16)
    }
#undef PIA_K8
    const int rc = check_launch("kv8_attention");
    if (rc) return rc;
  }
  return 0;
}
