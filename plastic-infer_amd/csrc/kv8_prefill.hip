// Attention of many query rows per sequence (prefill, chunked prefill) over the 8-bit KV pool on the
// matrix cores: bf16 or fp16 q (DT), head_dim to 128 (DP: 64, 96, 128), any page size of the pool.
//
// Work item (one workgroup of NW waves): one kv head and 32 NW / G consecutive query positions of one
// sequence, i.e. up to 32 NW (position, q head) rows that share the kv head's keys: row r is position
// s0 + r / G, head h * G + r % G. Wave w owns rows 32 w .. 32 w + 31, one 32 x 32 product block. The
// keys go by tiles of 64 tokens (four blocks); where there are few items, each is cut along its keys
// into pieces (workgroups of their own), whose outputs, maxima and sums a second kernel joins in order.
// Codes come from the pool into registers a tile ahead, and on their way into LDS, at the end of the
// tile before theirs, they are widened to DT: once for all rows, where an operand widened at its use
// would be widened by every wave. bf16 holds a code times its scale exactly. fp16 does only for scales of
// 2^-15 .. 2^7, so its K is codes, whose scale enters the scores in fp32 (1 to 2 % of the time); its V is
// within 2^-25 below those scales, and beyond 65504 counts as that. A head_dim below DP is made up with
// zeros of K and q; V's rows behind it are whatever LDS holds and end in outputs that nobody writes.
//
// Per tile each wave runs (v_mfma_f32_32x32x16: A rows and B columns are lane l % 32, k slots
// 8 (l / 32) + e; of C, lane l has column l % 32 and rows 8 i + 4 (l / 32) + j, i, j < 4)
//   S^T = K . q^T  lane l has the scores of row l % 32 for tokens 8 i + 4 (l / 32) + j of each 32
//   online softmax base 2, per row in fp32; a row's scores sit in two lanes (l, l ^ 32)
//   O^T += V^T . P^T  the probabilities are the B operand straight from the score registers: of a
//                  block's tokens, lane half hh holds 4 hh + j and 8 + 4 hh + j. Rows of the result are
//                  elements, so a lane has DP / 2 of them, all of its own row l % 32: what a row's
//                  maximum and sum do to it needs no exchange between lanes.
// The probabilities are rounded to DT once, and the sum is of the rounded ones: half a step of DT each,
// as much as the result's own rounding (bf16, the case below: 0.0020 of the norm from exact results,
// 0.0017 for exactly computed ones rounded). A second term would be half as many products again (fp16
// with two bf16 terms: 890 us, and 660 with one on the same machine). fp16 has 29 binades of normal numbers
// for them: a row's reference follows its maximum from tile to tile, up and down, so that a tile's largest
// has at least 25 of them below it (8 % of the time where heads' scores spread unlike). What the rest loses
// is bounded at the end of an item, which is done again where that is too much: 3.3 times as long.
// LDS tiles (16-byte units, XORed with a term of their row): K [token][d], 16 units to a token also at
// DP 96: unit u (d 8 u .. + 7) of token t at u ^ t % 16 (DP 64: 8 units, u ^ t / 2 % 8); V [d][token]:
// unit 2 m + hh (block m, tokens 4 hh + j, then 8 + 4 hh + j) of element d at
// (2 m + hh) ^ (d / 4 % 8) ^ (d / 2 % 2). With the bank rules of gfx950 (stores: 8 lanes over 32 banks;
// 16-byte reads: lanes {0-3, 12-15, 20-27} or the others over 64) all of them are conflict-free but K
// stores at DP 64.
//
// Measured: 8 sequences of 1024 new rows on 4096 keys, causal, 32 heads of 128 over 8, bf16: 625 to
// 645 us on several machines, 0.96 to 0.99 PFLOP/s of 619 GFLOP (a large library product of this card:
// 1.3). No one unit bounds it: the matrix cores are busy 46 % of the time, and of the rest a wave's
// exponentials and packing cost 50 us, the widening and its LDS stores 90, the loads 15, the operands'
// LDS reads 35 (each taken out alone).
// Scores a tile ahead brought it there from 700; loads two tiles ahead with exact waits, the widening
// between the two products and half-tile turns of the waves left it as it is.
#include <algorithm>
#include <type_traits>

#include "attn_tiles.h"
#include "kv8.h"

namespace pia {
namespace {

typedef float f32x16_t __attribute__((ext_vector_type(16)));

constexpr int P8_KT = 64;            // keys per tile: four blocks
constexpr int P8_MAX_SEQS = 1024;    // sequences per launch (tile prefix in LDS)
constexpr int P8_AHEAD = 4;           // LDS operands read ahead of their product
constexpr int P8_PV_VALU = 2;         // vector instructions after each product of the outputs
constexpr int P8_MAX_CUTS = 64;      // pieces of an item
constexpr int P8_RSRC_WORD3 = 0x00020000;
constexpr float P8_RESCALE = 8.0f;   // log2: how far a row's maximum may run ahead of its reference
// fp16, where a tile's largest probability has to be near the top of the type's range: how far a row's
// maximum in the tile may be from its reference, on either side, the exponent of the reference's
// probability, and how far below the largest maximum so far a reference may be (fp32 outputs hold
// 2^(13 + 60) times 2^31 keys of 2^16)
constexpr float P8_NEAR_HALF = 2.0f, P8_UP_HALF = 13.0f, P8_FLOOR_HALF = 60.0f;
constexpr float P8_LEAST_HALF = 6.103515625e-5f;  // 2^-14: the least normal number
constexpr float P8_REST = 16777216.f;             // 2^24, one over the least number
constexpr float P8_V_HALF = 0.0625f;              // the largest V scale that the rounding below takes

struct PrefillArgs {
  void* out;
  const void* q;
  int64_t q_stride;
  const uint8_t *kp, *vp;
  const float *ks, *vs;
  const int32_t* bt;
  int64_t bt_stride;
  const int32_t *lens, *cu, *offs;
  int64_t rows, num_pages;
  float scale_log2;
  int B, Hq, Hkv, G, D, P, ppt, cuts;
  float* parts;
};

template <int DT>
__device__ __forceinline__ f32x16_t mfma32(const uint4& a, const uint4& b, f32x16_t c) {
  if constexpr (DT == PIA_DTYPE_F16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(tile::f16x8_t, a),
                                                  __builtin_bit_cast(tile::f16x8_t, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(tile::bf16x8_t, a),
                                                   __builtin_bit_cast(tile::bf16x8_t, b), c, 0, 0,
                                                   0);
}

// fp16 infinities as the largest values: what no fp16 holds of a code times its scale (fp16 tensors
// round to 65536 at most, half a step from there). An infinity would be NaN in rows that do not see it.
__device__ __forceinline__ uint32_t finite16(uint32_t w) {
  return w - ((w & 0x7fffu) == 0x7c00u ? 1u : 0u) - ((w & 0x7fff0000u) == 0x7c000000u ? 0x10000u : 0u);
}
// a uint4 of DT values as it is, or finite
template <bool FIX>
__device__ __forceinline__ uint4 kept(const uint4& x) {
  if constexpr (FIX)
    return make_uint4(finite16(x.x), finite16(x.y), finite16(x.z), finite16(x.w));
  else
    return x;
}

// sum of a pair of DT values onto c
template <int DT>
__device__ __forceinline__ float add_pair(uint32_t x, float c) {
  typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
  typedef _Float16 h2 __attribute__((ext_vector_type(2)));
  if constexpr (DT == PIA_DTYPE_F16)
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(h2, x), __builtin_bit_cast(h2, 0x3c003c00u), c,
                                  false);
  else
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf2, x),
                                           __builtin_bit_cast(bf2, 0x3f803f80u), c, false);
}

__device__ __forceinline__ float swap_halves(float x) {  // the value of lane l ^ 32
  const unsigned u = __float_as_uint(x);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __uint_as_float((threadIdx.x & 32) ? r[0] : r[1]);
}

template <int DP, int NW, int DT>
__global__ __launch_bounds__(64 * NW, 8 / NW) void kv8_prefill_kernel(PrefillArgs a) {
  constexpr int NT = 64 * NW, KS = DP / 16, NB = DP / 32;
  constexpr int UK = DP > 64 ? 16 : 8;  // 16-byte units of a K row in LDS
  constexpr bool SPLIT = NW == 8;  // waves 0-3 stage K, 4-7 V; with four waves each stages both
  constexpr uint32_t K_BUF = P8_KT * UK * 16, V_BUF = DP * 128;  // bytes
  __shared__ __align__(16) unsigned char lds[2 * (K_BUF + V_BUF)];
  __shared__ int tile_pref[P8_MAX_SEQS + 1];
  __shared__ int wsum[NW];
  __shared__ int nan_seen;
  // fp16: the K scales of four tiles' blocks. A tile's are read while the one before it is computed, and
  // those two tiles on are put down meanwhile.
  constexpr bool HALF = DT == PIA_DTYPE_F16;
  __shared__ __align__(16) float k_scale[HALF ? 4 : 1][4];
  __shared__ uint32_t v_most[4];  // fp16: the largest V scale of each block of the tiles so far
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

  // work items per sequence and their prefix
  if (threadIdx.x == 0) tile_pref[0] = 0;
  if (threadIdx.x == 0) nan_seen = 0;
  if (threadIdx.x < 4) v_most[threadIdx.x] = 0;
  int carry = 0;
  for (int c0 = 0; c0 < a.B; c0 += NT) {
    const int i = c0 + threadIdx.x;
    int incl = 0;
    if (i < a.B) {
      const int64_t r0 = a.cu[i], n = min(int64_t(a.cu[i + 1]), a.rows) - r0;
      incl = r0 >= 0 && n > 0 ? int((n + a.ppt - 1) / a.ppt) : 0;
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int y = __shfl_up(incl, o, 64);
      if (lane >= o) incl += y;
    }
    if (lane == 63) wsum[wave] = incl;
    __syncthreads();
    int base = carry;
    for (int x = 0; x < wave; ++x) base += wsum[x];
    if (i < a.B) tile_pref[i + 1] = base + incl;
#pragma unroll
    for (int x = 0; x < NW; ++x) carry += wsum[x];
    __syncthreads();
  }
  int h, j;
  if (!xcd_item(blockIdx.x, carry * a.cuts, a.Hkv, h, j)) return;
  const int piece = a.cuts == 1 ? 0 : uint32_t(j) % uint32_t(a.cuts);  // of the item's keys
  if (a.cuts > 1) j = uint32_t(j) / uint32_t(a.cuts);
  int lo = 0, hi = a.B - 1;  // the sequence holding the item: the last with tile_pref[b] <= j
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (tile_pref[mid] <= j) lo = mid; else hi = mid - 1;
  }
  const int b = __builtin_amdgcn_readfirstlane(lo);
  h = __builtin_amdgcn_readfirstlane(h);
  // the last positions of a sequence, which see the most keys, first
  const int s0 = __builtin_amdgcn_readfirstlane((tile_pref[b + 1] - 1 - j) * a.ppt);
  const int64_t row0 = a.cu[b];
  const int n_b = int(min(int64_t(a.cu[b + 1]), a.rows) - row0);
  const int kv_len =
      int(min(int64_t(max(a.lens[b], 0)), min(a.bt_stride * a.P, int64_t(0x7ffffff0))));
  const int off = a.offs ? a.offs[b] : 0;
  const int s_last = min(s0 + a.ppt, n_b) - 1;
  const int kmax = a.offs ? kv8::seen(kv_len, off, s_last) : kv_len;
  // its tiles kt0 .. nkt - 1: all, or the piece's
  int kt0 = 0, nkt = (kmax + P8_KT - 1) / P8_KT;
  if (a.cuts > 1) {
    const uint32_t n = nkt;  // times 64 pieces: 2^31 at most
    kt0 = int(n * uint32_t(piece) / uint32_t(a.cuts));
    nkt = int(n * uint32_t(piece + 1) / uint32_t(a.cuts));
  }
  kt0 = __builtin_amdgcn_readfirstlane(kt0);
  nkt = __builtin_amdgcn_readfirstlane(nkt);
  const int nblk = (kv_len + 15) >> 4, PB = a.P / 16;
  const int32_t* btb = a.bt + int64_t(b) * a.bt_stride;

  // this lane's row and its q operands, d = 16 ks + 8 (l / 32) .. + 7
  const int D = NW == 8 ? DP : a.D;  // 8 waves: as a constant, it takes 1 % less
  const int hh = lane >> 5, n32 = lane & 31, G = a.G;
  const int r = 32 * wave + n32, pos = s0 + r / G;
  const bool live = r < a.ppt * G && pos < n_b;
  const int lim = !live ? 0 : a.offs ? kv8::seen(kv_len, off, pos) : kv_len;
  uint4 qr[KS];
  {
    const uint16_t* qp = static_cast<const uint16_t*>(a.q) + (row0 + (live ? pos : 0)) * a.q_stride +
                         int64_t(h * G + (live ? r % G : 0)) * D;
#pragma unroll
    for (int k = 0; k < KS; ++k)
      qr[k] = live && 16 * k < D ? *reinterpret_cast<const uint4*>(qp + 16 * k + 8 * hh)
                   : make_uint4(0u, 0u, 0u, 0u);
  }
  // every row of the item sees at least the keys below lim_min (its first position's limit)
  const int lim_min = a.offs ? kv8::seen(kv_len, off, s0) : kv_len;

  // staging: wave w (of four) moves block w of a tile, K by lanes (token l % 16, chunks l / 16 and
  // l / 16 + 4), V by lanes (elements 4 (l % 32) .. + 3, token groups l / 32 and l / 32 + 2). What a
  // wave has of either: its loads' offset, and a base of its LDS addresses (the rest enters by XOR).
  const int blk = wave & 3;
  const int VL = D / 4;  // lanes of a token group of V
  const int64_t tile_bytes = int64_t(D) * a.P;
  struct Part {
    uint4 x[2];
    float scale;  // of a block that is not there: any block's, NaN perhaps
    bool there;
    uint32_t off, base;
  };
  auto k_part = [&]() {
    const int t = 16 * blk + (lane & 15), c = lane >> 4, sw = DP > 64 ? t & 15 : (t >> 1) & 7;
    return Part{{}, 1.f, false, uint32_t((c * a.P + (lane & 15)) * 16),
                uint32_t(t * UK * 16 + 16 * ((2 * c) ^ sw))};
  };
  auto v_part = [&]() {
    const int x = lane & 31;  // below VL; the others load and drop
    return Part{{}, 1.f, false, uint32_t(hh * 4 * D + 16 * x),
                2 * K_BUF + uint32_t(x * 4 * 128 + 16 * ((2 * blk + hh) ^ (x & 7)))};
  };
  const bool first4 = wave < 4;
  Part pa = SPLIT && !first4 ? v_part() : k_part(), pb = v_part();  // pb: with four waves only
  // Pages of the blocks of a tile in lanes 0 .. 3 (-1 where there is none) and the blocks' places in
  // them. The ids are as loaded: what is made of them is made where they are used, tiles later, so
  // that no tile waits for them (and with them for every load before).
  struct Where {
    int id, sub;
  };
  const uint32_t np = a.num_pages > 0x7fffffff ? 0x7fffffffu : uint32_t(a.num_pages);
  auto where = [&](int kt) {
    Where w{-1, 0};
    const int kb = 4 * kt + lane, slot = PB == 1 ? kb : kb / PB;
    w.sub = kb - slot * PB;
    if (lane < 4 && kb < nblk) w.id = btb[slot];
    return w;
  };
  auto fetch_part = [&](Part& p, bool is_k, int id, int sub) {
    const bool ok = uint32_t(id) < np;
    const int64_t head = int64_t(id) * a.Hkv + h;
    const int64_t at = (ok ? head : 0) * tile_bytes + (is_k ? sub * 256 : sub * 16 * D);
    const int bytes = is_k ? int(tile_bytes) - sub * 256 : 16 * D;
    const uint32_t step = is_k ? uint32_t(64 * a.P) : uint32_t(8 * D);
    const auto rs = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint8_t*>((is_k ? a.kp : a.vp) + at), 0, ok ? bytes : 0, P8_RSRC_WORD3);
    p.x[0] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rs, p.off, 0, 0));
    if (DP > 64 || !is_k)
      p.x[1] =
          __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rs, p.off + step, 0, 0));
    p.scale = (is_k ? a.ks : a.vs)[ok ? head * PB + sub : 0];
    p.there = ok;
  };
  // K of one tile and V of another (with eight waves a wave has one of them)
  auto fetch_next = [&](const Where& wk, const Where& wv) {
    if constexpr (SPLIT) {
      const int id = __builtin_amdgcn_readlane(first4 ? wk.id : wv.id, blk);
      const int sub = __builtin_amdgcn_readlane(first4 ? wk.sub : wv.sub, blk);
      fetch_part(pa, first4, id, sub);
    } else {
      fetch_part(pa, true, __builtin_amdgcn_readlane(wk.id, blk),
                 __builtin_amdgcn_readlane(wk.sub, blk));
      fetch_part(pb, false, __builtin_amdgcn_readlane(wv.id, blk),
                 __builtin_amdgcn_readlane(wv.sub, blk));
    }
  };
  auto put = [&](uint32_t at, const uint4& x) {
    *reinterpret_cast<uint4*>(lds + at) = x;
  };
  // a block whose values may pass 65504 (448 times its scale): the same for the whole wave
  auto large = [&](float scale) {
    return DT == PIA_DTYPE_F16 && __builtin_amdgcn_readfirstlane(int(scale > 128.f));
  };
  auto stage_k = [&](const Part& p, int buf, int kt) {
    const uint32_t base = p.base + buf * K_BUF;
    const float scale = HALF && p.scale == p.scale ? 1.f : p.scale;  // NaN stays, in K
#pragma unroll
    for (int i = 0; i < UK / 8; ++i) {
      put(base ^ (128 * i), kv8::widen8<DT>(p.x[i].x, p.x[i].y, scale));
      put(base ^ (128 * i + 16), kv8::widen8<DT>(p.x[i].z, p.x[i].w, scale));
    }
    if (HALF && lane == 0) k_scale[kt & 3][blk] = p.there ? p.scale : 1.f;
  };
  auto stage_v = [&](Part& p, int buf, int kt, bool places) {
    // tokens past the context hold whatever the page held: zeros
    if (64 * kt + 64 > kv_len) {
      const int nv = kv_len - (64 * kt + 16 * blk + 4 * hh);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int n = nv - 8 * i;
        const uint32_t keep = n >= 4 ? 0xffffffffu : n <= 0 ? 0u : (1u << (8 * n)) - 1u;
        p.x[i].x &= keep;
        p.x[i].y &= keep;
        p.x[i].z &= keep;
        p.x[i].w &= keep;
      }
    }
    // Zero times NaN is NaN, so a NaN of V would reach the rows that may not see its token. On tiles
    // that not every row sees whole it is staged as zero; the end of the item puts it where it
    // belongs, from tiles of the NaNs' places (places: a one for each).
    float scale = p.there ? p.scale : 1.f;  // times zeros (K's scores are hidden, whatever they are)
    if (HALF && lane == 0 && p.there)
      __hip_atomic_fetch_max(&v_most[blk], __float_as_uint(scale), __ATOMIC_RELAXED,
                             __HIP_MEMORY_SCOPE_WORKGROUP);
    if (places || 64 * kt + 64 > lim_min) {
      uint32_t any = 0;
      uint32_t* w = &p.x[0].x;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t n = kv8::nan_codes(w[e]);
        any |= n;
        w[e] = places ? n * 0x38u : w[e] & ~(n * 0xffu);  // 0x38: the code of 1
      }
      if (places) scale = 1.f;
      else if (any && (lane & 31) < VL) nan_seen = 1;
    }
    auto all = [&](auto fix) {
      const uint32_t base = p.base + buf * V_BUF;
      put(base, kept<fix()>(kv8::widen8<DT>(p.x[0].x, p.x[1].x, scale)));
      put(base + 128, kept<fix()>(kv8::widen8<DT>(p.x[0].y, p.x[1].y, scale)));
      put((base ^ 16) + 256, kept<fix()>(kv8::widen8<DT>(p.x[0].z, p.x[1].z, scale)));
      put((base ^ 16) + 384, kept<fix()>(kv8::widen8<DT>(p.x[0].w, p.x[1].w, scale)));
    };
    if ((lane & 31) < VL) {
      if (large(scale)) all(std::true_type{});
      else all(std::false_type{});
    }
  };
  auto stage = [&](int buf, int kt, bool places) {
    if constexpr (SPLIT) {
      if (first4) stage_k(pa, buf, kt);
      else stage_v(pa, buf, kt, places);
    } else {
      stage_k(pa, buf, kt);
      stage_v(pb, buf, kt, places);
    }
  };
  // Operand addresses (bytes): the swizzle terms of rows 32 apart are the same, and the unit's upper
  // bits enter by XOR, so one base per lane and a constant give any of them; bases of a buffer, so
  // that they are computed where they are used and not kept.
  const uint32_t k_base = n32 * UK * 16 + 16 * (hh ^ (DP > 64 ? n32 & 15 : (n32 >> 1) & 7));
  const uint32_t v_base = n32 * 128 + 16 * (hh ^ (((n32 >> 2) & 7) ^ ((n32 >> 1) & 1)));
  auto kread = [&](int buf, int tb, int k) {
    const uint32_t at = ((k_base + buf * K_BUF) ^ (32 * k)) + 32 * tb * UK * 16;
    return *reinterpret_cast<const uint4*>(lds + at);
  };
  auto vread = [&](int buf, int nb, int s) {
    const uint32_t at = ((v_base + buf * V_BUF) ^ (32 * s)) + 32 * nb * 128;
    return *reinterpret_cast<const uint4*>(lds + 2 * K_BUF + at);
  };

  // bf16: the row's reference point m is in units of the products q . K. fp16: K is codes, and m, like
  // `unit`, what a block's products have to be multiplied by, in those of the exponent.
  float m = -INFINITY, l = 0.f;  // l: the lane's sum
  float4 unit = make_float4(0.f, 0.f, 0.f, 0.f);  // fp16: of the tile whose scores are there
  auto unit_of = [&](int kt) {
    if constexpr (HALF) {
      // never 0: hidden scores are -inf
      auto f = [&](float x) { return fmaxf(x * a.scale_log2, 1.17549435e-38f); };
      const float4 x = *reinterpret_cast<const float4*>(k_scale[kt & 3]);
      unit = make_float4(f(x.x), f(x.y), f(x.z), f(x.w));
    }
  };
  f32x16_t acc[NB];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int v = 0; v < 16; ++v) acc[nb][v] = 0.f;

  // scores of a tile from its K, on their own
  auto scores = [&](f32x16_t (&sc)[2], int buf) {
#pragma unroll
    for (int tb = 0; tb < 2; ++tb)
#pragma unroll
      for (int v = 0; v < 16; ++v) sc[tb][v] = 0.f;
#pragma unroll
    for (int i = 0; i < 2 * KS; ++i)
      sc[i & 1] = mfma32<DT>(kread(buf, i & 1, i >> 1), qr[i >> 1], sc[i & 1]);
  };
  auto largest = [&](const f32x16_t (&sc)[2]) {
    if constexpr (HALF) {
      float b[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int v = 0; v < 8; ++v)
          b[s] = __builtin_elementwise_maximum(b[s], sc[s >> 1][8 * (s & 1) + v]);
      return __builtin_elementwise_maximum(
          __builtin_elementwise_maximum(b[0] * unit.x, b[1] * unit.y),
          __builtin_elementwise_maximum(b[2] * unit.z, b[3] * unit.w));
    }
    float mx = -INFINITY;
#pragma unroll
    for (int tb = 0; tb < 2; ++tb)
#pragma unroll
      for (int v = 0; v < 16; ++v) mx = __builtin_elementwise_maximum(mx, sc[tb][v]);
    return mx;
  };
  const float m_unit = HALF ? 1.f : a.scale_log2;
  auto minus = [&](float x) {  // what a score takes to its probability's exponent
    return x == -INFINITY ? 0.f : HALF ? P8_UP_HALF - x : -x * m_unit;
  };
  float top = -INFINITY;  // fp16: the largest of the row's maxima
  auto reference = [&](float mx) {
    if constexpr (!HALF) return (mx - m) * m_unit > P8_RESCALE || mx != mx ? mx : m;
    top = __builtin_elementwise_maximum(top, mx);
    const float d = mx - m;
    return fabsf(d) <= P8_NEAR_HALF || mx == -INFINITY
               ? m : __builtin_elementwise_maximum(mx, top - P8_FLOOR_HALF);
  };
  auto unit_at = [&](int s) {
    return !HALF ? a.scale_log2 : s == 0 ? unit.x : s == 1 ? unit.y : s == 2 ? unit.z : unit.w;
  };
  auto hide = [&](f32x16_t (&sc)[2], int kt, int there) {  // what the row may not see
    const int rel = lim - (kt * P8_KT + 4 * hh);
#pragma unroll
    for (int tb = 0; tb < 2; ++tb)
#pragma unroll
      for (int v = 0; v < 16; ++v)
        if (!(32 * tb + 8 * (v >> 2) + (v & 3) < rel && ((there >> (2 * tb + (v >> 3))) & 1)))
          sc[tb][v] = -INFINITY;
  };
  // One tile. sc: its scores, mx: the largest of them (of the lane's) where none is hidden; sn, mx:
  // the next tile's on return. A wave keeps its matrix core and its vector ALU busy at once: the
  // next tile's scores are multiplied while this one's become probabilities, and this one's
  // outputs while the tile after is staged.
  auto turn = [&](f32x16_t (&sc)[2], f32x16_t (&sn)[2], float& mx, int kt, int buf, int there) {
    if (!(there == 0xf && (kt + 1) * P8_KT <= lim_min)) {
      hide(sc, kt, there);
      mx = largest(sc);
    }
    mx = __builtin_elementwise_maximum(mx, swap_halves(mx));
    const float mref = reference(mx);
    const float nm = minus(mref);
    if (__ballot(m != mref)) {
      const float alpha = m == mref ? 1.f : __builtin_amdgcn_exp2f((m - mref) * m_unit);
      l *= alpha;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int v = 0; v < 16; ++v) acc[nb][v] *= alpha;
    }
    m = mref;
    scores(sn, buf ^ 1);
    uint4 pk[4];  // block s of the tile: the B operand of its 16 tokens, the probabilities
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const float u = unit_at(s);
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int v = 8 * (s & 1) + 2 * i;
        const float p0 = __builtin_amdgcn_exp2f(fmaf(sc[s >> 1][v], u, nm));
        const float p1 = __builtin_amdgcn_exp2f(fmaf(sc[s >> 1][v + 1], u, nm));
        w[i] = tile::pack16x2<DT>(p0, p1);
        l = add_pair<DT>(w[i], l);
      }
      pk[s] = make_uint4(w[0], w[1], w[2], w[3]);
    }
#pragma unroll
    for (int i = 0; i < 4 * NB; ++i)
      acc[i % NB] = mfma32<DT>(vread(buf, i % NB, i / NB), pk[i / NB], acc[i % NB]);
    unit_of(kt + 1);
    mx = largest(sn);
    // kept so through the scheduler: operands read P8_AHEAD products ahead of their use, the vector
    // work of the probabilities among the scores' products, the next maximum's among the outputs'
    constexpr int QK = 2 * KS, PV = 4 * NB;
    __builtin_amdgcn_sched_group_barrier(0x100, P8_AHEAD, 0);
#pragma unroll
    for (int i = 0; i < QK; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x402, 96 / QK, 0);
    }
#pragma unroll
    for (int i = 0; i < PV; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      if (i + P8_AHEAD < PV) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x402, P8_PV_VALU, 0);
    }
  };

  // K is staged two tiles ahead of the outputs, for scores are a tile ahead, V one. With two buffers
  // each, what a tile stages replaces what the tile before it has read, with a barrier between.
  auto stage_next = [&](int kt, int buf) {
    if constexpr (SPLIT) {
      if (first4) stage_k(pa, buf, kt + 2);
      else stage_v(pa, buf ^ 1, kt + 1, false);
    } else {
      stage_k(pa, buf, kt + 2);
      stage_v(pb, buf ^ 1, kt + 1, false);
    }
  };
  Where w0 = where(kt0), w1 = where(kt0 + 1), w2 = where(kt0 + 2), w3 = where(kt0 + 3);  // kt .. kt + 3
  fetch_next(w0, w0);
  stage(0, kt0, false);
  if (!SPLIT || first4) {  // K of tile 1; the other waves have nothing of it
    fetch_part(pa, true, __builtin_amdgcn_readlane(w1.id, blk),
               __builtin_amdgcn_readlane(w1.sub, blk));
    stage_k(pa, 1, kt0 + 1);
  }
  fetch_next(w2, w1);
  __syncthreads();
  f32x16_t sa[2], sb[2];
  scores(sa, 0);
  unit_of(kt0);
  float mx = largest(sa);
  __syncthreads();  // the first step stages K where these scores were read
  auto step = [&](f32x16_t (&sc)[2], f32x16_t (&sn)[2], int kt, int buf) {
    const int there = int(__ballot(lane < 4 && uint32_t(w0.id) < np)) & 0xf;
    const Where w4 = where(kt + 4);
    turn(sc, sn, mx, kt, buf, there);
    stage_next(kt, buf);
    fetch_next(w3, w2);
    __syncthreads();
    w0 = w1;
    w1 = w2;
    w2 = w3;
    w3 = w4;
  };
  for (int kt = kt0; kt < nkt; kt += 2) {
    step(sa, sb, kt, 0);
    if (kt + 1 >= nkt) break;
    step(sb, sa, kt + 1, 1);
  }

  // fp16: rounding takes up to 2^-25 from each probability below the normal numbers, where the largest of
  // its tile is 2^11 at least. The lost ones of 64 keys are 2^-30 of that largest one then, and those of all
  // keys 2^-30 of the row's sum: times values of up to 28 (448 times the limit), less than half of the least
  // fp16 number. For larger values the item is done again with its row's own maximum, each probability below
  // the normal numbers as two: what fp16 holds of it, and 2^24 times the rest.
  if constexpr (HALF) {
    const float most = __uint_as_float(max(max(v_most[0], v_most[1]), max(v_most[2], v_most[3])));
    if (!(most <= P8_V_HALF)) {  // the same for all waves
      m = top;
      const float nm = minus(m);
      l = 0.f;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int v = 0; v < 16; ++v) acc[nb][v] = 0.f;
#pragma unroll 1
      for (int i = 2 * kt0; i < 2 * nkt; ++i) {  // the rests of all tiles first
        const bool rest = i < kt0 + nkt;
        const int kt = rest ? i - kt0 : i - nkt;
        __syncthreads();
        const Where w = where(kt);
        fetch_next(w, w);
        stage(0, kt, false);
        __syncthreads();
        if (i == kt0 + nkt)
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int v = 0; v < 16; ++v) acc[nb][v] *= 1.f / P8_REST;
        scores(sa, 0);
        unit_of(kt);
        hide(sa, kt, int(__ballot(lane < 4 && uint32_t(w.id) < np)) & 0xf);
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          uint32_t x[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            float r[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float p = __builtin_amdgcn_exp2f(
                  fmaf(sa[s >> 1][8 * (s & 1) + 2 * k + e], unit_at(s), nm));
              const float less = p < P8_LEAST_HALF ? (p - half_to_f32(f32_to_half(p))) * P8_REST : 0.f;
              r[e] = rest ? less : p;
              l += rest ? p : 0.f;
            }
            x[k] = tile::pack16x2<DT>(r[0], r[1]);
          }
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
            acc[nb] = mfma32<DT>(vread(0, nb, s), make_uint4(x[0], x[1], x[2], x[3]), acc[nb]);
        }
      }
    }
  }

  if (nan_seen) {  // the same for every wave: all stores to it are barriers ago
#pragma unroll 1
    for (int kt = max(kt0, lim_min / P8_KT); kt < nkt; ++kt) {
      __syncthreads();
      const Where w = where(kt);
      fetch_next(w, w);
      stage(0, kt, true);
      __syncthreads();
      const int there = int(__ballot(lane < 4 && uint32_t(w.id) < np)) & 0xf;
      const int rel = lim - (kt * P8_KT + 4 * hh);
      constexpr uint32_t ONE = DT == PIA_DTYPE_F16 ? 0x3c00u : 0x3f80u;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        f32x16_t hit;
#pragma unroll
        for (int v = 0; v < 16; ++v) hit[v] = 0.f;
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          __builtin_amdgcn_sched_barrier(0);  // one operand at a time (registers)
          uint32_t see[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int t = 16 * s + 8 * (i >> 1) + 2 * (i & 1);
            const bool here = (there >> s) & 1;
            see[i] = (here && t < rel ? ONE : 0u) | (here && t + 1 < rel ? ONE << 16 : 0u);
          }
          hit = mfma32<DT>(vread(0, nb, s), make_uint4(see[0], see[1], see[2], see[3]), hit);
        }
#pragma unroll
        for (int v = 0; v < 16; ++v)
          if (hit[v] > 0.f) acc[nb][v] = __builtin_nanf("");
      }
    }
  }

  l += swap_halves(l);
  if (!live) return;
  if (a.cuts > 1) {  // the piece as it is, to be joined: its outputs, then its maximum and sum
    const int64_t R = a.rows * a.Hq, at = piece * R + (row0 + pos) * a.Hq + h * G + r % G;
    float* o = a.parts + at * D + 4 * hh;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (32 * nb + 8 * i < D)
          *reinterpret_cast<float4*>(o + 32 * nb + 8 * i) = make_float4(
              acc[nb][4 * i], acc[nb][4 * i + 1], acc[nb][4 * i + 2], acc[nb][4 * i + 3]);
    if (hh == 0)
      reinterpret_cast<float2*>(a.parts + a.cuts * R * D)[at] = make_float2(m * m_unit, l);
    return;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  uint16_t* o = static_cast<uint16_t*>(a.out) + ((row0 + pos) * a.Hq + h * G + r % G) * D + 4 * hh;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (32 * nb + 8 * i >= D) continue;
      uint32_t w[2];
#pragma unroll
      for (int e = 0; e < 2; ++e)
        w[e] = tile::pack16x2<DT>(l == 0.f ? 0.f : acc[nb][4 * i + 2 * e] * inv,
                                  l == 0.f ? 0.f : acc[nb][4 * i + 2 * e + 1] * inv);
      *reinterpret_cast<uint2*>(o + 32 * nb + 8 * i) = make_uint2(w[0], w[1]);
    }
}

// The pieces of every row joined, in order: a thread has four elements of one.
template <int DT>
__global__ __launch_bounds__(256) void kv8_prefill_join_kernel(PrefillArgs a) {
  const int D = a.D;
  const int64_t x = int64_t(blockIdx.x) * 256 + threadIdx.x, R = a.rows * a.Hq;
  const int64_t at = uint32_t(x) / uint32_t(D / 4);  // below 2^31
  const int d = 4 * int(x - at * (D / 4));
  const int64_t row = uint32_t(at) / uint32_t(a.Hq);
  if (at >= R || row < a.cu[0] || row >= a.cu[a.B]) return;
  const float2* ml = reinterpret_cast<const float2*>(a.parts + a.cuts * R * D);
  float M = -INFINITY, L = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  constexpr int N = 4;  // pieces on their way at once; past the end: the last again, without weight
  for (int p0 = 0; p0 < a.cuts; p0 += N) {
    float2 pm[N];
    float4 po[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int64_t i = min(p0 + k, a.cuts - 1) * R + at;
      pm[k] = ml[i];
      po[k] = *reinterpret_cast<const float4*>(a.parts + i * D + d);
    }
#pragma unroll
    for (int k = 0; k < N; ++k) {
      if (p0 + k >= a.cuts) break;
      const float to = __builtin_elementwise_maximum(M, pm[k].x);
      const float f0 = M == to ? 1.f : __builtin_amdgcn_exp2f(M - to);
      const float f = pm[k].x == to ? 1.f : __builtin_amdgcn_exp2f(pm[k].x - to);
      L = L * f0 + pm[k].y * f;
      o = make_float4(fmaf(po[k].x, f, o.x * f0), fmaf(po[k].y, f, o.y * f0),
                      fmaf(po[k].z, f, o.z * f0), fmaf(po[k].w, f, o.w * f0));
      M = to;
    }
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
  const uint2 w = make_uint2(tile::pack16x2<DT>(L == 0.f ? 0.f : o.x * inv, L == 0.f ? 0.f : o.y * inv),
                             tile::pack16x2<DT>(L == 0.f ? 0.f : o.z * inv, L == 0.f ? 0.f : o.w * inv));
  *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + at * D + d) = w;
}

template <int DP, int NW, int DT>
void launch(const PrefillArgs& a, unsigned blocks, hipStream_t s) {
  hipLaunchKernelGGL((kv8_prefill_kernel<DP, NW, DT>), dim3(blocks), dim3(64 * NW), 0, s, a);
  if (a.cuts > 1)
    hipLaunchKernelGGL((kv8_prefill_join_kernel<DT>),
                       dim3(unsigned(ceil_div(a.rows * a.Hq * (a.D / 4), 256))), dim3(256), 0, s, a);
}

}  // namespace

// Against the kernel that streams codes to each 16 rows: that one takes 2.4 us for 1M rows x keys at
// head_dim 128 (1.3 at 64), this one 0.6 (0.5) where its items are full and long, and their rows cost
// the same when most are missing. In us there and here, 4096 keys, 8 kv heads of 128, rows of a kv head
// and sequence: one sequence, 32 rows 20.0 and 19.5, 64 rows 25 and 20, 256 rows 30 and 25, 4096 rows
// 175 and 87; 16 sequences, 32 rows 39 and 52, 64 rows 61 and 48, 4096 rows 1694 and 530. Only a few rows
// on few heads lose a microsecond or two from 64 rows on (one sequence, 512 keys: 13.7 and 15.3); below
// two rows to a compute unit there would not be pieces enough for all of them.
bool kv8_prefill_path(int dtype, int Hq, int Hkv, int D, int num_seqs, int64_t total_q_rows,
                      const int32_t* cu_q, float scale) {
  const int G = Hq / Hkv;
  // scale > 0: the kernel keeps its running max in raw score units
  return (dtype == PIA_DTYPE_BF16 || dtype == PIA_DTYPE_F16) && D <= 128 &&
         scale > 0.f && G <= 128 && cu_q != nullptr && num_seqs <= P8_MAX_SEQS &&
         total_q_rows * G >= 64 * int64_t(num_seqs) &&
         total_q_rows * Hq >= 2 * int64_t(device_cus());
}

int launch_kv8_prefill(int dtype, void* out, const void* q, int64_t q_stride, const uint8_t* kp,
                       const uint8_t* vp, const float* ks, const float* vs, const int32_t* bt,
                       int64_t bt_stride, const int32_t* lens, const int32_t* cu,
                       const int32_t* offs, int num_seqs, int64_t total_q_rows, int Hq, int Hkv,
                       int D, int P, int64_t num_pages, float scale_log2, float* parts,
                       int64_t part_rows, hipStream_t s) {
  const int G = Hq / Hkv;
  // Items of 256 rows halve what is widened for a row but come half as many: for long contexts that
  // fill the CUs all the same. 32 sequences, 32 heads, 64 rows each: 90 us and 86 at 2048 keys, 322 and
  // 279 at 8192; 128 rows: 95 and 101 at 1024 keys, 164 and 158 at 2048, 300 and 276 at 4096. At
  // head_dim 64, where a tile's products are half, they lose everywhere (390 and 430 at 4096 keys).
  const int64_t cus = device_cus(), tiles = ceil_div(bt_stride * P, P8_KT);
  const int64_t items = std::max<int64_t>(1, (ceil_div(total_q_rows, 128 / G) + num_seqs / 2) * Hkv);
  const bool wide = D == 128 && bt_stride * P >= 2048 && items >= 2 * cus;
  const int ppt = (wide ? 256 : 128) / G;
  // Fewer items than CUs: their keys are cut into pieces, to two on every CU of 16 tiles each (if the
  // table is full), or one of 4, as far as the workspace has rows for them. One sequence of 32 heads of
  // 128 on 32768 keys: 128 rows 650 us whole and 88 cut, 512 rows 666 and 288. 64 pieces of 8 tiles a
  // row take 52 us there where 32 of 16 take 43; pieces of 2 tiles cost more than they bring (4096 keys,
  // 2048 rows of 64 heads: 34 us, and 25 with 8), and so does a cut of items that fill the CUs (512
  // keys, 32768 rows: 30 and 21). Under a table that is not full the pieces are shorter than that: 128 rows on
  // 512 keys take 18 us with their own table, 23 with one of 4096 tokens, 31 of 32768.
  const int64_t most = std::max(std::min(2 * cus / items, tiles / 16), std::min(cus / items, tiles / 4));
  const int cuts = int(std::max<int64_t>(
      1, std::min(std::min<int64_t>(most, P8_MAX_CUTS), part_rows / (total_q_rows * Hq))));
  const int64_t blocks = ceil_div((ceil_div(total_q_rows, ppt) + num_seqs) * cuts * Hkv, 8) * 8;
  if (blocks > 0x7fffffff) return fail(PIA_EINVAL, "kv8_attention: too many query rows");
  PrefillArgs a{out, q, q_stride, kp, vp, ks, vs, bt, bt_stride, lens, cu, offs, total_q_rows,
                num_pages, scale_log2, num_seqs, Hq, Hkv, G, D, P, ppt, cuts, parts};
#define PIA_P8(DT)                                                 \
  {                                                                \
    if (wide) launch<128, 8, DT>(a, unsigned(blocks), s);          \
    else if (D > 96) launch<128, 4, DT>(a, unsigned(blocks), s);   \
    else if (D > 64) launch<96, 4, DT>(a, unsigned(blocks), s);    \
    else launch<64, 4, DT>(a, unsigned(blocks), s);                \
  }
  if (dtype == PIA_DTYPE_F16) PIA_P8(PIA_DTYPE_F16) else PIA_P8(PIA_DTYPE_BF16)
#undef PIA_P8
  return check_launch("kv8_prefill");
}

}  // namespace pia
