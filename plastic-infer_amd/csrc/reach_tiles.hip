// Windowed attention and attention behind a shared prefix for many query rows per key, on tiles in LDS:
// bf16 or fp16 (DT), head_dim to 256 (DP: 64, 96, 128, 256), pages in multiples of 16 tokens.
//
// Work item (one workgroup of NW waves): one kv head and 32 NW / G consecutive query positions of one
// sequence, i.e. up to 32 NW (position, q head) rows that share the kv head's keys: row r is position
// s0 + r / G, head h * G + r % G; or those of a group, one position a sequence, over its prefix. Wave w owns
// rows 32 w .. 32 w + 31, one 32 x 32 product block. The keys go by tiles of 64 tokens (four blocks of 16): first
// those of the sinks or of the prefix, then the sequence's own that some row of the item sees. Where there are
// few items, each is cut along its tiles into pieces (workgroups of their own) that are joined in order.
//
// Bound by the matrix cores, the exponentials and the LDS reads of both products, which a wave runs against each
// other: 2.0 us for a tile of 256 rows on a CU, 1.07 PFLOP/s (a large product of the library: 1.22), and 13 us
// around a workgroup's tiles: its search for its item, the first ids, rows and tiles one after the other, the
// results. No LDS bank conflicts. 8 x 1024 rows, 32 / 8 heads, 8192 keys each: head_dim 128 1111 us in bf16 (0.99
// PFLOP/s) and 1210 in fp16, 96 970 and 1083, 64 754 and 835 (half the products for the same exponentials); 16 / 4
// heads of 256 1914 and 2120 (one wave to a SIMD). A window of 2048 of the chunks' own and earlier tokens: 360.
//
// Per tile each wave runs (v_mfma_f32_32x32x16: A rows and B columns are lane l % 32, k slots
// 8 (l / 32) + e; of C, lane l has column l % 32 and rows 8 i + 4 (l / 32) + j, i, j < 4; hh = l / 32)
//   S^T = K . q^T  K rows lie in LDS with bits 2 and 3 of the token exchanged, so that a lane has the
//                  scores of tokens 8 hh .. + 7 of each block
//   online softmax base 2, per row in fp32; a row's scores sit in two lanes (l, l ^ 32)
//   O^T += V^T . P^T  the probabilities are the B operand straight from the score registers. A lane has
//                  DP / 2 outputs, all of its own row l % 32: what a row's maximum and sum do to them
//                  needs no exchange between lanes.
// The probabilities are rounded to DT once, and the sum is of the rounded ones: half a step of DT each, as much as
// the result's own rounding. Results are 1.25 times as far from their exact values as those that are rounded once at
// the end (bf16: 0.0021 of the norm and 0.00166). A second term of each, as the streaming kernel has, brings them
// there for half as many products again: 8 x 1024 rows on 8192 keys 1400 us for 1085, in a window of 2048 455 for
// 362. fp16 numbers are scaled by up to 2^15 and normal to 2^-25 of the
// reference; a tile with smaller ones multiplies what rounding took of them too.
//
// LDS tiles (16-byte units, XORed with a term of their row). The pool's rows are [d][token]. V is staged as
// it is: [d][64 tokens], unit u (tokens 8 u .. + 7) at u ^ d / 2 % 8; a wave's lanes take the rows of 1 KB in the
// order that stores without conflicts. K is turned on its way: a lane loads TL tokens of eight rows and
// stores, for each token, a unit of eight elements. Those are the elements u, u + NU, u + 2 NU, ... (NU = DP / 8
// units to a row), for that makes a wave's loads whole lines, and q's operands are taken in the same
// order once an item. K [token][d]: unit u of row r at u ^ r % 16 (DP 64: 8 units, u ^ r / 2 % 8).
#include <algorithm>

#include "attn_tiles.h"
#include "reach.h"

// A lambda that is not inlined keeps all that it captures in memory: the compiler left the largest of DP 256 as
// calls (8 x 1024 rows, 16 heads, 8192 keys each: 9200 us with them, 1914 without)
#define RT_INLINE __attribute__((always_inline))

namespace pia {
namespace {

using reach::Args;
using reach::Seq;

typedef float f32x16_t __attribute__((ext_vector_type(16)));

constexpr int RT_KT = 64;            // keys per tile: four blocks
constexpr int RT_MAX_SEQS = 1024;    // sequences per launch (item prefix in LDS)
constexpr int RT_AHEAD = 4;          // LDS operands read ahead of their product
constexpr int RT_PV_VALU = 2;        // vector instructions after each product of the outputs
constexpr int RT_MAX_CUTS = 64;      // pieces of an item
constexpr int RT_MAX_BLOCKS = 1 << 22;  // items of a call (a launch of 2^32 threads is refused)
constexpr int RT_RSRC_WORD3 = 0x00020000;
// log2: how far a row's maximum may run ahead of its reference, and what the reference's probability is
template <int DT>
constexpr float RT_RESCALE = DT == PIA_DTYPE_F16 ? 4.0f : 8.0f;
template <int DT>
constexpr float RT_SHIFT = DT == PIA_DTYPE_F16 ? 11.0f : 0.0f;
constexpr float RT_LEAST_HALF = 6.103515625e-5f;  // 2^-14: the least normal number
constexpr float RT_REST = 0x1p38f;  // what such numbers' rounding takes, 2^-25, is 2^13 of its units
constexpr uint32_t RT_PUT = 0xf400u;  // minus the least number, 2^-24, in them: -2^14

struct TileArgs : Args {
  int ppt, cuts;
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
__global__ __launch_bounds__(64 * NW, DP > 128 ? 1 : 8 / NW) void reach_tiles_kernel(TileArgs a) {
  constexpr int NT = 64 * NW, KS = DP / 16, NB = DP / 32, NU = DP / 8;
  constexpr int UK = DP > 128 ? 32 : DP > 64 ? 16 : 8;  // 16-byte units of a K row in LDS
  constexpr int TL = DP > 128 ? 8 : DP > 64 ? 4 : 2;    // tokens of a lane's K loads
  constexpr bool SPLIT = NW == 8;  // waves 0-3 stage K, 4-7 V; with four waves each stages both
  constexpr bool HALF = DT == PIA_DTYPE_F16;
  constexpr uint32_t K_BUF = RT_KT * UK * 16, V_BUF = DP * 128;  // bytes
  __shared__ __align__(16) unsigned char lds[2 * (K_BUF + V_BUF)];
  __shared__ int item_pref[RT_MAX_SEQS + 1];
  __shared__ int wsum[NW];
  __shared__ int odd_seen;
  __shared__ int4 sees[32 * NW];  // of each row: lowest, limit, and how much of the head
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  auto seq_at = [&](int b) {
    return a.by_group ? reach::group(a, a.first + b) : reach::sequence(a, a.first + b);
  };

  // work items per sequence, those before each, and this workgroup's: item `j` of sequence `b`
  if (threadIdx.x == 0) odd_seen = 0;
  int h, j, b, piece;
  auto mine = [&](int items) {  // of all sequences' items
    if (!xcd_item(blockIdx.x, items * a.cuts, a.Hkv, h, j)) return false;
    piece = a.cuts == 1 ? 0 : uint32_t(j) % uint32_t(a.cuts);  // of the item's tiles
    if (a.cuts > 1) j = uint32_t(j) / uint32_t(a.cuts);
    return true;
  };
  auto items_at = [&](int i) {
    const int n = i < a.count ? seq_at(i).n : 0;
    return n > 0 ? (n + a.ppt - 1) / a.ppt : 0;
  };
  auto scan = [&](int x) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int y = __shfl_up(x, o, 64);
      if (lane >= o) x += y;
    }
    return x;
  };
  if (a.count <= 64) {  // each wave for itself
    const int own = items_at(lane), incl = scan(own);
    if (!mine(__builtin_amdgcn_readlane(incl, 63))) return;
    b = __builtin_ctzll(__ballot(incl > j));  // the first with more items up to it
    j = __builtin_amdgcn_readlane(incl, b) - 1 - j;
  } else {
    if (threadIdx.x == 0) item_pref[0] = 0;
    int carry = 0;
    for (int c0 = 0; c0 < a.count; c0 += NT) {
      const int i = c0 + threadIdx.x;
      const int incl = scan(items_at(i));
      if (lane == 63) wsum[wave] = incl;
      __syncthreads();
      int base = carry;
      for (int x = 0; x < wave; ++x) base += wsum[x];
      if (i < a.count) item_pref[i + 1] = base + incl;
#pragma unroll
      for (int x = 0; x < NW; ++x) carry += wsum[x];
      __syncthreads();
    }
    if (!mine(carry)) return;
    int lo_b = 0, hi_b = a.count - 1;  // the last with item_pref[b] <= j
    while (lo_b < hi_b) {
      const int mid = (lo_b + hi_b + 1) >> 1;
      if (item_pref[mid] <= j) lo_b = mid; else hi_b = mid - 1;
    }
    b = lo_b;
    j = item_pref[b + 1] - 1 - j;
  }
  b = __builtin_amdgcn_readfirstlane(b);
  piece = __builtin_amdgcn_readfirstlane(piece);
  h = __builtin_amdgcn_readfirstlane(h);
  // the last positions of a sequence, which see the most keys, first
  const int s0 = __builtin_amdgcn_readfirstlane(j * a.ppt);
  const Seq s = seq_at(b);
  const int64_t row0 = s.row0;
  const int s_last = min(s0 + a.ppt, s.n) - 1;
  // the two stretches of tiles: of the sinks or the prefix (head), then of the sequence's own table
  const bool grouped = a.by_group != 0;
  const int32_t* own = grouped ? a.pt + int64_t(a.first + b) * a.pt_stride
                               : a.bt + int64_t(a.first + b) * a.bt_stride;
  const int32_t* head_table = own;
  int head = 0;  // tokens of the head
  bool prefixed = false;
  if (a.window) head = min(a.sinks, reach::limit(s, s_last));
  else if (!grouped) {
    const int g = reach::group_of(a, a.first + b);
    if (g >= 0) {
      prefixed = true;
      head_table = a.pt + g * a.pt_stride;
      head = reach::held(a.plens[g], a.pt_stride, a.P);
    }
  }
  const int lim_any = reach::limit(s, s_last), lim_all = reach::limit(s, s0);
  const int lo_any = reach::lowest(a, s, s0), lo_all = reach::lowest(a, s, s_last);
  const int hs_all = a.window ? min(head, lim_all) : head;
  const int nh = (head + RT_KT - 1) / RT_KT;
  const int t0 = a.window ? max(nh, lo_any / RT_KT) : 0;
  const int n_own = max(0, (lim_any + RT_KT - 1) / RT_KT - t0);
  // its tiles kt0 .. nkt - 1: all, or the piece's
  int kt0 = 0, nkt = nh + n_own;
  if (a.cuts > 1) {
    const uint32_t n = nkt;  // times 64 pieces: 2^32 at most
    kt0 = int(uint64_t(n) * uint32_t(piece) / uint32_t(a.cuts));
    nkt = int(uint64_t(n) * uint32_t(piece + 1) / uint32_t(a.cuts));
  }
  kt0 = __builtin_amdgcn_readfirstlane(kt0);
  nkt = __builtin_amdgcn_readfirstlane(nkt);

  // rows, and what they see: in LDS, for the tiles that not all rows see whole
  const int D = a.D;
  const int hh = lane >> 5, n32 = lane & 31, G = a.G;
  struct Row {
    int r, pos;
    bool live;
  };
  auto row_now = [&]() {
    int x = lane & 31;
    asm volatile("" : "+v"(x));
    const int r = 32 * wave + x, pos = s0 + r / G;
    return Row{r, pos, r < a.ppt * G && pos < s.n};
  };

  if (threadIdx.x < 32 * NW) {
    const int r = threadIdx.x, pos = s0 + r / G, lim = reach::limit(s, pos);
    const bool live = r < a.ppt * G && pos < s.n;
    sees[r] = live ? make_int4(reach::lowest(a, s, pos), lim, a.window ? min(head, lim) : head, 0)
                   : make_int4(0, 0, 0, 0);
  }

  // q: unit u of a row is its elements u, NU + u, ..., and a lane's units 2 k + hh are the elements hh of all its
  // words. So a lane loads its whole row and takes half of each word.
  uint4 qr[KS];
  {
    const Row x = row_now();
    const uint16_t* q = static_cast<const uint16_t*>(a.q) +
                        (row0 + (x.live ? x.pos : 0)) * a.q_stride +
                        int64_t(h * G + (x.live ? x.r % G : 0)) * D;
    uint4 z[DP / 8];
#pragma unroll
    for (int i = 0; i < DP / 8; ++i) {  // rows that are none take the first one's, and are not written
      const bool ok = 8 * i < D;
      z[i] = *reinterpret_cast<const uint4*>(q + (ok ? 8 * i : 0));
      z[i].x = ok ? z[i].x : 0u;
      z[i].y = ok ? z[i].y : 0u;
      z[i].z = ok ? z[i].z : 0u;
      z[i].w = ok ? z[i].w : 0u;
    }
    const uint32_t half = hh ? 0x07060302u : 0x05040100u;
    auto of = [&](int d) {  // the word of element d
      const uint4& y = z[d / 8];
      const int i = d % 8 / 2;
      return i == 0 ? y.x : i == 1 ? y.y : i == 2 ? y.z : y.w;
    };
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      uint32_t w[4];
#pragma unroll
      for (int f = 0; f < 4; ++f)
        w[f] = __builtin_amdgcn_perm(of(NU * (2 * f + 1) + 2 * k), of(NU * 2 * f + 2 * k), half);
      qr[k] = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }

  // tile `it` of the item's list: its first token, and whether it is of the head
  auto in_head = [&](int it) { return it < nh; };
  auto first_token = [&](int it) { return (it < nh ? it : t0 + it - nh) * RT_KT; };
  // Of a tile's tokens: those of [from, to) of the sequence, and in the head's tiles those below `below`. A
  // prefix's tiles have no others.
  struct Reach {
    int from, to, below;
  };
  auto reach_of = [&](int it, int from, int to, int below) {
    const int base = first_token(it);
    const bool head_tile = in_head(it);
    return Reach{from - base, (head_tile && prefixed ? 0 : to) - base, (head_tile ? below : 0) - base};
  };
  // 8 tokens from token t of the tile on, as bits
  auto bits8 = [](const Reach& x, int t) {
    auto first = [](int n) { return (1u << min(max(n, 0), 8)) - 1u; };
    return (first(x.to - t) & ~first(x.from - t)) | first(x.below - t);
  };
  auto reach_of_row = [&](int it) {
    const int4 x = sees[32 * wave + n32];
    return reach_of(it, x.x, x.y, x.z);
  };
  // whether every row sees all of a tile (of the blocks that are there)
  auto seen_whole = [&](int it) {
    const Reach x = reach_of(it, lo_all, lim_all, hs_all);
    return x.below >= RT_KT || (x.from <= 0 && x.to >= RT_KT);
  };
  // Pages of the blocks of a tile in lanes 0 .. 3 (-1 where no row sees any of it). The ids are as
  // loaded: what is made of them is made where they are used, tiles later, so that no tile waits for them
  // (and with them for every load before).
  const uint32_t np = uint32_t(a.num_pages);
  const int PB = a.P / 16;
  auto where = [&](int it) {
    const Reach x = reach_of(it, lo_any, lim_any, head);
    const int t = 16 * lane, kb = (first_token(it) >> 4) + lane, slot = PB == 1 ? kb : kb / PB;
    const bool in = (it < nkt) & (lane < 4) &
                    (((t + 16 > x.from) & (t < x.to)) | (t < x.below));
    int id = -1;
    if (in) id = (in_head(it) ? head_table : own)[slot];
    return id;
  };

  // staging: wave w (of four) moves block w of a tile
  const int blk = wave & 3;
  constexpr int KL = 8, VL = DP / 32;  // loads of a lane
  struct Part {
    uint32_t w[DP > 128 ? 32 : 16];
  };
  const int du = lane % NU, tg = lane / NU;  // K: unit and token group
  const bool k_lane = DP != 96 || tg < 4;
  const uint32_t row_bytes = 2 * a.P;
  const uint32_t k_off = uint32_t(du) * row_bytes + uint32_t(k_lane ? tg : 0) * TL * 2;
  // V: lanes 8 c + 2 x + half take row c % 4 + 4 x + 16 (c / 4), and those 32 on
  const int vd = ((lane >> 3) & 3) + 4 * ((lane >> 1) & 3) + 16 * (lane >> 5), vh = lane & 1;
  const uint32_t v_off = uint32_t(vd) * row_bytes + 16 * vh;
  // where they go: K's first token (bits 2 and 3 of the token exchanged), V's first row
  const int k_tok = TL * tg, k_row = 16 * blk + ((k_tok & 3) | ((k_tok & 4) << 1) | ((k_tok & 8) >> 1));
  const uint32_t k_st = k_row * UK * 16 + 16 * (du ^ (DP > 64 ? k_row & 15 : (k_row >> 1) & 7));
  const uint32_t v_st = 2 * K_BUF + vd * 128 + 16 * ((2 * blk + vh) ^ ((vd >> 1) & 7));
  const int tile_bytes = D * a.P * 2;
  const int64_t page_bytes = int64_t(tile_bytes) * a.Hkv;
  const char* kp = static_cast<const char*>(a.kp) + int64_t(h) * tile_bytes;
  const char* vp = static_cast<const char*>(a.vp) + int64_t(h) * tile_bytes;
  auto rsrc = [&](const char* pool, int ids, int it) {
    const int id = __builtin_amdgcn_readlane(ids, blk), kb = (first_token(it) >> 4) + blk;
    const int sub = PB == 1 ? 0 : kb % PB;
    const bool ok = uint32_t(id) < np;
    // elements behind head_dim lie past the descriptor's end, and are zeros. In scalar registers by force: the
    // compiler kept the descriptors of DP 256 in vector registers, with a loop around every load
    const uint64_t at = reinterpret_cast<uint64_t>(pool) + (ok ? id : 0) * page_bytes + sub * 32;
    const uint32_t lo = __builtin_amdgcn_readfirstlane(uint32_t(at)),
                   hi = __builtin_amdgcn_readfirstlane(uint32_t(at >> 32));
    return __builtin_amdgcn_make_buffer_rsrc(
        reinterpret_cast<void*>(uint64_t(hi) << 32 | lo), 0,
        __builtin_amdgcn_readfirstlane(ok ? tile_bytes - sub * 32 : 0), RT_RSRC_WORD3);
  };
  // a lane's term, hidden, so that what is added to it is added at its use: kept for all uses, the sums were
  // spilled, and a wait for a spilled register is one for every load before it
  auto now = [](uint32_t x) {
    asm volatile("" : "+v"(x));
    return x;
  };
  auto fetch_k = [&](Part& p, int ids, int it) RT_INLINE {
    const auto rs = rsrc(kp, ids, it);
    const uint32_t o = now(k_off);
#pragma unroll
    for (int e = 0; e < KL; ++e) {
      const uint32_t at = o + uint32_t(e * NU) * row_bytes;
      if constexpr (TL == 8) {
        const auto y = __builtin_amdgcn_raw_buffer_load_b128(rs, at, 0, 0);
#pragma unroll
        for (int c = 0; c < 4; ++c) p.w[4 * e + c] = y[c];
      } else if constexpr (TL == 4) {
        const auto y = __builtin_amdgcn_raw_buffer_load_b64(rs, at, 0, 0);
        p.w[2 * e] = y[0];
        p.w[2 * e + 1] = y[1];
      } else {
        p.w[e] = __builtin_amdgcn_raw_buffer_load_b32(rs, at, 0, 0);
      }
    }
  };
  auto fetch_v = [&](Part& p, int ids, int it) RT_INLINE {
    const auto rs = rsrc(vp, ids, it);
    const uint32_t o = now(v_off);
#pragma unroll
    for (int i = 0; i < VL; ++i) {
      const auto y =
          __builtin_amdgcn_raw_buffer_load_b128(rs, o + uint32_t(32 * i) * row_bytes, 0, 0);
#pragma unroll
      for (int c = 0; c < 4; ++c) p.w[4 * i + c] = y[c];
    }
  };
  auto put = [&](uint32_t at, const uint4& x) { *reinterpret_cast<uint4*>(lds + at) = x; };
  auto stage_k = [&](Part& p, int buf) RT_INLINE {
    if (!k_lane) return;
    const uint32_t o = now(k_st) + buf * K_BUF;
#pragma unroll
    for (int t = 0; t < TL; ++t) {
      uint32_t w[4];
#pragma unroll
      for (int f = 0; f < 4; ++f)
        w[f] = __builtin_amdgcn_perm(p.w[(2 * f + 1) * (TL / 2) + (t >> 1)],
                                     p.w[2 * f * (TL / 2) + (t >> 1)],
                                     (t & 1) ? 0x07060302u : 0x05040100u);
      // so many rows on, by which the swizzle differs too (DP 64: by none)
      const int c = (t & 3) + 2 * (t & 4);
      put(((o ^ (DP > 64 ? 16 * c : 0)) + c * UK * 16), make_uint4(w[0], w[1], w[2], w[3]));
    }
  };
  // kind 0: V itself, but zeros for what is not finite on tiles that some row does not see whole (zero
  // times it would be NaN there; the end of the item puts it where it belongs); 1, 2, 3: a one where V is
  // NaN, infinite, minus infinite
  constexpr uint32_t EXP = HALF ? 0x7c00u : 0x7f80u, ONE = HALF ? 0x3c00u : 0x3f80u;
  auto stage_v = [&](Part& p, int buf, int it, int kind) RT_INLINE {
    bool look = kind != 0;
    if (!kind && !seen_whole(it)) {
      // a half that is not finite carries into its top bit: |x| + 2^(mantissa bits) >= 2^15
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < 4 * VL; ++i)
        top |= (p.w[i] & 0x7fff7fffu) + (HALF ? 0x04000400u : 0x00800080u);
      look = __ballot((top & 0x80008000u) != 0) != 0;
    }
    if (look) {
      const uint32_t any = bits8(reach_of(it, lo_any, lim_any, head), 16 * blk + 8 * vh);
      uint32_t odd = 0;
#pragma unroll
      for (int i = 0; i < 4 * VL; ++i) {
        uint32_t& w = p.w[i];
        // 0xffff for each half that is not finite
        const uint32_t bad = ((w & EXP) == EXP ? 0xffffu : 0u) |
                             ((w & (EXP << 16)) == EXP << 16 ? 0xffff0000u : 0u);
        const uint32_t see = (any >> (2 * (i & 3))) & 3u;
        odd |= bad & ((see & 1u) | ((see & 2u) << 15));
        if (kind == 0) {
          w &= ~bad;
        } else {
          const uint32_t nan = ((w & 0x7fffu) != EXP ? 0xffffu : 0u) |
                               ((w & 0x7fff0000u) != EXP << 16 ? 0xffff0000u : 0u);
          const uint32_t neg = ((w >> 15) & 0x00010001u) * 0xffffu;
          const uint32_t hit = kind == 1 ? nan : kind == 2 ? ~nan & ~neg : ~nan & neg;
          w = bad & hit & (ONE | ONE << 16);
        }
      }
      if (odd) odd_seen = 1;
    }
    const uint32_t o = now(v_st) + buf * V_BUF;
#pragma unroll
    for (int i = 0; i < VL; ++i)
      put(o + 4096 * i, make_uint4(p.w[4 * i], p.w[4 * i + 1], p.w[4 * i + 2], p.w[4 * i + 3]));
  };
  // Operand addresses (bytes): the swizzle terms of rows 32 apart are the same, and the unit's upper
  // bits enter by XOR, so one base per lane and a constant give any of them
  const uint32_t k_base = n32 * UK * 16 + 16 * (hh ^ (DP > 64 ? n32 & 15 : (n32 >> 1) & 7));
  const uint32_t v_base = n32 * 128 + 16 * (hh ^ ((n32 >> 1) & 7));
  auto kread = [&](int buf, int tb, int k) {
    const uint32_t at = ((k_base + buf * K_BUF) ^ (32 * k)) + 32 * tb * UK * 16;
    return *reinterpret_cast<const uint4*>(lds + at);
  };
  auto vread = [&](int buf, int nb, int s4) {
    const uint32_t at = ((v_base + buf * V_BUF) ^ (32 * s4)) + 32 * nb * 128;
    return *reinterpret_cast<const uint4*>(lds + 2 * K_BUF + at);
  };

  float m = -INFINITY, l = 0.f;  // m: the row's reference, in units of the products q . K; l: the lane's sum
  f32x16_t acc[NB];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int v = 0; v < 16; ++v) acc[nb][v] = 0.f;

  // scores of a tile from its K, on their own
  auto scores = [&](f32x16_t (&sc)[2], int buf) RT_INLINE {
#pragma unroll
    for (int tb = 0; tb < 2; ++tb)
#pragma unroll
      for (int v = 0; v < 16; ++v) sc[tb][v] = 0.f;
#pragma unroll
    for (int i = 0; i < 2 * KS; ++i)
      sc[i & 1] = mfma32<DT>(kread(buf, i & 1, i >> 1), qr[i >> 1], sc[i & 1]);
  };
  auto largest = [&](const f32x16_t (&sc)[2]) {
    float mx = -INFINITY;
#pragma unroll
    for (int tb = 0; tb < 2; ++tb)
#pragma unroll
      for (int v = 0; v < 16; ++v) mx = __builtin_elementwise_maximum(mx, sc[tb][v]);
    return mx;
  };
  auto hide = [&](f32x16_t (&sc)[2], int it, int there) RT_INLINE {  // what the row may not see
    const Reach x = reach_of_row(it);
#pragma unroll
    for (int tb = 0; tb < 2; ++tb)
#pragma unroll
      for (int v = 0; v < 16; v += 8) {
        const int s4 = 2 * tb + (v >> 3);
        const uint32_t see = (there >> s4) & 1 ? bits8(x, 16 * s4 + 8 * hh) : 0u;
#pragma unroll
        for (int e = 0; e < 8; ++e) {  // all bits of `keep`, or none: v_bfe_i32, v_bfi_b32
          const uint32_t keep = uint32_t(int32_t(see << (31 - e)) >> 31);
          sc[tb][v + e] = __uint_as_float((keep & __float_as_uint(sc[tb][v + e])) |
                                          (~keep & 0xff800000u));
        }
      }
  };
  // One tile. sc: its scores, mx: the largest of them (of the lane's) where none is hidden; sn, mx:
  // the next tile's on return. A wave keeps its matrix core and its vector ALU busy at once: the
  // next tile's scores are multiplied while this one's become probabilities, and this one's
  // outputs while the tile after is staged.
  auto turn = [&](f32x16_t (&sc)[2], f32x16_t (&sn)[2], float& mx, int it, int buf, int there) RT_INLINE {
    if (!(there == 0xf && seen_whole(it))) {
      hide(sc, it, there);
      mx = largest(sc);
    }
    mx = __builtin_elementwise_maximum(mx, swap_halves(mx));
    const float mref = (mx - m) * a.scale_log2 > RT_RESCALE<DT> || mx != mx ? mx : m;
    const float nm = mref == -INFINITY ? 0.f : RT_SHIFT<DT> - mref * a.scale_log2;
    if (__ballot(m != mref)) {
      const float alpha = m == mref ? 1.f : __builtin_amdgcn_exp2f((m - mref) * a.scale_log2);
      l *= alpha;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int v = 0; v < 16; ++v) acc[nb][v] *= alpha;
    }
    m = mref;
    __builtin_amdgcn_s_setprio(1);  // a wave at its products before one that stages (1 to 7 %)
    scores(sn, buf ^ 1);
    uint4 pk[4];  // block s of the tile: the B operand of its 16 tokens, the probabilities
    float least = INFINITY;  // fp16: hidden ones' zeros too, so that tiles which have some look for the rest of none
#pragma unroll
    for (int s4 = 0; s4 < 4; ++s4) {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int v = 8 * (s4 & 1) + 2 * i;
        const float p0 = __builtin_amdgcn_exp2f(fmaf(sc[s4 >> 1][v], a.scale_log2, nm));
        const float p1 = __builtin_amdgcn_exp2f(fmaf(sc[s4 >> 1][v + 1], a.scale_log2, nm));
        w[i] = tile::pack16x2<DT>(p0, p1);
        l = add_pair<DT>(w[i], l);
        if constexpr (HALF) {
          sc[s4 >> 1][v] = p0;
          sc[s4 >> 1][v + 1] = p1;
          least = fminf(least, fminf(p0, p1));
        }
      }
      pk[s4] = make_uint4(w[0], w[1], w[2], w[3]);
    }
    // kept so through the scheduler: operands read RT_AHEAD products ahead of their use, the vector
    // work of the probabilities among the scores' products, the next maximum's among the outputs'
    constexpr int QK = 2 * KS, PV = 4 * NB;
    auto order_scores = [&]() {
      __builtin_amdgcn_sched_group_barrier(0x100, RT_AHEAD, 0);
#pragma unroll
      for (int i = 0; i < QK; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x402, 96 / QK, 0);
      }
    };
    if constexpr (HALF) {
      order_scores();
      // What rounding took of probabilities below the normal numbers, in 2^38ths. Where V is not finite, a
      // positive one may not be 0, which would make NaN of an infinity: the least number is put in for it,
      // and taken off again where V is finite.
      if (__builtin_expect(__ballot(least < RT_LEAST_HALF) != 0, 0)) {
#pragma unroll
        for (int s4 = 0; s4 < 4; ++s4) {
          __builtin_amdgcn_sched_barrier(0);  // one operand at a time (registers)
          uint32_t z[4];
          uint32_t any = 0;
          auto word = [&](int i) -> uint32_t& {
            return i == 0 ? pk[s4].x : i == 1 ? pk[s4].y : i == 2 ? pk[s4].z : pk[s4].w;
          };
          auto p = [&](int i) { return sc[s4 >> 1][8 * (s4 & 1) + i]; };
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t w = word(i);
            auto left = [&](float x, uint32_t half) {
              return x < RT_LEAST_HALF ? (x - half_to_f32(uint16_t(half))) * RT_REST : 0.f;
            };
            z[i] = tile::pack16x2<DT>(left(p(2 * i), w), left(p(2 * i + 1), w >> 16));
            any |= z[i] & 0x7fff7fffu;
          }
          if (!__ballot(any != 0)) continue;
          bool odd = false;
          auto add = [&]() {
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
              __builtin_amdgcn_sched_barrier(0);
              f32x16_t t;
#pragma unroll
              for (int v = 0; v < 16; ++v) t[v] = 0.f;
              t = mfma32<DT>(vread(buf, nb, s4), make_uint4(z[0], z[1], z[2], z[3]), t);
#pragma unroll
              for (int v = 0; v < 16; ++v) {
                const bool fine = fabsf(t[v]) < INFINITY;
                odd |= !fine;
                acc[nb][v] += fine ? t[v] * (1.f / RT_REST) : 0.f;
              }
            }
          };
          add();
          if (__ballot(odd)) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint32_t& w = word(i);
              const uint32_t put = (p(2 * i) > 0.f && !(w & 0xffffu) ? 1u : 0u) |
                                   (p(2 * i + 1) > 0.f && !(w >> 16) ? 0x10000u : 0u);
              w |= put;
              z[i] = put * RT_PUT;
            }
            add();
          }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 4 * NB; ++i)
      acc[i % NB] = mfma32<DT>(vread(buf, i % NB, i / NB), pk[i / NB], acc[i % NB]);
    __builtin_amdgcn_s_setprio(0);
    mx = largest(sn);
    if constexpr (!HALF) order_scores();
#pragma unroll
    for (int i = 0; i < PV; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      if (i + RT_AHEAD < PV) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x402, RT_PV_VALU, 0);
    }
  };

  // K is staged two tiles ahead of the outputs, for scores are a tile ahead, V one. With two buffers
  // each, what a tile stages replaces what the tile before it has read, with a barrier between.
  const bool first4 = wave < 4;
  Part pa, pb;  // SPLIT: K or V in pa; else K in pa, V in pb
  int w0 = where(kt0), w1 = where(kt0 + 1), w2 = where(kt0 + 2), w3 = where(kt0 + 3);
  // K of tile it_k and V of the one before (with eight waves a wave has one of them)
  auto fetch = [&](int wk, int wv, int it_k) RT_INLINE {
    if constexpr (SPLIT) {
      if (first4) fetch_k(pa, wk, it_k);
      else fetch_v(pa, wv, it_k - 1);
    } else {
      fetch_k(pa, wk, it_k);
      fetch_v(pb, wv, it_k - 1);
    }
  };
  auto stage = [&](int buf_k, int buf_v, int it_v) RT_INLINE {
    if constexpr (SPLIT) {
      if (first4) stage_k(pa, buf_k);
      else stage_v(pa, buf_v, it_v, 0);
    } else {
      stage_k(pa, buf_k);
      stage_v(pb, buf_v, it_v, 0);
    }
  };
  {  // the first tile's K and V and the second's K, all on their way at once
    Part pc;
    fetch(w1, w0, kt0 + 1);
    if (!SPLIT || first4) fetch_k(pc, w0, kt0);
    __syncthreads();  // odd_seen is cleared
    stage(1, 0, kt0);
    if (!SPLIT || first4) stage_k(pc, 0);
  }
  fetch(w2, w1, kt0 + 2);
  __syncthreads();
  f32x16_t sa[2], sb[2];
  scores(sa, 0);
  float mx = largest(sa);
  __syncthreads();  // the first step stages K where these scores were read
  auto step = [&](f32x16_t (&sc)[2], f32x16_t (&sn)[2], int it, int buf) RT_INLINE {
    const int there = int(__ballot(lane < 4 && uint32_t(w0) < np)) & 0xf;
    const int w4 = where(it + 4);
    turn(sc, sn, mx, it, buf, there);
    stage(buf, buf ^ 1, it + 1);
    fetch(w3, w2, it + 3);
    __syncthreads();
    w0 = w1;
    w1 = w2;
    w2 = w3;
    w3 = w4;
  };
  for (int it = kt0; it < nkt; it += 2) {
    step(sa, sb, it, 0);
    if (it + 1 >= nkt) break;
    step(sb, sa, it + 1, 1);
  }

  if (odd_seen) {  // the same for every wave: all stores to it are barriers ago
#pragma unroll 1
    for (int it = kt0; it < nkt; ++it) {
      if (seen_whole(it)) continue;
      const int w = where(it);
      const int there = int(__ballot(lane < 4 && uint32_t(w) < np)) & 0xf;
      const Reach x = reach_of_row(it);
#pragma unroll 1
      for (int kind = 1; kind <= 3; ++kind) {
        __syncthreads();
        if (!SPLIT || !first4) {
          fetch_v(SPLIT ? pa : pb, w, it);
          stage_v(SPLIT ? pa : pb, 0, it, kind);
        }
        __syncthreads();
        const float z = kind == 1 ? __builtin_nanf("") : kind == 2 ? INFINITY : -INFINITY;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          f32x16_t hit;
#pragma unroll
          for (int v = 0; v < 16; ++v) hit[v] = 0.f;
#pragma unroll
          for (int s4 = 0; s4 < 4; ++s4) {
            __builtin_amdgcn_sched_barrier(0);  // one operand at a time (registers)
            const uint32_t bits = (there >> s4) & 1 ? bits8(x, 16 * s4 + 8 * hh) : 0u;
            uint32_t see[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
              see[i] = ((bits >> (2 * i)) & 1u ? ONE : 0u) | ((bits >> (2 * i)) & 2u ? ONE << 16 : 0u);
            hit = mfma32<DT>(vread(0, nb, s4), make_uint4(see[0], see[1], see[2], see[3]), hit);
          }
#pragma unroll
          for (int v = 0; v < 16; ++v)
            if (hit[v] > 0.f) acc[nb][v] += z;
        }
      }
    }
  }

  l += swap_halves(l);
  const Row own_row = row_now();
  if (!own_row.live) return;
  const int64_t at = (row0 + own_row.pos) * a.Hq + h * G + own_row.r % G, R = a.rows * a.Hq;
  if (a.dst) {  // the piece as it is, to be joined: its outputs, then its reference and sum
    float* o = a.dst + (piece * R + at) * D + 4 * hh;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (32 * nb + 8 * i < D)
          *reinterpret_cast<float4*>(o + 32 * nb + 8 * i) = make_float4(
              acc[nb][4 * i], acc[nb][4 * i + 1], acc[nb][4 * i + 2], acc[nb][4 * i + 3]);
    if (hh == 0)
      a.dst_ml[piece * R + at] =
          make_float2(m == -INFINITY ? m : m * a.scale_log2 - RT_SHIFT<DT>, l);
    return;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  uint16_t* o = static_cast<uint16_t*>(a.out) + at * D + 4 * hh;
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
__global__ __launch_bounds__(256) void reach_tiles_join_kernel(TileArgs a) {
  const int D = a.D;
  const int64_t x = a.first_row + int64_t(blockIdx.x) * 256 + threadIdx.x, R = a.rows * a.Hq;
  const int64_t at = x / (D / 4);
  const int d = 4 * int(x - at * (D / 4));
  const int64_t row = at / a.Hq;
  if (at >= R || row < a.cu[a.first] || row >= a.cu[a.first + a.count]) return;
  float M = -INFINITY, L = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  constexpr int N = 4;  // pieces on their way at once; past the end: the last again, without weight
  for (int p0 = 0; p0 < a.cuts; p0 += N) {
    float2 pm[N];
    float4 po[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int64_t i = min(p0 + k, a.cuts - 1) * R + at;
      pm[k] = a.dst_ml[i];
      po[k] = *reinterpret_cast<const float4*>(a.dst + i * D + d);
    }
#pragma unroll
    for (int k = 0; k < N; ++k) {
      if (p0 + k >= a.cuts) break;
      const float to = __builtin_elementwise_maximum(M, pm[k].x);
      const float f0 = reach::weight(M, to), f = reach::weight(pm[k].x, to);
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
void launch(const TileArgs& a, unsigned blocks, hipStream_t s) {
  hipLaunchKernelGGL((reach_tiles_kernel<DP, NW, DT>), dim3(blocks), dim3(64 * NW), 0, s, a);
}

}  // namespace

bool reach_tiles_shape(const Args& a, int dtype) {
  // scale > 0: the kernel keeps its references in units of the products
  return dtype != PIA_DTYPE_F32 && a.D <= 256 && a.scale_log2 > 0.f && a.G <= 128 &&
         (ceil_div(a.rows, 128 / a.G) + std::max(a.B, a.groups)) * a.Hkv <= RT_MAX_BLOCKS;
}

reach::TilePlan reach_tiles_plan(const Args& a, int64_t tokens, int64_t most) {
  const int64_t cus = device_cus(), tiles = ceil_div(tokens, RT_KT), n = a.by_group ? a.groups : a.B;
  auto items_of = [&](int rows) {
    return std::max<int64_t>(1, (ceil_div(a.rows, rows / a.G) + n / 2) * a.Hkv);
  };
  // Items of 256 rows, one on a CU, halve what is staged for a row, where there is work for 16 tiles on
  // every CU (8 x 1024 rows, window of 2048: 362 us, by 128 rows 398; 256 rows on a prefix of 32768: 213
  // for 235); else of 128 rows, two on a CU, of which one stages while the other starts.
  const int64_t items8 = items_of(256), items4 = items_of(128);
  const bool wide = a.D == 128 && a.G <= 128 && a.rows * a.G >= 192 * n && items8 * tiles >= 16 * cus;
  // Fewer items than CUs: their keys are cut into pieces, of 16 tiles at least, or of 4 to one on every CU
  const int64_t cuts =
      wide ? std::min(cus / items8, tiles / 16)
           : std::max(std::min(2 * cus / items4, tiles / 16), std::min(cus / items4, tiles / 4));
  return {wide, int(std::max<int64_t>(1, std::min(std::min<int64_t>(cuts, RT_MAX_CUTS), most)))};
}

int launch_reach_tiles(const Args& args, int dtype, reach::TilePlan plan, hipStream_t s) {
  TileArgs a;
  static_cast<Args&>(a) = args;
  const int cuts = a.cuts = plan.cuts;
  const bool wide = plan.wide;
  const int n = a.by_group ? a.groups : a.B;
  a.ppt = (wide ? 256 : 128) / a.G;
  const bool joined = cuts > 1 && !a.by_group;
  for (int b0 = 0; b0 < n; b0 += RT_MAX_SEQS) {
    a.first = b0;
    a.count = std::min(n - b0, RT_MAX_SEQS);
    const int64_t blocks =
        ceil_div((ceil_div(a.rows, a.ppt) + a.count) * cuts * a.Hkv, 8) * 8;
#define PIA_RT(DT)                                                 \
  {                                                                \
    if (wide) launch<128, 8, DT>(a, unsigned(blocks), s);          \
    else if (a.D > 128) launch<256, 4, DT>(a, unsigned(blocks), s); \
    else if (a.D > 96) launch<128, 4, DT>(a, unsigned(blocks), s); \
    else if (a.D > 64) launch<96, 4, DT>(a, unsigned(blocks), s);  \
    else launch<64, 4, DT>(a, unsigned(blocks), s);                \
  }
    if (dtype == PIA_DTYPE_F16) PIA_RT(PIA_DTYPE_F16) else PIA_RT(PIA_DTYPE_BF16)
#undef PIA_RT
    int rc = check_launch("reach_tiles");
    if (rc) return rc;
    if (joined) {
      const int64_t all = a.rows * a.Hq * (a.D / 4), part = int64_t(1) << 31;
      for (a.first_row = 0; a.first_row < all; a.first_row += part) {
        const dim3 grid{unsigned(ceil_div(std::min(part, all - a.first_row), 256)), 1u, 1u};
        if (dtype == PIA_DTYPE_F16)
          hipLaunchKernelGGL((reach_tiles_join_kernel<PIA_DTYPE_F16>), grid, dim3(256), 0, s, a);
        else
          hipLaunchKernelGGL((reach_tiles_join_kernel<PIA_DTYPE_BF16>), grid, dim3(256), 0, s, a);
        rc = check_launch("reach_tiles_join");
        if (rc) return rc;
      }
    }
  }
  return 0;
}

}  // namespace pia
