// Appending a batch's new tokens to a paged cache with the rotary positions applied on the way, into
// pools of the model's type or 8-bit ones, and reading contexts back from the 8-bit pool.
//
// Rows cu_new[b] .. cu_new[b + 1] of q, k and v are the last tokens of sequence b, whose context_lens
// counts them; a token's position is its place in the context. q is rotated into q_out, k rotated
// into its slot, v copied into its slot.
//
// The unit of work is an aligned block of 16 positions of one sequence: one wave then sees all the new
// tokens that share an 8-bit scale. Some workgroups rotate a block's q heads, others take four of its
// K and V heads, one a wave, so that a single token's chain of loads is as short as it can be; each
// computes the (cos, sin) of its tokens once. Blocks are numbered without a scan: sequence b's start at
// cu_new[b] / 16 + 2 b, which leaves room for every block that its rows can touch. Bound by HBM for
// prompts (each element once) and by latency for single tokens.
//
// Measured, 8 prompts: 4964 tokens of 16 + 8 heads of 128, bf16 pool: 21.5 us, 3.8 TB/s; 10000 tokens of
// 32 + 8 heads, fp16, 8-bit pool: 47 us, 4.7 TB/s (a large copy of this card: 5.2). 256 single tokens
// of 32 + 8 heads, 8-bit pool: 7.4 us.
#include <algorithm>
#include <cmath>

#include "kv8.h"
#include "rope.h"

namespace pia {
namespace {

constexpr int KA_THREADS = 256;
constexpr int KA_WAVES = KA_THREADS / 64;

// bytes of a wave's tile: 16 tokens of 128 elements
template <int DT>
constexpr int KA_TILE = 16 * 128 * int(sizeof(typename Elem<DT>::T));

struct AppendArgs {
  void* q_out;
  const void *q, *k, *v;
  int64_t q_tok, q_head, k_tok, k_head, v_tok, v_head;
  void *k_pages, *v_pages;
  float *k_scale, *v_scale;
  const int32_t* bt;
  int64_t bt_stride;
  const int32_t *lens, *cu;
  int64_t num_tokens;
  const double* turns;
  int64_t num_pages;
  int num_seqs, pairs, inter, Hq, Hkv, D, P;
  double factor;
  float k_bound;
  int k_vec, v_vec, k_pair, v_pair, whole, q_shares, stream;
};

// N consecutive elements as they are, in words; VEC: p is a vector of them (16 bytes at most)
template <int DT, int N>
struct Raw {
  using T = typename Elem<DT>::T;
  static constexpr int PER = 4 / int(sizeof(T)), W = N / PER;  // elements of a word, words
  uint32_t w[W];
  __device__ __forceinline__ void load(const T* p, bool vec) {
    if (vec) {
      if constexpr (W >= 4) {
#pragma unroll
        for (int i = 0; i < W; i += 4) {
          const uint4 x = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint32_t*>(p) + i);
          w[i] = x.x;
          w[i + 1] = x.y;
          w[i + 2] = x.z;
          w[i + 3] = x.w;
        }
      } else {
        const uint2 x = *reinterpret_cast<const uint2*>(p);
        w[0] = x.x;
        w[1] = x.y;
      }
    } else {
#pragma unroll
      for (int i = 0; i < W; ++i) {
        if constexpr (PER == 2) w[i] = uint32_t(p[2 * i]) | uint32_t(p[2 * i + 1]) << 16;
        else w[i] = __float_as_uint(p[i]);
      }
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < W; ++i) w[i] = 0;
  }
  __device__ __forceinline__ float at(int e) const {
    if constexpr (DT == PIA_DTYPE_F32) return __uint_as_float(w[e]);
    else if constexpr (DT == PIA_DTYPE_BF16) return (e & 1) ? bf16_hi(w[e / 2]) : bf16_lo(w[e / 2]);
    else return half_to_f32(uint16_t((e & 1) ? w[e / 2] >> 16 : w[e / 2]));
  }
  // most (magnitudes as whole numbers, in halves of a word for 16-bit types) with these elements
  __device__ __forceinline__ uint32_t larger(uint32_t most) const {
    typedef unsigned short u16x2_t __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int i = 0; i < W; ++i) {
      if constexpr (PER == 2)
        most = __builtin_bit_cast(
            uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2_t, most),
                                                __builtin_bit_cast(u16x2_t, w[i] & 0x7fff7fffu)));
      else
        most = max(most, w[i] & 0x7fffffffu);
    }
    return most;
  }
  // the largest finite magnitude
  __device__ __forceinline__ float finite(float most) const {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float x = fabsf(at(e));
      most = fmaxf(most, x < INFINITY ? x : 0.f);
    }
    return most;
  }
};

// The wave's largest finite magnitude: of whole numbers first, and only if that is not finite one
// element after the other.
template <int DT, int N, int C>
__device__ __forceinline__ float largest(const Raw<DT, N> (&x)[C]) {
  uint32_t most = 0;
#pragma unroll
  for (int i = 0; i < C; ++i) most = x[i].larger(most);
  if constexpr (Raw<DT, N>::PER == 2) most = max(most & 0xffffu, most >> 16);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) most = max(most, uint32_t(__shfl_xor(int(most), o, 64)));
  float r = DT == PIA_DTYPE_F32 ? __uint_as_float(most)
            : DT == PIA_DTYPE_BF16 ? bf16_to_f32(uint16_t(most)) : half_to_f32(uint16_t(most));
  if (r < INFINITY) return r;
  r = 0.f;
#pragma unroll
  for (int i = 0; i < C; ++i) r = x[i].finite(r);
  return wave_max(r);
}

// The K codes of one (block, kv head) of the 8-bit pool by one wave: lane (t, g) has token t's
// elements 16 c .. 16 c + 15 for c = g, g + 4, ... (NC of them). o0: the block's offset of its first
// new token, n: how many; r0: their first row; was: the block's scale, 0 where it holds no earlier
// tokens.
template <int DT, int NC>
__device__ __forceinline__ void append8_k(const AppendArgs& a, const float2* tab, int tab_row, int h,
                                          int64_t r0, int o0, int n, int64_t head, int sub,
                                          float was) {
  using T = typename Elem<DT>::T;
  const int lane = threadIdx.x & 63, D = a.D, P = a.P, rd = 2 * a.pairs;
  const int t = lane & 15, g = lane >> 4;
  const bool fresh = t >= o0 && t < o0 + n, old = t < o0;
  const T* x = static_cast<const T*>(a.k) + (r0 + (fresh ? t - o0 : 0)) * a.k_tok + h * a.k_head;
  uint4* codes =
      reinterpret_cast<uint4*>(static_cast<uint8_t*>(a.k_pages) + head * D * P) + sub * 16 + t;
  Raw<DT, 16> v[NC];
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int c = g + 4 * i;
    if (fresh && 16 * c < D) v[i].load(x + 16 * c, a.k_vec);
    else v[i].zero();
  }
  const float now = fmaxf(was, kv8::scale_of(largest(v) * a.k_bound));
  const float inv = kv8::inverse(now), ratio = was * inv;
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int c = g + 4 * i;
    if (16 * c >= D) continue;
    if (fresh) {
      float r[16];
      const float2* cs = tab + (t - o0) * tab_row;
      if (16 * c >= rd) {
#pragma unroll
        for (int e = 0; e < 16; ++e) r[e] = v[i].at(e);
      } else if (a.inter) {
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
          const float v0 = v[i].at(e), v1 = v[i].at(e + 1);
          const bool in = 16 * c + e < rd;
          const float2 f = in ? cs[8 * c + e / 2] : make_float2(1.f, 0.f);
          r[e] = in ? rope::turn(v0, -v1, f.x, f.y) : v0;
          r[e + 1] = in ? rope::turn(v1, v0, f.x, f.y) : v1;
        }
      } else if (a.pairs % 16 == 0) {
        const bool first = 16 * c < a.pairs;
        const int other = first ? 16 * c + a.pairs : 16 * c - a.pairs;
        const float sign = first ? -1.f : 1.f;
        // the partners: in this lane where they are 64 or 128 elements on, else from the cache
        Raw<DT, 16> p;
        if (NC >= 2 && a.pairs == 64) p = v[i ^ (NC >= 2 ? 1 : 0)];
        else if (NC == 4 && a.pairs == 128) p = v[i ^ (NC == 4 ? 2 : 0)];
        else p.load(x + other, a.k_vec);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float2 f = cs[(first ? 16 * c : other) + e];
          r[e] = rope::turn(v[i].at(e), sign * p.at(e), f.x, f.y);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int d = 16 * c + e;
          r[e] = v[i].at(e);
          if (d < rd) {
            const bool first = d < a.pairs;
            const float2 f = cs[first ? d : d - a.pairs];
            const float p = Elem<DT>::load(x, first ? d + a.pairs : d - a.pairs);
            r[e] = rope::turn(r[e], first ? -p : p, f.x, f.y);
          }
        }
      }
      codes[c * P] = make_uint4(kv8::encode4(r[0], r[1], r[2], r[3], inv),
                                kv8::encode4(r[4], r[5], r[6], r[7], inv),
                                kv8::encode4(r[8], r[9], r[10], r[11], inv),
                                kv8::encode4(r[12], r[13], r[14], r[15], inv));
    } else if (old && now != was) {
      uint4 w = codes[c * P];
      w.x = kv8::rescale4(w.x, ratio);
      w.y = kv8::rescale4(w.y, ratio);
      w.z = kv8::rescale4(w.z, ratio);
      w.w = kv8::rescale4(w.w, ratio);
      codes[c * P] = w;
    }
  }
  if (lane == 0) a.k_scale[head * (P / 16) + sub] = now;
}

// Its V codes: lane (x, tg) has elements 64 i + 4 x .. + 3 of tokens 4 tg .. 4 tg + 3, one word of codes
// for each element; a word that also holds earlier or stale tokens keeps theirs.
template <int DT, int NC>
__device__ __forceinline__ void append8_v(const AppendArgs& a, int h, int64_t r0, int o0, int n,
                                          int64_t head, int sub, float was) {
  using T = typename Elem<DT>::T;
  const int lane = threadIdx.x & 63, D = a.D, P = a.P;
  const int x4 = (lane & 15) * 4, t0 = (lane >> 4) * 4;
  uint4* codes = reinterpret_cast<uint4*>(static_cast<uint8_t*>(a.v_pages) + head * D * P +
                                          (sub * 4 + (lane >> 4)) * 4 * D);
  Raw<DT, 4> v[4 * NC];
#pragma unroll
  for (int i = 0; i < NC; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int t = t0 + j, d = 64 * i + x4;
      if (d < D && t >= o0 && t < o0 + n)
        v[4 * i + j].load(
            static_cast<const T*>(a.v) + (r0 + t - o0) * a.v_tok + h * a.v_head + d, a.v_vec);
      else
        v[4 * i + j].zero();
    }
  // bytes of a word: new tokens, and earlier ones that the scale moves
  uint32_t fresh = 0, old = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int t = t0 + j;
    fresh |= t >= o0 && t < o0 + n ? 0xffu << (8 * j) : 0u;
    old |= t < o0 ? 0xffu << (8 * j) : 0u;
  }
  // codes that share their words with new ones: on their way while the scale is found
  const bool part = (fresh | old) != 0 && fresh != 0xffffffffu;
  uint4 before[NC];
#pragma unroll
  for (int i = 0; i < NC; ++i)
    if (part && 64 * i + x4 < D) before[i] = codes[(64 * i + x4) / 4];
  const float now = fmaxf(was, kv8::scale_of(largest(v)));
  const float inv = kv8::inverse(now), ratio = was * inv;
  const bool moved = old != 0 && now != was;
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    if (64 * i + x4 >= D || (fresh == 0 && !moved)) continue;
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e)
      w[e] = kv8::encode4(v[4 * i].at(e), v[4 * i + 1].at(e), v[4 * i + 2].at(e),
                          v[4 * i + 3].at(e), inv);
    if (part) {
      const uint32_t was4[4] = {before[i].x, before[i].y, before[i].z, before[i].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        uint32_t b = was4[e];
        if (moved) b = (kv8::rescale4(b, ratio) & old) | (b & ~old);
        w[e] = (w[e] & fresh) | (b & ~fresh);
      }
    }
    codes[(64 * i + x4) / 4] = make_uint4(w[0], w[1], w[2], w[3]);
  }
  if (lane == 0) a.v_scale[head * (P / 16) + sub] = now;
}

// K (which = 0) or V of one (block, kv head) of a pool of the model's type by one wave: a lane has
// E consecutive elements of the block's n tokens (NT at most; all loads go out before any is used, those
// past n are the last token's again). A whole block goes out in the pool's order, 16 bytes a lane and
// a KB of consecutive ones a store, through a tile in LDS (K and V of 5000 tokens, 8 heads of 128 in
// bf16: 20 us, and 22 straight from the lanes that have them, 64 bytes apart); of others each element
// goes to its place. Token by token, with a page looked up and a row loaded for each, a prompt's
// ragged ends took longer than all its blocks: the same call is 12.5 us, 3.3 TB/s, without.
template <int DT, int E, int NT>
__device__ __forceinline__ void append_plain(const AppendArgs& a, const float2* tab, int tab_row,
                                             int which, int h, int64_t r0, int64_t p0, int n,
                                             const int32_t* row, unsigned char* tile) {
  using T = typename Elem<DT>::T;
  constexpr int TV = 16 / int(sizeof(T)), N = 2 * 16 / TV;
  const int lane = threadIdx.x & 63, D = a.D, P = a.P, rd = which ? 0 : 2 * a.pairs;
  const int64_t tok = which ? a.v_tok : a.k_tok;
  const T* x = static_cast<const T*>(which ? a.v : a.k) + r0 * tok + h * (which ? a.v_head : a.k_head);
  T* pool = static_cast<T*>(which ? a.v_pages : a.k_pages);
  struct alignas(E * sizeof(T)) Part {
    T v[E];
  };
  struct alignas(16) Pack {
    T x[TV];
  };
  // lane t: where token t's first element goes, -1 where its page is not in the pool
  int64_t to = -1;
  if (lane < n) {
    const uint32_t pos = uint32_t(p0 + lane), slot = pos / uint32_t(P);
    const int32_t page = row[slot];
    if (uint32_t(page) < uint64_t(a.num_pages))
      to = (int64_t(page) * a.Hkv + h) * D * P + (pos - slot * uint32_t(P));
  }
  auto to_of = [&](int t) {
    return int64_t(uint64_t(uint32_t(__builtin_amdgcn_readlane(int(to >> 32), t))) << 32 |
                   uint32_t(__builtin_amdgcn_readlane(int(to), t)));
  };
  for (int d0 = 0; d0 < D; d0 += 64 * E) {
    const bool in = d0 + E * lane < D;
    const int d = in ? d0 + E * lane : 0;
    const bool turned = d < rd, first = a.inter ? !(d & 1) : d < a.pairs;
    const int od = a.inter ? (E == 2 ? d : d ^ 1) : first ? d + a.pairs : d - a.pairs;
    Part own[NT], other[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
      own[t] = *reinterpret_cast<const Part*>(x + min(t, n - 1) * tok + d);
    if (turned && !(E == 2 && a.inter)) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
        other[t] = *reinterpret_cast<const Part*>(x + min(t, n - 1) * tok + od);
    }
    if (turned && E == 2 && a.inter) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const float2 f = tab[t * tab_row + d / 2];
        const float v0 = Elem<DT>::load(own[t].v, 0), v1 = Elem<DT>::load(own[t].v, E - 1);
        own[t].v[0] = rope::narrow<DT>(rope::turn(v0, -v1, f.x, f.y));
        own[t].v[E - 1] = rope::narrow<DT>(rope::turn(v1, v0, f.x, f.y));
      }
    } else if (turned) {
      const float2* cs = tab + (a.inter ? d >> 1 : first ? d : od);
      const float sign = first ? -1.f : 1.f;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float2 f = cs[t * tab_row + e];
          own[t].v[e] = rope::narrow<DT>(rope::turn(Elem<DT>::load(own[t].v, e),
                                                    sign * Elem<DT>::load(other[t].v, e), f.x, f.y));
        }
    }
    if constexpr (E == 2 && NT == 16) {
      if (n == 16 && a.whole) {
        const int64_t base = to_of(0);  // one page: P is a multiple of 16
        if (base < 0) return;
        // 16-byte units of the tile, in the pool's order; a lane writes N of them in a row. The order
        // within N is XORed so that eight lanes' units fall into different banks either way (K and V
        // alone count no conflict; those of the whole call, 6 cycles to an instruction, are of q's
        // lanes, which read 32 or 64 bytes of the table each).
        auto place = [&](int u) {
          return reinterpret_cast<Pack*>(tile) + ((u & ~(N - 1)) | ((u ^ (u >> 3)) & (N - 1)));
        };
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int i = 0; i < 16 / TV; ++i) {
            Pack o;
#pragma unroll
            for (int j = 0; j < TV; ++j) o.x[j] = own[TV * i + j].v[e];
            *place(N * lane + e * (16 / TV) + i) = o;
          }
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int u = lane + 64 * i, at = d0 + u / (16 / TV);
          if (at < D)
            reinterpret_cast<Pack*>(pool + base + int64_t(at) * P)[u % (16 / TV)] = *place(u);
        }
        __builtin_amdgcn_wave_barrier();
        continue;
      }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int64_t base = t < n ? to_of(t) : -1;
      if (base < 0 || !in) continue;
#pragma unroll
      for (int e = 0; e < E; ++e) pool[base + int64_t(d + e) * P] = own[t].v[e];
    }
  }
}

template <int DT, bool INTER, bool VEC>
__device__ __forceinline__ void turn_q(const AppendArgs& a, const float2* tab, int tab_row,
                                       int64_t r0, int n, int h0, int h1) {
  using T = typename Elem<DT>::T;
  using U = rope::Units<DT, INTER, VEC>;
  const unsigned per_head = U::count(a.pairs, a.D), per_tok = per_head * (h1 - h0);
  for (unsigned i = threadIdx.x; i < per_tok * n; i += KA_THREADS) {
    const unsigned t = i / per_tok, r = i - t * per_tok, hh = r / per_head;
    const int h = h0 + int(hh);
    const T* x = static_cast<const T*>(a.q) + (r0 + t) * a.q_tok + h * a.q_head;
    T* o = static_cast<T*>(a.q_out) + ((r0 + t) * a.Hq + h) * a.D;
    U::run(o, x, int(r - hh * per_head), tab + t * tab_row, a.pairs, a.D, 1.f,
           a.stream != 0);
  }
}

// NC: 64-element parts of an 8-bit pool's head; 0: pools of the model's type
template <int DT, int NC, bool QVEC>
__global__ __launch_bounds__(KA_THREADS) void kv_append_kernel(AppendArgs a) {
  extern __shared__ float2 tab[];
  int64_t id = blockIdx.x;
  int b = int(id), row_lo = int(id), n_b = 1;
  if (a.cu) {
    b = kv8::last_at(a.num_seqs, id, [&](int i) { return (a.cu[i] >> 4) + int64_t(2) * i; });
    row_lo = a.cu[b];
    n_b = a.cu[b + 1] - row_lo;
    id -= (row_lo >> 4) + int64_t(2) * b;
  } else {
    id = 0;
  }
  // the block's new tokens: positions p0 .. p0 + n - 1, rows r0 ..
  const int64_t end = a.lens[b], start = end - n_b;
  const int64_t blk = (start >> 4) + id;
  const int64_t p0 = max(start, blk * 16);
  const int64_t r0 = row_lo + (p0 - start);
  const int n = int(min(min(end, blk * 16 + 16) - p0, a.num_tokens - r0));
  if (n <= 0 || row_lo < 0 || id < 0) return;
  const int y = blockIdx.y, wave = threadIdx.x >> 6;
  const bool for_q = y < a.q_shares;
  // keys and values: what a wave needs of tables and scales is on its way before the angles
  const uint32_t slot = uint32_t(max(p0, int64_t(0))) / uint32_t(a.P);
  const bool slots = !for_q && p0 >= 0 && slot < a.bt_stride;  // else no position has one
  const int32_t* row = a.bt + b * a.bt_stride;
  // K heads first, in workgroups of their own: those of V need no angles
  const int k_shares = (a.Hkv + KA_WAVES - 1) / KA_WAVES;
  const int which = !for_q && y - a.q_shares >= k_shares;
  const int h = (y - a.q_shares - (which ? k_shares : 0)) * KA_WAVES + wave;
  int64_t head = -1;
  float was = 0.f;
  const int sub = int(uint32_t(p0) - slot * uint32_t(a.P)) >> 4, o0 = int(p0 & 15);
  if constexpr (NC > 0) {
    if (slots && h < a.Hkv) {
      const int32_t page = row[slot];
      if (uint32_t(page) < uint64_t(a.num_pages)) {
        head = int64_t(page) * a.Hkv + h;
        if (o0 > 0) was = (which ? a.v_scale : a.k_scale)[head * (a.P / 16) + sub];
      }
    }
  }
  // a row of the table more than the pairs: 16 tokens' entries of one pair then sit in 16 banks
  const int tab_row = a.pairs + 1;
  if (for_q || !which) {
    for (int i = threadIdx.x; i < n * a.pairs; i += KA_THREADS) {
      const int t = i / a.pairs, p = i - t * a.pairs;
      tab[t * tab_row + p] = rope::cos_sin(a.turns[p], p0 + t, a.factor);
    }
    __syncthreads();
  }
  if (for_q) {
    const int h0 = int(int64_t(a.Hq) * y / a.q_shares);
    const int h1 = int(int64_t(a.Hq) * (y + 1) / a.q_shares);
    if (a.inter) turn_q<DT, true, QVEC>(a, tab, tab_row, r0, n, h0, h1);
    else turn_q<DT, false, QVEC>(a, tab, tab_row, r0, n, h0, h1);
    return;
  }
  if (!slots || h >= a.Hkv) return;
  const int m = int(min(int64_t(n), a.bt_stride * a.P - p0));
  if constexpr (NC > 0) {
    if (head < 0) return;
    if (which) append8_v<DT, NC>(a, h, r0, o0, m, head, sub, was);
    else append8_k<DT, NC>(a, tab, tab_row, h, r0, o0, m, head, sub, was);
  } else {
    unsigned char* tile = reinterpret_cast<unsigned char*>(tab + 16 * tab_row) + wave * KA_TILE<DT>;
    const bool two = which ? a.v_pair : a.k_pair;
    if (m == 1) {
      if (two) append_plain<DT, 2, 1>(a, tab, tab_row, which, h, r0, p0, m, row, tile);
      else append_plain<DT, 1, 1>(a, tab, tab_row, which, h, r0, p0, m, row, tile);
    } else {
      if (two) append_plain<DT, 2, 16>(a, tab, tab_row, which, h, r0, p0, m, row, tile);
      else append_plain<DT, 1, 16>(a, tab, tab_row, which, h, r0, p0, m, row, tile);
    }
  }
}

// Contexts of the 8-bit pool in logical order: one wave for each (block of 16 tokens, kv head). The
// codes come in whole 256-byte runs, become values, and leave as whole rows: through LDS, because
// the runs hold pieces of many rows, and lines that are written in pieces cost a third more. Measured:
// 16 contexts of 512 to 8192 tokens, 8 heads of 128, to bf16: 88 us, 4.9 TB/s.
template <int DT>
__global__ __launch_bounds__(256) void kv8_gather_kernel(
    typename Elem<DT>::T* __restrict__ k_out, typename Elem<DT>::T* __restrict__ v_out,
    const uint8_t* __restrict__ k_pages, const uint8_t* __restrict__ v_pages,
    const float* __restrict__ k_scale, const float* __restrict__ v_scale,
    const int32_t* __restrict__ bt, int64_t bt_stride, const int64_t* __restrict__ cu, int num_seqs,
    int64_t total, int Hkv, int D, int P, int64_t num_pages, int stream) {
  using T = typename Elem<DT>::T;
  extern __shared__ __align__(16) unsigned char rows_lds[];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t w = blockIdx.x * (blockDim.x >> 6) + wave;  // 32-bit quotients: the long ones took longer
  const uint32_t id = w / uint32_t(Hkv);                     // than the copy
  const int h = int(w - id * Hkv);
  const int b = kv8::last_at(num_seqs, id, [&](int i) { return (cu[i] >> 4) + i; });
  const int64_t first = cu[b], blk = id - ((first >> 4) + b);
  const int64_t len = min(cu[b + 1], total) - first;
  const int64_t n64 = min(len, bt_stride * P) - blk * 16;
  if (n64 <= 0 || first < 0 || blk < 0) return;
  const int n = int(min(n64, int64_t(16)));
  const uint32_t slot = uint32_t(blk) / uint32_t(P / 16);
  const int sub = int(uint32_t(blk) - slot * uint32_t(P / 16));
  const int32_t page = bt[b * bt_stride + slot];
  const bool ok = uint32_t(page) < uint64_t(num_pages);
  const int64_t head = int64_t(ok ? page : 0) * Hkv + h;
  const int64_t row0 = first + blk * 16;
  const int t = lane & 15, g = lane >> 4;
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
  // a row of the tile: D elements and 16 bytes, which spreads neighbouring rows over the banks
  const int pitch = D * int(sizeof(T)) + 16, parts = D * int(sizeof(T)) / 16;
  unsigned char* tile = rows_lds + wave * 16 * pitch;
  uint4 kx[4], vx[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    kx[i] = vx[i] = zero;
    const int c = g + 4 * i, d = 64 * i + 4 * t;
    if (ok && 16 * c < D)
      kx[i] = reinterpret_cast<const uint4*>(k_pages + head * D * P)[c * P + sub * 16 + t];
    if (ok && d < D)
      vx[i] = reinterpret_cast<const uint4*>(v_pages + head * D * P + (sub * 4 + g) * 4 * D)[d / 4];
  }
  const float ks = ok ? k_scale[head * (P / 16) + sub] : 0.f;
  const float vs = ok ? v_scale[head * (P / 16) + sub] : 0.f;
  auto leave = [&](T* out) {
    for (int u = lane; u < n * parts; u += 64) {
      const int r = u / parts, p = u - r * parts;
      const auto x = *reinterpret_cast<const rope::u32x4_t*>(tile + r * pitch + 16 * p);
      auto* to = reinterpret_cast<rope::u32x4_t*>(out + ((row0 + r) * Hkv + h) * D) + p;
      if (stream) __builtin_nontemporal_store(x, to);
      else *to = x;
    }
  };
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = g + 4 * i;
    if (16 * c < D) {
      const uint32_t q[4] = {kx[i].x, kx[i].y, kx[i].z, kx[i].w};
      float r[16];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float f[4];
        kv8::decode4(q[e], f);
#pragma unroll
        for (int j = 0; j < 4; ++j) r[4 * e + j] = f[j] * ks;
      }
      rope::store<DT, 16, true>(reinterpret_cast<T*>(tile + t * pitch) + 16 * c, r);
    }
  }
  __builtin_amdgcn_wave_barrier();  // one wave's LDS operations are done in order
  leave(k_out);
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int d = 64 * i + 4 * t;
    if (d < D) {
      float f[4][4];
      kv8::decode4(vx[i].x, f[0]);
      kv8::decode4(vx[i].y, f[1]);
      kv8::decode4(vx[i].z, f[2]);
      kv8::decode4(vx[i].w, f[3]);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float r[4] = {f[0][j] * vs, f[1][j] * vs, f[2][j] * vs, f[3][j] * vs};
        rope::store<DT, 4, true>(reinterpret_cast<T*>(tile + (4 * g + j) * pitch) + d, r);
      }
    }
  }
  __builtin_amdgcn_wave_barrier();
  leave(v_out);
}

}  // namespace
}  // namespace pia

using namespace pia;

extern "C" int pia_kv_append(void* q_out, const void* q, int64_t q_token_stride,
                             int64_t q_head_stride, const void* k, int64_t k_token_stride,
                             int64_t k_head_stride, const void* v, int64_t v_token_stride,
                             int64_t v_head_stride, void* k_pages, void* v_pages, float* k_scales,
                             float* v_scales, const int32_t* block_tables, int64_t bt_stride,
                             const int32_t* context_lens, const int32_t* cu_new,
                             int64_t num_tokens, int num_seqs, const double* turns, int pairs,
                             double factor, int interleaved, int num_heads, int num_kv_heads,
                             int head_dim, int page_size, int64_t num_pages, int dtype,
                             void* stream) {
  if (dtype != PIA_DTYPE_F32 && dtype != PIA_DTYPE_F16 && dtype != PIA_DTYPE_BF16)
    return fail(PIA_EUNSUPPORTED, "kv_append: dtype must be bf16, fp16 or fp32");
  if (num_tokens < 0 || num_seqs < 0 || num_heads < 0 || num_kv_heads <= 0 || head_dim <= 0 ||
      page_size <= 0 || num_pages < 0 || num_pages > 0x7fffffff || bt_stride < 0 || pairs < 0 ||
      2 * int64_t(pairs) > head_dim)
    return fail(PIA_EINVAL, "kv_append: invalid size");
  if (head_dim > 512) return fail(PIA_EUNSUPPORTED, "kv_append: head_dim over 512");
  const bool kv8 = k_scales != nullptr;
  if (kv8 != (v_scales != nullptr)) return fail(PIA_EINVAL, "kv_append: one scale array of two");
  if (kv8 && !kv8::pool_shape(head_dim, page_size))
    return fail(PIA_EUNSUPPORTED,
                "kv_append: 8-bit pools take head_dim and page_size in multiples of 16, up to 256 "
                "and 4096");
  if (num_tokens > 0x7fffffff || int64_t(num_heads) * head_dim > (1 << 24))
    return fail(PIA_EINVAL, "kv_append: too many tokens or heads");
  if (!cu_new && num_tokens != num_seqs)
    return fail(PIA_EINVAL, "kv_append: without cu_new one token per sequence");
  if (num_tokens == 0 || num_seqs == 0) return 0;
  if (!k || !v || !k_pages || !v_pages || !context_lens || (bt_stride && !block_tables) ||
      (pairs && !turns) || !q != !q_out)
    return fail(PIA_EINVAL, "kv_append: null pointer");
  const int elem = dtype == PIA_DTYPE_F32 ? 4 : 2;
  const bool inter = interleaved != 0;
  if (kv8 && (!aligned(k_pages, 16) || !aligned(v_pages, 16) || !aligned(k_scales, 4) ||
              !aligned(v_scales, 4)))
    return fail(PIA_EINVAL, "kv_append: pools must be 16-byte aligned");
  const int64_t v16 = 16 / elem;
  // c: a rotated element is at most sqrt(2) times the factor's size times the head's largest element
  const float bound = pairs ? float(1.4142135623730951 * std::abs(factor)) : 1.f;
  AppendArgs a{q_out, q, k, v, q_token_stride, q_head_stride, k_token_stride, k_head_stride,
               v_token_stride, v_head_stride, k_pages, v_pages, k_scales, v_scales, block_tables,
               bt_stride, context_lens, cu_new, num_tokens, turns, num_pages, num_seqs, pairs,
               interleaved != 0, q ? num_heads : 0, num_kv_heads, head_dim, page_size, factor,
               bound};
  a.k_vec = aligned(k, 16) && k_token_stride % v16 == 0 && k_head_stride % v16 == 0;
  a.whole = page_size % 16 == 0 && aligned(k_pages, 16) && aligned(v_pages, 16);
  a.v_vec = aligned(v, 4 * elem) && v_token_stride % 4 == 0 && v_head_stride % 4 == 0;
  a.k_pair = pairs % 2 == 0 && head_dim % 2 == 0 && aligned(k, 2 * elem) &&
             k_token_stride % 2 == 0 && k_head_stride % 2 == 0;
  a.v_pair = head_dim % 2 == 0 && aligned(v, 2 * elem) && v_token_stride % 2 == 0 &&
             v_head_stride % 2 == 0;
  const bool qvec = q && rope::vectors(elem, inter, pairs, head_dim, q, q_out, q_token_stride,
                                       q_head_stride);
  const int64_t blocks = cu_new ? num_tokens / 16 + 2 * int64_t(num_seqs) : num_seqs;
  if (blocks > 0x7fffffff) return fail(PIA_EINVAL, "kv_append: too many sequences");
  // Workgroups of a block: some for q, about four vectors for each thread, and one for every four of
  // the K and V heads, a wave each. Each computes the table of its tokens.
  const int per_wg = KA_THREADS * 4 * (qvec ? int(v16) : 1) * (inter ? 1 : 2);
  a.q_shares = a.Hq ? int(std::min<int64_t>(
      a.Hq, ceil_div(int64_t(cu_new ? 16 : 1) * a.Hq * head_dim, per_wg))) : 0;
  const int64_t shares = a.q_shares + 2 * ceil_div(int64_t(num_kv_heads), KA_WAVES);
  a.stream = num_tokens * a.Hq * head_dim * elem >= rope::kStreamBytes;
  if (shares > 65535) return fail(PIA_EINVAL, "kv_append: too many heads");
  const dim3 grid{unsigned(blocks), unsigned(shares), 1u};
  size_t lds = sizeof(float2) * size_t(cu_new ? 16 : 1) * size_t(pairs + 1);
  if (cu_new && !kv8 && a.whole) {  // and the tiles, if a launch may have that much (pairs to 255)
    const size_t tiles = size_t(KA_WAVES) * 16 * 128 * elem;
    if (lds + tiles <= 65536) lds += tiles;
    else a.whole = 0;
  }
  hipStream_t s = as_stream(stream);
#define PIA_KA(DT, NC, QV) \
  hipLaunchKernelGGL((kv_append_kernel<DT, NC, QV>), grid, dim3(KA_THREADS), lds, s, a)
#define PIA_KA_Q(DT, NC) \
  if (qvec) PIA_KA(DT, NC, true); else PIA_KA(DT, NC, false)
#define PIA_KA_D(DT)                           \
  if (!kv8) {                                  \
    PIA_KA_Q(DT, 0);                           \
  } else if (head_dim <= 64) {                 \
    PIA_KA_Q(DT, 1);                           \
  } else if (head_dim <= 128) {                \
    PIA_KA_Q(DT, 2);                           \
  } else {                                     \
    PIA_KA_Q(DT, 4);                           \
  }
  if (dtype == PIA_DTYPE_F32) {
    PIA_KA_D(PIA_DTYPE_F32)
  } else if (dtype == PIA_DTYPE_F16) {
    PIA_KA_D(PIA_DTYPE_F16)
  } else {
    PIA_KA_D(PIA_DTYPE_BF16)
  }
#undef PIA_KA_D
#undef PIA_KA_Q
#undef PIA_KA
  return check_launch("kv_append");
}

extern "C" int pia_kv8_gather(void* k_out, void* v_out, const void* k_pages, const void* v_pages,
                              const float* k_scales, const float* v_scales,
                              const int32_t* block_tables, int64_t bt_stride,
                              const int64_t* cu_seqlens, int num_seqs, int64_t total_tokens,
                              int num_kv_heads, int head_dim, int page_size, int64_t num_pages,
                              int dtype, void* stream) {
  if (dtype != PIA_DTYPE_F32 && dtype != PIA_DTYPE_F16 && dtype != PIA_DTYPE_BF16)
    return fail(PIA_EUNSUPPORTED, "kv8_gather: dtype must be bf16, fp16 or fp32");
  if (num_seqs < 0 || total_tokens < 0 || num_kv_heads <= 0 || num_pages <= 0 ||
      num_pages > 0x7fffffff || bt_stride < 0)
    return fail(PIA_EINVAL, "kv8_gather: invalid size");
  if (!kv8::pool_shape(head_dim, page_size))
    return fail(PIA_EUNSUPPORTED,
                "kv8_gather: head_dim and page_size in multiples of 16, up to 256 and 4096");
  if (num_seqs == 0 || total_tokens == 0 || bt_stride == 0) return 0;
  if (!k_out || !v_out || !k_pages || !v_pages || !k_scales || !v_scales || !block_tables ||
      !cu_seqlens)
    return fail(PIA_EINVAL, "kv8_gather: null pointer");
  if (!aligned(k_out, 16) || !aligned(v_out, 16) || !aligned(k_pages, 16) || !aligned(v_pages, 16))
    return fail(PIA_EINVAL, "kv8_gather: pools and outputs must be 16-byte aligned");
  const int64_t waves = (total_tokens / 16 + num_seqs) * int64_t(num_kv_heads);
  if (waves > 0x7fffffff) return fail(PIA_EINVAL, "kv8_gather: too many tokens");
  const int elem = dtype == PIA_DTYPE_F32 ? 4 : 2;
  const size_t tile = size_t(16) * (size_t(head_dim) * elem + 16);
  const int per_wg = tile > 16384 ? 2 : 4;  // waves; their tiles stay within 64 KB
  const size_t lds = per_wg * tile;
  const int64_t wgs = ceil_div(waves, per_wg);
  hipStream_t s = as_stream(stream);
  const int stream_out =
      2 * total_tokens * num_kv_heads * head_dim * elem >= rope::kStreamBytes;
#define PIA_KG(DT)                                                                              \
  hipLaunchKernelGGL((kv8_gather_kernel<DT>), dim3(unsigned(wgs)), dim3(64 * per_wg), lds, s,   \
                     static_cast<Elem<DT>::T*>(k_out), static_cast<Elem<DT>::T*>(v_out),        \
                     static_cast<const uint8_t*>(k_pages), static_cast<const uint8_t*>(v_pages), \
                     k_scales, v_scales, block_tables, bt_stride, cu_seqlens, num_seqs,         \
                     total_tokens, num_kv_heads, head_dim, page_size, num_pages, stream_out)
  if (dtype == PIA_DTYPE_F32) PIA_KG(PIA_DTYPE_F32);
  else if (dtype == PIA_DTYPE_F16) PIA_KG(PIA_DTYPE_F16);
  else PIA_KG(PIA_DTYPE_BF16);
#undef PIA_KG
  return check_launch("kv8_gather");
}
