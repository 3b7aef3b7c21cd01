// The 8-bit KV pool: e4m3 codes and one power-of-two scale for every block of 16 tokens of a head.
//
//   K codes [num_pages, Hkv, D / 16, P, 16]   a token's 16 elements together, tokens next to each
//                                             other: the operand of K . q^T, whose lanes are tokens
//   V codes [num_pages, Hkv, P / 4, D, 4]     an element's 4 tokens together: the operand of P . V,
//                                             whose lanes hold 4 tokens of each block
//   scales  fp32 [num_pages, Hkv, P / 16]
//
// A block of either pool is 16 D bytes; a wave loads it in whole 256-byte runs straight into matrix
// operands, with no transposing and no LDS. With scales that are powers of two a code times its
// scale is exact in bf16, and a block whose scale grows keeps its codes' digits: only the exponent
// moves (but for codes that fall below 2^-6 of the new scale, which keep 2^-9 of it).
#pragma once

#include "pia_internal.h"

namespace pia {
namespace kv8 {

constexpr int BLOCK = 16;
constexpr float LARGEST = 448.f;

// The smallest power of two whose multiple by 448 = 1.75 * 2^8 is at least bound (finite, >= 0),
// within 2^-100 .. 2^119.
__device__ __forceinline__ float scale_of(float bound) {
  const uint32_t u = __float_as_uint(bound);
  // exponent field of bound / 2^8, one more where its mantissa is over 1.75 (denormals: the least)
  const int e = int(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return __uint_as_float(uint32_t(min(max(e, 27), 246)) << 23);
}

// Four values times inv (the inverse of a scale) as the e4m3 codes of a word, nearest even. A scale holds
// its values within 448, so nothing is clipped; NaN and infinities become the NaN code, and so would
// a finite value beyond 464 (only the largest fp32 values are, over a scale of 2^119).
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d, float inv) {
  const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(a * inv, b * inv, 0, false);
  return uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(c * inv, d * inv, lo, true));
}
__device__ __forceinline__ void decode4(uint32_t w, float (&x)[4]) {
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(int(w), false);
  const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(int(w), true);
  x[0] = lo[0];
  x[1] = lo[1];
  x[2] = hi[0];
  x[3] = hi[1];
}
// two codes (the low or high half of a word) times scale as two 16-bit values of type T
template <int T, bool HI>
__device__ __forceinline__ uint32_t widen(uint32_t w, float scale) {
  if constexpr (T == PIA_DTYPE_F16)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, HI));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, HI));
}
template <int T>
__device__ __forceinline__ uint4 widen8(uint32_t a, uint32_t b, float scale = 1.f) {
  return make_uint4(widen<T, false>(a, scale), widen<T, true>(a, scale),
                    widen<T, false>(b, scale), widen<T, true>(b, scale));
}
// the bytes of a word of codes that hold the NaN code, as 1 each
__device__ __forceinline__ uint32_t nan_codes(uint32_t w) {
  return (((w & 0x7f7f7f7fu) + 0x01010101u) >> 7) & 0x01010101u;
}
// a word's codes times ratio (a power of two, at most 1), rounded to codes again
__device__ __forceinline__ uint32_t rescale4(uint32_t w, float ratio) {
  float x[4];
  decode4(w, x);
  return encode4(x[0], x[1], x[2], x[3], ratio);
}

// 1 / a scale that scale_of gave (a power of two within 2^-100 .. 2^119): exact
__device__ __forceinline__ float inverse(float scale) {
  return __uint_as_float((254u << 23) - __float_as_uint(scale));
}

// Multi-row attention on tiles in LDS (kv8_prefill.hip): whether a call takes it, and its launch
// (arguments already checked by pia_kv8_attention).
}  // namespace kv8
bool kv8_prefill_path(int dtype, int Hq, int Hkv, int D, int num_seqs, int64_t total_q_rows,
                      const int32_t* cu_q, float scale);
int launch_kv8_prefill(int dtype, void* out, const void* q, int64_t q_stride, const uint8_t* kp,
                       const uint8_t* vp, const float* ks, const float* vs, const int32_t* bt,
                       int64_t bt_stride, const int32_t* lens, const int32_t* cu,
                       const int32_t* offs, int num_seqs, int64_t total_q_rows, int Hq, int Hkv,
                       int D, int P, int64_t num_pages, float scale_log2, float* parts,
                       int64_t part_rows, hipStream_t s);
namespace kv8 {

// The last of n numbers base(0) <= base(1) <= ... that is at or before id (the first where none is): 64
// of them at once, one a lane; base reads what it needs. id is the same in all lanes.
template <class Base>
__device__ __forceinline__ int last_at(int n, int64_t id, Base base) {
  const int lane = threadIdx.x & 63;
  int lo = 0;
  while (n > 1) {
    const int step = (n + 63) >> 6, at = lane * step;
    const uint64_t in = __ballot(at < n && base(lo + at) <= id);
    const int last = in ? 63 - __builtin_clzll(in) : 0;
    lo += last * step;
    n = min(step, n - last * step);
  }
  return lo;
}

// Keys that row `pos` of a sequence sees of the first `keys`, with its first row at position off (any int)
__device__ __forceinline__ int seen(int keys, int off, int pos) {
  return int(max(int64_t(0), min(int64_t(keys), int64_t(off) + pos + 1)));
}

inline bool pool_shape(int D, int P) {
  return D > 0 && D % 16 == 0 && D <= 256 && P > 0 && P % BLOCK == 0 && P <= 4096;
}

}  // namespace kv8
}  // namespace pia
