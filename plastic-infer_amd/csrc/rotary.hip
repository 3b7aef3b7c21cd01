// Rotary positions of q and k: rotate-half or interleaved pairs, in the whole head or its first part,
// from frequencies in fp64 (any scaling of them is the caller's), forward and transposed.
//
//   (a, b) -> (a c - b s, b c + a s), c = factor cos(2 pi p f), s = factor sin(2 pi p f)
//
// With several axes (time, height, width of images and video) a token has a position on each, and p is
// that of the pair's own axis: only the table of (cos, sin) differs, by two loads for each of its entries (64
// tokens, 32 + 4 heads of 128, three axes: 3.5 us, one axis 3.0; 8192 tokens, 32 + 8 heads: 30 us, 5.6 TB/s).
//
// The transposed map (the gradient's) is the same with s negated. Bound by HBM: every element is read
// and written once. A workgroup takes a few tokens, computes their (cos, sin) into LDS once for all
// heads of q and k, and then streams the heads in 16-byte vectors; fp32 arithmetic, one rounding. 8192
// tokens of 32 + 8 heads of 128, bf16: 29 to 35 us, 4.8 to 5.8 TB/s (40 us with ordinary stores).
#include <algorithm>

#include "rope.h"

namespace pia {
namespace {

constexpr int RT_THREADS = 256;
constexpr int RT_MAX_PAIRS = 2048;

struct RotaryArgs {
  void *q_out, *k_out;
  const void *q, *k;
  int64_t q_tok, q_head, k_tok, k_head;
  const void* positions;
  const int32_t* axes;  // several axes: the axis of each pair, positions [num_axes, tokens]
  const double* turns;
  int64_t tokens;
  int num_axes, wide, pairs, Hq, Hkv, D, per_wg, stream;
  double factor;
  float sin_sign;
};

template <int DT, bool INTER, bool VEC, bool AXES>
__global__ __launch_bounds__(RT_THREADS) void rotary_kernel(RotaryArgs a) {
  using T = typename Elem<DT>::T;
  using U = rope::Units<DT, INTER, VEC>;
  extern __shared__ float2 tab[];
  const int64_t t0 = int64_t(blockIdx.x) * a.per_wg;
  const int nt = int(min(int64_t(a.per_wg), a.tokens - t0));
  for (int i = threadIdx.x; i < nt * a.pairs; i += RT_THREADS) {
    const int t = i / a.pairs, p = i - t * a.pairs;
    int64_t at = t0 + t;
    bool there = true;
    if constexpr (AXES) {
      const int axis = a.axes[p];
      there = axis >= 0 && axis < a.num_axes;
      at += (there ? axis : 0) * a.tokens;
    }
    int64_t pos = a.wide ? static_cast<const int64_t*>(a.positions)[at]
                         : int64_t(static_cast<const int32_t*>(a.positions)[at]);
    if (AXES && !there) pos = 0;
    tab[i] = rope::cos_sin(a.turns[p], pos, a.factor);
  }
  __syncthreads();
  const unsigned per_head = U::count(a.pairs, a.D), H = a.Hq + a.Hkv;
  const unsigned per_tok = per_head * H, total = per_tok * nt;
  for (unsigned i = blockIdx.y * RT_THREADS + threadIdx.x; i < total;
       i += gridDim.y * RT_THREADS) {
    const unsigned t = i / per_tok, r = i - t * per_tok, hh = r / per_head;
    const int h = int(hh), u = int(r - hh * per_head);
    const int64_t tok = t0 + t;
    const T* x;
    T* o;
    if (h < a.Hq) {
      x = static_cast<const T*>(a.q) + tok * a.q_tok + h * a.q_head;
      o = static_cast<T*>(a.q_out) + (tok * a.Hq + h) * a.D;
    } else {
      x = static_cast<const T*>(a.k) + tok * a.k_tok + (h - a.Hq) * a.k_head;
      o = static_cast<T*>(a.k_out) + (tok * a.Hkv + h - a.Hq) * a.D;
    }
    U::run(o, x, u, tab + t * a.pairs, a.pairs, a.D, a.sin_sign, a.stream != 0);
  }
}

int rotate(void* q_out, void* k_out, const void* q, const void* k, int64_t q_token_stride,
           int64_t q_head_stride, int64_t k_token_stride, int64_t k_head_stride,
           const void* positions, int positions_i64, const int32_t* axes, int num_axes,
           const double* turns, int pairs, double factor, int interleaved, int transposed,
           int64_t num_tokens, int num_heads, int num_kv_heads, int head_dim, int dtype,
           void* stream) {
  if (dtype != PIA_DTYPE_F32 && dtype != PIA_DTYPE_F16 && dtype != PIA_DTYPE_BF16)
    return fail(PIA_EUNSUPPORTED, "rotary: dtype must be bf16, fp16 or fp32");
  if (num_tokens < 0 || num_heads < 0 || num_kv_heads < 0 || head_dim <= 0 || pairs < 0 ||
      2 * int64_t(pairs) > head_dim)
    return fail(PIA_EINVAL, "rotary: invalid size");
  if (pairs > RT_MAX_PAIRS) return fail(PIA_EUNSUPPORTED, "rotary: more than 4096 rotated elements");
  const int64_t H = int64_t(num_heads) + num_kv_heads;
  if (num_tokens == 0 || H == 0) return 0;
  if (H * head_dim > (1 << 24) || num_tokens > 0x7fffffff)
    return fail(PIA_EINVAL, "rotary: too many heads or tokens");
  if ((num_heads && (!q || !q_out)) || (num_kv_heads && (!k || !k_out)) || !positions ||
      (pairs && !turns))
    return fail(PIA_EINVAL, "rotary: null pointer");
  const int elem = dtype == PIA_DTYPE_F32 ? 4 : 2;
  const bool inter = interleaved != 0;
  const bool vec =
      (!num_heads || rope::vectors(elem, inter, pairs, head_dim, q, q_out, q_token_stride,
                                   q_head_stride)) &&
      (!num_kv_heads || rope::vectors(elem, inter, pairs, head_dim, k, k_out, k_token_stride,
                                      k_head_stride));
  RotaryArgs a{q_out, k_out, q, k, q_token_stride, q_head_stride, k_token_stride, k_head_stride,
               positions, axes, turns, num_tokens, num_axes, positions_i64 != 0, pairs, num_heads, num_kv_heads,
               head_dim, 1, num_tokens * H * head_dim * elem >= rope::kStreamBytes, factor,
               transposed ? -1.f : 1.f};
  // tokens of a workgroup: one, or four where that still leaves four workgroups
  // for every compute unit (and the table 32 KiB)
  a.per_wg = num_tokens >= 16 * int64_t(device_cus()) ? 4 : 1;
  if (int64_t(a.per_wg) * pairs > 4096) a.per_wg = 1;
  // few tokens: their heads over several workgroups, two vectors for each thread
  const int64_t bytes = H * head_dim * elem;
  const int gy = num_tokens < device_cus()
                     ? int(std::min<int64_t>(8, ceil_div(bytes, 32 * RT_THREADS))) : 1;
  const dim3 grid{unsigned(ceil_div(num_tokens, a.per_wg)), unsigned(gy), 1u};
  const size_t lds = sizeof(float2) * size_t(a.per_wg) * size_t(pairs);
  hipStream_t s = as_stream(stream);
#define PIA_RT(DT, I, V)                                                                      \
  if (axes)                                                                                   \
    hipLaunchKernelGGL((rotary_kernel<DT, I, V, true>), grid, dim3(RT_THREADS), lds, s, a);   \
  else                                                                                        \
    hipLaunchKernelGGL((rotary_kernel<DT, I, V, false>), grid, dim3(RT_THREADS), lds, s, a)
#define PIA_RT_D(DT)                                                   \
  if (inter) {                                                         \
    if (vec) { PIA_RT(DT, true, true); } else { PIA_RT(DT, true, false); }     \
  } else {                                                             \
    if (vec) { PIA_RT(DT, false, true); } else { PIA_RT(DT, false, false); }   \
  }
  if (dtype == PIA_DTYPE_F32) {
    PIA_RT_D(PIA_DTYPE_F32)
  } else if (dtype == PIA_DTYPE_F16) {
    PIA_RT_D(PIA_DTYPE_F16)
  } else {
    PIA_RT_D(PIA_DTYPE_BF16)
  }
#undef PIA_RT_D
#undef PIA_RT
  return check_launch("rotary");
}

}  // namespace
}  // namespace pia

using namespace pia;

extern "C" int pia_rotary(void* q_out, void* k_out, const void* q, const void* k,
                          int64_t q_token_stride, int64_t q_head_stride, int64_t k_token_stride,
                          int64_t k_head_stride, const void* positions, int positions_i64,
                          const double* turns, int pairs, double factor, int interleaved,
                          int transposed, int64_t num_tokens, int num_heads, int num_kv_heads,
                          int head_dim, int dtype, void* stream) {
  return rotate(q_out, k_out, q, k, q_token_stride, q_head_stride, k_token_stride, k_head_stride,
                positions, positions_i64, nullptr, 1, turns, pairs, factor, interleaved, transposed,
                num_tokens, num_heads, num_kv_heads, head_dim, dtype, stream);
}

extern "C" int pia_rotary_axes(void* q_out, void* k_out, const void* q, const void* k,
                               int64_t q_token_stride, int64_t q_head_stride,
                               int64_t k_token_stride, int64_t k_head_stride,
                               const void* positions, int positions_i64, const int32_t* axes,
                               int num_axes, const double* turns, int pairs, double factor,
                               int interleaved, int transposed, int64_t num_tokens, int num_heads,
                               int num_kv_heads, int head_dim, int dtype, void* stream) {
  if (num_axes <= 0) return fail(PIA_EINVAL, "rotary: invalid number of axes");
  if (pairs > 0 && num_tokens > 0 && !axes) return fail(PIA_EINVAL, "rotary: null pointer");
  return rotate(q_out, k_out, q, k, q_token_stride, q_head_stride, k_token_stride, k_head_stride,
                positions, positions_i64, pairs > 0 ? axes : nullptr, num_axes, turns, pairs, factor,
                interleaved, transposed, num_tokens, num_heads, num_kv_heads, head_dim, dtype, stream);
}
