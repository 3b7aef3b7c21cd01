// Rotary positions: what the kernels that rotate share.
//
// Pair i of a head turns by angle 2 pi * position * turns[i], with turns[i] = frequency / 2 pi in
// fp64. The product is taken in fp64: in fp32 a position of 100000 would leave an error of 0.01
// turns in the fastest pair. So are cos and sin, from their Taylor series within an eighth of a turn
// of the nearest quarter (sin to x^9, cos to x^10: below 2e-9), which costs no more vector
// instructions than the fp32 functions and gives them to half a step of fp32. That matters where
// the result is rounded to 8 bits: two computations of it then differ as rarely as can be.
#pragma once

#include "pia_internal.h"

namespace pia {
namespace rope {

// (cos, sin) of a pair at a position, both times factor
__device__ __forceinline__ float2 cos_sin(double turns, int64_t pos, double factor) {
  double t = double(pos) * turns;
  t -= rint(t);
  const double quarter = rint(4.0 * t);
  const double x = fma(-0.25, quarter, t) * 6.283185307179586, y = x * x;
  double s = fma(y, 1.0 / 362880, -1.0 / 5040), c = fma(y, -1.0 / 3628800, 1.0 / 40320);
  s = fma(y, s, 1.0 / 120);
  c = fma(y, c, -1.0 / 720);
  s = fma(y, s, -1.0 / 6);
  c = fma(y, c, 1.0 / 24);
  s = fma(x * y, s, x);
  c = fma(y, c, -0.5);
  c = fma(y, c, 1.0);
  const int q = int(quarter);  // -2 .. 2: quarters of a turn, (c, s) -> (-s, c) each
  double u = (q & 1) ? -s : c, v = (q & 1) ? c : s;
  if (q & 2) {
    u = -u;
    v = -v;
  }
  return make_float2(float(u * factor), float(v * factor));
}

// x c + y s by one fused product: the same bits wherever a pair is turned (a c - b s is turn(a, -b)).
// The sum is held as an fp32 value: folded into its rounding to fp16, as the compiler does in some
// places, it would be rounded once there and twice elsewhere.
__device__ __forceinline__ float turn(float x, float y, float c, float s) {
  float r = fmaf(x, c, y * s);
  asm("" : "+v"(r));
  return r;
}

// x rounded to nearest even, by the instruction that does it (bf16: two elements at once; in integer
// arithmetic with a branch for NaN it is ten, and the rotation bound by them)
template <int DT>
__device__ __forceinline__ typename Elem<DT>::T narrow(float x) {
  if constexpr (DT == PIA_DTYPE_BF16) return __builtin_bit_cast(uint16_t, static_cast<__bf16>(x));
  else if constexpr (DT == PIA_DTYPE_F16) return f32_to_half(x);
  else return x;
}

// V consecutive elements of a 16- or 32-bit row as floats, by 16-byte vectors (VEC) or one by one
template <int DT, int V, bool VEC>
__device__ __forceinline__ void load(const typename Elem<DT>::T* p, float (&x)[V]) {
  using T = typename Elem<DT>::T;
  if constexpr (VEC) {
    constexpr int W = V * int(sizeof(T)) < 16 ? V * int(sizeof(T)) : 16;
    struct alignas(W) Pack {
      T v[W / sizeof(T)];
    };
#pragma unroll
    for (int i = 0; i < V; i += W / int(sizeof(T))) {
      const Pack a = *reinterpret_cast<const Pack*>(p + i);
#pragma unroll
      for (int j = 0; j < W / int(sizeof(T)); ++j) x[i + j] = Elem<DT>::load(a.v, j);
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = Elem<DT>::load(p, i);
  }
}
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
// stream: past the caches' usual order, for results larger than they are
template <int DT, int V, bool VEC>
__device__ __forceinline__ void store(typename Elem<DT>::T* p, const float (&x)[V],
                                      bool stream = false) {
  using T = typename Elem<DT>::T;
  if constexpr (VEC) {
    constexpr int W = V * int(sizeof(T)) < 16 ? V * int(sizeof(T)) : 16;
    struct alignas(W) Pack {
      T v[W / sizeof(T)];
    };
#pragma unroll
    for (int i = 0; i < V; i += W / int(sizeof(T))) {
      Pack a;
#pragma unroll
      for (int j = 0; j < W / int(sizeof(T)); ++j) a.v[j] = narrow<DT>(x[i + j]);
      if constexpr (W == 16) {
        if (stream) {
          __builtin_nontemporal_store(__builtin_bit_cast(u32x4_t, a),
                                      reinterpret_cast<u32x4_t*>(p + i));
          continue;
        }
      }
      *reinterpret_cast<Pack*>(p + i) = a;
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) p[i] = narrow<DT>(x[i]);
  }
}

// Units of a head: what one thread turns (or copies) at a time. Half layout: V elements and their V
// partners; interleaved: V elements, V / 2 pairs; behind the rotated part: V elements copied. VEC:
// V elements are a 16-byte vector; else V = 1 (half), 2 (interleaved).
template <int DT, bool INTER, bool VEC>
struct Units {
  using T = typename Elem<DT>::T;
  static constexpr int V = VEC ? 16 / int(sizeof(T)) : INTER ? 2 : 1;
  __host__ __device__ static int turned(int pairs) { return INTER ? 2 * pairs / V : pairs / V; }
  __host__ __device__ static int count(int pairs, int D) {
    return turned(pairs) + (D - 2 * pairs + V - 1) / V;
  }
  // unit u of the head at x into the head at o; tab: the token's (cos, sin) of every pair
  __device__ __forceinline__ static void run(T* o, const T* x, int u, const float2* tab, int pairs,
                                             int D, float sin_sign, bool stream) {
    const int nt = turned(pairs);
    if (u >= nt) {
      const int d = 2 * pairs + (u - nt) * V;
      if (!VEC && d + V > D) {  // an odd element at the end
        o[d] = x[d];
        return;
      }
      float a[V];
      load<DT, V, VEC>(x + d, a);
      store<DT, V, VEC>(o + d, a, stream);
      return;
    }
    float a[V];
    load<DT, V, VEC>(x + u * V, a);
    if constexpr (INTER) {
      float r[V];
#pragma unroll
      for (int i = 0; i < V; i += 2) {
        const float2 cs = tab[(u * V + i) / 2];
        const float s = cs.y * sin_sign;
        r[i] = turn(a[i], -a[i + 1], cs.x, s);
        r[i + 1] = turn(a[i + 1], a[i], cs.x, s);
      }
      store<DT, V, VEC>(o + u * V, r, stream);
    } else {
      float b[V], r0[V], r1[V];
      load<DT, V, VEC>(x + pairs + u * V, b);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float2 cs = tab[u * V + i];
        const float s = cs.y * sin_sign;
        r0[i] = turn(a[i], -b[i], cs.x, s);
        r1[i] = turn(b[i], a[i], cs.x, s);
      }
      store<DT, V, VEC>(o + u * V, r0, stream);
      store<DT, V, VEC>(o + pairs + u * V, r1, stream);
    }
  }
};

// Results from this size on are stored past the caches' usual order: the L2s together hold 32 MB
constexpr int64_t kStreamBytes = int64_t(32) << 20;

// Whether a head's units are whole vectors at every stride (elements; bytes for the pointers)
inline bool vectors(int elem, bool inter, int pairs, int D, const void* a, const void* b,
                    int64_t s0, int64_t s1) {
  const int v = 16 / elem;
  return (inter ? 2 * pairs : pairs) % v == 0 && (D - 2 * pairs) % v == 0 && D % v == 0 &&
         s0 % v == 0 && s1 % v == 0 && aligned(a, 16) && aligned(b, 16);
}

}  // namespace rope
}  // namespace pia
