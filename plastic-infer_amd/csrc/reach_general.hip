// Windowed attention and attention behind a shared prefix for every shape: one wave for each row and q
// head, which walks the keys that the row sees, 64 at a time, and no others. All products and sums in fp32.
//
// QK: a lane has a key (tokens are innermost in the pool, so lanes read neighbours), q is in LDS. PV: a
// lane has elements lane + 64 i, the probabilities come from LDS. Nothing is shared between rows or heads, so it
// is bound by its loads of single elements, which every head of a group repeats (32 / 8 heads of 128, bf16, a window
// of 1024 over pages of 8 tokens: 64 single rows 636 us, 8 x 128 rows 6.8 ms; with pages of 16, which the faster
// kernels take, 49 and 42 us). It takes what they do not: head_dim over 256 or not in multiples of 16, pages not in
// multiples of 16, addresses that are not aligned to 16 bytes.
#include <algorithm>

#include "reach.h"

namespace pia {
namespace {

using reach::Args;

template <int DT, int ND>
__global__ __launch_bounds__(64) void reach_general_kernel(Args a) {
  using T = typename Elem<DT>::T;
  __shared__ float qs[64 * ND];
  __shared__ float ps[64];
  __shared__ int64_t at[64];  // of the chunk's keys: (page, head) tile and token, -1: no key
  const int lane = threadIdx.x;
  const unsigned r = blockIdx.x / unsigned(a.Hq);
  const int head = int(blockIdx.x - r * unsigned(a.Hq)), h = head / a.G;
  const int64_t row = a.first_row + r;
  int b = int(row);
  if (a.cu) {
    if (row < a.cu[0] || row >= a.cu[a.B]) return;
    int lo = 0, hi = a.B - 1;  // the last sequence that begins at or before the row
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (a.cu[mid] <= row) lo = mid; else hi = mid - 1;
    }
    b = lo;
  }
  const reach::Seq s = reach::sequence(a, b);
  const int pos = int(row - s.row0);
  if (pos < 0 || pos >= s.n) return;
  const T* qp = static_cast<const T*>(a.q) + row * a.q_stride + int64_t(head) * a.D;
  for (int d = lane; d < 64 * ND; d += 64) qs[d] = d < a.D ? Elem<DT>::load(qp, d) : 0.f;
  __syncthreads();

  float m = -INFINITY, l = 0.f, acc[ND];
#pragma unroll
  for (int i = 0; i < ND; ++i) acc[i] = 0.f;
  const int64_t tile = int64_t(a.D) * a.P;
  const T* kp = static_cast<const T*>(a.kp);
  const T* vp = static_cast<const T*>(a.vp);

  auto walk = [&](const int32_t* table, int from, int to) {
    for (int t0 = from; t0 < to; t0 += 64) {
      const int t = t0 + lane, n = min(64, to - t0);
      int64_t where = -1;
      if (lane < n) {
        const int id = table[t / a.P];
        if (id >= 0 && id < a.num_pages)
          where = (int64_t(id) * a.Hkv + h) * tile + t % a.P;
      }
      float sc = -INFINITY;
      if (where >= 0) {
        float x = 0.f;
        for (int d = 0; d < a.D; ++d) x = fmaf(qs[d], Elem<DT>::load(kp, where + int64_t(d) * a.P), x);
        sc = x * a.scale_log2;
      }
      const float mn = fmaxf(m, wave_max(sc));  // a NaN score makes its probability and the row NaN
      const float alpha = m == mn ? 1.f : __builtin_amdgcn_exp2f(m - mn);
      const float p = where < 0 ? 0.f : __builtin_amdgcn_exp2f(sc - (mn == -INFINITY ? 0.f : mn));
      m = mn;
      l = l * alpha + wave_sum(p);
      __syncthreads();
      ps[lane] = p;
      at[lane] = where;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < ND; ++i) acc[i] *= alpha;
      for (int k = 0; k < n; ++k) {
        const int64_t w = at[k];
        if (w < 0) continue;
        const float pk = ps[k];
#pragma unroll
        for (int i = 0; i < ND; ++i) {
          const int d = lane + 64 * i;
          if (d < a.D) acc[i] = fmaf(pk, Elem<DT>::load(vp, w + int64_t(d) * a.P), acc[i]);
        }
      }
    }
  };
  const int lim = reach::limit(s, pos), lo = reach::lowest(a, s, pos);
  const int g = reach::group_of(a, b);
  if (g >= 0) walk(a.pt + g * a.pt_stride, 0, reach::held(a.plens[g], a.pt_stride, a.P));
  const int32_t* own = a.bt + int64_t(b) * a.bt_stride;
  const int sinks = a.window ? min(a.sinks, lim) : 0;
  walk(own, 0, min(sinks, lo));
  walk(own, lo, lim);

  const float inv = l == 0.f ? 0.f : 1.f / l;
  T* o = static_cast<T*>(a.out) + (row * a.Hq + head) * a.D;
#pragma unroll
  for (int i = 0; i < ND; ++i) {
    const int d = lane + 64 * i;
    if (d < a.D) Elem<DT>::store(o, d, l == 0.f ? 0.f : acc[i] * inv);
  }
}

template <int DT>
int launch(Args a, hipStream_t s) {
  // parts of rows, so that a launch has fewer than 2^32 threads
  const int64_t most = std::max<int64_t>(1, (int64_t(1) << 25) / a.Hq);
  for (a.first_row = 0; a.first_row < a.rows; a.first_row += most) {
    const dim3 grid{unsigned(std::min(most, a.rows - a.first_row) * a.Hq), 1u, 1u};
    if (a.D <= 64) hipLaunchKernelGGL((reach_general_kernel<DT, 1>), grid, dim3(64), 0, s, a);
    else if (a.D <= 128) hipLaunchKernelGGL((reach_general_kernel<DT, 2>), grid, dim3(64), 0, s, a);
    else if (a.D <= 256) hipLaunchKernelGGL((reach_general_kernel<DT, 4>), grid, dim3(64), 0, s, a);
    else hipLaunchKernelGGL((reach_general_kernel<DT, 8>), grid, dim3(64), 0, s, a);
    const int rc = check_launch("reach_general");
    if (rc) return rc;
  }
  return 0;
}

}  // namespace

int launch_reach_general(const reach::Args& a, int dtype, hipStream_t s) {
  return dtype == PIA_DTYPE_F32   ? launch<PIA_DTYPE_F32>(a, s)
         : dtype == PIA_DTYPE_F16 ? launch<PIA_DTYPE_F16>(a, s)
                                  : launch<PIA_DTYPE_BF16>(a, s);
}

}  // namespace pia
