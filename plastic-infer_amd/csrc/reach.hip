// Entry points of windowed attention and of attention behind a shared prefix: checks of the arguments
// and the choice of a kernel.
#include <algorithm>

#include "reach.h"

namespace pia {
namespace {

// Whether `out` (bytes) holds any byte of n rows of `row` bytes, `stride` bytes apart from q on
bool holds_rows(uintptr_t out, int64_t bytes, uintptr_t q, int64_t n, int64_t row, int64_t stride) {
  if (stride <= 0) n = 1;
  // the first row that ends behind out's beginning
  const int64_t to = int64_t(out) - int64_t(q) - row;
  const int64_t r = to < 0 || n == 1 ? 0 : to / stride + 1;
  const int64_t from = int64_t(q) + r * stride;
  return r < n && from < int64_t(out) + bytes && from + row > int64_t(out);
}

int elem_bytes(int dtype) { return dtype == PIA_DTYPE_F32 ? 4 : 2; }

// What both entry points ask of their arguments; 0: the call can run, 1: there is nothing to do
int check(const reach::Args& a, int dtype, const char* name) {
  if (dtype != PIA_DTYPE_F32 && dtype != PIA_DTYPE_F16 && dtype != PIA_DTYPE_BF16) {
    set_error("%s: dtype must be bf16, fp16 or fp32", name);
    return PIA_EUNSUPPORTED;
  }
  auto bad = [&](const char* what) {
    set_error("%s: %s", name, what);
    return PIA_EINVAL;
  };
  if (a.B < 0 || a.rows < 0 || a.Hq <= 0 || a.Hkv <= 0 || a.num_pages <= 0 || a.bt_stride < 0 ||
      a.D <= 0 || a.P <= 0)
    return bad("invalid size");
  if (a.Hq % a.Hkv) return bad("num_heads % num_kv_heads != 0");
  if (a.D > 512 || a.P > 4096) {
    set_error("%s: head_dim to 512 and page_size to 4096", name);
    return PIA_EUNSUPPORTED;
  }
  if (!a.cu && a.rows != a.B) return bad("without cu_q one row per sequence");
  if (a.B == 0 || a.rows == 0) return 1;
  if (a.num_pages > 0x7fffffff || a.num_pages * a.Hkv > 0x7fffffff || a.rows > 0x3fffffff ||
      a.rows * a.Hq > 0x7ffffff0)
    return bad("pool or rows too large");
  if (!a.out || !a.q || !a.kp || !a.vp || !a.lens || (a.bt_stride && !a.bt))
    return bad("null pointer");
  const int e = elem_bytes(dtype);
  const int64_t row = int64_t(a.Hq) * a.D * e;
  // every row is read before it is written, by whoever writes it, but not before others are
  if (!(a.out == a.q && a.q_stride * e == row) &&
      holds_rows(uintptr_t(a.out), a.rows * row, uintptr_t(a.q), a.rows, row, a.q_stride * e))
    return bad("out overlaps q");
  return 0;
}

}  // namespace
}  // namespace pia

using namespace pia;

extern "C" int64_t pia_window_attention_workspace_bytes(int head_dim) { return 0; }

extern "C" int pia_window_attention(void* out, const void* q, int64_t q_stride, const void* k_pages,
                                    const void* v_pages, const int32_t* block_tables,
                                    int64_t bt_stride, const int32_t* kv_lens, const int32_t* cu_q,
                                    const int32_t* q_pos_offsets, int window, int sinks,
                                    int num_seqs, int64_t total_q_rows, int num_heads,
                                    int num_kv_heads, int head_dim, int page_size,
                                    int64_t num_pages, float scale, int dtype, void* workspace,
                                    int64_t workspace_bytes, void* stream) {
  if (window <= 0 || sinks < 0)
    return fail(PIA_EINVAL, "window_attention: window must be positive and sinks not negative");
  const reach::Args a{out, q, q_stride, k_pages, v_pages, block_tables, bt_stride, kv_lens, cu_q,
                      q_pos_offsets, total_q_rows, num_pages, 0, scale * 1.4426950408889634f, num_seqs,
                      num_heads, num_kv_heads, num_kv_heads > 0 ? num_heads / num_kv_heads : 0,
                      head_dim, page_size, window, sinks, nullptr, 0, nullptr, nullptr, 0};
  const int rc = check(a, dtype, "window_attention");
  if (rc) return rc < 0 ? rc : 0;
  return launch_reach_general(a, dtype, as_stream(stream));
}

extern "C" int64_t pia_prefix_attention_workspace_bytes(int64_t total_q_rows, int num_heads,
                                                        int head_dim) {
  return 0;
}

extern "C" int pia_prefix_attention(void* out, const void* q, int64_t q_stride, const void* k_pages,
                                    const void* v_pages, const int32_t* prefix_tables,
                                    int64_t pt_stride, const int32_t* prefix_lens,
                                    const int32_t* cu_seqs, int num_groups,
                                    const int32_t* block_tables, int64_t bt_stride,
                                    const int32_t* kv_lens, const int32_t* cu_q,
                                    const int32_t* q_pos_offsets, int num_seqs,
                                    int64_t total_q_rows, int num_heads, int num_kv_heads,
                                    int head_dim, int page_size, int64_t num_pages, float scale,
                                    int dtype, void* workspace, int64_t workspace_bytes,
                                    void* stream) {
  if (num_groups < 0 || pt_stride < 0)
    return fail(PIA_EINVAL, "prefix_attention: invalid size");
  if (!cu_seqs && num_groups > 1)
    return fail(PIA_EINVAL, "prefix_attention: without cu_seqs one group");
  const bool some = num_groups > 0 && pt_stride > 0;
  if (some && (!prefix_tables || !prefix_lens))
    return fail(PIA_EINVAL, "prefix_attention: null pointer");
  const reach::Args a{out, q, q_stride, k_pages, v_pages, block_tables, bt_stride, kv_lens, cu_q,
                      q_pos_offsets, total_q_rows, num_pages, 0, scale * 1.4426950408889634f, num_seqs,
                      num_heads, num_kv_heads, num_kv_heads > 0 ? num_heads / num_kv_heads : 0,
                      head_dim, page_size, 0, 0, some ? prefix_tables : nullptr, pt_stride,
                      prefix_lens, cu_seqs, some ? num_groups : 0};
  const int rc = check(a, dtype, "prefix_attention");
  if (rc) return rc < 0 ? rc : 0;
  return launch_reach_general(a, dtype, as_stream(stream));
}
