// Entry points of windowed attention and of attention behind a shared prefix: checks of the arguments
// and the choice of a kernel.
#include <algorithm>
#include <atomic>
#include <random>

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

// (position, head) rows of a kv head and sequence (group) from which tiles in LDS take the call: a tile's 128
// rows cost the same however few there are, the streaming kernel reads K and V again for every 16. 8 sequences of
// 4096 tokens, 32 / 8 heads of 128, us (tiles, streaming): 32 rows 44 and 39, 64 rows 42 and 68.
constexpr int64_t TILE_ROWS = 64;
// the same for windows where there are sequences' heads for half of the compute units: 64 sequences of 2048
// tokens, 24 rows 105 and 181 (window of 64: 17 and 45). One number for every head_dim: with heads of 64 streaming
// is ahead at 16 rows (60 and 56), with heads of 128 it is not (111 and 135, which such calls pay).
constexpr int64_t TILE_ROWS_MANY = 24;
// (position, head) rows whose pieces a workspace has room for at least: 128 pieces of 128 rows and 4 heads
constexpr int64_t PREFIX_ROWS = 65536;

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

int check_workspace(const void* ws, int64_t bytes, int64_t need, const char* name) {
  if (need == 0) return 0;
  if (!ws || bytes < need || !aligned(ws, 16)) {
    set_error("%s: workspace missing, too small or not 16-byte aligned", name);
    return PIA_EINVAL;
  }
  return 0;
}
// Whether the streaming kernel takes a call; what it does not is the general kernel's
bool streams(const reach::Args& a, int dtype) {
  const int64_t e = elem_bytes(dtype);
  return a.D % 16 == 0 && a.D <= 256 && a.P % 16 == 0 && aligned(a.q, 16) && aligned(a.out, 16) &&
         a.q_stride * e % 16 == 0 && aligned(a.kp, 16) && aligned(a.vp, 16) &&
         // workgroups of the joining kernel
         ((a.rows * a.G >> 4) + a.B + a.groups + 2) * a.Hkv < (1 << 25);
}
int stream_call(const reach::Args& a, int dtype, int64_t tokens, hipStream_t s) {
  return dtype == PIA_DTYPE_F32   ? launch_reach_stream_f32(a, tokens, s)
         : dtype == PIA_DTYPE_F16 ? launch_reach_stream_f16(a, tokens, s)
                                  : launch_reach_stream_bf16(a, tokens, s);
}
// A workspace: the streaming kernel's numbers, its pieces by wave, and (prefix) pieces of rows
void place(reach::Args& a, void* workspace) {
  char* p = static_cast<char*>(workspace);
  a.pref = reinterpret_cast<int64_t*>(p);
  a.parts = reinterpret_cast<float*>(p + reach_stream_pref_bytes());
}
int64_t piece_bytes(int64_t rows, int Hq, int D) {  // of one piece of all rows
  return rows * Hq * (D + 2) * int64_t(sizeof(float));
}
// Room for pieces of the prefix and one of the rest: two of all rows, or as many as bring the prefix's
// items onto all compute units
int64_t prefix_bytes(int64_t rows, int Hq, int D) {
  return std::max(2 * piece_bytes(rows, Hq, D), piece_bytes(PREFIX_ROWS, 1, D));
}

// Whether n sequences (groups) have rows enough for tiles in LDS: on average, for the lengths are known on the
// device alone. A call of 128 single rows and one chunk of 512 (window of 1024, 2048 tokens, 32 / 8 heads of 128)
// streams them all, 178 us; apart the two take 139 and 39, the single rows without cu_q 108.
bool tiled(const reach::Args& a, int dtype, int64_t n) {
  // not behind prefixes: there few rows of many sequences share the prefix's tiles as a group
  const bool many = a.window && 2 * n * a.Hkv >= device_cus();
  return reach_tiles_shape(a, dtype) && a.rows * a.G >= (many ? TILE_ROWS_MANY : TILE_ROWS) * n;
}
// Tiles for the sequences of a call, with the plan's pieces from dst on
int tile_call(reach::Args a, int dtype, reach::TilePlan plan, float* dst, hipStream_t s) {
  if (plan.cuts > 1) {
    a.dst = dst;
    a.dst_ml = reinterpret_cast<float2*>(dst + plan.cuts * a.rows * a.Hq * a.D);
  }
  return launch_reach_tiles(a, dtype, plan, s);
}

// How a prefix call runs, and the workspace that it takes. general: no workspace. tiles: for the sequences, the
// prefix and their own keys as one list; a workspace for items that are cut, of which there are few rows.
// Else the prefix's part of all rows as pieces of rows (by tiles or streaming), then the rest.
struct PrefixRoute {
  bool general, tiles, group_tiles;
  reach::TilePlan plan;
  int64_t bytes;
};
PrefixRoute prefix_route(reach::Args a, int dtype, bool ragged) {
  PrefixRoute r{!streams(a, dtype), false, false, {false, 1}, 0};
  if (r.general) return r;
  const int64_t piece = piece_bytes(a.rows, a.Hq, a.D), parts = reach_stream_parts_bytes(a.D),
                shared = prefix_bytes(a.rows, a.Hq, a.D);
  const int64_t prefix_tokens = a.pt_stride * a.P;
  r.tiles = ragged && tiled(a, dtype, a.B);
  if (r.tiles) {  // they share their own keys' tiles too
    r.plan = reach_tiles_plan(a, prefix_tokens + a.bt_stride * a.P, (parts + shared) / piece);
    r.bytes = r.plan.cuts > 1 ? reach_stream_pref_bytes() + r.plan.cuts * piece : 0;
    return r;
  }
  r.bytes = reach_stream_pref_bytes() + parts;
  if (!a.groups) return r;
  r.bytes += shared;
  r.group_tiles = tiled(a, dtype, a.groups);
  a.by_group = 1;
  if (r.group_tiles) r.plan = reach_tiles_plan(a, prefix_tokens, shared / piece - 1);
  return r;
}

}  // namespace

unsigned long long reach_token() {
  static std::atomic<unsigned long long> next{[] {
    std::random_device r;
    return (static_cast<unsigned long long>(r()) << 32) | r();
  }()};
  return next.fetch_add(1, std::memory_order_relaxed) << 16;
}

}  // namespace pia

using namespace pia;

extern "C" int64_t pia_window_attention_workspace_bytes(int head_dim) {
  if (head_dim <= 0 || head_dim > 256 || head_dim % 16) return 0;
  return reach_stream_pref_bytes() + reach_stream_parts_bytes(head_dim);
}

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
  reach::Args a{out, q, q_stride, k_pages, v_pages, block_tables, bt_stride, kv_lens, cu_q,
                q_pos_offsets, total_q_rows, num_pages, 0, scale * 1.4426950408889634f, num_seqs,
                num_heads, num_kv_heads, num_kv_heads > 0 ? num_heads / num_kv_heads : 0,
                head_dim, page_size, window, sinks};
  int rc = check(a, dtype, "window_attention");
  if (!rc)
    rc = check_workspace(workspace, workspace_bytes, pia_window_attention_workspace_bytes(head_dim),
                         "window_attention");
  if (rc) return rc < 0 ? rc : 0;
  if (!streams(a, dtype)) return launch_reach_general(a, dtype, as_stream(stream));
  place(a, workspace);
  // tokens that an item walks: the sinks' and the window's, of the table's
  const int64_t tokens = std::min(bt_stride * page_size,
                                  int64_t(window) + sinks + std::min<int64_t>(total_q_rows, 16));
  if (cu_q && tiled(a, dtype, num_seqs)) {
    const reach::TilePlan plan = reach_tiles_plan(
        a, tokens, reach_stream_parts_bytes(head_dim) / piece_bytes(a.rows, a.Hq, a.D));
    return tile_call(a, dtype, plan, a.parts, as_stream(stream));
  }
  return stream_call(a, dtype, tokens, as_stream(stream));
}

extern "C" int64_t pia_prefix_attention_workspace_bytes(int64_t total_q_rows, int num_heads,
                                                        int head_dim) {
  if (head_dim <= 0 || head_dim > 256 || head_dim % 16 || total_q_rows <= 0 || num_heads <= 0)
    return 0;
  return reach_stream_pref_bytes() + reach_stream_parts_bytes(head_dim) +
         prefix_bytes(total_q_rows, num_heads, head_dim);
}

extern "C" int64_t pia_prefix_attention_call_workspace_bytes(
    int num_groups, int64_t pt_stride, int64_t bt_stride, int ragged, int num_seqs,
    int64_t total_q_rows, int num_heads, int num_kv_heads, int head_dim, int page_size, float scale,
    int dtype) {
  if (num_seqs <= 0 || total_q_rows <= 0 || num_heads <= 0 || num_kv_heads <= 0 ||
      num_heads % num_kv_heads || head_dim <= 0 || page_size <= 0 || pt_stride < 0 || bt_stride < 0)
    return 0;
  reach::Args a{};
  a.rows = total_q_rows;
  a.B = num_seqs;
  a.Hq = num_heads;
  a.Hkv = num_kv_heads;
  a.G = num_heads / num_kv_heads;
  a.D = head_dim;
  a.P = page_size;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.pt_stride = pt_stride;
  a.bt_stride = bt_stride;
  a.groups = num_groups > 0 && pt_stride > 0 ? num_groups : 0;
  return prefix_route(a, dtype, ragged != 0).bytes;
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
  reach::Args a{out, q, q_stride, k_pages, v_pages, block_tables, bt_stride, kv_lens, cu_q,
                q_pos_offsets, total_q_rows, num_pages, 0, scale * 1.4426950408889634f, num_seqs,
                num_heads, num_kv_heads, num_kv_heads > 0 ? num_heads / num_kv_heads : 0,
                head_dim, page_size, 0, 0, some ? prefix_tables : nullptr, pt_stride, prefix_lens,
                cu_seqs, some ? num_groups : 0};
  int rc = check(a, dtype, "prefix_attention");
  if (rc) return rc < 0 ? rc : 0;
  const PrefixRoute r = prefix_route(a, dtype, cu_q != nullptr);
  rc = check_workspace(workspace, workspace_bytes, r.bytes, "prefix_attention");
  if (rc) return rc;
  hipStream_t s = as_stream(stream);
  if (r.general) return launch_reach_general(a, dtype, s);
  if (r.bytes) place(a, workspace);
  if (r.tiles) return tile_call(a, dtype, r.plan, a.parts, s);
  if (some) {
    reach::Args g = a;
    g.by_group = 1;
    const int64_t R = total_q_rows * num_heads;
    const int cuts = r.plan.cuts;
    g.dst = a.parts + reach_stream_parts_bytes(head_dim) / int64_t(sizeof(float));
    g.dst_ml = reinterpret_cast<float2*>(g.dst + (cuts + 1) * R * head_dim);
    rc = r.group_tiles ? launch_reach_tiles(g, dtype, r.plan, s)
                       : stream_call(g, dtype, pt_stride * page_size, s);
    if (rc) return rc;
    a.src = g.dst;
    a.src_ml = g.dst_ml;
    a.src_cuts = cuts;
    a.dst = g.dst + cuts * R * head_dim;
    a.dst_ml = g.dst_ml + cuts * R;
  }
  return stream_call(a, dtype, bt_stride * page_size, s);
}
