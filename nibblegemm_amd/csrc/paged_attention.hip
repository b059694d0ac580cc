// Attention of the newest tokens of several sequences over a paged cache, with a
// window and first tokens that stay visible, on 16-bit or 8-bit pages.
//
// Sequence b holds lengths[b] rows before the call, its token i is row r = lengths[b] +
// i and sees the rows j <= r, of these, under a window, those with r - j < window or
// j < sinks; rows without a page are not seen:
//   out = sum_j p(j) v(j) / sum_j p(j),  p(j) = exp(scale q . k(j) - top),
// in one pass over the rows with a running top and running sums in fp32.  A token that
// sees nothing, and tokens behind a sequence's last, give zeros.
//
// The queries of a kv head's group (tokens x query heads, `rows`) go to the matrix cores
// together: up to 32 to rows_kernel, which memory bounds (a decode step's tokens: 4 to
// 256 operations for each byte of the cache), more to prompt_kernel, which matrix and
// vector instructions bound.  In both keys are a product's rows and queries its columns, so that a lane
// has scores of one query and its probabilities are already where the second product (V^T
// P^T, queries as columns again) wants them, if that product's k index runs over a lane's
// keys in turn.  V is read transposed from LDS (ds_read_b64_tr_b16, _tr_b8).  8-bit rows
// stay 8-bit in LDS and are converted, exactly, with their page's power of two, on their
// way into the products' operands.
//
// What it reads, writes and computes: the visible rows once a kv head and 128 query
// rows, 4 rows keys D operations, and, where the rows are split, D + 2 floats a query
// row and share.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "nibble_common.h"
#include "paged_prompt.h"
#include "paged_rows.h"

namespace nibble {

int check_paged(const nibble_paged_cache* c, int64_t dtype, int64_t batch);

namespace {

struct PagedPlan {
  int rows = 16, row_tiles = 1, shares = 0, slots = 0;
  size_t counter_bytes = 0, workspace_bytes = 0;
};

int plan_paged(int64_t batch, int64_t tokens, int64_t n_heads, int64_t n_kv, int64_t head_dim,
               int64_t max_rows, PagedPlan* p) {
  NIBBLE_CHECK(head_dim == 64 || head_dim == 128, "head_dim must be 64 or 128, got %lld",
               (long long)head_dim);
  NIBBLE_CHECK(n_kv >= 1 && n_kv <= 65535, "n_kv_heads must be in [1, 65535], got %lld",
               (long long)n_kv);
  NIBBLE_CHECK(n_heads >= n_kv && n_heads <= 65535 && n_heads % n_kv == 0,
               "n_heads (%lld) must be a multiple of n_kv_heads (%lld), at most 65535",
               (long long)n_heads, (long long)n_kv);
  NIBBLE_CHECK(batch >= 0 && tokens >= 0 && batch <= 65535 && tokens <= (1 << 20),
               "batch must be in [0, 65535] and tokens in [0, 2^20]");
  NIBBLE_CHECK(max_rows >= 0 && max_rows < (int64_t(1) << 30),
               "a sequence's pages must have less than 2^30 rows, got %lld", (long long)max_rows);
  if (batch == 0 || tokens == 0) return NIBBLE_OK;
  const int64_t rows = tokens * (n_heads / n_kv);
  NIBBLE_CHECK(rows * batch * n_kv <= (int64_t(1) << 30), "more than 2^30 query rows");
  p->rows = rows <= 16 ? 16 : rows <= 32 ? 32 : 128;
  p->row_tiles = static_cast<int>(ceil_div(rows, p->rows));
  NIBBLE_CHECK(ceil_div(batch, 8) * 8 * n_kv * p->row_tiles * kPagedThreads < (int64_t(1) << 32),
               "%lld sequences of %lld kv heads: a launch ends at 2^32 threads", (long long)batch,
               (long long)n_kv);
  // Room for more workgroups than there are (sequence, kv head, row tile)s: the
  // cached rows are split, unless there are but a few tiles of them.
  const int64_t room = kSplitWorkgroups / (n_kv * p->row_tiles);
  const bool line = p->rows <= 32;  // rows_kernel's
  // (the line's length, in tiles and gaps, has to stay far below 2^31)
  if (line ? room > 0 && batch <= kSplitWorkgroups && batch * n_kv < 4 * kSplitWorkgroups &&
                 batch * (max_rows / kPagedKeys + 8) < (int64_t(1) << 30)
           : room > batch && batch < kSplitWorkgroups) {
    if (max_rows <= 4 * kPagedKeys) return NIBBLE_OK;
    p->shares = static_cast<int>(room);
    p->slots = static_cast<int>(line ? 2 * room : room);
    p->counter_bytes = line ? 4 * kSplitWorkgroups * sizeof(int) : 0;  // a sequence and kv head
    p->workspace_bytes = p->counter_bytes +
                         static_cast<size_t>(n_kv * p->slots * rows) * (head_dim + 2) * 4 +
                         static_cast<size_t>(line ? 0 : batch) * 8;
  }
  return NIBBLE_OK;
}

template <class E, int D, bool Q8>
hipError_t launch_paged(const AttendArgs& a, const PagedPlan& p, hipStream_t stream) {
  const int64_t pieces = p.shares > 0 ? p.shares : a.B;
  if (p.rows <= 32) {
    const dim3 grid(static_cast<unsigned>(ceil_div(pieces, 8) * 8 * a.n_kv));
    if (p.rows == 16) rows_kernel<E, D, 1, Q8><<<grid, kPagedThreads, 0, stream>>>(a);
    else rows_kernel<E, D, 2, Q8><<<grid, kPagedThreads, 0, stream>>>(a);
    return hipGetLastError();
  }
  const dim3 grid(static_cast<unsigned>(ceil_div(pieces * a.n_kv, 8) * 8 * p.row_tiles));
  prompt_kernel<E, D, Q8><<<grid, kPagedThreads, 0, stream>>>(a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.shares == 0) return e;
  const int64_t parts = ceil_div(static_cast<int64_t>(a.T) * a.qpk, kSplitThreads / (D / 4));
  join_kernel<E, D><<<dim3(static_cast<unsigned>(a.B * a.n_kv * parts)), kSplitThreads, 0,
                      stream>>>(a);
  return hipGetLastError();
}

template <class E>
hipError_t launch_paged(const AttendArgs& a, const PagedPlan& p, int D, hipStream_t stream) {
  const bool q8 = a.k_scales != nullptr;
  if (D == 64) return q8 ? launch_paged<E, 64, true>(a, p, stream) : launch_paged<E, 64, false>(a, p, stream);
  return q8 ? launch_paged<E, 128, true>(a, p, stream) : launch_paged<E, 128, false>(a, p, stream);
}

}  // namespace
}  // namespace nibble

using namespace nibble;

extern "C" size_t nibble_attention_paged_workspace_bytes(int64_t batch, int64_t tokens,
                                                         int64_t n_heads, int64_t n_kv_heads,
                                                         int64_t head_dim, int64_t max_rows) {
  PagedPlan p;
  if (plan_paged(batch, tokens, n_heads, n_kv_heads, head_dim, max_rows, &p) != NIBBLE_OK) return 0;
  return p.workspace_bytes;
}

extern "C" size_t nibble_attention_paged_counter_bytes(int64_t batch, int64_t tokens,
                                                       int64_t n_heads, int64_t n_kv_heads,
                                                       int64_t head_dim, int64_t max_rows) {
  PagedPlan p;
  if (plan_paged(batch, tokens, n_heads, n_kv_heads, head_dim, max_rows, &p) != NIBBLE_OK) return 0;
  return p.counter_bytes;
}

extern "C" int nibble_attention_paged(const void* Q, int64_t dtype, int64_t batch, int64_t tokens,
                                      int64_t n_heads, const nibble_paged_cache* cache,
                                      const void* lengths, const void* sizes, int64_t window,
                                      int64_t sinks, float scale, void* Out, void* workspace,
                                      size_t workspace_bytes, void* stream_) {
  int rc = check_paged(cache, dtype, batch);
  if (rc != NIBBLE_OK) return rc;
  const nibble_paged_cache& c = *cache;
  PagedPlan p;
  rc = plan_paged(batch, tokens, n_heads, c.n_kv_heads, c.head_dim, c.table_pages * c.page_rows, &p);
  if (rc != NIBBLE_OK) return rc;
  NIBBLE_CHECK(std::isfinite(scale * kLog2e), "scale must be finite, also times log2(e)");
  NIBBLE_CHECK(window >= 0 && window <= (1 << 30), "window must be in [0, 2^30], got %lld",
               (long long)window);
  NIBBLE_CHECK(sinks >= 0 && sinks <= (1 << 30), "sinks must be in [0, 2^30], got %lld",
               (long long)sinks);
  if (batch == 0 || tokens == 0) return ok();
  NIBBLE_CHECK(Q != nullptr && Out != nullptr && lengths != nullptr, "null pointer");
  NIBBLE_CHECK(aligned(Q, 16) && aligned(Out, 16), "q and output must be 16-byte aligned");
  NIBBLE_CHECK(aligned(lengths, 4) && aligned(sizes, 4), "lengths and sizes must be 4-byte aligned");
  if (p.workspace_bytes > 0) {
    if (workspace == nullptr || workspace_bytes < p.workspace_bytes)
      return fail(NIBBLE_ERR_WORKSPACE, "attention needs %zu bytes of workspace, got %zu",
                  p.workspace_bytes, workspace == nullptr ? size_t(0) : workspace_bytes);
    if (!aligned(workspace, 256))
      return fail(NIBBLE_ERR_WORKSPACE, "workspace must be 256-byte aligned");
  }
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  DeviceGuard guard;
  int dev = 0;
  NIBBLE_HIP(guard.enter(stream, &dev));
  const int64_t bytes = c.k_scales != nullptr ? 1 : 2, P = c.page_rows;
  AttendArgs a;
  a.q = Q;
  a.k = static_cast<const char*>(c.K);
  a.v = static_cast<const char*>(c.V);
  a.k_scales = static_cast<const uint8_t*>(c.k_scales);
  a.v_scales = static_cast<const uint8_t*>(c.v_scales);
  a.table = static_cast<const int32_t*>(c.table);
  a.lengths = static_cast<const int32_t*>(lengths);
  a.sizes = static_cast<const int32_t*>(sizes);
  a.out = Out;
  a.qpk = static_cast<int>(n_heads / c.n_kv_heads);
  a.counters = static_cast<int*>(workspace);
  a.partial = reinterpret_cast<float*>(static_cast<char*>(workspace) + p.counter_bytes);
  a.runs = reinterpret_cast<int*>(a.partial + static_cast<size_t>(c.n_kv_heads) * p.slots * tokens *
                                              a.qpk * (c.head_dim + 2));
  a.kp = c.k_page_stride * bytes, a.kh = c.k_head_stride * bytes, a.kr = c.k_row_stride * bytes;
  a.vp = c.v_page_stride * bytes, a.vh = c.v_head_stride * bytes, a.vr = c.v_row_stride * bytes;
  a.B = static_cast<int>(batch);
  a.T = static_cast<int>(tokens);
  a.n_heads = static_cast<int>(n_heads);
  a.n_kv = static_cast<int>(c.n_kv_heads);
  // (where there are no pages, there are no scales to read either)
  a.width = c.n_pages > 0 ? static_cast<int>(c.table_pages) : 0;
  a.n_pages = static_cast<int>(c.n_pages);
  a.shift = P == 16 ? 4 : P == 32 ? 5 : P == 64 ? 6 : P == 128 ? 7 : 8;
  a.window = window > 0 ? static_cast<int>(window) : 1 << 30;
  a.sinks = static_cast<int>(sinks);
  a.shares = p.shares;
  a.slots = p.slots;
  a.row_tiles = p.row_tiles;
  a.join_cost = kPagedShareCost + kPagedRowCost * static_cast<float>(tokens * n_heads);
  a.fold = batch * c.n_kv_heads * p.row_tiles <= kSplitWorkgroups;
  a.scale = scale == 0.0f ? 1.0f : std::fabs(scale) * kLog2e;
  a.sign = scale > 0.0f ? 1.0f : scale < 0.0f ? -1.0f : 0.0f;
  const hipError_t e = dtype == 0 ? launch_paged<Half>(a, p, static_cast<int>(c.head_dim), stream)
                                  : launch_paged<Bfloat>(a, p, static_cast<int>(c.head_dim), stream);
  if (e != hipSuccess) return hip_fail(e, "paged attention kernel launch");
  return ok();
}
