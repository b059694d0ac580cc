// Paged caches: the way of new tokens' keys and values into the pages, and the dense
// rows that a sequence's pages stand for.
//
// Sequence b holds lengths[b] rows; its token t goes to the row behind them, row
// r = lengths[b] + t, which lies in page table[b][r / P] at r % P.  A query or key head
// x of a token at position p becomes, in fp32 and rounded once,
//   n = x w / sqrt(mean(x^2) + eps)                       (where the heads have norms)
//   n[i] cos(p, k) - n[j] sin(p, k), n[j] cos(p, k) + n[i] sin(p, k)
// for the pairs k of its first R elements, (i, j) = (k, k + R / 2) or (2k, 2k + 1);
// values go through as they are.
//
// A page of 8-bit floats has a power of two for each head, 2^(e - 127), the least (of
// those whose products with the codes are values of the 16-bit type) under which the
// new rows fit; where the page holds earlier rows, the larger of theirs and the new
// one's, and when that rises their codes are halved as often, exactly but for those
// that end below the smallest normal one.
//
// Memory bounds both: every value is read once and written once.  What is written goes
// past the caches (nt), which keep what is read, the product before, instead: 4 x 2000
// tokens of 32 + 2 x 8 heads of 128 take 36 to 39 us in place of 41 (44 if the reads go
// past them, too).  A decode step, whose q and new rows the attention reads next, is the
// same either way: 1 over 1000 rows 14.1 us (14.0 without), 64 over 300 17.3 (17.5), 16
// over 2000 25.9 (25.9).
#include <cmath>

#include "nibble_common.h"
#include "nibble_float8.h"
#include "nibble_reduce.h"

namespace nibble {
namespace {

constexpr int kPagedThreads = 256;

struct PagedArgs {
  const void* qkv;  // [B, T, n_heads + 2 n_kv, D]
  char* k;          // element (page, h, r, d) at page kp + h kh + r kr + d elements
  char* v;
  uint8_t* k_scales;       // [n_pages, n_kv] or null: 16-bit pages
  uint8_t* v_scales;
  const int32_t* table;    // [B, width]
  const int32_t* lengths;  // [B]
  const int32_t* sizes;    // [B] or null: T each
  const int32_t* positions;  // [B, T] or null: a token's row
  const void* q_weight;      // [D] or null
  const void* k_weight;
  const float* cos;  // [rope_rows, R / 2] or null
  const float* sin;
  void* q_out;  // [B, T, n_heads, D]
  int64_t kp, kh, kr, vp, vh, vr;  // in bytes
  uint32_t heads;                  // those that a lane group has each: B T (n_heads [+ 2 n_kv])
  uint32_t T;
  int B, n_heads, n_kv, width, n_pages, shift, rope_rows, R;
  uint32_t tasks, spans;  // 8-bit: (sequence, page, head, k or v)s, pages that a run of tokens may reach
  unsigned head_blocks;
  float eps;
  bool interleaved;
};

// What there is of a sequence, and where its tokens go.
struct Rows {
  int len, live;
  __device__ __forceinline__ Rows(const PagedArgs& a, int b) {
    const int room = a.width << a.shift;
    len = min(max(a.lengths[b], 0), room);
    const int T = static_cast<int>(a.T);
    live = min(a.sizes != nullptr ? min(max(a.sizes[b], 0), T) : T, room - len);
  }
};

// The page of a sequence's row, or -1.
__device__ __forceinline__ int page_of(const int32_t* table, int b, int width, int n_pages, int m) {
  const int page = table[static_cast<int64_t>(b) * width + m];
  return page >= 0 && page < n_pages ? page : -1;
}

// A token's position in the tables, or -1 where they do not have it.
__device__ __forceinline__ int position(const PagedArgs& a, int b, int t, int row) {
  const int pos = a.positions != nullptr ? a.positions[static_cast<int64_t>(b) * a.T + t] : row;
  return a.cos == nullptr || (pos >= 0 && pos < a.rope_rows) ? pos : -1;
}

// A head is held by D / 16 lanes, 16 elements each in two runs of 8: under the half
// layout lanes of the rotated part hold a run and its partners.
struct Runs {
  int lo, hi;
  bool turns;
  __device__ __forceinline__ Runs(const PagedArgs& a, int j) {
    turns = a.cos != nullptr && 16 * j < a.R;
    const bool halves = turns && !a.interleaved;
    lo = halves ? 8 * j : 16 * j;
    hi = halves ? 8 * j + a.R / 2 : 16 * j + 8;
  }
};

// Norm and rotation of a query or key head: f and g are this lane's runs.
template <class E, int D>
__device__ __forceinline__ void turn(const PagedArgs& a, const void* weight, const Runs& runs,
                                     int j, int pos, float (&f)[8], float (&g)[8]) {
  using T = typename E::type;
  using vec8 = typename E::vec8;
  const T* w = static_cast<const T*>(weight);
  if (w != nullptr) {
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = __builtin_fmaf(f[i], f[i], ss);
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = __builtin_fmaf(g[i], g[i], ss);
    ss += dpp<kDppXor1>(ss);
    ss += dpp<kDppXor2>(ss);
    if (D == 128) ss += dpp<kDppHalfMirror>(ss);
    const float r = rms_scale(ss, D, a.eps);
    const vec8 wl = *reinterpret_cast<const vec8*>(w + runs.lo);
    const vec8 wh = *reinterpret_cast<const vec8*>(w + runs.hi);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      f[i] *= r * static_cast<float>(wl[i]);
      g[i] *= r * static_cast<float>(wh[i]);
    }
  }
  if (!runs.turns) return;
  const int64_t at = static_cast<int64_t>(max(pos, 0)) * (a.R / 2) + 8 * j;
  f4_t c[2], s[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    c[e] = *reinterpret_cast<const f4_t*>(a.cos + at + 4 * e);
    s[e] = *reinterpret_cast<const f4_t*>(a.sin + at + 4 * e);
  }
  auto pair = [&](float& x, float& y, int k) {
    const float cc = c[k / 4][k % 4], si = s[k / 4][k % 4];
    const float n = x * cc - y * si;
    y = y * cc + x * si;
    x = n;
  };
  if (a.interleaved) {
#pragma unroll
    for (int i = 0; i < 4; ++i) pair(f[2 * i], f[2 * i + 1], i), pair(g[2 * i], g[2 * i + 1], i + 4);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) pair(f[i], g[i], i);
  }
}

// Heads of D / 16 lanes each: the queries, and with 16-bit pages keys and values too.
template <class E, int D, bool Q8>
__device__ __forceinline__ void append_heads(const PagedArgs& a) {
  using T = typename E::type;
  using vec8 = typename E::vec8;
  constexpr int LANES = D / 16;
  const int j = threadIdx.x % LANES;
  const uint32_t x = blockIdx.x * (kPagedThreads / LANES) + threadIdx.x / LANES;
  // (heads behind the last take part in the reductions, as copies of it)
  const uint32_t at = min(x, a.heads - 1);
  const uint32_t all = a.n_heads + 2 * a.n_kv, some = Q8 ? a.n_heads : all;
  const uint32_t token = at / some, in_batch = token / a.T;
  const int head = static_cast<int>(at - token * some);
  const int b = static_cast<int>(in_batch), t = static_cast<int>(token - in_batch * a.T);
  const Runs runs(a, j);
  const T* from = static_cast<const T*>(a.qkv) + (static_cast<int64_t>(token) * all + head) * D;
  vec8 lo = *reinterpret_cast<const vec8*>(from + runs.lo);
  vec8 hi = *reinterpret_cast<const vec8*>(from + runs.hi);
  const Rows rows(a, b);
  const int row = rows.len + t, pos = position(a, b, t, row);
  const int page = t < rows.live ? page_of(a.table, b, a.width, a.n_pages, row >> a.shift) : -1;
  const bool live = page >= 0 && (a.cos == nullptr || pos >= 0);
  const bool query = head < a.n_heads, value = head >= a.n_heads + a.n_kv;
  if (!value) {
    float f[8], g[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = static_cast<float>(lo[i]), g[i] = static_cast<float>(hi[i]);
    turn<E, D>(a, query ? a.q_weight : a.k_weight, runs, j, pos, f, g);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      lo[i] = static_cast<T>(query && !live ? 0.0f : f[i]);
      hi[i] = static_cast<T>(query && !live ? 0.0f : g[i]);
    }
  }
  if (x >= a.heads || !(query || live)) return;
  T* o;
  if (query) {
    o = static_cast<T*>(a.q_out) + (static_cast<int64_t>(token) * a.n_heads + head) * D;
  } else {
    const int h = head - a.n_heads - (value ? a.n_kv : 0), r = row & ((1 << a.shift) - 1);
    o = reinterpret_cast<T*>(value ? a.v + page * a.vp + h * a.vh + r * a.vr
                                   : a.k + page * a.kp + h * a.kh + r * a.kr);
  }
  __builtin_nontemporal_store(lo, reinterpret_cast<vec8*>(o + runs.lo));
  __builtin_nontemporal_store(hi, reinterpret_cast<vec8*>(o + runs.hi));
}

// The new rows of one page, one head, keys or values: a task of one wave, two or four, by
// the page's size.  A lane holds its rows' values from the first look, for the largest
// magnitude, to their rounding.  (4 x 2000 tokens of 32 + 2 x 8 heads of 128 on pages of 64
// 45 us; a wave a page, its values worked out twice, 71 us.)
template <class E, int D, int P>
__device__ __forceinline__ void append_page(const PagedArgs& a) {
  using T = typename E::type;
  using vec8 = typename E::vec8;
  constexpr int LANES = D / 16;
  constexpr int WAVES = P * LANES <= 128 ? 1 : P * LANES <= 256 ? 2 : 4;
  constexpr int STEP = WAVES * 64 / LANES;  // rows at once
  constexpr int N = P > STEP ? P / STEP : 1;
  const int me = threadIdx.x % (WAVES * 64);  // within the task
  const uint32_t task = (blockIdx.x - a.head_blocks) * (4 / WAVES) + threadIdx.x / (WAVES * 64);
  __shared__ float part[4];
  const uint32_t rest = (task >> 1) / a.n_kv, in_batch = rest / a.spans;
  const int which = static_cast<int>(task & 1), h = static_cast<int>((task >> 1) - rest * a.n_kv);
  const int b = static_cast<int>(in_batch), m = static_cast<int>(rest - in_batch * a.spans);
  int len = 0, index = 0, first = 0, begin = 0, end = 0, page = -1;
  if (task < a.tasks) {
    const Rows rows(a, b);
    len = rows.len, index = (len >> a.shift) + m, first = index * P;  // the page's first row
    begin = max(len, first), end = min(len + rows.live, first + P);
    if (begin < end) page = page_of(a.table, b, a.width, a.n_pages, index);
  }
  const int j = me % LANES, r0 = me / LANES;
  Runs runs(a, j);
  if (which != 0) runs.turns = false, runs.lo = 16 * j, runs.hi = 16 * j + 8;
  const int all = a.n_heads + 2 * a.n_kv;
  float f[N][8], g[N][8], top = -1.0f;  // below zero: no row
  bool live[N];  // a row with a place, whose position the tables have
  uint8_t* scale = nullptr;
  int was = 0;
  if (page >= 0) {
    const T* const from = static_cast<const T*>(a.qkv) +
                          (static_cast<int64_t>(b) * a.T * all + a.n_heads + which * a.n_kv + h) * D;
    scale = (which != 0 ? a.v_scales : a.k_scales) + static_cast<int64_t>(page) * a.n_kv + h;
    was = *scale;
    int pos[N];
    vec8 raw[N][2];
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int row = first + r0 + n * STEP;
      const bool in = row >= begin && row < end;
      pos[n] = in ? position(a, b, row - len, row) : -1;
      live[n] = in && (a.cos == nullptr || pos[n] >= 0);
      const T* x = from + static_cast<int64_t>((in ? row : begin) - len) * all * D;
      raw[n][0] = *reinterpret_cast<const vec8*>(x + runs.lo);
      raw[n][1] = *reinterpret_cast<const vec8*>(x + runs.hi);
    }
#pragma unroll
    for (int n = 0; n < N; ++n) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        f[n][i] = static_cast<float>(raw[n][0][i]), g[n][i] = static_cast<float>(raw[n][1][i]);
      if (which == 0) turn<E, D>(a, a.k_weight, runs, j, pos[n], f[n], g[n]);
      if (!live[n]) continue;
      top = fmaxf(top, 0.0f);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        // (an infinity or a NaN has no part in the scale)
        const float x = fabsf(f[n][i]), y = fabsf(g[n][i]);
        top = fmaxf(top, x < INFINITY ? fminf(x, kLargest<E>) : 0.0f);
        top = fmaxf(top, y < INFINITY ? fminf(y, kLargest<E>) : 0.0f);
      }
    }
    top = wave_max(top);
  }
  if (WAVES > 1) {  // (every wave has read the scale, too)
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
    __syncthreads();
    const int wave0 = threadIdx.x / (WAVES * 64) * WAVES;
#pragma unroll
    for (int x = 0; x < WAVES; ++x) top = fmaxf(top, part[wave0 + x]);
  }
  if (top < 0.0f) return;

  char* const base = which != 0 ? a.v + page * a.vp + h * a.vh : a.k + page * a.kp + h * a.kh;
  const int64_t stride = which != 0 ? a.vr : a.kr;
  const int need = exponent_for<E>(top);
  const bool fresh = begin == first, none = was == 255;  // no power: earlier rows are NaN
  const int e = fresh || none ? need : max(need, was);
  if (!fresh && e != was) {  // earlier rows, on the new power of two
    const float by = none ? __builtin_nanf("") : power(max(127 + was - e, 1));
#pragma unroll 1
    for (int i = me; i < (begin - first) * LANES; i += WAVES * 64) {
      u4_t* const at = reinterpret_cast<u4_t*>(base + (i / LANES) * stride + 16 * (i % LANES));
      u4_t x = *at;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(x[w]), false);
        const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(x[w]), true);
        x[w] = to_float8(lo[0] * by, lo[1] * by, hi[0] * by, hi[1] * by);
      }
      *at = x;
    }
  }
  if (me == 0 && e != was) *scale = static_cast<uint8_t>(e);
  // (2^-127, the inverse of a caller's scale of 254, is subnormal)
  const float inverse = e == 254 ? 0x1p-127f : power(254 - e);
  const float most = e >= kHighExponent<E> ? kFloat8LastMax : kFloat8Max;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    if (!live[n]) continue;
    auto code = [&](float x) {
      const float y = x * inverse;
      // (an infinity or a NaN becomes NaN)
      return fabsf(x) < INFINITY ? fminf(fmaxf(y, -most), most) : __builtin_nanf("");
    };
    char* const o = base + (r0 + n * STEP) * stride;
    typedef uint32_t u2_t __attribute__((ext_vector_type(2)));
    const float(&x)[8] = f[n];
    const float(&y)[8] = g[n];
    *reinterpret_cast<u2_t*>(o + runs.lo) =
        u2_t{to_float8(code(x[0]), code(x[1]), code(x[2]), code(x[3])),
             to_float8(code(x[4]), code(x[5]), code(x[6]), code(x[7]))};
    *reinterpret_cast<u2_t*>(o + runs.hi) =
        u2_t{to_float8(code(y[0]), code(y[1]), code(y[2]), code(y[3])),
             to_float8(code(y[4]), code(y[5]), code(y[6]), code(y[7]))};
  }
}

template <class E, int D>
__global__ __launch_bounds__(kPagedThreads) void append_kernel(PagedArgs a) {
  append_heads<E, D, false>(a);
}
template <class E, int D, int P>
__global__ __launch_bounds__(kPagedThreads) void append8_kernel(PagedArgs a) {
  if (blockIdx.x < a.head_blocks) append_heads<E, D, true>(a);
  else append_page<E, D, P>(a);
}

template <class E, int D>
hipError_t launch_append(const PagedArgs& a, bool q8, dim3 grid, hipStream_t stream) {
  if (!q8) append_kernel<E, D><<<grid, kPagedThreads, 0, stream>>>(a);
  else if (a.shift == 4) append8_kernel<E, D, 16><<<grid, kPagedThreads, 0, stream>>>(a);
  else if (a.shift == 5) append8_kernel<E, D, 32><<<grid, kPagedThreads, 0, stream>>>(a);
  else if (a.shift == 6) append8_kernel<E, D, 64><<<grid, kPagedThreads, 0, stream>>>(a);
  else if (a.shift == 7) append8_kernel<E, D, 128><<<grid, kPagedThreads, 0, stream>>>(a);
  else append8_kernel<E, D, 256><<<grid, kPagedThreads, 0, stream>>>(a);
  return hipGetLastError();
}

struct ValuesArgs {
  const char* k;
  const char* v;
  const uint8_t* k_scales;
  const uint8_t* v_scales;
  const int32_t* table;
  const int32_t* lengths;
  void* k_out;  // [B, n_kv, rows, D]
  void* v_out;
  int64_t kp, kh, kr, vp, vh, vr;  // in bytes
  uint32_t units;                  // B n_kv rows D / 16, of keys (and as many of values)
  uint32_t n_kv, rows;
  int width, n_pages, shift;
};

// Sixteen values a thread, keys and values side by side.
template <class E, int D, bool Q8>
__global__ __launch_bounds__(kPagedThreads) void values_kernel(ValuesArgs a) {
  using vec8 = typename E::vec8;
  constexpr int UNITS = D / 16;
  const uint32_t unit = blockIdx.x * kPagedThreads + threadIdx.x;
  if (unit >= a.units) return;
  const uint32_t at = unit / UNITS, pair = at / a.rows, in_batch = pair / a.n_kv;
  const int u = static_cast<int>(unit % UNITS), row = static_cast<int>(at - pair * a.rows);
  const int b = static_cast<int>(in_batch), h = static_cast<int>(pair - in_batch * a.n_kv);
  const int m = row >> a.shift, r = row & ((1 << a.shift) - 1);
  const int page = row < a.lengths[b] && m < a.width ? page_of(a.table, b, a.width, a.n_pages, m) : -1;
  vec8 y[2][2] = {};
  if (page >= 0) {
    const char* const x[2] = {a.k + page * a.kp + h * a.kh + r * a.kr,
                              a.v + page * a.vp + h * a.vh + r * a.vr};
    if constexpr (Q8) {
      const int64_t s = static_cast<int64_t>(page) * a.n_kv + h;
      const float scale[2] = {power(a.k_scales[s]), power(a.v_scales[s])};
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const u4_t c = *reinterpret_cast<const u4_t*>(x[i] + 16 * u);
        y[i][0] = from_float8<E>(c[0], c[1], scale[i], scale[i]);
        y[i][1] = from_float8<E>(c[2], c[3], scale[i], scale[i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          y[i][e] = *reinterpret_cast<const vec8*>(x[i] + 32 * u + 16 * e);
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int e = 0; e < 2; ++e)
      static_cast<vec8*>(i == 0 ? a.k_out : a.v_out)[2 * static_cast<int64_t>(unit) + e] = y[i][e];
}

template <class E>
hipError_t launch_values(const ValuesArgs& a, int D, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(ceil_div(a.units, kPagedThreads)));
  if (a.k_scales == nullptr) {
    if (D == 64) values_kernel<E, 64, false><<<grid, kPagedThreads, 0, stream>>>(a);
    else values_kernel<E, 128, false><<<grid, kPagedThreads, 0, stream>>>(a);
  } else {
    if (D == 64) values_kernel<E, 64, true><<<grid, kPagedThreads, 0, stream>>>(a);
    else values_kernel<E, 128, true><<<grid, kPagedThreads, 0, stream>>>(a);
  }
  return hipGetLastError();
}

}  // namespace

int check_paged(const nibble_paged_cache* c, int64_t dtype, int64_t batch) {
  NIBBLE_CHECK(c != nullptr, "null cache");
  NIBBLE_CHECK(dtype == 0 || dtype == 1, "dtype must be 0 (fp16) or 1 (bf16), got %lld",
               (long long)dtype);
  NIBBLE_CHECK(c->head_dim == 64 || c->head_dim == 128, "head_dim must be 64 or 128, got %lld",
               (long long)c->head_dim);
  NIBBLE_CHECK(c->n_kv_heads >= 1 && c->n_kv_heads <= 65535,
               "n_kv_heads must be in [1, 65535], got %lld", (long long)c->n_kv_heads);
  NIBBLE_CHECK(c->page_rows == 16 || c->page_rows == 32 || c->page_rows == 64 ||
                   c->page_rows == 128 || c->page_rows == 256,
               "a page must have 16, 32, 64, 128 or 256 rows, got %lld", (long long)c->page_rows);
  NIBBLE_CHECK(c->n_pages >= 0 && c->n_pages <= 0x7fffffff, "n_pages must be in [0, 2^31), got %lld",
               (long long)c->n_pages);
  NIBBLE_CHECK(c->table_pages >= 0 && c->table_pages < (int64_t(1) << 30) / c->page_rows,
               "a sequence's pages must have less than 2^30 rows, got %lld pages of %lld",
               (long long)c->table_pages, (long long)c->page_rows);
  NIBBLE_CHECK(batch >= 0 && batch <= 65535, "batch must be in [0, 65535], got %lld",
               (long long)batch);
  NIBBLE_CHECK((c->k_scales == nullptr) == (c->v_scales == nullptr),
               "k_scales and v_scales must both be given or both be null");
  const int64_t unit = c->k_scales != nullptr ? 16 : 8;  // elements of 16 bytes
  for (int64_t s : {c->k_page_stride, c->k_head_stride, c->k_row_stride, c->v_page_stride,
                    c->v_head_stride, c->v_row_stride})
    NIBBLE_CHECK(s >= 0 && s % unit == 0 && s < (int64_t(1) << 58),
                 "cache strides must be multiples of 16 bytes, got %lld elements", (long long)s);
  // 32-bit offsets within the rows of one tile
  NIBBLE_CHECK(c->k_row_stride <= (1 << 22) && c->v_row_stride <= (1 << 22),
               "row strides must be at most 2^22 elements");
  NIBBLE_CHECK(batch == 0 || c->n_pages == 0 || (c->K != nullptr && c->V != nullptr), "null pointer");
  NIBBLE_CHECK(batch == 0 || c->table_pages == 0 || c->table != nullptr, "null pointer");
  NIBBLE_CHECK(aligned(c->K, 16) && aligned(c->V, 16), "caches must be 16-byte aligned");
  NIBBLE_CHECK(aligned(c->table, 4), "the table must be 4-byte aligned");
  return NIBBLE_OK;
}

}  // namespace nibble

using namespace nibble;

extern "C" int nibble_paged_append(const void* QKV, int64_t dtype, int64_t batch, int64_t tokens,
                                   int64_t n_heads, const nibble_paged_cache* cache,
                                   const void* lengths, const void* sizes, const void* positions,
                                   const void* q_weight, const void* k_weight, float eps,
                                   const void* rope_cos, const void* rope_sin, int64_t rope_rows,
                                   int64_t rope_dim, int64_t interleaved, void* Q_out,
                                   void* stream_) {
  const int rc = check_paged(cache, dtype, batch);
  if (rc != NIBBLE_OK) return rc;
  const nibble_paged_cache& c = *cache;
  NIBBLE_CHECK(n_heads >= 1 && n_heads <= 65535, "n_heads must be in [1, 65535], got %lld",
               (long long)n_heads);
  NIBBLE_CHECK(tokens >= 0 && tokens <= (1 << 20), "tokens must be in [0, 2^20], got %lld",
               (long long)tokens);
  NIBBLE_CHECK((rope_cos == nullptr) == (rope_sin == nullptr),
               "rope_cos and rope_sin must both be given or both be null");
  NIBBLE_CHECK(rope_cos == nullptr || (rope_rows >= 1 && rope_rows <= 0x7fffffff),
               "rope tables must have between 1 and 2^31 - 1 rows, got %lld", (long long)rope_rows);
  NIBBLE_CHECK(rope_cos == nullptr ||
                   (rope_dim >= 16 && rope_dim <= c.head_dim && rope_dim % 16 == 0),
               "the rotated part of a head must be a multiple of 16 of its %lld elements, got %lld",
               (long long)c.head_dim, (long long)rope_dim);
  NIBBLE_CHECK(interleaved == 0 || interleaved == 1, "interleaved must be 0 or 1, got %lld",
               (long long)interleaved);
  NIBBLE_CHECK(std::isfinite(eps) && eps >= 0.0f, "eps must be finite and >= 0");
  if (batch == 0 || tokens == 0) return ok();
  NIBBLE_CHECK(QKV != nullptr && Q_out != nullptr && lengths != nullptr, "null pointer");
  NIBBLE_CHECK(aligned(QKV, 16) && aligned(Q_out, 16) && aligned(q_weight, 16) &&
                   aligned(k_weight, 16),
               "qkv, weights and output must be 16-byte aligned");
  NIBBLE_CHECK(aligned(rope_cos, 16) && aligned(rope_sin, 16), "rope tables must be 16-byte aligned");
  NIBBLE_CHECK(aligned(lengths, 4) && aligned(sizes, 4) && aligned(positions, 4),
               "lengths, sizes and positions must be 4-byte aligned");
  const bool q8 = c.k_scales != nullptr;
  const int64_t bytes = q8 ? 1 : 2, P = c.page_rows;
  PagedArgs a;
  const int64_t heads = batch * tokens * (n_heads + (q8 ? 0 : 2 * c.n_kv_heads));
  const int64_t head_blocks = ceil_div(heads, kPagedThreads / (c.head_dim / 16));
  // pages that a run of tokens reaches, wherever it begins
  const int64_t spans = (tokens + P - 2) / P + 1;
  const int64_t tasks = q8 ? batch * spans * c.n_kv_heads * 2 : 0;
  const int64_t lanes = P * (c.head_dim / 16);  // of a task: a wave, two or four
  const int64_t blocks = head_blocks + ceil_div(tasks, lanes <= 128 ? 4 : lanes <= 256 ? 2 : 1);
  // (a launch ends at 2^32 threads; heads and tasks are fewer)
  NIBBLE_CHECK(blocks < (int64_t(1) << 32) / kPagedThreads, "too many tokens: %lld x %lld",
               (long long)batch, (long long)tokens);
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  DeviceGuard guard;
  int dev = 0;
  NIBBLE_HIP(guard.enter(stream, &dev));
  a.qkv = QKV;
  a.k = static_cast<char*>(c.K);
  a.v = static_cast<char*>(c.V);
  a.k_scales = static_cast<uint8_t*>(c.k_scales);
  a.v_scales = static_cast<uint8_t*>(c.v_scales);
  a.table = static_cast<const int32_t*>(c.table);
  a.lengths = static_cast<const int32_t*>(lengths);
  a.sizes = static_cast<const int32_t*>(sizes);
  a.positions = static_cast<const int32_t*>(positions);
  a.q_weight = q_weight;
  a.k_weight = k_weight;
  a.cos = static_cast<const float*>(rope_cos);
  a.sin = static_cast<const float*>(rope_sin);
  a.q_out = Q_out;
  a.kp = c.k_page_stride * bytes, a.kh = c.k_head_stride * bytes, a.kr = c.k_row_stride * bytes;
  a.vp = c.v_page_stride * bytes, a.vh = c.v_head_stride * bytes, a.vr = c.v_row_stride * bytes;
  a.B = static_cast<int>(batch);
  a.heads = static_cast<uint32_t>(heads);
  a.T = static_cast<uint32_t>(tokens);
  a.n_heads = static_cast<int>(n_heads);
  a.n_kv = static_cast<int>(c.n_kv_heads);
  a.width = static_cast<int>(c.table_pages);
  a.n_pages = static_cast<int>(c.n_pages);
  a.shift = P == 16 ? 4 : P == 32 ? 5 : P == 64 ? 6 : P == 128 ? 7 : 8;
  a.rope_rows = rope_cos != nullptr ? static_cast<int>(rope_rows) : 0;
  a.R = rope_cos != nullptr ? static_cast<int>(rope_dim) : 0;
  a.tasks = static_cast<uint32_t>(tasks);
  a.spans = static_cast<uint32_t>(spans);
  a.head_blocks = static_cast<unsigned>(head_blocks);
  a.eps = eps;
  a.interleaved = interleaved != 0;
  const dim3 grid(static_cast<unsigned>(blocks));
  const hipError_t e = dtype == 0 ? (c.head_dim == 64 ? launch_append<Half, 64>(a, q8, grid, stream)
                                                      : launch_append<Half, 128>(a, q8, grid, stream))
                                  : (c.head_dim == 64 ? launch_append<Bfloat, 64>(a, q8, grid, stream)
                                                      : launch_append<Bfloat, 128>(a, q8, grid, stream));
  if (e != hipSuccess) return hip_fail(e, "paged append kernel launch");
  return ok();
}

extern "C" int nibble_paged_values(const nibble_paged_cache* cache, int64_t dtype, int64_t batch,
                                   const void* lengths, int64_t rows, void* K_out, void* V_out,
                                   void* stream_) {
  const int rc = check_paged(cache, dtype, batch);
  if (rc != NIBBLE_OK) return rc;
  const nibble_paged_cache& c = *cache;
  NIBBLE_CHECK(rows >= 0 && rows < (int64_t(1) << 30), "rows must be in [0, 2^30), got %lld",
               (long long)rows);
  if (batch == 0 || rows == 0) return ok();
  NIBBLE_CHECK(K_out != nullptr && V_out != nullptr && lengths != nullptr, "null pointer");
  NIBBLE_CHECK(aligned(K_out, 16) && aligned(V_out, 16), "outputs must be 16-byte aligned");
  NIBBLE_CHECK(aligned(lengths, 4), "lengths must be 4-byte aligned");
  ValuesArgs a;
  const int64_t units = batch * c.n_kv_heads * rows * (c.head_dim / 16);
  NIBBLE_CHECK(units < (int64_t(1) << 32) - kPagedThreads, "too many rows: %lld x %lld x %lld",
               (long long)batch, (long long)c.n_kv_heads, (long long)rows);
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  DeviceGuard guard;
  int dev = 0;
  NIBBLE_HIP(guard.enter(stream, &dev));
  const int64_t bytes = c.k_scales != nullptr ? 1 : 2, P = c.page_rows;
  a.k = static_cast<const char*>(c.K);
  a.v = static_cast<const char*>(c.V);
  a.k_scales = static_cast<const uint8_t*>(c.k_scales);
  a.v_scales = static_cast<const uint8_t*>(c.v_scales);
  a.table = static_cast<const int32_t*>(c.table);
  a.lengths = static_cast<const int32_t*>(lengths);
  a.k_out = K_out;
  a.v_out = V_out;
  a.kp = c.k_page_stride * bytes, a.kh = c.k_head_stride * bytes, a.kr = c.k_row_stride * bytes;
  a.vp = c.v_page_stride * bytes, a.vh = c.v_head_stride * bytes, a.vr = c.v_row_stride * bytes;
  a.units = static_cast<uint32_t>(units);
  a.n_kv = static_cast<uint32_t>(c.n_kv_heads);
  a.rows = static_cast<uint32_t>(rows);
  a.width = static_cast<int>(c.table_pages);
  a.n_pages = static_cast<int>(c.n_pages);
  a.shift = P == 16 ? 4 : P == 32 ? 5 : P == 64 ? 6 : P == 128 ? 7 : 8;
  const hipError_t e = dtype == 0 ? launch_values<Half>(a, static_cast<int>(c.head_dim), stream)
                                  : launch_values<Bfloat>(a, static_cast<int>(c.head_dim), stream);
  if (e != hipSuccess) return hip_fail(e, "paged values kernel launch");
  return ok();
}
