// Attention of a tree of drafted tokens over a KV cache.
//
// Sequence b holds lengths[b] tokens before the call; its tree's sizes[b]
// tokens lie in the cache rows behind them.  Query head h of tree token i sees
// every row before the tree and the tree rows its mask row names (itself and
// its ancestors), or, without a mask, those up to its own:
//   out = sum_t p(t) v(t) / sum_t p(t),  p(t) = exp(scale q . k(t) - top),
// in one pass over the rows with a running top and running sums in fp32.  A
// token that sees nothing, and tokens behind a sequence's last, give zeros.
//
// The queries of a kv head's group (tokens x query heads, `rows`) go to the
// matrix cores together.  A 16x16x32 product takes keys as rows and queries as
// columns, so lane (g = l / 16, c = l % 16) gets the scores of query c for keys
// 4g .. 4g + 3 of a 16-key tile: a query's statistics need two lane swaps, and
// its probabilities are already where the second product (V^T P^T, queries as
// columns again) wants them, if that product's k index runs over a lane's keys
// of two tiles in turn.  V is read transposed from LDS (ds_read_b64_tr_b16).
#include <algorithm>
#include <cmath>

#include "nibble_common.h"
#include "nibble_copy.h"
#include "nibble_reduce.h"

namespace nibble {
namespace {

constexpr int kTreeThreads = 256;
constexpr int kTreeKeys = 64;  // keys of a tile
constexpr int kTreeMaxSplits = 64;
constexpr float kLog2e = 1.4426950408889634f;
// A query's reference maximum moves only when a score passes it by this much
// (in powers of two): until then its probabilities stay below 2^8, which the
// 16-bit types hold, and its sums need no rescaling.
constexpr float kTreeSlack = 8.0f;

struct TreeArgs {
  const void* q;  // [B, T, n_heads, D]
  const void* k;  // element (b, h, s, d) at b kb + h kh + s ks + d
  const void* v;
  const int32_t* lengths;  // [B]
  const int32_t* sizes;    // [B] or null: T each
  const uint8_t* mask;     // [B or 1, T, T] or null: causal
  void* out;               // [B, T, n_heads, D]
  float* partial;          // [B n_kv][splits][rows][D], then [..][2] (top, sum), when splits > 1
  int64_t kb, kh, ks, vb, vh, vs;
  int64_t mask_batch;  // bytes between two sequences' masks
  int B, T, n_heads, n_kv, qpk, seq;
  int splits, row_tiles;
  float scale;  // its magnitude times log2(e); 1 for a scale of zero
  float sign;   // its sign
};

// Unit (16 bytes) u of LDS row r lies at unit u ^ tree_swizzle(r): eight rows of
// a K read, and four rows' 32-byte pieces of a V read, cover 32 banks once.
template <int UNITS>
__device__ __forceinline__ int tree_swizzle(int r) {
  return ((r & 3) << 1 | (r >> 2 & 1) | (r & 8)) & (UNITS - 1);
}

// A lane's value and the one of the lane 32 (16) away, in either order.
struct Pair {
  float a, b;
};
template <int DIST>
__device__ __forceinline__ Pair swap_pair(float v) {
  const uint32_t i = __builtin_bit_cast(uint32_t, v);
  const auto r = DIST == 32 ? __builtin_amdgcn_permlane32_swap(i, i, false, false)
                            : __builtin_amdgcn_permlane16_swap(i, i, false, false);
  const uint32_t x = r[0], y = r[1];  // (a bit cast of r[1] itself takes r[0])
  return {__builtin_bit_cast(float, x), __builtin_bit_cast(float, y)};
}
__device__ __forceinline__ float swap_max(float v) {
  const Pair a = swap_pair<32>(v);
  const Pair b = swap_pair<16>(fmaxf(a.a, a.b));
  return fmaxf(b.a, b.b);
}
__device__ __forceinline__ float swap_sum(float v) {
  const Pair a = swap_pair<32>(v);
  const Pair b = swap_pair<16>(a.a + a.b);
  return b.a + b.b;
}

// What of sequence b there is: cached tokens and tree tokens within the cache.
struct TreeSpan {
  int len, live, total;
  __device__ __forceinline__ TreeSpan(const TreeArgs& a, int b) {
    len = min(max(a.lengths[b], 0), a.seq);
    live = a.sizes != nullptr ? min(max(a.sizes[b], 0), a.T) : a.T;
    total = min(len + live, a.seq);
  }
};

// One workgroup: 16 QT WQ query rows of one kv head (WQ = 4 / WK waves along
// the rows, WK along the keys), one split of the cached rows, in tiles of 64
// keys.  A tile's rows of k and v are copied straight into one of two LDS
// buffers while the tile before it is computed; two workgroups share a CU, so
// one's softmax runs beside the other's products.
template <class E, int D, int QT, int WK>
__global__ __launch_bounds__(kTreeThreads, 2) void tree_kernel(TreeArgs a) {
  using T = typename E::type;
  using vec8 = typename E::vec8;
  constexpr int WQ = 4 / WK, KT = kTreeKeys, ROWS = 16 * QT * WQ;
  constexpr int KPW = KT / WK < 32 ? KT / WK : 32;    // keys of a wave's step: 16 or 32
  constexpr int KS = KPW / 16, STEPS = KT / (KPW * WK);
  constexpr int UNITS = D / 8;                        // 16-byte units of a row
  constexpr int COPIES = KT * UNITS / kTreeThreads;   // of K or V, a wave and tile
  constexpr int CROWS = 64 / UNITS;                   // rows of a copy
  typedef short s4_t __attribute__((ext_vector_type(4)));
  typedef short s8_t __attribute__((ext_vector_type(8)));
  typedef __attribute__((address_space(3))) s4_t lds4_t;
  __shared__ __attribute__((aligned(16))) T kv[2][2][KT * D];  // buffer, k or v
  __shared__ float stat[2][WK][WQ * QT * 16];
  static_assert(sizeof(kv) >= sizeof(float) * WK * WQ * 16 * D, "the sums fit");

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  const int wq = wave / WK, wk = wave % WK;
  const int g = lane >> 4, c = lane & 15;
  // Workgroup -> (sequence and kv head, split), row tile: the row tiles that
  // read the same cache rows run on one XCD (id % 8) and share its L2.
  const int slot = blockIdx.x >> 3;
  const int pair = slot / a.row_tiles * 8 + (blockIdx.x & 7);
  if (pair >= a.B * a.n_kv * a.splits) return;
  const int row_tile = a.row_tiles - 1 - slot % a.row_tiles;  // the longest of a run first
  const int unit = pair / a.splits, split = pair - unit * a.splits;
  const int b = unit / a.n_kv, h = unit - b * a.n_kv;
  const TreeSpan span(a, b);
  const int rows_all = a.T * a.qpk, rows = span.live * a.qpk;
  const int r0 = row_tile * ROWS;
  const int rw = r0 + wq * 16 * QT;  // this wave's first row

  // Keys up to `end` matter to this workgroup, of which this split takes
  // [first, last), whole tiles of them.
  int end = r0 < rows ? span.total : 0;
  if (a.mask == nullptr && end > 0)
    end = min(end, span.len + (min(r0 + ROWS, rows) - 1) / a.qpk + 1);
  const int tiles = (end + KT - 1) / KT, per = (tiles + a.splits - 1) / a.splits;
  const int first = min(split * per, tiles) * KT, last = min(end, min((split + 1) * per, tiles) * KT);

  const T* const kbase = static_cast<const T*>(a.k) + b * a.kb + h * a.kh;
  const T* const vbase = static_cast<const T*>(a.v) + b * a.vb + h * a.vh;
  const uint32_t lds0 = lds_address(kv) + wave * COPIES * 1024u;
  const uint32_t kpitch = static_cast<uint32_t>(a.ks) * 2u, vpitch = static_cast<uint32_t>(a.vs) * 2u;
  constexpr uint32_t kTile = KT * D * 2;  // bytes of a tile of k or v
  auto copy = [&](int key0, int buf) {
    // Rows behind the sequence's last read as zeros.
    const int here = last - key0;
    const T* const kt = kbase + key0 * a.ks;
    const T* const vt = vbase + key0 * a.vs;
#pragma unroll
    for (int u = 0; u < COPIES; ++u) {
      const int r = (wave * COPIES + u) * CROWS + lane / UNITS;
      const uint32_t unit16 = ((lane % UNITS) ^ tree_swizzle<UNITS>(r)) * 16u;
      const uint32_t dst = lds0 + buf * 2 * kTile + u * 1024u;
      lds_copy16(kt, 0x7fffffffu, dst, r < here ? r * kpitch + unit16 : kOutOfRange);
      lds_copy16(vt, 0x7fffffffu, dst + kTile, r < here ? r * vpitch + unit16 : kOutOfRange);
    }
  };
  if (first < last) copy(first, 0);

  // Queries: lane (g, c) holds elements 32 s + 8 g .. + 7 of row c of a tile.
  vec8 q[QT][D / 32];
  int node[QT];
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const int r = rw + 16 * t + c;
    const bool in = r < rows;
    node[t] = in ? r / a.qpk : 0;
    const int64_t at = ((static_cast<int64_t>(b) * a.T + node[t]) * a.n_heads + h * a.qpk +
                        (in ? r - node[t] * a.qpk : 0)) * D + 8 * g;
#pragma unroll
    for (int s = 0; s < D / 32; ++s)
      q[t][s] = in ? *reinterpret_cast<const vec8*>(static_cast<const T*>(a.q) + at + 32 * s)
                   : vec8{};
  }
  if (a.sign != 1.0f) {  // a scale that is not positive: its sign goes into q, exactly
#pragma unroll
    for (int t = 0; t < QT; ++t)
#pragma unroll
      for (int s = 0; s < D / 32; ++s)
#pragma unroll
        for (int i = 0; i < 8; ++i)
          q[t][s][i] = static_cast<T>(static_cast<float>(q[t][s][i]) * a.sign);
  }

  f4_t acc[QT][D / 16];
  float top[QT], sum[QT];  // of query c, top times the scale; sum over this lane's keys
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    top[t] = -INFINITY;
    sum[t] = 0.0f;
#pragma unroll
    for (int d = 0; d < D / 16; ++d) acc[t][d] = f4_t{0.0f, 0.0f, 0.0f, 0.0f};
  }

  // Byte offsets within a tile (rows 16 apart share the swizzle): of row c, k
  // elements 8 g .. of each 32; of row 4 g + c / 4, v elements 4 (c % 4) .. of
  // each 16.
  const int krow = c * D * 2 + ((g ^ tree_swizzle<UNITS>(c)) * 16);
  const int vr = 4 * g + (c >> 2);
  const int vrow = vr * D * 2 + (((c >> 1 & 1) ^ tree_swizzle<UNITS>(vr)) * 16) + (c & 1) * 8;
  int buf = 0;
  for (int key0 = first; key0 < last; key0 += KT, buf ^= 1) {
    __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));
    lds_barrier();
    if (key0 + KT < last) copy(key0 + KT, buf ^ 1);
    const char* const kt = reinterpret_cast<const char*>(kv[buf][0]);
    const uint32_t vt = lds_address(kv[buf][1]);
#pragma unroll
    for (int st = 0; st < STEPS; ++st) {
      const int kb = (st * WK + wk) * KPW;  // this step's first key in the tile
      f4_t s[KS][QT];
#pragma unroll
      for (int kt16 = 0; kt16 < KS; ++kt16) {
#pragma unroll
        for (int t = 0; t < QT; ++t) s[kt16][t] = f4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int ss = 0; ss < D / 32; ++ss) {
          const vec8 ka = *reinterpret_cast<const vec8*>(kt + (kb + 16 * kt16) * D * 2 +
                                                         (krow ^ (64 * ss)));
#pragma unroll
          for (int t = 0; t < QT; ++t) s[kt16][t] = E::mfma(ka, q[t][ss], s[kt16][t]);
        }
      }
      const bool tail = key0 + kb + KPW > span.len;
      if (tail) {
        const int k0 = key0 + kb + 4 * g;  // key of s[0][.][0]
#pragma unroll
        for (int t = 0; t < QT; ++t)
#pragma unroll
          for (int i = 0; i < 4 * KS; ++i) {
            const int key = k0 + 16 * (i / 4) + i % 4, other = key - span.len;
            bool seen = key < last;
            if (seen && other >= 0)
              seen = a.mask == nullptr
                         ? other <= node[t]
                         : a.mask[b * a.mask_batch + static_cast<int64_t>(node[t]) * a.T + other] != 0;
            if (!seen) s[i / 4][t][i % 4] = -INFINITY;
          }
      }
      vec8 p[QT];
#pragma unroll
      for (int t = 0; t < QT; ++t) {
        float m = s[0][t][0];
#pragma unroll
        for (int i = 1; i < 4 * KS; ++i) m = fmaxf(m, s[i / 4][t][i % 4]);
        m = swap_max(m) * a.scale;
        if (__any(m > top[t] + kTreeSlack)) {
          const float up = fmaxf(m, top[t]);
          const float keep = up == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(top[t] - up);
          top[t] = up;
          sum[t] *= keep;
#pragma unroll
          for (int d = 0; d < D / 16; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[t][d][i] *= keep;
        }
        const float base = top[t] == -INFINITY ? 0.0f : top[t];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float e = i < 4 * KS
                              ? __builtin_amdgcn_exp2f(__builtin_fmaf(s[i / 4 % KS][t][i % 4], a.scale, -base))
                              : 0.0f;
          sum[t] += e;
          p[t][i] = static_cast<T>(e);
        }
      }
      // A masked row's infinity or NaN must not meet its zero probability.
      bool strange = false;
#pragma unroll
      for (int d = 0; d < D / 16; ++d) {
        s4_t v2[2] = {};
#pragma unroll
        for (int kt16 = 0; kt16 < KS; ++kt16)
          v2[kt16] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (lds4_t*)(uintptr_t)(vt + (kb + 16 * kt16) * D * 2 + (vrow ^ (32 * d))));
        s8_t vv = {v2[0][0], v2[0][1], v2[0][2], v2[0][3], v2[1][0], v2[1][1], v2[1][2], v2[1][3]};
        if (tail) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if ((vv[i] & E::kExponent) == E::kExponent) {
              strange = true;
              vv[i] = 0;
            }
        }
#pragma unroll
        for (int t = 0; t < QT; ++t)
          acc[t][d] = E::mfma(__builtin_bit_cast(vec8, vv), p[t], acc[t][d]);
      }
      if (tail && __any(strange)) {
        // Key by key, the rows that see the key only.
        for (int kk = 0; kk < KPW; ++kk) {
          const int from = (kk % 16 / 4) * 16 + c, i = kk / 16 * 4 + kk % 4;
          const int r = kb + kk;
#pragma unroll
          for (int t = 0; t < QT; ++t) {
            float w = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (e == i) w = static_cast<float>(p[t][e]);
            w = __shfl(w, from);
#pragma unroll
            for (int d = 0; d < D / 16; ++d)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int dim = 16 * d + 4 * g + e;
                const T x = kv[buf][1][r * D + ((dim / 8) ^ tree_swizzle<UNITS>(r)) * 8 + dim % 8];
                const bool odd = (__builtin_bit_cast(unsigned short, x) & E::kExponent) == E::kExponent;
                if (odd && w != 0.0f) acc[t][d][e] += w * static_cast<float>(x);
              }
          }
        }
      }
    }
  }
  __syncthreads();

  // The waves along the keys meet: statistics first, then the sums on the
  // common maximum, 16 rows of each wave at a time through LDS.
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    sum[t] = swap_sum(sum[t]);
    if (rw + 16 * t + c >= rows) top[t] = -INFINITY, sum[t] = 0.0f;  // behind the last token
    if (g == 0) {
      stat[0][wk][(wq * QT + t) * 16 + c] = top[t];
      stat[1][wk][(wq * QT + t) * 16 + c] = sum[t];
    }
  }
  __syncthreads();
  float* const red = reinterpret_cast<float*>(&kv[0][0][0]);  // [WK][WQ 16][D]
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    float m = stat[0][0][(wq * QT + t) * 16 + c];
#pragma unroll
    for (int w = 1; w < WK; ++w) m = fmaxf(m, stat[0][w][(wq * QT + t) * 16 + c]);
    const float mine = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(top[t] - m);
#pragma unroll
    for (int d = 0; d < D / 16; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        red[(wk * WQ * 16 + wq * 16 + c) * D + 16 * d + 4 * g + i] = acc[t][d][i] * mine;
    __syncthreads();
    for (int e = threadIdx.x; e < WQ * 16 * (D / 4); e += kTreeThreads) {
      const int rr = e / (D / 4), d = e % (D / 4) * 4;
      const int slot16 = (rr / 16 * QT + t) * 16 + rr % 16;
      const int r = r0 + rr / 16 * 16 * QT + 16 * t + rr % 16;
      if (r >= rows_all) continue;
      f4_t o = *reinterpret_cast<const f4_t*>(&red[rr * D + d]);
      float mr = stat[0][0][slot16];
#pragma unroll
      for (int w = 1; w < WK; ++w) {
        o += *reinterpret_cast<const f4_t*>(&red[(w * WQ * 16 + rr) * D + d]);
        mr = fmaxf(mr, stat[0][w][slot16]);
      }
      float l = 0.0f;
#pragma unroll
      for (int w = 0; w < WK; ++w)
        l += mr == -INFINITY ? 0.0f
                             : stat[1][w][slot16] * __builtin_amdgcn_exp2f(stat[0][w][slot16] - mr);
      if (a.splits == 1) {
        const int i = r / a.qpk;
        T* out = static_cast<T*>(a.out) +
                 ((static_cast<int64_t>(b) * a.T + i) * a.n_heads + h * a.qpk + (r - i * a.qpk)) * D + d;
        typedef T vec4 __attribute__((ext_vector_type(4)));
        vec4 y;
#pragma unroll
        for (int x = 0; x < 4; ++x) y[x] = static_cast<T>(l == 0.0f ? 0.0f : o[x] / l);
        *reinterpret_cast<vec4*>(out) = y;
      } else {
        const int64_t rec = (static_cast<int64_t>(unit) * a.splits + split) * rows_all + r;
        *reinterpret_cast<f4_t*>(a.partial + rec * D + d) = o;
        if (d == 0) {
          float* st = a.partial +
                      static_cast<int64_t>(a.B) * a.n_kv * a.splits * rows_all * D + rec * 2;
          st[0] = mr;
          st[1] = l;
        }
      }
    }
    __syncthreads();
  }
}

// Joins the splits of a row: one group of D / 4 lanes a row.
template <class E, int D>
__global__ __launch_bounds__(kTreeThreads) void tree_join_kernel(TreeArgs a) {
  using T = typename E::type;
  const int rows_all = a.T * a.qpk;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (kTreeThreads / (D / 4)) +
                      threadIdx.x / (D / 4);
  const int64_t units = static_cast<int64_t>(a.B) * a.n_kv;
  if (row >= units * rows_all) return;
  const int d = threadIdx.x % (D / 4) * 4;
  const int64_t unit = row / rows_all;
  const int r = static_cast<int>(row - unit * rows_all);
  const float* st = a.partial + units * a.splits * rows_all * D;
  const int64_t rec0 = unit * a.splits * rows_all + r;
  float m = -INFINITY;
  for (int s = 0; s < a.splits; ++s)
    m = fmaxf(m, st[(rec0 + static_cast<int64_t>(s) * rows_all) * 2]);
  f4_t o = {0.0f, 0.0f, 0.0f, 0.0f};
  float l = 0.0f;
  for (int s = 0; s < a.splits; ++s) {
    const int64_t rec = rec0 + static_cast<int64_t>(s) * rows_all;
    const float x = st[rec * 2];
    if (x == -INFINITY) continue;  // saw nothing: its sums are zeros
    const float w = __builtin_amdgcn_exp2f(x - m);
    l += st[rec * 2 + 1] * w;
    const f4_t v = *reinterpret_cast<const f4_t*>(a.partial + rec * D + d);
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] += v[i] * w;
  }
  const int i = r / a.qpk;
  const int b = static_cast<int>(unit / a.n_kv), h = static_cast<int>(unit - b * a.n_kv);
  typedef T vec4 __attribute__((ext_vector_type(4)));
  vec4 y;
#pragma unroll
  for (int x = 0; x < 4; ++x) y[x] = static_cast<T>(l == 0.0f ? 0.0f : o[x] / l);
  *reinterpret_cast<vec4*>(static_cast<T*>(a.out) +
                           ((static_cast<int64_t>(b) * a.T + i) * a.n_heads + h * a.qpk +
                            (r - i * a.qpk)) * D + d) = y;
}

struct TreePlan {
  int qt = 1, wk = 4, rows = 16, row_tiles = 1, splits = 1;
  size_t workspace_bytes = 0;
};

int plan_tree(int64_t batch, int64_t tokens, int64_t n_heads, int64_t n_kv, int64_t head_dim,
              int64_t max_seq, TreePlan* p) {
  NIBBLE_CHECK(head_dim == 64 || head_dim == 128, "head_dim must be 64 or 128, got %lld",
               (long long)head_dim);
  NIBBLE_CHECK(n_kv >= 1 && n_kv <= 65535, "n_kv_heads must be in [1, 65535], got %lld",
               (long long)n_kv);
  NIBBLE_CHECK(n_heads >= n_kv && n_heads <= 65535 && n_heads % n_kv == 0,
               "n_heads (%lld) must be a multiple of n_kv_heads (%lld), at most 65535",
               (long long)n_heads, (long long)n_kv);
  NIBBLE_CHECK(batch >= 0 && tokens >= 0 && batch <= 65535 && tokens <= (1 << 20),
               "batch must be in [0, 65535] and tokens in [0, 2^20]");
  NIBBLE_CHECK(max_seq >= 0 && max_seq < (int64_t(1) << 30), "max_seq must be in [0, 2^30), got %lld",
               (long long)max_seq);
  if (batch == 0 || tokens == 0) return NIBBLE_OK;
  const int64_t rows = tokens * (n_heads / n_kv);
  NIBBLE_CHECK(rows * batch * n_kv <= (int64_t(1) << 30), "more than 2^30 query rows");
  p->qt = rows <= 16 ? 1 : 2;
  p->wk = rows <= 32 ? 4 : rows <= 64 ? 2 : 1;
  p->rows = 16 * p->qt * (4 / p->wk);
  p->row_tiles = static_cast<int>(ceil_div(rows, p->rows));
  const int64_t units = batch * n_kv * p->row_tiles;
  // As many splits as make two rounds of the CUs, each of two tiles at least.
  const int64_t tiles = ceil_div(std::max<int64_t>(max_seq, 1), kTreeKeys);
  int64_t splits = std::min<int64_t>({ceil_div(512, units), ceil_div(tiles, 2), kTreeMaxSplits});
  p->splits = static_cast<int>(std::max<int64_t>(splits, 1));
  if (p->splits > 1)
    p->workspace_bytes = static_cast<size_t>(batch * n_kv * p->splits * rows) * (head_dim + 2) * 4;
  return NIBBLE_OK;
}

template <class E, int D>
hipError_t launch_tree(const TreeArgs& a, const TreePlan& p, hipStream_t stream) {
  const int64_t pairs = static_cast<int64_t>(a.B) * a.n_kv * p.splits;
  const dim3 grid(static_cast<unsigned>(ceil_div(pairs, 8) * 8 * p.row_tiles));
  if (p.qt == 1) tree_kernel<E, D, 1, 4><<<grid, kTreeThreads, 0, stream>>>(a);
  else if (p.wk == 4) tree_kernel<E, D, 2, 4><<<grid, kTreeThreads, 0, stream>>>(a);
  else if (p.wk == 2) tree_kernel<E, D, 2, 2><<<grid, kTreeThreads, 0, stream>>>(a);
  else tree_kernel<E, D, 2, 1><<<grid, kTreeThreads, 0, stream>>>(a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.splits == 1) return e;
  const int64_t rows = static_cast<int64_t>(a.B) * a.n_kv * a.T * a.qpk;
  tree_join_kernel<E, D><<<dim3(static_cast<unsigned>(ceil_div(rows, kTreeThreads / (D / 4)))),
                           kTreeThreads, 0, stream>>>(a);
  return hipGetLastError();
}

}  // namespace
}  // namespace nibble

using namespace nibble;

extern "C" size_t nibble_attention_tree_workspace_bytes(int64_t batch, int64_t tokens,
                                                        int64_t n_heads, int64_t n_kv_heads,
                                                        int64_t head_dim, int64_t max_seq) {
  TreePlan p;
  if (plan_tree(batch, tokens, n_heads, n_kv_heads, head_dim, max_seq, &p) != NIBBLE_OK) return 0;
  return p.workspace_bytes;
}

extern "C" int nibble_attention_tree(const void* Q, int64_t dtype, int64_t batch, int64_t tokens,
                                     int64_t n_heads, int64_t n_kv_heads, int64_t head_dim,
                                     const void* K_cache, int64_t k_batch_stride,
                                     int64_t k_head_stride, int64_t k_row_stride,
                                     const void* V_cache, int64_t v_batch_stride,
                                     int64_t v_head_stride, int64_t v_row_stride, int64_t max_seq,
                                     const void* lengths, const void* mask, int64_t mask_batches,
                                     const void* sizes, float scale, void* Out, void* workspace,
                                     size_t workspace_bytes, void* stream_) {
  NIBBLE_CHECK(dtype == 0 || dtype == 1, "dtype must be 0 (fp16) or 1 (bf16), got %lld",
               (long long)dtype);
  TreePlan p;
  const int rc = plan_tree(batch, tokens, n_heads, n_kv_heads, head_dim, max_seq, &p);
  if (rc != NIBBLE_OK) return rc;
  NIBBLE_CHECK(std::isfinite(scale), "scale must be finite");
  if (batch == 0 || tokens == 0) return ok();
  for (int64_t s : {k_batch_stride, k_head_stride, k_row_stride, v_batch_stride, v_head_stride,
                    v_row_stride})
    NIBBLE_CHECK(s >= 0 && s % 8 == 0, "cache strides must be multiples of 8 elements, got %lld",
                 (long long)s);
  // 32-bit offsets within the rows of one tile
  NIBBLE_CHECK(k_row_stride <= (1 << 22) && v_row_stride <= (1 << 22),
               "row strides must be at most 2^22 elements");
  NIBBLE_CHECK(mask == nullptr || mask_batches == 1 || mask_batches == batch,
               "the mask must have 1 or %lld batches, got %lld", (long long)batch,
               (long long)mask_batches);
  NIBBLE_CHECK(Q != nullptr && Out != nullptr && lengths != nullptr &&
                   (max_seq == 0 || (K_cache != nullptr && V_cache != nullptr)),
               "null pointer");
  NIBBLE_CHECK(aligned(Q, 16) && aligned(K_cache, 16) && aligned(V_cache, 16) && aligned(Out, 16),
               "q, caches and output must be 16-byte aligned");
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
  TreeArgs a;
  a.q = Q;
  a.k = K_cache;
  a.v = V_cache;
  a.lengths = static_cast<const int32_t*>(lengths);
  a.sizes = static_cast<const int32_t*>(sizes);
  a.mask = static_cast<const uint8_t*>(mask);
  a.out = Out;
  a.partial = static_cast<float*>(workspace);
  a.kb = k_batch_stride, a.kh = k_head_stride, a.ks = k_row_stride;
  a.vb = v_batch_stride, a.vh = v_head_stride, a.vs = v_row_stride;
  a.mask_batch = mask_batches == 1 ? 0 : tokens * tokens;
  a.B = static_cast<int>(batch);
  a.T = static_cast<int>(tokens);
  a.n_heads = static_cast<int>(n_heads);
  a.n_kv = static_cast<int>(n_kv_heads);
  a.qpk = static_cast<int>(n_heads / n_kv_heads);
  a.seq = static_cast<int>(max_seq);
  a.splits = p.splits;
  a.row_tiles = p.row_tiles;
  a.scale = scale == 0.0f ? 1.0f : std::fabs(scale) * kLog2e;
  a.sign = scale > 0.0f ? 1.0f : scale < 0.0f ? -1.0f : 0.0f;
  const hipError_t e = dtype == 0 ? (head_dim == 64 ? launch_tree<Half, 64>(a, p, stream)
                                                    : launch_tree<Half, 128>(a, p, stream))
                                  : (head_dim == 64 ? launch_tree<Bfloat, 64>(a, p, stream)
                                                    : launch_tree<Bfloat, 128>(a, p, stream));
  if (e != hipSuccess) return hip_fail(e, "tree attention kernel launch");
  return ok();
}
