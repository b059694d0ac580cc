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
//
// What it reads, writes and computes: the cached rows once a kv head and 128
// query rows, 4 rows keys D operations, and, where the rows are split, D + 2
// floats a query row and share.  Times are of 32 heads on 8, head_dim 128.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "nibble_common.h"
#include "nibble_copy.h"
#include "nibble_split.h"

namespace nibble {
namespace {

constexpr int kTreeThreads = 256;
constexpr int kTreeKeys = 64;        // keys of a tile
// What a share more costs, in the time of a tile: the join's turn, and a query
// row's sums written and read again.  us with these / with as many shares as there
// is room for: 1 x 100 tokens (32 heads on 8) over 1000 21.8 / 27.7, 1 x 64 over 4000
// 27 / 30, 1 x 16 over 8000 20 / 25.5, 4 x 30 over 1000 23.8 / 29.4, 1 x 1 over 4000
// 10.6 / 13.9 (13.8 with half the first); half the second -7 to +19%, twice it 2 to
// 14% slower.
constexpr float kTreeShareCost = 0.08f, kTreeRowCost = 4.8e-4f;
// Probabilities are relative to a query's reference, 2^lift below a maximum.  It
// moves only when a score passes that maximum by more than the slack (in powers of
// two): until then they are at most 2^(slack + lift), and the sums need no
// rescaling.  fp16 ends at 2^16 and has steps of 2^-24 at least, so its reference
// lies as low as it can: weights down to 2^-21 of the largest keep all their bits,
// and thousands of 2^-25, which a sink leaves to the rest, are not lost.  (A slack
// of 4 and a lift of 11: 4 x 8 tokens over 3000, 32 heads of 64 on 4, 16.2 us in
// place of 15.7; 16 x 27 over 8100 105.8 in place of 103.)  bf16 has the range of
// fp32.  The slack is measured by a difference, which is exact: a sum would round to
// the steps of a large maximum.  (Below 2^28, in powers of two, that is; beyond it a
// score's own rounding in fp32 passes what fp16 has left.)
constexpr float kTreeSlack = 8.0f;
template <class E>
constexpr float kTreeLift = std::is_same_v<E, Half> ? 7.0f : 0.0f;

struct TreeArgs {
  const void* q;  // [B, T, n_heads, D]
  const void* k;  // element (b, h, s, d) at b kb + h kh + s ks + d
  const void* v;
  const int32_t* lengths;  // [B]
  const int32_t* sizes;    // [B] or null: T each
  const uint8_t* mask;     // [B or 1, T, T] or null: causal
  void* out;               // [B, T, n_heads, D]
  float* partial;          // [n_kv][shares][rows][D], then [..][2] (top, sum), when shares > 0
  int* runs;               // [B][2]: a sequence's first share and their number
  int64_t kb, kh, ks, vb, vh, vs;
  int64_t mask_batch;  // bytes between two sequences' masks
  int B, T, n_heads, n_kv, qpk, seq;
  int shares, row_tiles;  // shares: 0 where no sequence's rows are split
  float join_cost;        // of one share, in tiles
  bool fold;              // row tiles from both ends to the middle
  float scale;  // its magnitude times log2(e); 1 for a scale of zero
  float sign;   // its sign
  __device__ int tiles(int b) const;  // of a sequence's rows
};

// Unit (16 bytes) u of LDS row r lies at unit u ^ tree_swizzle(r): eight rows of
// a K read, and four rows' 32-byte pieces of a V read, cover 32 banks once.
template <int UNITS>
__device__ __forceinline__ int tree_swizzle(int r) {
  return ((r & 3) << 1 | (r >> 2 & 1) | (r & 8)) & (UNITS - 1);
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
__device__ __forceinline__ int TreeArgs::tiles(int b) const {
  return (TreeSpan(*this, b).total + kTreeKeys - 1) / kTreeKeys;
}

// One workgroup: 16 QT WQ query rows of one kv head (WQ = 4 / WK waves along
// the rows, WK along the keys), one share of the cached rows, in tiles of 64
// keys.  A tile's rows of k and v are copied straight into one of two LDS
// buffers while the tile before it is computed; two workgroups share a CU.
//
// What bounds it: 64 tokens over 65000 take 86 us of this kernel (16 sequences of
// 27 over up to 8100 85, 4.2 TB/s; 2048 over 2048 112, 0.92 PFLOP/s).  A tile of
// a wave is 68 products of 16 cycles and 32 exponentials of 16 beside some 130
// plain vector operations of 4; for the two waves of a SIMD that adds up to 4300
// cycles, and a tile takes 4375: the two hardly overlap.  Neither a priority for
// the products or the softmax, a fixed one by workgroup, nor a late start of one
// of the two changed that (1 to 10% slower).  LDS is busy for 40% of the time.
// Some of it is power: with queries, keys and values of zero, the same
// instructions, 2048 over 2048 take 102 us in place of 121, 64 over 65000 83 in
// place of 100 (with the join).
// Three workgroups a CU (smaller tiles) took 283 us for the last of those, 64
// queries a wave, which would halve the reads of LDS, 519 (registers spilt).  The
// form for 128 rows of head_dim 128 takes all 256 registers and spills 26; its loops
// reach those only in the pass for infinities and NaN.
//
// One call of 16 tokens over 1000 is latency: 8.6 us, of which finding its share
// and loading the queries take 2.3, the copies 0.9, each of two tiles 1.2, the
// meeting of the waves and the stores 2.9 (4.5 with a barrier for each 16 rows).
template <class E, int D, int QT, int WK>
__global__ __launch_bounds__(kTreeThreads, 2) void tree_kernel(TreeArgs a) {
  using T = typename E::type;
  using vec8 = typename E::vec8;
  constexpr int WQ = 4 / WK, ROWS = 16 * QT * WQ;
  constexpr int KT = kTreeKeys, KPW = KT / WK, KS = KPW / 16;  // a wave's keys of a tile
  constexpr int PS = (KS + 1) / 2;                    // products of 32 keys (or 16 and zeros)
  constexpr int UNITS = D / 8;                        // 16-byte units of a row
  constexpr int COPIES = KT * UNITS / kTreeThreads;   // of K or V, a wave and tile
  constexpr int CROWS = 64 / UNITS;                   // rows of a copy
  typedef short s4_t __attribute__((ext_vector_type(4)));
  typedef unsigned short us4_t __attribute__((ext_vector_type(4)));
  typedef unsigned short us8_t __attribute__((ext_vector_type(8)));
  typedef __attribute__((address_space(3))) s4_t lds4_t;
  __shared__ __attribute__((aligned(16))) T kv[2][2][KT * D];  // buffer; k, v
  __shared__ float stat[2][WK][WQ * QT * 16];
  __shared__ int place[WQ * QT * 16];  // of a row's output, in heads
  static_assert(sizeof(kv) >= sizeof(float) * WK * WQ * QT * 16 * D, "the sums fit");

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  const int wq = wave / WK, wk = wave % WK;
  const int g = lane >> 4, c = lane & 15;
  // Workgroup -> (share, kv head), row tile: the row tiles that read the same
  // cache rows run on one XCD (id % 8) and share its L2.  Without a mask the
  // later row tiles are longer: longest first, or, where all are on the CUs at
  // once, two a CU, each with its counterpart.
  const int slot = blockIdx.x >> 3;
  const int pair = slot / a.row_tiles * 8 + (blockIdx.x & 7);
  const int rt = slot % a.row_tiles;
  const int row_tile = a.fold && rt >= (a.row_tiles + 1) / 2 ? rt - (a.row_tiles + 1) / 2
                                                             : a.row_tiles - 1 - rt;
  const int w = pair / a.n_kv, h = pair - w * a.n_kv;
  int b = w, share = 0, per = 0x3fffffff;  // the whole sequence
  if (a.shares > 0) {
    if (w >= a.shares) return;
    const Shares<TreeArgs> shares(a, w);
    if (shares.found < 0) return;
    b = shares.found, share = w - shares.first, per = shares.per;
    // (for the kernel that joins them)
    if (share == 0 && h == 0 && rt == 0 && threadIdx.x == 0)
      a.runs[2 * b] = shares.first, a.runs[2 * b + 1] = shares.count;
  } else if (w >= a.B) {
    return;
  }
  const TreeSpan span(a, b);
  const int rows_all = a.T * a.qpk, rows = span.live * a.qpk;
  const int r0 = row_tile * ROWS;
  const int rw = r0 + wq * 16 * QT;  // this wave's first row

  // Keys up to `end` matter to this workgroup, of which it takes [first, last).
  int end = r0 < rows ? span.total : 0;
  if (a.mask == nullptr && end > 0)
    end = min(end, span.len + (min(r0 + ROWS, rows) - 1) / a.qpk + 1);
  const int tiles = (end + KT - 1) / KT;
  const int first = min(share * per, tiles) * KT;
  const int last = min(end, min(share * per + per, tiles) * KT);
  const int count = (last - first + KT - 1) / KT;  // tiles

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

  const T* const kbase = static_cast<const T*>(a.k) + b * a.kb + h * a.kh;
  const T* const vbase = static_cast<const T*>(a.v) + b * a.vb + h * a.vh;
  constexpr uint32_t kTile = KT * D * 2;  // bytes of a tile of k or v
  const uint32_t lds0 = lds_address(kv) + wave * COPIES * 1024u;
  // This wave's copies of tile i; rows behind the share's last, and whole tiles
  // there, read as zeros.
  auto copy = [&](int i) {
    const int key0 = first + i * KT, here = last - key0, from = here > 0 ? key0 : 0;
    const T* const kt = kbase + from * a.ks;
    const T* const vt = vbase + from * a.vs;
    const uint32_t dst = lds0 + (i & 1) * 2 * kTile;
#pragma unroll
    for (int u = 0; u < COPIES; ++u) {
      const int r = (wave * COPIES + u) * CROWS + lane / UNITS;
      const uint32_t unit16 = ((lane % UNITS) ^ tree_swizzle<UNITS>(r)) * 16u;
      lds_copy16(kt, 0x7fffffffu, dst + u * 1024u,
                 r < here ? r * static_cast<uint32_t>(a.ks) * 2u + unit16 : kOutOfRange);
      lds_copy16(vt, 0x7fffffffu, dst + kTile + u * 1024u,
                 r < here ? r * static_cast<uint32_t>(a.vs) * 2u + unit16 : kOutOfRange);
    }
  };
  copy(0);

  f4_t acc[QT][D / 16];
  float top[QT];  // the reference of query c, in powers of two
  f4_t sum[QT];   // of the probabilities: four copies
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    top[t] = -INFINITY;
    sum[t] = f4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int d = 0; d < D / 16; ++d) acc[t][d] = f4_t{0.0f, 0.0f, 0.0f, 0.0f};
  }

  // Byte offsets within a tile (rows 16 apart share the swizzle): of row c, k
  // elements 8 g .. of each 32; of row 4 g + c / 4, v elements 4 (c % 4) .. of
  // each 16.
  const int krow = c * D * 2 + ((g ^ tree_swizzle<UNITS>(c)) * 16);
  const int vr = 4 * g + (c >> 2);
  const int vrow = vr * D * 2 + (((c >> 1 & 1) ^ tree_swizzle<UNITS>(vr)) * 16) + (c & 1) * 8;
  struct Scores {
    f4_t s[KS][QT];
  };
  auto multiply = [&](Scores& x, int buf) {
    const char* const kt = reinterpret_cast<const char*>(kv[buf][0]) + wk * KPW * D * 2;
#pragma unroll
    for (int j = 0; j < KS; ++j) {
#pragma unroll
      for (int ss = 0; ss < D / 32; ++ss) {
        const vec8 ka = *reinterpret_cast<const vec8*>(kt + j * 16 * D * 2 + (krow ^ (64 * ss)));
#pragma unroll
        for (int t = 0; t < QT; ++t)
          x.s[j][t] = E::mfma(ka, q[t][ss], ss == 0 ? f4_t{0.0f, 0.0f, 0.0f, 0.0f} : x.s[j][t]);
      }
    }
  };
  // What this lane's queries see of a tail's keys, a bit for each of its scores;
  // whether any lane's sees anything.  Four neighbouring keys are four bytes of the
  // mask in one load, from a place in the row, and shifted to theirs.  The choice of
  // loads by T stands in every turn of the loops, so the KS QT loads of a tile wait
  // for one another, ahead of the tile's barrier.  A wave leaves a tile out that it
  // sees nothing of.  (15 trees of 444 tokens 95 to 99 us, 134 with single bytes,
  // loaded behind the products, and no tile left out.)
  uint32_t seen[QT];
  auto look = [&](int i) {
    typedef uint32_t word_t __attribute__((aligned(1)));
    const int k0 = first + i * KT + wk * KPW + 4 * g;  // key of bit 0
    auto upto = [](int n) { return (1u << min(max(n, 0), 4)) - 1u; };
    uint32_t some = 0;
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      const uint8_t* const row =
          a.mask + (a.mask != nullptr
                        ? b * a.mask_batch + static_cast<int64_t>(node[t]) * a.T : 0);
      seen[t] = 0;
#pragma unroll
      for (int j = 0; j < KS; ++j) {
        const int key = k0 + 16 * j, n = key - span.len;
        uint32_t bits;
        if (a.mask != nullptr) {
          uint32_t bytes = 0;
          if (a.T >= 4) {
            const int from = min(max(n, 0), a.T - 4);
            bytes = *reinterpret_cast<const word_t*>(row + from);
            const int by = 8 * min(abs(n - from), 3);  // (farther off: cached keys, or none)
            bytes = n > from ? bytes >> by : bytes << by;
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              bytes |= static_cast<uint32_t>(row[min(max(n + e, 0), a.T - 1)]) << (8 * e);
          }
          // bit 7 of every byte that is not zero, then the four side by side
          const uint32_t on = (((bytes & 0x7f7f7f7fu) + 0x7f7f7f7fu) | bytes) >> 7 & 0x01010101u;
          bits = on * 0x01020408u >> 24 & 15u;
        } else {
          bits = upto(node[t] - n + 1);
        }
        seen[t] |= ((bits | upto(span.len - key)) & upto(last - key)) << (4 * j);
      }
      some |= seen[t];
    }
    return __any(some != 0) != 0;
  };
  auto hide = [&](Scores& x) {
#pragma unroll
    for (int t = 0; t < QT; ++t)
#pragma unroll
      for (int e = 0; e < 4 * KS; ++e)
        if ((seen[t] >> e & 1u) == 0) x.s[e / 4][t][e % 4] = -INFINITY;
  };
  float m[QT];  // the largest of a lane's scores of a query, times the scale
  auto largest = [&](const Scores& x) {
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      m[t] = x.s[0][t][0];
#pragma unroll
      for (int i = 1; i < 4 * KS; ++i) m[t] = fmaxf(m[t], x.s[i / 4][t][i % 4]);
      m[t] *= a.scale;
    }
  };
  auto move = [&]() {
    bool moves = false;
#pragma unroll
    for (int t = 0; t < QT; ++t) moves |= m[t] - top[t] > kTreeSlack + kTreeLift<E>;
    if (!__any(moves)) return;
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      const float up = fmaxf(swap_max(m[t]) - kTreeLift<E>, top[t]);
      const float keep = up == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(top[t] - up);
      top[t] = up;
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[t][i] *= keep;
#pragma unroll
      for (int d = 0; d < D / 16; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[t][d][i] *= keep;
    }
  };
  vec8 p[PS][QT], ones;
#pragma unroll
  for (int i = 0; i < 8; ++i) ones[i] = static_cast<T>(1.0f);
  auto weigh = [&](const Scores& x) {
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      const float base = top[t] == -INFINITY ? 0.0f : top[t];
#pragma unroll
      for (int i = 0; i < 8 * PS; ++i) {
        p[i / 8][t][i % 8] = static_cast<T>(
            i < 4 * KS ? __builtin_amdgcn_exp2f(
                             __builtin_fmaf(x.s[i / 4 % KS][t][i % 4], a.scale, -base))
                       : 0.0f);
      }
      // (The probabilities are rounded to 16 bits because the matrix cores take
      // them so: each is off by half a step at most, in fp16 of 2^-24 at least, and the
      // sum is of the rounded.)
      // The sum of the probabilities as they are multiplied, by the matrix cores
      // too: ones times P^T, a tile's keys at once, in fp32.
#pragma unroll
      for (int j = 0; j < PS; ++j) sum[t] = E::mfma(ones, p[j][t], sum[t]);
    }
  };
  // Whether this wave's v rows of a tile hold an infinity or a NaN.
  auto strange = [&](int i) {
    const u4_t* const vt = reinterpret_cast<const u4_t*>(kv[i & 1][1] + wk * KPW * D);
    us8_t most = {};
#pragma unroll
    for (int e = 0; e < KPW * UNITS / 64; ++e) {
      const u4_t bits = vt[e * 64 + lane] & 0x7fff7fffu;
      most = __builtin_elementwise_max(most, __builtin_bit_cast(us8_t, bits));
    }
    bool odd = false;
#pragma unroll
    for (int e = 0; e < 8; ++e) odd |= most[e] >= E::kExponent;
    return __any(odd) != 0;
  };
  // V^T of 32 keys (16 where a wave has no more) for 16 elements.
  auto values = [&](uint32_t vt, int d, int j) {
    s4_t v2[2] = {};
#pragma unroll
    for (int e = 0; e < (KS == 1 ? 1 : 2); ++e)
      v2[e] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (lds4_t*)(uintptr_t)(vt + (2 * j + e) * 16 * D * 2 + (vrow ^ (32 * d))));
    return us8_t(__builtin_shufflevector(__builtin_bit_cast(us4_t, v2[0]),
                                         __builtin_bit_cast(us4_t, v2[1]), 0, 1, 2, 3, 4, 5, 6, 7));
  };
  // The sums.  A hidden row's infinity or NaN must not meet its zero
  // probability: with `careful` they are left out of the products and counted,
  // over the rows a query sees, by products of their own: infinities of either
  // sign, a NaN as both.  A query and element that met one gets that infinity
  // added, and of both the NaN that they make; a weight that rounds to zero takes
  // neither away (in a tile that all see it makes NaN of an infinity).
  auto add = [&](int buf, auto careful) {
    constexpr bool kCareful = decltype(careful)::value;
    const uint32_t vt = lds_address(kv[buf][1]) + wk * KPW * D * 2;
#pragma unroll
    for (int d = 0; d < D / 16; ++d)
#pragma unroll
      for (int j = 0; j < PS; ++j) {
        us8_t v = values(vt, d, j);
        if constexpr (kCareful) v = (v & E::kExponent) == E::kExponent ? us8_t{} : v;
#pragma unroll
        for (int t = 0; t < QT; ++t)
          acc[t][d] = E::mfma(__builtin_bit_cast(vec8, v), p[j][t], acc[t][d]);
        if constexpr (kCareful) __builtin_amdgcn_sched_barrier(0);  // one at a time: registers
      }
    if constexpr (kCareful) {
#pragma unroll
      for (int j = 0; j < PS; ++j)
#pragma unroll
        for (int t = 0; t < QT; ++t)
#pragma unroll
          for (int e = 0; e < 8; ++e)
            p[j][t][e] = static_cast<T>(
                8 * j + e < 4 * KS && (seen[t] >> (8 * j + e) & 1u) != 0 ? 1.0f : 0.0f);
      const us8_t one = __builtin_bit_cast(us8_t, ones);
#pragma unroll
      for (int d = 0; d < D / 16; ++d)
#pragma unroll
        for (int sign = 0; sign < 2; ++sign) {
          f4_t n[QT] = {};
#pragma unroll
          for (int j = 0; j < PS; ++j) {
            const us8_t v = values(vt, d, j);
            const us8_t inf = us8_t{} + static_cast<unsigned short>(E::kExponent | sign << 15);
            const us8_t is = v == inf || (v & 0x7fff) > E::kExponent ? one : us8_t{};
#pragma unroll
            for (int t = 0; t < QT; ++t) n[t] = E::mfma(__builtin_bit_cast(vec8, is), p[j][t], n[t]);
          }
          const float met = sign == 0 ? INFINITY : -INFINITY;
#pragma unroll
          for (int t = 0; t < QT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[t][d][e] += n[t][e] != 0.0f ? met : 0.0f;
          __builtin_amdgcn_sched_barrier(0);
        }
    }
  };
  // (`buf`, the tile's buffer, is a constant in the plain loop: the reads' addresses
  // then take it in as immediates, 2048 over 2048 125 -> 122 us with the statistics'
  // swaps left to tiles whose maximum moves.)
  auto turn = [&](int i, int buf, auto tail) {
    bool any = true;
    if constexpr (decltype(tail)::value) any = look(i);
    __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));
    lds_barrier();
    copy(i + 1);
    if (!any) return;
    Scores x;
    multiply(x, buf);
    if constexpr (decltype(tail)::value) hide(x);
    largest(x);
    move();
    weigh(x);
    if constexpr (decltype(tail)::value) {
      if (strange(i)) {
        look(i);  // (again, so that its bits need no registers meanwhile: 15 x 444 -2.5%)
        add(buf, std::true_type{});
        return;
      }
    }
    add(buf, std::false_type{});
    // Eight reads of v, the exponentials, then each read two pairs of products
    // ahead of its own.
    __builtin_amdgcn_sched_group_barrier(0x100, 8, 0);
    __builtin_amdgcn_sched_group_barrier(0x402, 64 * PS * QT, 0);
#pragma unroll
    for (int n = 0; n < PS * (D / 16 + 1); ++n) {
      __builtin_amdgcn_sched_group_barrier(0x008, QT, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
    }
  };
  // A tile with rows that some query does not see, or behind the last, is a tail.
  const int common = a.mask != nullptr ? span.len : span.len + r0 / a.qpk + 1;
  const int plain = max(0, min(common, last) - first) / KT;
  int i = 0;
  for (; i + 1 < plain; i += 2) {
    turn(i, 0, std::false_type{});
    turn(i + 1, 1, std::false_type{});
  }
  if (i < plain) turn(i, 0, std::false_type{}), ++i;
  for (; i < count; ++i) turn(i, i & 1, std::true_type{});
  __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));  // no copy may land in what follows
  lds_barrier();

  // The waves along the keys meet: statistics and sums through LDS, then each
  // wave's sums on the common maximum.  Unit (16 bytes) u of row c of 16 lies at
  // unit u ^ (c % 8): eight rows of a write cover 32 banks once.
  constexpr int QUADS = D / 4, ALL = QT * WQ * 16;
  f4_t* const red = reinterpret_cast<f4_t*>(&kv[0][0][0]);  // [WK][ALL][QUADS]
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const int at = (wq * QT + t) * 16 + c, r = rw + 16 * t + c;
    const bool behind = r >= rows;  // the last token
    if (behind) top[t] = -INFINITY;
    else if (top[t] == -INFINITY && sum[t][0] != 0.0f) top[t] = 0.0f;  // NaN scores alone
    if (g == 0) {
      stat[0][wk][at] = top[t];
      stat[1][wk][at] = behind ? 0.0f : sum[t][0];
      if (wk == 0) {
        const int i = behind ? r / a.qpk : node[t];
        place[at] = i * a.n_heads + r - i * a.qpk;
      }
    }
#pragma unroll
    for (int d = 0; d < D / 16; ++d)
      red[(wk * ALL + at) * QUADS + ((4 * d + g) ^ (c & 7))] = acc[t][d];
  }
  lds_barrier();
  const int64_t rec0 = (static_cast<int64_t>(h) * a.shares + w) * rows_all + r0;
  float* const sums = a.partial + rec0 * D;
  float* const stats = a.partial + static_cast<int64_t>(a.n_kv) * a.shares * rows_all * D + rec0 * 2;
  T* const out = static_cast<T*>(a.out) +
                 (static_cast<int64_t>(b) * a.T * a.n_heads + h * a.qpk) * D;
  const int u = threadIdx.x % QUADS;
#pragma unroll
  for (int e = 0; e < ALL * QUADS / kTreeThreads; ++e) {
    const int at = e * (kTreeThreads / QUADS) + threadIdx.x / QUADS;
    if (r0 + at >= rows_all) break;
    float mr = stat[0][0][at], l = 0.0f;
#pragma unroll
    for (int x = 1; x < WK; ++x) mr = fmaxf(mr, stat[0][x][at]);
    f4_t o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int x = 0; x < WK; ++x) {
      const float keep = mr == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(stat[0][x][at] - mr);
      l += stat[1][x][at] * keep;
      const f4_t v = red[(x * ALL + at) * QUADS + (u ^ (at & 7))];
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] += v[i] * keep;
    }
    if (a.shares == 0) {
      typedef T vec4 __attribute__((ext_vector_type(4)));
      vec4 y;
#pragma unroll
      for (int x = 0; x < 4; ++x) y[x] = static_cast<T>(l == 0.0f ? 0.0f : o[x] / l);
      *reinterpret_cast<vec4*>(out + static_cast<int64_t>(place[at]) * D + 4 * u) = y;
    } else {
      if (mr != -INFINITY) *reinterpret_cast<f4_t*>(sums + static_cast<int64_t>(at) * D + 4 * u) = o;
      if (u == 0) stats[2 * at] = mr, stats[2 * at + 1] = l;
    }
  }
}

struct TreePlan {
  int form = 0, rows = 16, row_tiles = 1, shares = 0;
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
  p->form = rows <= 16 ? 0 : rows <= 32 ? 1 : rows <= 64 ? 2 : 3;
  p->rows = 16 << p->form;
  p->row_tiles = static_cast<int>(ceil_div(rows, p->rows));
  NIBBLE_CHECK(ceil_div(batch * n_kv, 8) * 8 * p->row_tiles * kTreeThreads < (int64_t(1) << 32),
               "%lld sequences of %lld kv heads: a launch ends at 2^32 threads", (long long)batch,
               (long long)n_kv);
  // Room for more workgroups than there are (sequence, kv head, row tile)s: the
  // cached rows are split, unless there are but a few tiles of them.
  const int64_t room = kSplitWorkgroups / (n_kv * p->row_tiles);
  if (room > batch && batch < kSplitWorkgroups && max_seq > 4 * kTreeKeys) {
    p->shares = static_cast<int>(room);
    p->workspace_bytes =
        static_cast<size_t>(n_kv * room * rows) * (head_dim + 2) * 4 + static_cast<size_t>(batch) * 8;
  }
  return NIBBLE_OK;
}

template <class E, int D>
hipError_t launch_tree(const TreeArgs& a, const TreePlan& p, hipStream_t stream) {
  const int64_t pairs = static_cast<int64_t>(p.shares > 0 ? p.shares : a.B) * a.n_kv;
  const dim3 grid(static_cast<unsigned>(ceil_div(pairs, 8) * 8 * p.row_tiles));
  if (p.form == 0) tree_kernel<E, D, 1, 4><<<grid, kTreeThreads, 0, stream>>>(a);
  else if (p.form == 1) tree_kernel<E, D, 2, 4><<<grid, kTreeThreads, 0, stream>>>(a);
  else if (p.form == 2) tree_kernel<E, D, 2, 2><<<grid, kTreeThreads, 0, stream>>>(a);
  else tree_kernel<E, D, 2, 1><<<grid, kTreeThreads, 0, stream>>>(a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.shares == 0) return e;
  const int64_t parts = ceil_div(static_cast<int64_t>(a.T) * a.qpk, kTreeThreads / (D / 4));
  join_kernel<E, D><<<dim3(static_cast<unsigned>(a.B * a.n_kv * parts)), kTreeThreads, 0,
                           stream>>>(a);
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
  NIBBLE_CHECK(std::isfinite(scale * kLog2e), "scale must be finite, also times log2(e)");
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
  a.runs = reinterpret_cast<int*>(a.partial + static_cast<size_t>(n_kv_heads) * p.shares * tokens *
                                              (n_heads / n_kv_heads) * (head_dim + 2));
  a.kb = k_batch_stride, a.kh = k_head_stride, a.ks = k_row_stride;
  a.vb = v_batch_stride, a.vh = v_head_stride, a.vs = v_row_stride;
  a.mask_batch = mask_batches == 1 ? 0 : tokens * tokens;
  a.B = static_cast<int>(batch);
  a.T = static_cast<int>(tokens);
  a.n_heads = static_cast<int>(n_heads);
  a.n_kv = static_cast<int>(n_kv_heads);
  a.qpk = static_cast<int>(n_heads / n_kv_heads);
  a.seq = static_cast<int>(max_seq);
  a.shares = p.shares;
  a.row_tiles = p.row_tiles;
  a.join_cost = kTreeShareCost + kTreeRowCost * static_cast<float>(tokens * n_heads);
  a.fold = mask == nullptr && batch * n_kv_heads * p.row_tiles <= kSplitWorkgroups;
  a.scale = scale == 0.0f ? 1.0f : std::fabs(scale) * kLog2e;
  a.sign = scale > 0.0f ? 1.0f : scale < 0.0f ? -1.0f : 0.0f;
  const hipError_t e = dtype == 0 ? (head_dim == 64 ? launch_tree<Half, 64>(a, p, stream)
                                                    : launch_tree<Half, 128>(a, p, stream))
                                  : (head_dim == 64 ? launch_tree<Bfloat, 64>(a, p, stream)
                                                    : launch_tree<Bfloat, 128>(a, p, stream));
  if (e != hipSuccess) return hip_fail(e, "tree attention kernel launch");
  return ok();
}
