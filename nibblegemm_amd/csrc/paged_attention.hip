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
// The queries of a kv head's group (tokens x query heads, `rows`) go to the matrix
// cores together.  A 16x16x32 product takes keys as rows and queries as columns, so lane
// (g = l / 16, c = l % 16) gets the scores of query c for keys 4g .. 4g + 3 of a 16-key
// tile; its probabilities are already where the second product (V^T P^T, queries as
// columns again) wants them, if that product's k index runs over a lane's keys of two
// tiles in turn.  V is read transposed from LDS (ds_read_b64_tr_b16, _tr_b8).  8-bit
// rows stay 8-bit in LDS and are converted, exactly, with their page's power of two,
// on their way into the products' operands.
//
// What it reads, writes and computes: the visible rows once a kv head and 128 query
// rows, 4 rows keys D operations, and, where the rows are split, D + 2 floats a query
// row and share.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "paged_prompt.h"
#include "paged_rows.h"

namespace nibble {

int check_paged(const nibble_paged_cache* c, int64_t dtype, int64_t batch);

namespace {

// One workgroup: 16 QT WQ query rows of one kv head (WQ = 4 / WK waves along the
// rows, WK along the keys), one share of the rows, in tiles of 64 keys.  A tile's rows
// of k and v are copied straight into one of two LDS buffers while the tile before it is
// computed; two workgroups share a CU.  Wave w copies the tile's w-th 16 rows, which
// lie in one page.
template <class E, int D, int QT, int WK, bool Q8>
__global__ __launch_bounds__(kPagedThreads, 2) void paged_kernel(AttendArgs a) {
  using T = typename E::type;
  using vec8 = typename E::vec8;
  constexpr int WQ = 4 / WK, ROWS = 16 * QT * WQ;
  constexpr int KT = kPagedKeys, KPW = KT / WK, KS = KPW / 16;  // a wave's keys of a tile
  constexpr int PS = (KS + 1) / 2;               // products of 32 keys (or 16 and zeros)
  constexpr int BYTES = Q8 ? D : 2 * D;          // of a row
  constexpr int UNITS = BYTES / 16;              // 16-byte units of a row
  constexpr int CROWS = 64 / UNITS;              // rows of a copy
  constexpr int COPIES = 16 / CROWS;             // of K or V, a wave and tile
  constexpr uint32_t kTile = KT * BYTES;         // bytes of a tile of k or v
  typedef short s4_t __attribute__((ext_vector_type(4)));
  typedef int i2_t __attribute__((ext_vector_type(2)));
  typedef unsigned short us4_t __attribute__((ext_vector_type(4)));
  typedef unsigned short us8_t __attribute__((ext_vector_type(8)));
  typedef __attribute__((address_space(3))) s4_t lds4_t;
  typedef __attribute__((address_space(3))) i2_t lds2_t;
  constexpr int kSums = 4 * WK * WQ * QT * 16 * D;  // bytes
  __shared__ __attribute__((aligned(16))) char kv[4 * kTile > kSums ? 4 * kTile : kSums];
  __shared__ float stat[2][WK][WQ * QT * 16];
  __shared__ int place[WQ * QT * 16];  // of a row's output, in heads

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  const int wq = wave / WK, wk = wave % WK;
  const int g = lane >> 4, c = lane & 15;
  // Workgroup -> (share, kv head), row tile: the row tiles that read the same cache
  // rows run on one XCD (id % 8) and share its L2.  The later row tiles are longer:
  // longest first, or, where all are on the CUs at once, two a CU, each with its
  // counterpart.
  const int slot = blockIdx.x >> 3;
  const int pair = slot / a.row_tiles * 8 + (blockIdx.x & 7);
  const int rt = slot % a.row_tiles;
  const int row_tile = a.fold && rt >= (a.row_tiles + 1) / 2 ? rt - (a.row_tiles + 1) / 2
                                                             : a.row_tiles - 1 - rt;
  const int w = pair / a.n_kv, h = pair - w * a.n_kv;
  int b = w, share = 0, per = 0x3fffffff;  // the whole sequence
  if (a.shares > 0) {
    if (w >= a.shares) return;
    const Shares<AttendArgs> shares(a, w);
    if (shares.found < 0) return;
    b = shares.found, share = w - shares.first, per = shares.per;
    // (for the kernel that joins them)
    if (share == 0 && h == 0 && rt == 0 && threadIdx.x == 0)
      a.runs[2 * b] = shares.first, a.runs[2 * b + 1] = shares.count;
  } else if (w >= a.B) {
    return;
  }
  const PagedSpan span = PagedSpan(a, b).uniform();
  const int rows_all = a.T * a.qpk, rows = span.live * a.qpk;
  const int r0 = row_tile * ROWS;
  const int rw = r0 + wq * 16 * QT;  // this wave's first row

  // Rows of the cache [low, end) and those before a.sinks matter to this workgroup's
  // tokens, early to late; of their tiles it takes those of its share: [a0, a0 + na)
  // and [b0, b0 + nb).
  const int early = r0 / a.qpk, late = (min(r0 + ROWS, rows) - 1) / a.qpk;
  const int end = r0 < rows ? min(span.total, span.len + late + 1) : 0;
  const int low = end > 0 ? max(span.len + early - a.window + 1, 0) : 0;
  int a0, na, b0, count;
  {
    const Seen all = span.seen(a), own(low, a.sinks, end);
    const int x0 = min(share * per, 0x3fffffff), x1 = x0 + min(per, 0x3fffffff);  // of all's tiles
    const int shift = all.from - all.first;  // from place to tile, behind the first
    a0 = x0;
    na = max(0, min(all.first > 0 ? min(x1, all.first) : x1, own.first) - a0);
    b0 = max(max(x0, all.first) + shift, own.from);
    count = na + max(0, min(x1 + shift, own.upto) - b0);
  }
  auto key_of = [&](int i) { return (i < na ? a0 + i : b0 + i - na) * KT; };

  // Queries: lane (g, c) holds of row c of a tile the elements that it multiplies with
  // those of a key: of 32 8 g .., or with 8-bit keys, of 64 16 g ...
  vec8 q[QT][D / 32];
  int pos[QT];  // the row of its token
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const int r = rw + 16 * t + c;
    const bool in = r < rows;
    const int node = in ? r / a.qpk : 0;
    pos[t] = span.len + node;
    const int64_t at = ((static_cast<int64_t>(b) * a.T + node) * a.n_heads + h * a.qpk +
                        (in ? r - node * a.qpk : 0)) * D;
#pragma unroll
    for (int s = 0; s < D / 32; ++s) {
      const int e = Q8 ? 64 * (s / 2) + 16 * g + 8 * (s % 2) : 32 * s + 8 * g;
      q[t][s] = in ? *reinterpret_cast<const vec8*>(static_cast<const T*>(a.q) + at + e) : vec8{};
    }
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

  // The pages of a tile's four 16-row groups: lane l has that of group l % 4.
  const int32_t* const table = a.table + static_cast<int64_t>(b) * a.width;
  auto entry = [&](int i) {
    return table[min((key_of(min(i, count - 1)) + 16 * (lane & 3)) >> a.shift, a.width - 1)];
  };
  auto is_page = [&](int page) { return page >= 0 && page < a.n_pages; };
  const char* const kbase = a.k + h * a.kh;
  const char* const vbase = a.v + h * a.vh;
  const uint32_t lds0 = lds_address(kv) + wave * COPIES * 1024u;
  // This wave's copies of tile i, whose pages are `pages`; rows that none of the
  // workgroup's tokens sees read as zeros.
  auto copy = [&](int i, int pages) {
    const int page = __builtin_amdgcn_readlane(pages, wave);
    const int key0 = key_of(i) + 16 * wave, in_page = key0 & ((1 << a.shift) - 1);
    const int64_t at = is_page(page) ? page : 0;
    const int here = is_page(page) ? end : 0;
    const char* const kt = kbase + at * a.kp + in_page * a.kr;
    const char* const vt = vbase + at * a.vp + in_page * a.vr;
    const uint32_t dst = lds0 + (i & 1) * 2 * kTile;
#pragma unroll
    for (int u = 0; u < COPIES; ++u) {
      const int r = u * CROWS + lane / UNITS, key = key0 + r;
      const bool in = key < here && (key >= low || key < a.sinks);
      const uint32_t unit16 = ((lane % UNITS) ^ paged_swizzle<UNITS, Q8>(16 * wave + r)) * 16u;
      lds_copy16(kt, 0x7fffffffu, dst + u * 1024u,
                 in ? r * static_cast<uint32_t>(a.kr) + unit16 : kOutOfRange);
      lds_copy16(vt, 0x7fffffffu, dst + kTile + u * 1024u,
                 in ? r * static_cast<uint32_t>(a.vr) + unit16 : kOutOfRange);
    }
  };

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

  // Byte offsets within a tile.  16 bits: of row c, k elements 8 g .. of each 32; of
  // row 4 g + c / 4, v elements 4 (c % 4) .. of each 16.  8 bits: of row c, k elements
  // 16 g .. of each 64; v elements 8 (c % 2) .. of each 16 of the row of 32 (or 16) whose
  // place in the products' order is 8 g + c / 2.  (Rows 16 apart share the swizzle of 16
  // bits; that of 8 bits differs in the highest bit.)
  const int krow = c * BYTES + ((g ^ paged_swizzle<UNITS, Q8>(c)) * 16);
  int vrow;
  if constexpr (Q8) {
    const int x = c >> 1, r = KS == 1 ? 4 * g + (x & 3) : 16 * (x >> 2) + 4 * g + (x & 3);
    vrow = r * BYTES + paged_swizzle<UNITS, Q8>(wk * KPW + r) * 16 + 8 * (c & 1);
  } else {
    const int r = 4 * g + (c >> 2);
    vrow = r * BYTES + (((c >> 1 & 1) ^ paged_swizzle<UNITS, Q8>(r)) * 16) + (c & 1) * 8;
  }
  constexpr int kHighBit = UNITS == 8 ? 64 : 32;  // of the 8-bit swizzle, in bytes
  float kscale[KS], vscale[KS];  // 8 bits: of this wave's 16-key tiles
  struct Scores {
    f4_t s[KS][QT];
  };
  auto multiply = [&](Scores& x, int buf) {
    const char* const kt = kv + buf * 2 * kTile + wk * KPW * BYTES;
    const f4_t zero = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < KS; ++j) {
      if constexpr (Q8) {
        const int flip = (wk * KS + j) & 1 ? kHighBit : 0;
#pragma unroll
        for (int s2 = 0; s2 < D / 64; ++s2) {
          const u4_t w4 = *reinterpret_cast<const u4_t*>(kt + j * 16 * BYTES +
                                                         ((krow ^ (64 * s2)) ^ flip));
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const vec8 ka = from_float8<E>(w4[2 * e], w4[2 * e + 1], kscale[j], kscale[j]);
#pragma unroll
            for (int t = 0; t < QT; ++t)
              x.s[j][t] = E::mfma(ka, q[t][2 * s2 + e], s2 + e == 0 ? zero : x.s[j][t]);
          }
        }
      } else {
#pragma unroll
        for (int ss = 0; ss < D / 32; ++ss) {
          const vec8 ka = *reinterpret_cast<const vec8*>(kt + j * 16 * BYTES + (krow ^ (64 * ss)));
#pragma unroll
          for (int t = 0; t < QT; ++t) x.s[j][t] = E::mfma(ka, q[t][ss], ss == 0 ? zero : x.s[j][t]);
        }
      }
    }
  };
  // What this lane's queries see of a tile's keys, a bit for each of its scores;
  // `there` has a bit for each of the tile's 16-row groups that has a page.
  uint32_t seen[QT];
  auto look = [&](int key0, uint32_t there) {
    auto upto = [](int n) { return (1u << min(max(n, 0), 4)) - 1u; };
    uint32_t some = 0;
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      seen[t] = 0;
#pragma unroll
      for (int j = 0; j < KS; ++j) {
        const int key = key0 + wk * KPW + 16 * j + 4 * g;  // of bit 0
        const uint32_t near = ~upto(pos[t] - a.window + 1 - key) | upto(a.sinks - key);
        const uint32_t bits = near & upto(min(pos[t] + 1, end) - key);
        seen[t] |= ((there >> (wk * KS + j) & 1u) != 0 ? bits : 0u) << (4 * j);
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
    for (int t = 0; t < QT; ++t) moves |= m[t] - top[t] > kPagedSlack + kPagedLift<E>;
    if (!__any(moves)) return;
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      const float up = fmaxf(swap_max(m[t]) - kPagedLift<E>, top[t]);
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
      // (The probabilities are rounded to 16 bits because the matrix cores take them so:
      // each is off by half a step at most, in fp16 of 2^-24 at least, and the sum, by
      // the matrix cores too, ones times P^T in fp32, is of the rounded.)
#pragma unroll
      for (int j = 0; j < PS; ++j) sum[t] = E::mfma(ones, p[j][t], sum[t]);
    }
  };
  // Whether this wave's v rows of a tile hold what is not finite, or may once they
  // are converted.
  auto strange = [&](int buf) {
    const u4_t* const vt =
        reinterpret_cast<const u4_t*>(kv + (buf * 2 + 1) * kTile + wk * KPW * BYTES);
    bool odd = false;
    if constexpr (Q8) {
#pragma unroll
      for (int j = 0; j < KS; ++j) odd |= vscale[j] > power(kHighExponent<E> - 1);
#pragma unroll
      for (int e = 0; e < KPW * UNITS / 64; ++e) {
        const u4_t bits = vt[e * 64 + lane];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          odd |= (((bits[i] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0;
      }
    } else {
      us8_t most = {};
#pragma unroll
      for (int e = 0; e < KPW * UNITS / 64; ++e)
        most = __builtin_elementwise_max(most,
                                         __builtin_bit_cast(us8_t, vt[e * 64 + lane] & 0x7fff7fffu));
#pragma unroll
      for (int e = 0; e < 8; ++e) odd |= most[e] >= E::kExponent;
    }
    return __any(odd) != 0;
  };
  // V^T of 32 keys (16 where a wave has no more) for 16 elements.
  auto values = [&](uint32_t vt, int d, int j) {
    if constexpr (Q8) {
      const i2_t v2 = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
          (lds2_t*)(uintptr_t)(vt + 2 * j * 16 * BYTES + (vrow ^ (16 * d))));
      return __builtin_bit_cast(
          us8_t, from_float8<E>(v2[0], KS == 1 ? 0 : v2[1], vscale[2 * j], vscale[KS == 1 ? 0 : 2 * j + 1]));
    } else {
      s4_t v2[2] = {};
#pragma unroll
      for (int e = 0; e < (KS == 1 ? 1 : 2); ++e)
        v2[e] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (lds4_t*)(uintptr_t)(vt + (2 * j + e) * 16 * BYTES + (vrow ^ (32 * d))));
      return us8_t(__builtin_shufflevector(__builtin_bit_cast(us4_t, v2[0]),
                                           __builtin_bit_cast(us4_t, v2[1]), 0, 1, 2, 3, 4, 5, 6, 7));
    }
  };
  // The sums.  A hidden row's infinity or NaN must not meet its zero probability: with
  // `careful` they are left out of the products and counted, over the rows a query sees,
  // by products of their own: infinities of either sign, a NaN as both.  A query and
  // element that met one gets that infinity added, and of both the NaN that they make.
  auto add = [&](int buf, auto careful) {
    constexpr bool kCareful = decltype(careful)::value;
    const uint32_t vt = lds_address(kv) + (buf * 2 + 1) * kTile + wk * KPW * BYTES;
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
  // A tile's turn: it is there, and the next one's copies begin.  `pages` are the next
  // tile's, `there` says which of this tile's groups have one.
  int pages = 0;
  uint32_t there = 0;
  int next_k = 0, next_v = 0;  // 8 bits: the scales of this lane's group of the next tile
  auto begin = [&](int i) {
    if constexpr (Q8) {
#pragma unroll
      for (int j = 0; j < KS; ++j) {
        kscale[j] = power(__builtin_amdgcn_readlane(next_k, wk * KS + j));
        vscale[j] = power(__builtin_amdgcn_readlane(next_v, wk * KS + j));
      }
    }
    there = __ballot(is_page(pages)) & 15u;  // of the next tile
    if (i < count) {
      copy(i, pages);
      if constexpr (Q8) {
        const int64_t at = static_cast<int64_t>(is_page(pages) ? pages : 0) * a.n_kv + h;
        next_k = a.k_scales[at], next_v = a.v_scales[at];
      }
      pages = entry(i + 1);
    }
  };
  auto turn = [&](int i, int buf, auto tail, uint32_t has) {
    bool any = true;
    const int key0 = key_of(i);
    if constexpr (decltype(tail)::value) any = look(key0, has);
    if (!any) return;
    Scores x;
    multiply(x, buf);
    if constexpr (decltype(tail)::value) hide(x);
    largest(x);
    move();
    weigh(x);
    if constexpr (decltype(tail)::value) {
      if (strange(buf)) {
        look(key0, has);  // (again, so that its bits need no registers meanwhile)
        add(buf, std::true_type{});
        return;
      }
    }
    add(buf, std::false_type{});
  };
  // A tile with rows that some query does not see is a tail.
  auto plain = [&](int i, uint32_t has) {
    const int key0 = key_of(i);
    return has == 15u && key0 + KT <= min(span.len + early + 1, end) &&
           (key0 > span.len + late - a.window || key0 + KT <= a.sinks);
  };
  if (count > 0) {
    pages = entry(0);
    begin(0);
    auto step = [&](int i, int buf) {
      const uint32_t has = there;
      __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));
      lds_barrier();
      begin(i + 1);
      if (plain(i, has)) turn(i, buf, std::false_type{}, has);
      else turn(i, buf, std::true_type{}, has);
    };
#pragma unroll 1
    for (int i = 0; i < count; i += 2) {
      step(i, 0);
      if (i + 1 < count) step(i + 1, 1);
    }
  }
  __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));  // no copy may land in what follows
  lds_barrier();

  // The waves along the keys meet: statistics and sums through LDS, then each wave's
  // sums on the common maximum.  Unit (16 bytes) u of row c of 16 lies at unit u ^ (c %
  // 8): eight rows of a write cover 32 banks once.
  constexpr int QUADS = D / 4, ALL = QT * WQ * 16;
  f4_t* const red = reinterpret_cast<f4_t*>(kv);  // [WK][ALL][QUADS]
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
        const int i = r / a.qpk;
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
  for (int e = 0; e < ALL * QUADS / kPagedThreads; ++e) {
    const int at = e * (kPagedThreads / QUADS) + threadIdx.x / QUADS;
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

struct PagedPlan {
  int form = 0, rows = 16, row_tiles = 1, shares = 0, slots = 0;
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
  p->form = rows <= 16 ? 0 : rows <= 32 ? 1 : rows <= 64 ? 2 : 3;
  p->rows = 16 << p->form;
  p->row_tiles = static_cast<int>(ceil_div(rows, p->rows));
  NIBBLE_CHECK(ceil_div(batch, 8) * 8 * n_kv * p->row_tiles * kPagedThreads < (int64_t(1) << 32),
               "%lld sequences of %lld kv heads: a launch ends at 2^32 threads", (long long)batch,
               (long long)n_kv);
  // Room for more workgroups than there are (sequence, kv head, row tile)s: the
  // cached rows are split, unless there are but a few tiles of them.
  const int64_t room = kSplitWorkgroups / (n_kv * p->row_tiles);
  const bool line = p->form <= 1;
  if (line ? room > 0 && batch <= kSplitWorkgroups && batch * n_kv < 4 * kSplitWorkgroups
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
  const int64_t pairs = static_cast<int64_t>(p.shares > 0 ? p.shares : a.B) * a.n_kv;
  const dim3 grid(static_cast<unsigned>(ceil_div(pairs, 8) * 8 * p.row_tiles));
  if (p.form <= 1) {
    const dim3 lines(static_cast<unsigned>(
        ceil_div(p.shares > 0 ? p.shares : a.B, 8) * 8 * a.n_kv));
    if (p.form == 0) rows_kernel<E, D, 1, Q8><<<lines, kPagedThreads, 0, stream>>>(a);
    else rows_kernel<E, D, 2, Q8><<<lines, kPagedThreads, 0, stream>>>(a);
    return hipGetLastError();
  }
  if (p.form == 2) paged_kernel<E, D, 2, 2, Q8><<<grid, kPagedThreads, 0, stream>>>(a);
  else prompt_kernel<E, D, 1, Q8><<<grid, kPagedThreads, 0, stream>>>(a);
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
  a.width = static_cast<int>(c.table_pages);
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
