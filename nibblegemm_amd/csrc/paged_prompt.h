// Attention over a paged cache for many query rows a kv head: prompts, and parts of them.
#pragma once

#include "paged_attention.h"

namespace nibble {
namespace {

typedef float f16_t __attribute__((ext_vector_type(16)));

template <class E>
__device__ __forceinline__ f16_t mfma32(typename E::vec8 a, typename E::vec8 b, f16_t c) {
  if constexpr (std::is_same_v<E, Half>) return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
// Unit (16 bytes) u of LDS row r lies at unit u ^ prompt_swizzle(r), so that eight rows of
// a K read, and the rows of a V read (four and 32 bytes of each, or, of 8 bits, 4h .. 4h +
// 3 and 8 + 4h .. and 16 bytes), cover 32 banks once.
template <int UNITS, bool Q8>
__device__ __forceinline__ int prompt_swizzle(int r) {
  if (!Q8) return paged_swizzle<UNITS>(r);
  const int high = (r >> 2 ^ r >> 3) & 1;
  return UNITS == 8 ? (r & 3) | high << 2 : (r >> 1 & 1) | high << 1;
}

// One workgroup: 128 query rows of one kv head, 32 a wave, and one share of the rows, in
// tiles of 64 keys, which are copied straight into LDS, v into one of two buffers while the
// tile before is computed, k, a tile ahead of it, into one of three.
//
// A 32x32x16 product takes keys as rows and queries as columns, so lane (f = l / 32, c = l
// % 32) gets the scores of query c for keys 8 a + 4 f .. + 3 (a = 0 .. 3) of a 32-key tile,
// and its probabilities are where the second product (V^T P^T) wants them, if its k runs
// over a lane's keys in turn.
//
// The SIMDs bound it, matrix and vector instructions together, and the clock that falls
// under them: of 2048 tokens of 32 + 2 x 8 heads of 128 the products alone would take 86 us
// at the rate of a large library product, and it takes 110 to 119.  By the counters the
// matrix cores are busy 54% of the cycles (a ninth of that with the sums of the
// probabilities) and other vector instructions issue in 39%, at 1.7 GHz: the two hardly
// overlap, though two waves share a SIMD.  What fills the time between products was taken
// out: exponentials run beside the next scores' products, the maximum beside the sums'
// products, addresses of 64 tiles are worked out at once.  Waves whose rows are behind the
// last copy alone (64 rows over 32 x 4096 of 8 bits: 5 us of 58 less than if they compute,
// too; as much as by workgroups of two waves, which take 4 more than these on 16 bits).
template <class E, int D, bool Q8>
__global__ __launch_bounds__(kPagedThreads, 2) void prompt_kernel(AttendArgs a) {
  using T = typename E::type;
  using vec8 = typename E::vec8;
  constexpr int KT = kPagedKeys, ROWS = 128;
  constexpr int BYTES = Q8 ? D : 2 * D, UNITS = BYTES / 16;  // of a row; its 16-byte units
  constexpr int CROWS = 64 / UNITS, COPIES = 16 / CROWS;     // rows of a copy; of k or v, a wave
  constexpr uint32_t kTile = KT * BYTES;                     // bytes of a tile of k or v
  typedef short s4_t __attribute__((ext_vector_type(4)));
  typedef int i2_t __attribute__((ext_vector_type(2)));
  typedef unsigned short us4_t __attribute__((ext_vector_type(4)));
  typedef unsigned short us8_t __attribute__((ext_vector_type(8)));
  typedef __attribute__((address_space(3))) s4_t lds4_t;
  typedef __attribute__((address_space(3))) i2_t lds2_t;
  __shared__ __attribute__((aligned(16))) char kv[5 * kTile];  // v, v, k, k, k

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  const int f = lane >> 5, c = lane & 31;
  // Workgroup -> (share, kv head), row tile: the row tiles that read the same cache rows
  // run on one XCD (id % 8) and share its L2.  The later row tiles are longer: longest
  // first, or, where all are on the CUs at once, two a CU, each with its counterpart.
  const int slot = blockIdx.x >> 3;
  const int pair = slot / a.row_tiles * 8 + (blockIdx.x & 7);
  const int rt = slot % a.row_tiles;
  const int row_tile = a.fold && rt >= (a.row_tiles + 1) / 2 ? rt - (a.row_tiles + 1) / 2
                                                             : a.row_tiles - 1 - rt;
  const int w = pair / a.n_kv, h = pair - w * a.n_kv;
  int b = w, share = 0, pieces = 1;
  if (a.shares > 0) {
    if (w >= a.shares) return;
    const Shares<AttendArgs> shares(a, w);
    if (shares.found < 0) return;
    b = shares.found, share = w - shares.first, pieces = shares.count;
    // (for the kernel that joins them)
    if (share == 0 && h == 0 && rt == 0 && threadIdx.x == 0)
      a.runs[2 * b] = shares.first, a.runs[2 * b + 1] = shares.count;
  } else if (w >= a.B) {
    return;
  }
  const PagedSpan span = PagedSpan(a, b).uniform();
  const int rows_all = a.T * a.qpk, rows = span.live * a.qpk;
  const int r0 = row_tile * ROWS;
  const bool idle = r0 + 32 * wave >= rows;  // a wave that copies alone

  // Rows of the cache [low, end) and those before a.sinks matter to this workgroup's
  // tokens, early to late; of their tiles it takes those of its share: [a0, a0 + na) and
  // those from b0 on.
  const int early = r0 / a.qpk, late = (min(r0 + ROWS, rows) - 1) / a.qpk;
  const int end = r0 < rows ? min(span.total, span.len + late + 1) : 0;
  const int low = end > 0 ? max(span.len + early - a.window + 1, 0) : 0;
  int a0, na, b0, count;
  {
    // (a sequence's shares are equal: with as many tiles as Shares allows and a rest, 64 rows
    // over 32 x 4096 take 66 us in place of 60, of 8 bits 58 in place of 52)
    const Seen all = span.seen(a), own(low, a.sinks, end);
    const int per = (all.first + all.upto - all.from + pieces - 1) / pieces;
    const int x0 = share * per, x1 = x0 + per;  // of all's tiles
    const int shift = all.from - all.first;  // from place to tile, behind the first
    a0 = x0;
    na = max(0, min(all.first > 0 ? min(x1, all.first) : x1, own.first) - a0);
    b0 = max(max(x0, all.first) + shift, own.from);
    count = na + max(0, min(x1 + shift, own.upto) - b0);
  }
  auto key_of = [&](int i) { return (i < na ? a0 + i : b0 + i - na) * KT; };

  // Queries: lane (f, c) holds of row c of 32 the elements that it multiplies with those of
  // a key: of 16 8 f .., or with 8-bit keys, of 32 16 f ...
  vec8 q[D / 16];
  int pos;  // the row of its token
  {
    const int r = r0 + 32 * wave + c;
    const bool in = r < rows;
    const int node = in ? r / a.qpk : 0;
    pos = span.len + node;
    const T* const from = static_cast<const T*>(a.q) +
                          ((static_cast<int64_t>(b) * a.T + node) * a.n_heads + h * a.qpk +
                           (in ? r - node * a.qpk : 0)) * D;
#pragma unroll
    for (int s = 0; s < D / 16; ++s) {
      const int e = Q8 ? 32 * (s / 2) + 16 * f + 8 * (s % 2) : 16 * s + 8 * f;
      q[s] = in ? *reinterpret_cast<const vec8*>(from + e) : vec8{};
    }
    if (a.sign != 1.0f) {  // a scale that is not positive: its sign goes into q, exactly
#pragma unroll
      for (int s = 0; s < D / 16; ++s)
#pragma unroll
        for (int i = 0; i < 8; ++i)
          q[s][i] = static_cast<T>(static_cast<float>(q[s][i]) * a.sign);
    }
  }

  // Where the tiles' rows are, of 64 tiles, one a lane: the addresses of the 16 rows that
  // this wave copies, whether all of those are seen by some token, which of a tile's 16-row
  // groups have a page, and the scales of the groups, a byte each.
  const int32_t* const table = a.table + static_cast<int64_t>(b) * a.width;
  auto is_page = [&](int page) { return page >= 0 && page < a.n_pages; };
  auto page_at = [&](int key) { return table[min(key >> a.shift, a.width - 1)]; };
  struct Places {
    uint64_t k, v;
    uint32_t has, k_scales, v_scales;
  };
  Places places = {};
  uint64_t whole = 0;
  auto look_up = [&](int i) {
    const int key0 = key_of(min(i + lane, count - 1)), mine = key0 + 16 * wave;
    const int page = page_at(mine);
    const uint64_t at = is_page(page) ? page : 0, in_page = mine & ((1 << a.shift) - 1);
    places.k = reinterpret_cast<uint64_t>(a.k) + h * a.kh + at * a.kp + in_page * a.kr;
    places.v = reinterpret_cast<uint64_t>(a.v) + h * a.vh + at * a.vp + in_page * a.vr;
    places.has = places.k_scales = places.v_scales = 0;
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const int of = page_at(key0 + 16 * n);
      places.has |= is_page(of) ? 1u << n : 0u;
      if constexpr (Q8) {
        // (of a group that no token sees the scale may be anything: 255 would make NaN of the
        // zeros that are read in its place)
        const int key = key0 + 16 * n;
        const bool is = is_page(of) && key < end && (key + 16 > low || key < a.sinks);
        const int64_t s = static_cast<int64_t>(is ? of : 0) * a.n_kv + h;
        const uint32_t ks = a.k_scales[s], vs = a.v_scales[s];
        places.k_scales |= (is ? ks : 127u) << (8 * n);
        places.v_scales |= (is ? vs : 127u) << (8 * n);
      }
    }
    whole = __ballot(is_page(page) && mine + 16 <= end && (mine >= low || mine + 16 <= a.sinks));
  };
  // Of one tile, in scalar registers.
  struct Tile {
    uint64_t k, v;
    uint32_t has, k_scales, v_scales;
    bool whole;
  };
  auto tile_of = [&](int i) {
    auto lane64 = [&](uint64_t x) {
      const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(x), i & 63);
      const uint32_t hi = __builtin_amdgcn_readlane(static_cast<int>(x >> 32), i & 63);
      return static_cast<uint64_t>(hi) << 32 | lo;
    };
    Tile t = {lane64(places.k), lane64(places.v), 0, 0, 0, (whole >> (i & 63) & 1u) != 0};
    t.has = __builtin_amdgcn_readlane(static_cast<int>(places.has), i & 63);
    if constexpr (Q8) {
      t.k_scales = __builtin_amdgcn_readlane(static_cast<int>(places.k_scales), i & 63);
      t.v_scales = __builtin_amdgcn_readlane(static_cast<int>(places.v_scales), i & 63);
    }
    return t;
  };
  const uint32_t lds0 = lds_address(kv) + wave * COPIES * 1024u;
  uint32_t from_k[COPIES], from_v[COPIES];  // a lane's byte in 16 rows of k and v
#pragma unroll
  for (int u = 0; u < COPIES; ++u) {
    const int r = u * CROWS + lane / UNITS;
    const uint32_t unit16 = ((lane % UNITS) ^ prompt_swizzle<UNITS, Q8>(16 * wave + r)) * 16u;
    from_k[u] = r * static_cast<uint32_t>(a.kr) + unit16;
    from_v[u] = r * static_cast<uint32_t>(a.vr) + unit16;
  }
  // This wave's copies of tile i's k (v), from `at`; rows that none of the workgroup's
  // tokens sees read as zeros.
  auto copy = [&](int i, const Tile& t, uint64_t at, const uint32_t (&from)[COPIES], uint32_t dst) {
    const void* const base = reinterpret_cast<const void*>(at);
    if (t.whole) {
#pragma unroll
      for (int u = 0; u < COPIES; ++u) lds_copy16(base, 0x7fffffffu, dst + u * 1024u, from[u]);
    } else {
      const int key0 = key_of(i) + 16 * wave, here = (t.has >> wave & 1u) != 0 ? end : 0;
#pragma unroll
      for (int u = 0; u < COPIES; ++u) {
        const int key = key0 + u * CROWS + lane / UNITS;
        const bool in = key < here && (key >= low || key < a.sinks);
        lds_copy16(base, 0x7fffffffu, dst + u * 1024u, in ? from[u] : kOutOfRange);
      }
    }
  };
  auto copy_k = [&](int i, const Tile& t, uint32_t buf) { copy(i, t, t.k, from_k, lds0 + buf); };
  auto copy_v = [&](int i, const Tile& t) { copy(i, t, t.v, from_v, lds0 + (i & 1) * kTile); };

  f16_t acc[D / 32] = {};
  float top = -INFINITY;  // the reference of query c, in powers of two
  f16_t sum = {};         // of the probabilities: sixteen copies

  // Byte offsets within a tile: of row c, k elements 8 f .. of each 16 (8 bits: 16 f .. of
  // each 32); v elements 4 (l % 4) .. of 16 of row 4 f + l / 4 % 4 (8 bits: 8 (l % 2) .. of
  // row 4 f + l / 2 % 4, + 8 for l / 8 % 2), the second 16 of 32 for l / 16 % 2.
  const int half = lane >> 4 & 1;
  const int krow = c * BYTES + ((f ^ prompt_swizzle<UNITS, Q8>(c)) * 16);
  int vrow;
  if constexpr (Q8) {
    const int x = lane >> 1 & 7, r = 8 * (x >> 2) + 4 * f + (x & 3);
    vrow = r * BYTES + ((half ^ prompt_swizzle<UNITS, true>(r)) * 16) + 8 * (lane & 1);
  } else {
    const int r = 4 * f + (lane >> 2 & 3);
    vrow = r * BYTES + (((2 * half + (lane >> 1 & 1)) ^ prompt_swizzle<UNITS, false>(r)) * 16) +
           8 * (lane & 1);
  }
  float kscale[4], vscale[4];  // 8 bits: of a tile's 16-row groups
  vec8 ones;
#pragma unroll
  for (int i = 0; i < 8; ++i) ones[i] = static_cast<T>(1.0f);
  // K's operands of 32 keys: the e-th product takes lane elements from LDS four products
  // ahead.
  constexpr int N = D / 16, AHEAD = 4;
  constexpr int kFree = Q8 ? AHEAD - 1 : AHEAD;  // product e leaves room for that of e + kFree
  struct Ahead {
    vec8 at[AHEAD];
  };
  // Places in LDS of its reads, of the tile that is read: the rest of an address is a
  // constant.
  constexpr int KA = Q8 ? D / 32 : D / 16, VA = Q8 ? D / 32 : D / 16;
  uint32_t ka[KA], va[VA];
#pragma unroll
  for (int e = 0; e < KA; ++e) ka[e] = lds_address(kv) + 2 * kTile + (krow ^ (32 * e));
#pragma unroll
  for (int e = 0; e < VA; ++e)
    va[e] = lds_address(kv) +
            (Q8 ? vrow ^ (32 * e) : vrow ^ (64 * (e / 2)) ^ (UNITS > 8 ? 128 * (e % 2) : 0));
  auto shift_by = [](auto& at, uint32_t by) {
#pragma unroll
    for (uint32_t& x : at) x += by;
  };
  typedef __attribute__((address_space(3))) const u4_t lds_u4_t;
  // (j: which 32 keys of the tile.  8 bits: two products' elements side by side)
  auto read_k = [&](Ahead& x, int e, int j) {
    if constexpr (Q8) {
      if (e % 2 == 1 || e >= N) return;
      const float s = c < 16 ? kscale[2 * j] : kscale[2 * j + 1];
      const u4_t w4 = *(lds_u4_t*)(uintptr_t)(ka[e / 2] + j * 32 * BYTES);
      x.at[e % AHEAD] = from_float8<E>(w4[0], w4[1], s, s);
      x.at[e % AHEAD + 1] = from_float8<E>(w4[2], w4[3], s, s);
    } else if (e < N) {
      x.at[e % AHEAD] = __builtin_bit_cast(vec8, *(lds_u4_t*)(uintptr_t)(ka[e] + j * 32 * BYTES));
    }
  };
  // V^T of the n-th 16 keys for 32 elements.
  auto values = [&](int d, int n) {
    if constexpr (Q8) {
      const i2_t v2 =
          __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds2_t*)(uintptr_t)(va[d] + n * 16 * BYTES));
      return from_float8<E>(v2[0], v2[1], vscale[n], vscale[n]);
    } else {
      s4_t v2[2];
#pragma unroll
      for (int e = 0; e < 2; ++e)
        v2[e] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (lds4_t*)(uintptr_t)(va[2 * d + e] + n * 16 * BYTES + e * 8 * BYTES));
      return __builtin_bit_cast(
          vec8, us8_t(__builtin_shufflevector(__builtin_bit_cast(us4_t, v2[0]),
                                              __builtin_bit_cast(us4_t, v2[1]), 0, 1, 2, 3, 4, 5, 6, 7)));
    }
  };
  // Hides what this lane's queries do not see of 32 keys; `has`: which of their two 16-row
  // groups has a page.
  auto hide = [&](f16_t& x, int key0, uint32_t has) {
    auto below = [](int n) { return (1u << min(max(n, 0), 4)) - 1u; };
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int key = key0 + 8 * u + 4 * f;
      const uint32_t near = ~below(pos - a.window + 1 - key) | below(a.sinks - key);
      uint32_t seen = near & below(min(pos + 1, end) - key);
      seen = (has >> (u / 2) & 1u) != 0 ? seen : 0u;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if ((seen >> e & 1u) == 0) x[4 * u + e] = -INFINITY;
    }
  };
  float m;  // the largest of a lane's scores of the next 32 keys, not scaled
  auto largest = [&](const f16_t& x) {
    m = x[0];
#pragma unroll
    for (int e = 1; e < 16; ++e) m = fmaxf(m, x[e]);
  };
  auto move = [&]() {
    if (!__any(m * a.scale - top > kPagedSlack + kPagedLift<E>)) return;
    const Pair both = swap_pair<32>(m * a.scale);
    const float up = fmaxf(fmaxf(both.a, both.b) - kPagedLift<E>, top);
    const float keep = up == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(top - up);
    top = up;
#pragma unroll
    for (int e = 0; e < 16; ++e) sum[e] *= keep;
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[d][e] *= keep;
  };
  // Probabilities and sums of the j-th 32 keys of a tile, whose scores are x, beside the
  // scores of the next 32 (the next_j-th of theirs): a product of the scores, two
  // exponentials, and so on, then the sums' products, beside them the next scores' maximum
  // and the first operands of the products after them (the after_j-th 32 keys where
  // `between` has left ka).
  Ahead k;
  auto turn = [&](const f16_t& x, f16_t& next, int j, int next_j, int after_j, auto between) {
    Ahead v;
    move();
    vec8 p[2];
    const float base = top == -INFINITY ? 0.0f : top;
    auto read_v = [&](int e) { v.at[e % AHEAD] = values(e % (D / 32), 2 * j + e / (D / 32)); };
    constexpr int PER = 16 / N;  // scores beside a product
#pragma unroll
    for (int e = 0; e < N; ++e) {
      next = mfma32<E>(k.at[e % AHEAD], q[e], e == 0 ? f16_t{} : next);
#pragma unroll
      for (int u = 0; u < PER; ++u) {
        const int at = e * PER + u;
        p[at / 8][at % 8] =
            static_cast<T>(__builtin_amdgcn_exp2f(__builtin_fmaf(x[at], a.scale, -base)));
      }
      read_k(k, e + kFree, next_j);
      if (e + AHEAD >= N) read_v(e + AHEAD - N);
      __builtin_amdgcn_sched_barrier(0);
    }
    between();
    // (The probabilities are rounded to 16 bits because the matrix cores take them so: each
    // is off by half a step at most, in fp16 of 2^-24 at least, and the sum, ones times P^T
    // in fp32, is of the rounded.  v_dot2, which would add pairs, takes the matrix cores'
    // turns: four beside each product and the two take 1.6 times as long.)
    constexpr int M = D / 16;
#pragma unroll
    for (int e = 0; e < M; ++e) {
      if (e % (D / 32) == 0) sum = mfma32<E>(ones, p[e / (D / 32)], sum);
      acc[e % (D / 32)] = mfma32<E>(v.at[e % AHEAD], p[e / (D / 32)], acc[e % (D / 32)]);
      if (e + AHEAD < M) read_v(e + AHEAD);
      if (e + AHEAD >= M) read_k(k, e + AHEAD - M, after_j);
      if (e == M / 2) largest(next);
      if (e < M / 2 || e == M - 1) __builtin_amdgcn_sched_barrier(0);
    }
  };
  // Takes what is not finite out of this wave's 16 rows of a tile's v, for a hidden row's
  // infinity or NaN must not meet its zero probability.  What tokens that see them are to
  // have is left for the end.
  bool cleaned = false;
  auto clean = [&](int buf) {
    u4_t* const vt = reinterpret_cast<u4_t*>(kv + buf * kTile + 16 * wave * BYTES);
    const float s = wave < 2 ? (wave == 0 ? vscale[0] : vscale[1])
                             : (wave == 2 ? vscale[2] : vscale[3]);
    bool any = false;
#pragma unroll
    for (int e = 0; e < 16 * UNITS / 64; ++e) {
      u4_t x = vt[e * 64 + lane];
      if constexpr (Q8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const us8_t y = __builtin_bit_cast(us8_t, from_float8<E>(x[i], 0, s, s));
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            const bool is = (y[n] & E::kExponent) == E::kExponent;
            any |= is;
            x[i] &= is ? ~(0xffu << (8 * n)) : ~0u;
          }
        }
      } else {
        const us8_t y = __builtin_bit_cast(us8_t, x);
        const us8_t fine = (y & E::kExponent) == E::kExponent ? us8_t{} : y;
        x = __builtin_bit_cast(u4_t, fine);
#pragma unroll
        for (int n = 0; n < 8; ++n) any |= fine[n] != y[n];
      }
      if (__any(any)) vt[e * 64 + lane] = x;
    }
    cleaned |= __any(any) != 0;
  };

  auto spread = [&](uint32_t bytes, float (&to)[4]) {
    if constexpr (Q8) {
#pragma unroll
      for (int n = 0; n < 4; ++n) to[n] = power(bytes >> (8 * n) & 255);
    }
  };
  // Every query sees all of a tile's keys.
  auto plain = [&](int i, uint32_t has) {
    const int key0 = key_of(i);
    return has == 15u && key0 + KT <= min(span.len + early + 1, end) &&
           (key0 > span.len + late - a.window || key0 + KT <= a.sinks);
  };
  f16_t x, y;  // scores of 32 keys
  uint32_t buf0 = 2 * kTile, buf1 = 3 * kTile, buf2 = 4 * kTile;  // of k of tiles i, i + 1, i + 2
  Tile now = {}, next = {};  // tiles i and i + 1
  if (count > 0) {
    look_up(0);
    now = tile_of(0), next = tile_of(1);
    copy_k(0, now, buf0);
    copy_v(0, now);
    if (count > 1) copy_k(1, next, buf1);
    __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));
    lds_barrier();
    spread(now.k_scales, kscale);
#pragma unroll
    for (int e = 0; e < AHEAD; ++e) read_k(k, e, 0);
#pragma unroll
    for (int e = 0; e < N; ++e) {
      x = mfma32<E>(k.at[e % AHEAD], q[e], e == 0 ? f16_t{} : x);
      read_k(k, e + kFree, 0);
    }
    largest(x);
#pragma unroll
    for (int e = 0; e < AHEAD; ++e) read_k(k, e, 1);
  }
#pragma unroll 1
  for (int i = 0; i < count; ++i) {
    __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));  // v of tile i and k of tile i + 1 are there
    lds_barrier();
    const uint32_t has = now.has;
    const int key0 = key_of(i);
    const bool all = plain(i, has);
    spread(now.v_scales, vscale);
    if (!all) {
      clean(i & 1);
      if constexpr (Q8) {  // (a scale of 255, too: under it a zero code is NaN)
        uint32_t bytes = now.v_scales;
#pragma unroll
        for (int n = 0; n < 4; ++n)
          if ((bytes >> (8 * n) & 255) == 255) bytes ^= 128u << (8 * n);
        spread(bytes, vscale);
      }
      lds_barrier();
    }
    if (i + 1 < count) copy_v(i + 1, next);
    now = next;
    if (i + 2 < count) {
      if (((i + 2) & 63) == 0) look_up(i + 2);
      next = tile_of(i + 2);
      copy_k(i + 2, next, buf2);
    }
    if (!idle) {
      if (!all) hide(x, key0, has), largest(x);
      turn(x, y, 0, 1, 0, [&]() {
        spread(now.k_scales, kscale);
        shift_by(ka, buf1 - buf0);
      });
      if (!all) hide(y, key0 + 32, has >> 2), largest(y);
      turn(y, x, 1, 0, 1, []() {});
      shift_by(va, i % 2 == 0 ? kTile : 0u - kTile);
    }
    const uint32_t free = buf0;
    buf0 = buf1, buf1 = buf2, buf2 = free;
  }

  // What was taken out comes back to the tokens that see it: an infinity as it is, a NaN as
  // both (which make a NaN).
  lds_barrier();
  if (lane == 0) reinterpret_cast<int*>(kv)[wave] = cleaned ? 1 : 0;
  lds_barrier();
  const int4 flags = *reinterpret_cast<const int4*>(kv);
  if (__builtin_amdgcn_readfirstlane(flags.x | flags.y | flags.z | flags.w) != 0) {
#pragma unroll 1
    for (int i = 0; i < count; ++i)
#pragma unroll 1
      for (int key = key_of(i); key < min(key_of(i) + KT, end); ++key) {
        const int page = __builtin_amdgcn_readfirstlane(page_at(key));
        const uint32_t has = __ballot(is_page(page_at(key_of(i) + 16 * (lane & 3)))) & 15u;
        if (!is_page(page) || plain(i, has)) continue;
        const char* const row = a.v + h * a.vh + page * a.vp + (key & ((1 << a.shift) - 1)) * a.vr;
        const float s = Q8 ? power(a.v_scales[static_cast<int64_t>(page) * a.n_kv + h]) : 1.0f;
        const bool sees = key <= pos && (key > pos - a.window || key < a.sinks);
#pragma unroll
        for (int n = 0; n < D / 8; ++n) {
          us4_t v;
          if constexpr (Q8) {
            const uint32_t w1 = *reinterpret_cast<const uint32_t*>(row + 8 * n + 4 * f);
            const us8_t z = __builtin_bit_cast(us8_t, from_float8<E>(w1, 0, s, s));
            v = __builtin_shufflevector(z, z, 0, 1, 2, 3);
          } else {
            v = *reinterpret_cast<const us4_t*>(row + 16 * n + 8 * f);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float z = (v[e] & E::kExponent) != E::kExponent ? 0.0f
                            : (v[e] & 0x7fff) != E::kExponent     ? __builtin_nanf("")
                            : (v[e] >> 15) != 0                   ? -INFINITY : INFINITY;
            acc[n / 4][4 * (n % 4) + e] += sees ? z : 0.0f;
          }
        }
      }
  }

  const int64_t rec0 = (static_cast<int64_t>(h) * a.shares + w) * rows_all;
  float* const sums = a.partial + rec0 * D;
  float* const stats = a.partial + static_cast<int64_t>(a.n_kv) * a.shares * rows_all * D + rec0 * 2;
  const int r = r0 + 32 * wave + c;
  const bool behind = r >= rows;  // the last token
  const float l = behind ? 0.0f : sum[0];
  if (behind) top = -INFINITY;
  else if (top == -INFINITY && l != 0.0f) top = 0.0f;  // NaN scores alone
  if (r >= rows_all) return;
  if (a.shares == 0) {
    const int node = r / a.qpk;
    T* const out = static_cast<T*>(a.out) +
                   ((static_cast<int64_t>(b) * a.T + node) * a.n_heads + h * a.qpk +
                    (r - node * a.qpk)) * D + 4 * f;
    typedef T vec4 __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int e = 0; e < D / 8; ++e) {
      vec4 y;
#pragma unroll
      for (int x = 0; x < 4; ++x)
        y[x] = static_cast<T>(l == 0.0f ? 0.0f : acc[e / 4][4 * (e % 4) + x] / l);
      *reinterpret_cast<vec4*>(out + 8 * e) = y;
    }
  } else {
    if (top != -INFINITY) {
#pragma unroll
      for (int e = 0; e < D / 8; ++e) {
        f4_t y;
#pragma unroll
        for (int x = 0; x < 4; ++x) y[x] = acc[e / 4][4 * (e % 4) + x];
        *reinterpret_cast<f4_t*>(sums + static_cast<int64_t>(r) * D + 8 * e + 4 * f) = y;
      }
    }
    if (f == 0) stats[2 * r] = top, stats[2 * r + 1] = l;
  }
}

}  // namespace
}  // namespace nibble
