// Attention over a paged cache for up to 32 query rows a kv head: the tokens of a
// decode step.
#pragma once

#include "paged_attention.h"

namespace nibble {
namespace {

// Products over 16 k.
typedef short s4_t __attribute__((ext_vector_type(4)));
template <class E>
__device__ __forceinline__ f4_t mfma16(s4_t a, s4_t b, f4_t c) {
  typedef _Float16 h4_t __attribute__((ext_vector_type(4)));
  if constexpr (std::is_same_v<E, Half>)
    return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(h4_t, a),
                                                 __builtin_bit_cast(h4_t, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(a, b, c, 0, 0, 0);
}

// Sum of the values of this lane and those before it.
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);  // row_shr:1, 2, 4, 8
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // row 0's to 1, 2's to 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);  // row 1's to 2 and 3
  return v;
}

// Sum of the values of a wave's lanes.
__device__ __forceinline__ int wave_total(int v) { return __builtin_amdgcn_readlane(wave_scan(v), 63); }

// What a sequence more costs a share, in tiles of one byte a value: its queries, pages
// and first rows come one behind the other, and its waves meet.  (Of 2 to 12 any will do:
// 32 to 100 sequences of up to 2000 to 8000 rows differ by 4%, and lose it at the ends.)
constexpr int kSequenceCost = 4;

// Which tiles of which sequences a share has.  Where it costs no more than a sequence's
// start, every sequence is cut by itself, into equal pieces (one, if that is as good):
// `per` tiles at most, the least of a few for which there are enough shares.  Else the
// sequences' tiles are laid one behind the other, a sequence's behind a gap of what it
// costs, and all that is cut into equal shares.  The lengths are on the GPU: every wave
// works it out alike, 64 sequences at a time, one a lane.
struct Line {
  int n = 0, upto = 0;       // of this lane's sequence, of the 64 from `from`: tiles and gap
  int from = 0, before = 0;  // (or pieces), those to its end, and those before the 64
  int per = 0, total = 0, gap = 0;
  bool alone = false;    // a share has a piece of one sequence
  bool empties = false;  // there are sequences without a tile
  __device__ __forceinline__ void cut(const AttendArgs& a, int sequence_cost) {
    gap = sequence_cost;
#pragma unroll 1
    for (int i = 0; i < a.B; i += 64) take(a, i, total), total = last();
    per = __builtin_amdgcn_readfirstlane(max((total + a.shares - 1) / a.shares, 1));
    if (a.B > 64) return;
    if (a.B == 1) {  // (the same without a look at other lanes)
      const int tiles = total > 0 ? total - gap : 0;
      const int worth = static_cast<int>(
          __builtin_amdgcn_sqrtf(a.join_cost * static_cast<float>(tiles)));
      const int size = max(max((tiles + a.shares - 1) / a.shares, worth), 1);
      alone = true, gap = 0;
      upto = total = __builtin_amdgcn_readfirstlane((tiles + size - 1) / size);
      return;
    }
    const int tiles = n > 0 ? n - gap : 0;
    const int all = wave_total(tiles);
    // `least` tiles in turn, and all / least pieces whose sums are written and joined
    const int worth = static_cast<int>(__builtin_amdgcn_sqrtf(a.join_cost * static_cast<float>(all)));
    const int least = __builtin_amdgcn_readfirstlane(
        max(max((all + a.shares - 1) / a.shares, worth), 1));
    // pieces of that many and a few more tiles, if there is room for them
#pragma unroll 1
    for (int k = 0; k <= 4; ++k) {
      const int size = least + (sequence_cost * k + 3) / 4;
      const int pieces = tiles > 0 ? (tiles + size - 1) / size : 0;
      if (wave_total(pieces) <= a.shares) {
        alone = true, gap = 0, n = pieces, upto = wave_scan(pieces), total = last();
        return;
      }
    }
  }
  __device__ __forceinline__ void take(const AttendArgs& a, int i, int tiles) {
    const int b = i + static_cast<int>(threadIdx.x & 63), t = b < a.B ? a.tiles(b) : 0;
    empties |= __any(b < a.B && t == 0) != 0;
    n = t > 0 ? t + gap : 0;
    from = i, before = tiles, upto = before + wave_scan(n);
  }
  __device__ __forceinline__ int last() const { return __builtin_amdgcn_readlane(upto, 63); }
  // The sequence at place x < total of the line, and the places [start, end) that it has.
  __device__ __forceinline__ int find(const AttendArgs& a, int x, int* start, int* end) {
    if (a.B > 64 && (x < before || x >= last())) {
      int tiles = 0;
#pragma unroll 1
      for (int i = 0; i < a.B && tiles <= x; i += 64) take(a, i, tiles), tiles = last();
    }
    const int at = __builtin_ctzll(__ballot(upto > x));
    *start = at > 0 ? __builtin_amdgcn_readlane(upto, at - 1) : before;
    *end = __builtin_amdgcn_readlane(upto, at);
    return from + at;
  }
};

// 8-bit rows of 64 or 128 bytes, units of 16: eight rows of a K read, and two units of
// rows 4g .. 4g + 3 of a V read, cover 32 banks once; 16-bit rows as in paged_swizzle.
template <int UNITS, bool Q8>
__device__ __forceinline__ int rows_swizzle(int r) {
  if (Q8 && UNITS == 4) return (r >> 1 & 1) << 1 | (r >> 2 & 1);
  return paged_swizzle<UNITS>(r);
}

// One workgroup: the query rows of one kv head, and a share of the line of tiles.  A
// wave has every tile's 16 rows that it copies itself, into LDS of its own: nothing
// waits for another wave before a sequence's end.  Of its ring of NB units (16 rows of k
// and v) all but the one that it reads are on their way.  The last of the workgroups that
// have a piece of a sequence joins them.
//
// Memory bounds it where there is much to read: a step of 32 sequences of 8-bit rows takes
// 66 us for 338 MB, one token over 65000 of 16 bits 51 for 266 MB, 5.2 TB/s of the 6.9 that
// a kernel reaches that only reads.  Where there is little, what comes one behind the other
// does: 4 us from the launch to the first rows (lengths, pages, rows), 4 to 5 from the
// last piece to the output (sums, counter, sums), of 13 us for one token over 4000 rows.
// 32 x one token over up to 8100 rows of 16 bits take 111 us (6.1 TB/s), of heads of 64 66
// (5.1), in 8 bits 47 to 51 (3.3 to 3.6: the least data a unit, and its instructions are as
// many); 32 x 6 tokens over 8000, two tiles of query rows, 140 us of 16 bits (4.8 TB/s) and
// 83 of 8 (4.1).  That form, of heads of 128, spills 18 (8 bits: 4) vector registers, in what
// it does once a sequence; all forms keep 84 to 141 scalars in lanes, which loops read back.
// The copies go past the caches (nt), for a row is read once a call: 15% more of the rate.
// 8 KB a wave are enough on their way; with 16 a step of 16 to 100 sequences takes 4 to 8%
// longer.
template <class E, int D, int QT, bool Q8>
__global__ __launch_bounds__(kPagedThreads, 2) void rows_kernel(AttendArgs a) {
  using T = typename E::type;
  using vec8 = typename E::vec8;
  constexpr int BYTES = Q8 ? D : 2 * D, UNITS = BYTES / 16;  // of a row; its 16-byte units
  constexpr int CROWS = 64 / UNITS, COPIES = 16 / CROWS;     // rows of a copy; of k or v, a unit
  constexpr int kUnit = 16 * BYTES;
  constexpr int NB = 8192 / (2 * kUnit);
  constexpr int kPending = (2 * NB - 1) * COPIES;  // copies behind those that are waited for
  constexpr int QUADS = D / 4, ALL = QT * 16;
  constexpr int ROWS = kPagedThreads / QUADS;  // rows of outputs at once
  typedef int i2_t __attribute__((ext_vector_type(2)));
  typedef unsigned short us4_t __attribute__((ext_vector_type(4)));
  typedef unsigned short us8_t __attribute__((ext_vector_type(8)));
  typedef T vec4 __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) s4_t lds4_t;
  typedef __attribute__((address_space(3))) i2_t lds2_t;
  constexpr int kRing = 4 * NB * 2 * kUnit, kSums = 4 * 4 * ALL * D;
  __shared__ __attribute__((aligned(16))) char ring[kRing > kSums ? kRing : kSums];
  __shared__ float stat[2][4][ALL > ROWS ? ALL : ROWS];
  __shared__ int arrived;

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  const int g = lane >> 4, c = lane & 15;
  // The heads of a share on one XCD (id % 8): they read the same pages.
  const int eight = blockIdx.x / (8 * a.n_kv), in_eight = blockIdx.x - eight * 8 * a.n_kv;
  const int w = 8 * eight + (in_eight & 7), h = in_eight >> 3;
  if (w >= (a.shares > 0 ? a.shares : a.B)) return;
  const int rows_all = a.T * a.qpk;
  const int u = threadIdx.x % QUADS, mine = threadIdx.x / QUADS;  // of an output: its quad, row
  f4_t* const red = reinterpret_cast<f4_t*>(ring);
  auto write = [&](int b, int row, f4_t o, float l) {
    vec4 y;
#pragma unroll
    for (int x = 0; x < 4; ++x) y[x] = static_cast<T>(l == 0.0f ? 0.0f : o[x] / l);
    const int node = row / a.qpk;
    T* const out = static_cast<T*>(a.out) +
                   ((static_cast<int64_t>(b) * a.T + node) * a.n_heads + h * a.qpk +
                    (row - node * a.qpk)) * D;
    *reinterpret_cast<vec4*>(out + 4 * u) = y;
  };
  typedef uint32_t u2_t __attribute__((ext_vector_type(2)));
  constexpr int kCoherent = 16;  // sc1: past this XCD's L2
  auto coherent = [&](float* p) { return make_rsrc(p, 0x7fffffffu); };
  auto share = [&](float top, float most) {
    return top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(top - most);
  };

  int at = 0, upto = 1;  // this share's places (or, where nothing is split, a sequence)
  Line line;
  if (a.shares > 0) {
    line.cut(a, Q8 ? kSequenceCost : kSequenceCost / 2);
    at = line.alone ? w : w * line.per, upto = min(line.alone ? w + 1 : at + line.per, line.total);
    if (line.empties)  // zeros for sequences of which nothing is seen
#pragma unroll 1
      for (int b = w; b < a.B; b += a.shares)
        if (__builtin_amdgcn_readfirstlane(a.tiles(b)) == 0)
          for (int row = mine; row < rows_all; row += ROWS)
            write(b, row, f4_t{0.0f, 0.0f, 0.0f, 0.0f}, 0.0f);
  }
#pragma unroll 1
  while (at < upto) {
    // The next sequence's tiles [x0, x0 + count), those that it sees counted: piece
    // `piece` of `pieces`, the first of which is of share `first`.
    int b = w, start = 0, stop = 0;
    if (a.shares > 0) b = line.find(a, at, &start, &stop);
    const PagedSpan span = PagedSpan(a, b).uniform();
    const Seen all = span.seen(a);
    int x0 = 0, count = all.first + all.upto - all.from, first = w, pieces = 1;
    if (line.alone) {
      first = start, pieces = stop - start;
      const int size = (count + pieces - 1) / pieces;
      x0 = (w - start) * size, count = min(size, count - x0);
      at = upto;
    } else if (a.shares > 0) {
      start += line.gap;
      const int begin = max(at, start);
      at = min(upto, stop);
      if (begin >= at) continue;
      first = start / line.per, pieces = (stop - 1) / line.per - first + 1;
      x0 = begin - start, count = at - begin;
    } else {
      at = upto;
    }
    const int rows = span.live * a.qpk, late = span.live - 1, end = span.total;
    const int low = max(span.len - a.window + 1, 0);
    auto key_of = [&](int i) {  // of this wave's unit of the i-th tile
      const int x = x0 + i;
      return (x < all.first ? x : x - all.first + all.from) * kPagedKeys + 16 * wave;
    };

    // Queries: lane (g, c) holds of row c of a tile the elements that it multiplies with
    // those of a key: of 32 8 g .., or with 8-bit keys, of 64 16 g ...
    vec8 q[QT][D / 32];
    int pos[QT];  // the row of its token
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      const int r = 16 * t + c;
      const bool in = r < rows;
      const int node = in ? r / a.qpk : 0;
      pos[t] = span.len + node;
      const T* const from = static_cast<const T*>(a.q) +
                            ((static_cast<int64_t>(b) * a.T + node) * a.n_heads + h * a.qpk +
                             (in ? r - node * a.qpk : 0)) * D;
#pragma unroll
      for (int s = 0; s < D / 32; ++s) {
        const int e = Q8 ? 64 * (s / 2) + 16 * g + 8 * (s % 2) : 32 * s + 8 * g;
        q[t][s] = in ? *reinterpret_cast<const vec8*>(from + e) : vec8{};
      }
    }

    // Pages (and scales) of 64 units, one a lane: of those that are copied, and of those
    // that are computed.  (The compiler counts its own loads alone: one that it thought
    // on its way would make it wait, inside the loop, for every copy.)
    const int32_t* const table = a.table + static_cast<int64_t>(b) * a.width;
    auto is_page = [&](int page) { return page >= 0 && page < a.n_pages; };
    int pages = 0, copied_k = 0, copied_v = 0, k_scales = 0, v_scales = 0;
    uint64_t there = 0;
    auto look_up = [&](int i) {
      pages = table[min(key_of(min(i + lane, count - 1)) >> a.shift, a.width - 1)];
      __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));
    };
    auto look_up_scales = [&]() {
      if constexpr (Q8) {
        const int64_t from = static_cast<int64_t>(is_page(pages) ? pages : 0) * a.n_kv + h;
        copied_k = a.k_scales[from], copied_v = a.v_scales[from];
        __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));
      }
    };
    auto next_64 = [&]() {
      there = __ballot(is_page(pages));
      k_scales = copied_k, v_scales = copied_v;
    };
    const uint32_t lds0 = lds_address(ring) + wave * NB * 2 * kUnit;
    // The copies of the i-th unit's k (v); rows that no token sees read as zeros.
    auto copy = [&](int i, const char* base, int64_t page_stride, int64_t row_stride, uint32_t dst) {
      const int page = __builtin_amdgcn_readlane(pages, i & 63), key0 = key_of(i);
      const bool is = i < count && is_page(page);
      const int here = is ? end : 0;
      const char* const from = base + (is ? page : 0) * page_stride +
                               (key0 & ((1 << a.shift) - 1)) * row_stride;
#pragma unroll
      for (int x = 0; x < COPIES; ++x) {
        const int r = x * CROWS + lane / UNITS, key = key0 + r;
        const bool in = key < here && (key >= low || key < a.sinks);
        const uint32_t unit16 = ((lane % UNITS) ^ rows_swizzle<UNITS, Q8>(r)) * 16u;
        lds_stream16(from, 0x7fffffffu, dst + x * 1024u,
                     in ? r * static_cast<uint32_t>(row_stride) + unit16 : kOutOfRange);
      }
    };
    const char* const kbase = a.k + h * a.kh;
    const char* const vbase = a.v + h * a.vh;
    auto copy_k = [&](int i) { copy(i, kbase, a.kp, a.kr, lds0 + (i % NB) * 2 * kUnit); };
    auto copy_v = [&](int i) { copy(i, vbase, a.vp, a.vr, lds0 + (i % NB) * 2 * kUnit + kUnit); };

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
    // Byte offsets within a unit: of row c, k elements 8 g .. of each 32 (8 bits: 16 g ..
    // of each 64); of row 4 g + c / 4 (c / 2 % 4), v elements 4 (c % 4) .. of each 16 (8
    // (c % 2) .. of each 16 of 32, the first for c < 8).
    const int krow = c * BYTES + ((g ^ rows_swizzle<UNITS, Q8>(c)) * 16);
    const int vr = Q8 ? 4 * g + (c >> 1 & 3) : 4 * g + (c >> 2);
    const int vrow = vr * BYTES + (((Q8 ? c >> 3 : c >> 1 & 1) ^ rows_swizzle<UNITS, Q8>(vr)) * 16) +
                     8 * (c & 1);
    const f4_t zero = {0.0f, 0.0f, 0.0f, 0.0f};
    const s4_t ones = __builtin_bit_cast(
        s4_t, std::is_same_v<E, Half> ? 0x3c003c003c003c00ull : 0x3f803f803f803f80ull);

    // Whether every query sees all of the i-th unit's keys.
    auto plain = [&](int i) {
      const int key0 = key_of(i);
      return (there >> (i & 63) & 1u) != 0 && key0 + 16 <= min(span.len + 1, end) &&
             (key0 > span.len + late - a.window || key0 + 16 <= a.sinks);
    };
    auto step = [&](int i, auto tail) {
      constexpr bool kTail = decltype(tail)::value;
      const int key0 = key_of(i), buf = (wave * NB + i % NB) * 2 * kUnit;
      uint32_t seen[QT] = {};  // a bit for each of a lane's scores
      bool any = true;
      if constexpr (kTail) {
        auto below = [](int n) { return (1u << min(max(n, 0), 4)) - 1u; };
        const bool has = (there >> (i & 63) & 1u) != 0;
        uint32_t some = 0;
#pragma unroll
        for (int t = 0; t < QT; ++t) {
          const int key = key0 + 4 * g;
          const uint32_t near = ~below(pos[t] - a.window + 1 - key) | below(a.sinks - key);
          seen[t] = has ? near & below(min(pos[t] + 1, end) - key) : 0;
          some |= seen[t];
        }
        any = __any(some != 0) != 0;
      }
      asm volatile("s_waitcnt vmcnt(%0)" : : "n"(kPending) : "memory");
      f4_t s[QT];
      const char* const kt = ring + buf;
      const float ks = power(Q8 ? __builtin_amdgcn_readlane(k_scales, i & 63) : 0);
      if constexpr (Q8) {
#pragma unroll
        for (int s2 = 0; s2 < D / 64; ++s2) {
          const u4_t w4 = *reinterpret_cast<const u4_t*>(kt + (krow ^ (64 * s2)));
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const vec8 ka = from_float8<E>(w4[2 * e], w4[2 * e + 1], ks, ks);
#pragma unroll
            for (int t = 0; t < QT; ++t)
              s[t] = E::mfma(ka, q[t][2 * s2 + e], s2 + e == 0 ? zero : s[t]);
          }
        }
      } else {
#pragma unroll
        for (int ss = 0; ss < D / 32; ++ss) {
          const vec8 ka = *reinterpret_cast<const vec8*>(kt + (krow ^ (64 * ss)));
#pragma unroll
          for (int t = 0; t < QT; ++t) s[t] = E::mfma(ka, q[t][ss], ss == 0 ? zero : s[t]);
        }
      }
      // The unit's k has been read: the next one takes its place.
      asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
      const bool refill = ((i + NB) & 63) == 0;
      if (refill) look_up(i + NB);
      copy_k(i + NB);
      s4_t p[QT];
      float m[QT];
      bool moves = false;
#pragma unroll
      for (int t = 0; t < QT; ++t) {
        if constexpr (kTail) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if ((seen[t] >> e & 1u) == 0) s[t][e] = -INFINITY;
        }
        m[t] = fmaxf(fmaxf(s[t][0], s[t][1]), fmaxf(s[t][2], s[t][3])) * a.scale;
        moves |= m[t] - top[t] > kPagedSlack + kPagedLift<E>;
      }
      if (__any(moves)) {
#pragma unroll
        for (int t = 0; t < QT; ++t) {
          const float up = fmaxf(swap_max(m[t]) - kPagedLift<E>, top[t]);
          const float keep = up == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(top[t] - up);
          top[t] = up;
#pragma unroll
          for (int e = 0; e < 4; ++e) sum[t][e] *= keep;
#pragma unroll
          for (int d = 0; d < D / 16; ++d)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[t][d][e] *= keep;
        }
      }
#pragma unroll
      for (int t = 0; t < QT; ++t) {
        const float base = top[t] == -INFINITY ? 0.0f : top[t];
        vec4 e4;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          e4[e] = static_cast<T>(__builtin_amdgcn_exp2f(__builtin_fmaf(s[t][e], a.scale, -base)));
        p[t] = __builtin_bit_cast(s4_t, e4);
        // (The probabilities are rounded to 16 bits because the matrix cores take them
        // so, and the sum, ones times P^T in fp32, is of the rounded.)
        sum[t] = mfma16<E>(ones, p[t], sum[t]);
      }
      asm volatile("s_waitcnt vmcnt(%0)" : : "n"(kPending) : "memory");
      const uint32_t vt = lds_address(ring) + buf + kUnit;
      const float vs = power(Q8 ? __builtin_amdgcn_readlane(v_scales, i & 63) : 0);
      // V^T of the unit's keys for two runs of 16 elements.
      auto values = [&](int d2, us4_t (&v)[2]) {
        if constexpr (Q8) {
          const i2_t v2 = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
              (lds2_t*)(uintptr_t)(vt + (vrow ^ (32 * d2))));
          const us8_t z = __builtin_bit_cast(us8_t, from_float8<E>(v2[0], v2[1], vs, vs));
          v[0] = __builtin_shufflevector(z, z, 0, 1, 2, 3);
          v[1] = __builtin_shufflevector(z, z, 4, 5, 6, 7);
        } else {
#pragma unroll
          for (int e = 0; e < 2; ++e)
            v[e] = __builtin_bit_cast(us4_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (lds4_t*)(uintptr_t)(vt + (vrow ^ (32 * (2 * d2 + e))))));
        }
      };
      // A hidden row's infinity or NaN must not meet its zero probability.  Rows that no
      // token sees read as zeros; where the tokens see different ones and a value is not
      // finite, every token has the products of its own rows alone.
      bool odd = false;
      if constexpr (kTail) {
        if (late > 0 && any) {
#pragma unroll
          for (int d2 = 0; d2 < D / 32; ++d2) {
            us4_t v[2];
            values(d2, v);
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
              for (int x = 0; x < 4; ++x) odd |= (v[e][x] & E::kExponent) == E::kExponent;
          }
          odd = __any(odd) != 0;
        }
      }
      if (!odd) {
        if (any) {
#pragma unroll
          for (int d2 = 0; d2 < D / 32; ++d2) {
            us4_t v[2];
            values(d2, v);
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
              for (int t = 0; t < QT; ++t)
                acc[t][2 * d2 + e] = mfma16<E>(__builtin_bit_cast(s4_t, v[e]), p[t], acc[t][2 * d2 + e]);
          }
        }
      } else {
#pragma unroll 1
        for (int n = 0; n <= late; ++n) {
          us4_t shows = {};  // which of this lane's four keys token n sees
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int key = key0 + 4 * g + x, row = span.len + n;
            shows[x] = key <= row && key < end && (key > row - a.window || key < a.sinks) ? 0xffff : 0;
          }
#pragma unroll
          for (int d2 = 0; d2 < D / 32; ++d2) {
            us4_t v[2];
            values(d2, v);
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
              for (int t = 0; t < QT; ++t) {
                const f4_t more = mfma16<E>(__builtin_bit_cast(s4_t, us4_t(v[e] & shows)), p[t], zero);
#pragma unroll
                for (int x = 0; x < 4; ++x)
                  acc[t][2 * d2 + e][x] += pos[t] == span.len + n ? more[x] : 0.0f;
              }
          }
        }
      }
      asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
      copy_v(i + NB);
      if (refill) look_up_scales();
      if (((i + 1) & 63) == 0) next_64();
    };

    if (count > 0) look_up(0);
    if (a.sign != 1.0f) {  // a scale that is not positive: its sign goes into q, exactly
#pragma unroll
      for (int t = 0; t < QT; ++t)
#pragma unroll
        for (int s = 0; s < D / 32; ++s)
#pragma unroll
          for (int i = 0; i < 8; ++i)
            q[t][s][i] = static_cast<T>(static_cast<float>(q[t][s][i]) * a.sign);
    }
#pragma unroll
    for (int t = 0; t < QT; ++t)
#pragma unroll
      for (int x = 0; x < D / 32; ++x) asm volatile("" : "+v"(q[t][x]));  // (here already, too)
    if (count > 0) {
#pragma unroll 1
      for (int i = 0; i < NB; ++i) copy_k(i), copy_v(i);
      look_up_scales();
      next_64();
    }
#pragma unroll 1
    for (int i = 0; i < count;) {
#pragma unroll 1
      for (; i < count && plain(i); ++i) step(i, std::false_type{});
#pragma unroll 1
      for (; i < count && !plain(i); ++i) step(i, std::true_type{});
    }
    asm volatile("s_waitcnt vmcnt(0)" : : : "memory");  // no copy may land in what follows
    lds_barrier();

    // The waves meet: statistics and sums through LDS, then each wave's sums on the
    // common maximum.  Unit (16 bytes) x of row c of 16 lies at unit x ^ (c % 8).
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      const int row = 16 * t + c;
      const bool behind = row >= rows;  // the last token
      if (behind) top[t] = -INFINITY;
      else if (top[t] == -INFINITY && sum[t][0] != 0.0f) top[t] = 0.0f;  // NaN scores alone
      if (g == 0) {
        stat[0][wave][row] = top[t];
        stat[1][wave][row] = behind ? 0.0f : sum[t][0];
      }
#pragma unroll
      for (int d = 0; d < D / 16; ++d)  // [4][ALL][QUADS]
        red[(wave * ALL + row) * QUADS + ((4 * d + g) ^ (c & 7))] = acc[t][d];
    }
    lds_barrier();
    // A piece's sums [rows][D], and its rows' (top, sum), seen by every XCD.  A share has
    // two places: the second for a sequence that begins within it, and goes on.
    auto slot_of = [&](int s) {
      return 2 * s + (!line.alone && s == first && s * line.per < start ? 1 : 0);
    };
    const int slot = slot_of(w);
    const bool whole = pieces == 1;
    auto sums_of = [&](int s) {
      const int64_t n = static_cast<int64_t>(rows_all) * D;
      return coherent(a.partial + (static_cast<int64_t>(h) * a.slots + s) * n);
    };
    auto stats_of = [&](int s) {
      const int64_t n = static_cast<int64_t>(a.n_kv) * a.slots * rows_all;
      return coherent(a.partial + n * D + (static_cast<int64_t>(h) * a.slots + s) * rows_all * 2);
    };
    for (int row = mine; row < rows_all; row += ROWS) {
      float mr = stat[0][0][row], l = 0.0f;
#pragma unroll
      for (int x = 1; x < 4; ++x) mr = fmaxf(mr, stat[0][x][row]);
      f4_t o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const float keep = share(stat[0][x][row], mr);
        l += stat[1][x][row] * keep;
        const f4_t v = red[(x * ALL + row) * QUADS + (u ^ (row & 7))];
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] += v[i] * keep;
      }
      if (whole) {
        write(b, row, o, l);
      } else {
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4_t, o), sums_of(slot),
                                               (row * D + 4 * u) * 4, 0, kCoherent);
        if (u == 0)
          __builtin_amdgcn_raw_buffer_store_b64(
              u2_t{__builtin_bit_cast(uint32_t, mr), __builtin_bit_cast(uint32_t, l)},
              stats_of(slot), row * 8, 0, kCoherent);
      }
    }
    if (!whole) {
      // The piece is written; the last of its sequence (and head) to be so joins them.
      wait_vm_stores();
      lds_barrier();
      int* const counter = a.counters + b * a.n_kv + h;
      if (threadIdx.x == 0)
        arrived = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      lds_barrier();
      if (arrived == pieces - 1) {
        if (threadIdx.x == 0)
          __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        // G groups of a row's lanes, every G-th piece each, meet in LDS.
        constexpr int N = 16;
        int G = 1;
        while (2 * G * rows_all <= ROWS) G *= 2;
        const int grp = mine % G, step = ROWS / G;
#pragma unroll 1
        for (int row0 = 0; row0 < rows_all; row0 += step) {
          const int row = min(row0 + mine / G, rows_all - 1);
          float mr = -INFINITY, l = 0.0f;
          f4_t o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 1
          for (int s0 = 0; s0 < pieces; s0 += N * G) {
            float tops[N], ls[N], most = mr;
            f4_t v[N];
            const auto sums = sums_of(2 * (first + s0)), stats = stats_of(2 * (first + s0));
#pragma unroll
            for (int e = 0; e < N; ++e) {
              const int s = min(e * G + grp, pieces - 1 - s0);
              const int at_row = (slot_of(first + s0 + s) - 2 * (first + s0)) * rows_all + row;
              const u2_t st = __builtin_bit_cast(
                  u2_t, __builtin_amdgcn_raw_buffer_load_b64(stats, at_row * 8, 0, kCoherent));
              tops[e] = __builtin_bit_cast(float, static_cast<uint32_t>(st[0]));
              ls[e] = __builtin_bit_cast(float, static_cast<uint32_t>(st[1]));
              v[e] = __builtin_bit_cast(f4_t, __builtin_amdgcn_raw_buffer_load_b128(
                                                  sums, (at_row * D + 4 * u) * 4, 0, kCoherent));
            }
#pragma unroll
            for (int e = 0; e < N; ++e) {
              if (s0 + e * G + grp >= pieces) tops[e] = -INFINITY;
              most = fmaxf(most, tops[e]);
            }
            const float keep = share(mr, most);
            l *= keep;
#pragma unroll
            for (int x = 0; x < 4; ++x) o[x] *= keep;
            mr = most;
#pragma unroll
            for (int e = 0; e < N; ++e) {
              // (A piece that saw nothing has no part; one of no weight has: an infinity or
              // a NaN in its sums must not be lost.)
              const float weight = share(tops[e], mr);
              l += tops[e] == -INFINITY ? 0.0f : ls[e] * weight;
#pragma unroll
              for (int x = 0; x < 4; ++x) o[x] += tops[e] == -INFINITY ? 0.0f : v[e][x] * weight;
            }
          }
          if (G > 1) {
            lds_barrier();  // (the sums of the row before have been read)
            red[mine * QUADS + u] = o;
            if (u == 0) stat[0][0][mine] = mr, stat[1][0][mine] = l;
            lds_barrier();
            for (int x = 0; x < G; ++x) mr = fmaxf(mr, stat[0][0][mine - grp + x]);
            o = f4_t{0.0f, 0.0f, 0.0f, 0.0f}, l = 0.0f;
            for (int x = 0; x < G; ++x) {
              const float top = stat[0][0][mine - grp + x], keep = share(top, mr);
              l += stat[1][0][mine - grp + x] * keep;
              const f4_t v = red[(mine - grp + x) * QUADS + u];
#pragma unroll
              for (int i = 0; i < 4; ++i) o[i] += v[i] * keep;
            }
          }
          if (grp == 0 && row0 + mine / G < rows_all) write(b, row, o, l);
        }
      }
    }
    if (at < upto) lds_barrier();  // the sums have been read
  }
}

}  // namespace
}  // namespace nibble
