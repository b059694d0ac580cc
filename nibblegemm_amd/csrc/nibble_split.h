// Attention whose cached rows are split over workgroups: how the rows of several
// sequences are shared out on the GPU, and the kernel that joins the shares.  Args
// names the call: B, T, n_heads, n_kv, qpk, shares, join_cost, partial ([n_kv]
// [shares][rows][D] sums, then [..][2] top and sum), runs ([B][2]: a sequence's
// first share and their number), out, and tiles(b), those of sequence b's rows.
#pragma once

#include "nibble_common.h"
#include "nibble_copy.h"
#include "nibble_reduce.h"

namespace nibble {
namespace {

constexpr int kSplitThreads = 256;
constexpr int kMaxSplits = 64;         // of one sequence
constexpr int kSplitWorkgroups = 512;  // two a CU
constexpr float kLog2e = 1.4426950408889634f;

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
// How the cached rows are split when there are fewer (sequence, kv head, row
// tile)s than room for workgroups.  The lengths are on the GPU, so every wave
// works it out alike: a share is at most `per` tiles of one sequence, and per is
// (to a 16th) the least for which all sequences' shares together are at most
// a.shares.  Shares are numbered in the order of the sequences, of which there
// are fewer than a.shares; one without rows keeps a share, which writes that it
// saw nothing.
template <class Args>
struct Shares {
  static constexpr int kChunks = kSplitWorkgroups / 64;  // of sequences, one a lane
  int per = 0, found = -1, first = 0, count = 0;
  // Finds the sequence that share `want` is of, and that sequence's shares.
  __device__ __forceinline__ Shares(const Args& a, int want) {
    if (a.B == 1) {
      const int all = a.tiles(0);
      per = max((all + a.shares - 1) / a.shares,
                max((all + kMaxSplits - 1) / kMaxSplits, worth(a, static_cast<float>(all))));
      count = shares_of(all);
      found = want < count ? 0 : -1;
      return;
    }
    const int lane = threadIdx.x & 63;
    int t[kChunks];  // tiles; 0 where there is no sequence
    float most_f = 0.0f, total = 0.0f;
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      t[i] = 0;
      if (64 * i < a.B) {
        t[i] = 64 * i + lane < a.B ? a.tiles(64 * i + lane) : 0;
        most_f = fmaxf(most_f, static_cast<float>(t[i]));  // (below 2^24: exact)
        total += static_cast<float>(t[i]);
      }
    }
    const int most = static_cast<int>(wave_max(most_f));
    total = wave_sum(total);
    per = static_cast<int>(ceilf(total / static_cast<float>(a.shares)));
    per = max(max(per, (most + kMaxSplits - 1) / kMaxSplits), worth(a, total));
    per = __builtin_amdgcn_readfirstlane(per);
    int high = max(per, most);  // enough: one share each
    for (int low = per; low < high;) {
      const bool close = high - low <= low / 16;
      const int mid = close ? low : low + (high - low) / 2;
      int n = 0;
#pragma unroll
      for (int i = 0; i < kChunks; ++i)
        if (64 * i < a.B) n += 64 * i + lane < a.B ? max(1, (t[i] + mid - 1) / mid) : 0;
      if (wave_sum(static_cast<float>(n)) <= static_cast<float>(a.shares)) high = mid;
      else low = close ? high : mid + 1;
    }
    per = high;
    int before = 0;
#pragma unroll
    for (int i = 0; i < kChunks; ++i)
      if (64 * i < a.B && found < 0) {
        const int n = 64 * i + lane < a.B ? shares_of(t[i]) : 0;
        int upto = n;
#pragma unroll
        for (int x = 1; x < 64; x *= 2) {
          const int y = __shfl_up(upto, x);
          if (lane >= x) upto += y;
        }
        const int start = before + upto - n;
        const uint64_t hit = __ballot(want >= start && want < start + n);
        if (hit != 0) {
          const int at = __builtin_ctzll(hit);
          found = 64 * i + at;
          first = __builtin_amdgcn_readlane(start, at);
          count = __builtin_amdgcn_readlane(n, at);
        }
        before += __builtin_amdgcn_readlane(upto, 63);
      }
  }
  // per tiles in turn, and total / per shares whose sums are written and joined:
  // the least of per + join_cost total / per.
  static __device__ __forceinline__ int worth(const Args& a, float total) {
    return max(static_cast<int>(__builtin_amdgcn_sqrtf(a.join_cost * total)), 1);
  }
  __device__ __forceinline__ int shares_of(int t) const { return max(1, (t + per - 1) / per); }
};

// Joins the shares of a row: D / 4 lanes a row, four outputs each, the rows of
// one (sequence, kv head) in a workgroup.  The lanes read the shares' statistics
// together; the sums are then loaded eight shares at a time, those of shares
// that saw nothing not at all (a share of no weight counts: an infinity or a NaN in
// its sums must not be lost).  Memory and latency bound it: 64 rows of 8 shares
// and 8 kv heads 3 us, 256 rows of 32 shares 8 us, 34 MB (loads begun before
// the statistics are there gained 0.6 us on the first, lost 2 on ragged trees).
template <class E, int D, class Args>
__global__ __launch_bounds__(kSplitThreads) void join_kernel(Args a) {
  using T = typename E::type;
  constexpr int LANES = D / 4, PER = kMaxSplits / LANES;  // splits a lane looks at
  const int rows_all = a.T * a.qpk;
  const int parts = (rows_all + kSplitThreads / LANES - 1) / (kSplitThreads / LANES);
  const int unit = blockIdx.x / parts;
  const int b = unit / a.n_kv, h = unit - b * a.n_kv;
  const int at = (blockIdx.x - unit * parts) * (kSplitThreads / LANES) + threadIdx.x / LANES;
  const bool in = at < rows_all;
  const int r = in ? at : 0;  // (lanes without a row shuffle along)
  const int lane = threadIdx.x % LANES, d = lane * 4;
  const int first = a.runs[2 * b], count = a.runs[2 * b + 1];
  const float* const st = a.partial + static_cast<int64_t>(a.n_kv) * a.shares * rows_all * D;
  const int64_t rec0 = (static_cast<int64_t>(h) * a.shares + first) * rows_all + r;
  float tops[PER], w[PER], m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    const int s = u * LANES + lane;
    const float* p = st + (rec0 + static_cast<int64_t>(s) * rows_all) * 2;
    tops[u] = s < count ? p[0] : -INFINITY;
    w[u] = s < count ? p[1] : 0.0f;
    m = fmaxf(m, tops[u]);
  }
#pragma unroll
  for (int x = LANES / 2; x > 0; x /= 2) m = fmaxf(m, __shfl_xor(m, x, LANES));
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    const float keep = tops[u] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(tops[u] - m);
    l += w[u] * keep;
    w[u] = tops[u] == -INFINITY ? -1.0f : keep;  // (negative: no sums)
  }
#pragma unroll
  for (int x = LANES / 2; x > 0; x /= 2) l += __shfl_xor(l, x, LANES);
  f4_t o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int u = 0; u < PER; ++u)
    for (int s0 = 0; s0 < LANES && u * LANES + s0 < count; s0 += 8) {
      f4_t v[8];
      float k[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        k[e] = __shfl(w[u], s0 + e, LANES);
        v[e] = f4_t{0.0f, 0.0f, 0.0f, 0.0f};
        if (!(k[e] < 0.0f))
          v[e] = *reinterpret_cast<const f4_t*>(
              a.partial + (rec0 + static_cast<int64_t>(u * LANES + s0 + e) * rows_all) * D + d);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] += v[e][i] * k[e];
    }
  if (!in) return;
  const int i = r / a.qpk;
  typedef T vec4 __attribute__((ext_vector_type(4)));
  vec4 y;
#pragma unroll
  for (int x = 0; x < 4; ++x) y[x] = static_cast<T>(l == 0.0f ? 0.0f : o[x] / l);
  *reinterpret_cast<vec4*>(static_cast<T*>(a.out) +
                           ((static_cast<int64_t>(b) * a.T + i) * a.n_heads + h * a.qpk +
                            (r - i * a.qpk)) * D + d) = y;
}

}  // namespace
}  // namespace nibble
