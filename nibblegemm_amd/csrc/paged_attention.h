// What the kernels of the attention over a paged cache have in common.
#pragma once

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "nibble_common.h"
#include "nibble_float8.h"
#include "nibble_split.h"

namespace nibble {
namespace {

constexpr int kPagedThreads = 256;
constexpr int kPagedKeys = 64;  // keys of a tile
// What the sums of a share cost that are written and joined, in tiles: of a call, and of
// its query rows.  (2 x 12 tokens of 32 + 2 x 4 heads over 20000 rows of 8 bits: 37 us, 35
// if it costs nothing, 54 if four times that; 4 x 60 of 8 + 2 x 8 over 2000: 20, 25, 27.)
constexpr float kPagedShareCost = 0.08f, kPagedRowCost = 4.8e-4f;
// Probabilities are relative to a query's reference, 2^lift below a maximum, which
// moves only when a score passes that maximum by more than the slack (in powers of two).
// fp16 ends at 2^16 and has steps of 2^-24 at least, so its reference lies as low as it
// can; bf16 has the range of fp32.
constexpr float kPagedSlack = 8.0f;
template <class E>
constexpr float kPagedLift = std::is_same_v<E, Half> ? 7.0f : 0.0f;

struct PagedSpan;

struct AttendArgs {
  const void* q;  // [B, T, n_heads, D]
  const char* k;  // element (page, h, r, d) at page kp + h kh + r kr bytes + d elements
  const char* v;
  const uint8_t* k_scales;  // [n_pages, n_kv], 8-bit pages
  const uint8_t* v_scales;
  const int32_t* table;    // [B, width]
  const int32_t* lengths;  // [B]
  const int32_t* sizes;    // [B] or null: T each
  void* out;               // [B, T, n_heads, D]
  float* partial;          // [n_kv][slots][rows][D], then [..][2] (top, sum), when shares > 0
  int* runs;               // [B][2]: a sequence's first share and their number
  int* counters;           // [B][n_kv], zero on entry and on exit: pieces that are written
  int64_t kp, kh, kr, vp, vh, vr;
  int B, T, n_heads, n_kv, qpk, width, n_pages, shift;
  int window, sinks;      // window: 2^30 where there is none
  int shares, row_tiles;  // shares: 0 where no sequence's rows are split
  int slots;              // of sums and statistics: one a share, or two (rows_kernel)
  float join_cost;        // of one share, in tiles
  bool fold;              // row tiles from both ends to the middle
  float scale;            // its magnitude times log2(e); 1 for a scale of zero
  float sign;             // its sign
  __device__ int tiles(int b) const;  // that some token of sequence b sees
};

__device__ __forceinline__ int tiles_of(int rows) { return (rows + kPagedKeys - 1) / kPagedKeys; }

// The tiles that a run of tokens sees: [0, first) and [from, upto).
struct Seen {
  int first, from, upto;
  // low, end: the first row in the window of the run's first token, and the row
  // behind the last token's own.
  __device__ __forceinline__ Seen(int low, int sinks, int end) {
    first = low > 0 ? tiles_of(min(sinks, end)) : 0;
    from = low / kPagedKeys;
    if (from <= first) first = from = 0;
    upto = tiles_of(end);
  }
};

// What of sequence b there is: earlier rows, tokens, and all rows.
struct PagedSpan {
  int len, live, total;
  __device__ __forceinline__ PagedSpan(const AttendArgs& a, int b) {
    const int room = a.width << a.shift;
    len = min(max(a.lengths[b], 0), room);
    live = a.sizes != nullptr ? min(max(a.sizes[b], 0), a.T) : a.T;
    total = live > 0 ? min(len + live, room) : 0;
  }
  // The same in scalar registers: of a sequence that is the same in every lane.
  __device__ __forceinline__ PagedSpan uniform() const {
    PagedSpan s = *this;
    s.len = __builtin_amdgcn_readfirstlane(len);
    s.live = __builtin_amdgcn_readfirstlane(live);
    s.total = __builtin_amdgcn_readfirstlane(total);
    return s;
  }
  __device__ __forceinline__ Seen seen(const AttendArgs& a) const {
    return Seen(total > 0 ? max(len - a.window + 1, 0) : 0, a.sinks, total);
  }
};
__device__ __forceinline__ int AttendArgs::tiles(int b) const {
  const Seen s = PagedSpan(*this, b).seen(*this);
  return s.first + s.upto - s.from;
}

// Unit (16 bytes) u of LDS row r, 16-bit values, lies at unit u ^ paged_swizzle(r): eight
// rows of a K read, and four rows' 32-byte pieces of a V read, cover 32 banks once.
template <int UNITS>
__device__ __forceinline__ int paged_swizzle(int r) {
  return ((r & 3) << 1 | (r >> 2 & 1) | (r & 8)) & (UNITS - 1);
}

}  // namespace
}  // namespace nibble
