// Norms of the query and key heads, their rotary embedding and the way of the
// keys and values into the cache, in one pass over the q|k|v projection's
// output.
//
// A head x of a token at position p becomes, in fp32 and rounded once,
//   n = x w / sqrt(mean(x^2) + eps)        (where the heads have norms)
//   n[i] cos(p, i) - n[i + D/2] sin(p, i), n[i + D/2] cos(p, i) + n[i] sin(p, i)
// (where there are rotary tables); values go through as they are.
//
// What bounds it: memory, every value read once and written once: 8000 tokens of
// 32 + 2 x 8 heads of 128 in 31.5 us, 6.2 TB/s; one token is a launch (2 us).  A
// head is held by D / 16 lanes: lane j has elements 8j .. 8j + 7 of each half, so
// an element and its rotary partner meet in one lane, and the sum of squares in
// three (two) DPP steps.
#include <cmath>

#include "nibble_common.h"
#include "nibble_copy.h"
#include "nibble_reduce.h"

namespace nibble {
namespace {

constexpr int kQkThreads = 256;

struct QkArgs {
  const void* qkv;         // [tokens, (n_heads + 2 n_kv) D]
  void* k_cache;           // element (b, h, s, d) at b kb + h kh + s ks + d
  void* v_cache;
  const int32_t* positions;  // [tokens]
  const int32_t* slots;      // [tokens]
  const void* q_weight;    // [D] or null
  const void* k_weight;    // [D] or null
  const float* cos;        // [table, D / 2] or null
  const float* sin;
  void* q_out;             // [tokens, n_heads D]
  int64_t vectors;         // tokens (n_heads + 2 n_kv)
  int64_t kb, kh, ks, vb, vh, vs;
  int T, n_heads, n_kv, seq, table;
  float eps;
};

template <class E, int D>
__global__ __launch_bounds__(kQkThreads) void qk_norm_kernel(QkArgs a) {
  using T = typename E::type;
  using vec8 = typename E::vec8;
  constexpr int LANES = D / 16, HALF = D / 2;
  const int j = threadIdx.x % LANES;
  const int64_t v = static_cast<int64_t>(blockIdx.x) * (kQkThreads / LANES) + threadIdx.x / LANES;
  // (vectors behind the last take part in the reductions, as copies of it)
  const int64_t vec = v < a.vectors ? v : a.vectors - 1;
  const int heads = a.n_heads + 2 * a.n_kv;
  const int64_t token = vec / heads;
  const int head = static_cast<int>(vec - token * heads);
  const int slot = a.slots[token], pos = a.positions[token];
  const T* x = static_cast<const T*>(a.qkv) + vec * D + 8 * j;
  const vec8 lo = *reinterpret_cast<const vec8*>(x), hi = *reinterpret_cast<const vec8*>(x + HALF);
  // A token whose cache row or angle does not exist is padding.
  const bool rope = a.cos != nullptr;
  const bool live = slot >= 0 && slot < a.seq && (!rope || (pos >= 0 && pos < a.table));
  const bool query = head < a.n_heads, value = head >= a.n_heads + a.n_kv;
  vec8 out_lo = lo, out_hi = hi;
  if (!value) {
    float f[8], g[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = static_cast<float>(lo[i]), g[i] = static_cast<float>(hi[i]);
    const T* w = static_cast<const T*>(query ? a.q_weight : a.k_weight);
    if (w != nullptr) {
      float ss = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = __builtin_fmaf(f[i], f[i], ss);
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = __builtin_fmaf(g[i], g[i], ss);
      ss += dpp<kDppXor1>(ss);
      ss += dpp<kDppXor2>(ss);
      if (LANES == 8) ss += dpp<kDppHalfMirror>(ss);
      const float r = rms_scale(ss, D, a.eps);
      const vec8 wl = *reinterpret_cast<const vec8*>(w + 8 * j);
      const vec8 wh = *reinterpret_cast<const vec8*>(w + HALF + 8 * j);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        f[i] *= r * static_cast<float>(wl[i]);
        g[i] *= r * static_cast<float>(wh[i]);
      }
    }
    if (rope) {
      const int64_t at = static_cast<int64_t>(live ? pos : 0) * HALF + 8 * j;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float c = a.cos[at + i], s = a.sin[at + i];
        const float n = f[i] * c - g[i] * s;
        g[i] = g[i] * c + f[i] * s;
        f[i] = n;
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      out_lo[i] = static_cast<T>(query && !live ? 0.0f : f[i]);
      out_hi[i] = static_cast<T>(query && !live ? 0.0f : g[i]);
    }
  }
  if (v >= a.vectors || !(query || live)) return;
  T* o;
  if (query) {
    o = static_cast<T*>(a.q_out) + (token * a.n_heads + head) * D;
  } else {
    const int64_t b = token / a.T;
    const int h = head - a.n_heads - (value ? a.n_kv : 0);
    o = value ? static_cast<T*>(a.v_cache) + b * a.vb + h * a.vh + slot * a.vs
              : static_cast<T*>(a.k_cache) + b * a.kb + h * a.kh + slot * a.ks;
  }
  *reinterpret_cast<vec8*>(o + 8 * j) = out_lo;
  *reinterpret_cast<vec8*>(o + HALF + 8 * j) = out_hi;
}

template <class E>
hipError_t launch_qk(const QkArgs& a, int D, hipStream_t stream) {
  const int per = kQkThreads / (D / 16);
  const dim3 grid(static_cast<unsigned>(ceil_div(a.vectors, per)));
  if (D == 64) qk_norm_kernel<E, 64><<<grid, kQkThreads, 0, stream>>>(a);
  else qk_norm_kernel<E, 128><<<grid, kQkThreads, 0, stream>>>(a);
  return hipGetLastError();
}

}  // namespace
}  // namespace nibble

using namespace nibble;

extern "C" int nibble_qk_norm_rope(const void* QKV, int64_t dtype, int64_t batch, int64_t tokens,
                                   int64_t n_heads, int64_t n_kv_heads, int64_t head_dim,
                                   void* K_cache, int64_t k_batch_stride, int64_t k_head_stride,
                                   int64_t k_row_stride, void* V_cache, int64_t v_batch_stride,
                                   int64_t v_head_stride, int64_t v_row_stride, int64_t max_seq,
                                   const void* positions, const void* slots, const void* q_weight,
                                   const void* k_weight, float eps, const void* rope_cos,
                                   const void* rope_sin, int64_t rope_rows, void* Q_out,
                                   void* stream_) {
  NIBBLE_CHECK(dtype == 0 || dtype == 1, "dtype must be 0 (fp16) or 1 (bf16), got %lld",
               (long long)dtype);
  NIBBLE_CHECK(head_dim == 64 || head_dim == 128, "head_dim must be 64 or 128, got %lld",
               (long long)head_dim);
  NIBBLE_CHECK(n_kv_heads >= 1 && n_heads >= 1 && n_heads <= 65535 && n_kv_heads <= 65535,
               "n_heads and n_kv_heads must be in [1, 65535], got %lld and %lld",
               (long long)n_heads, (long long)n_kv_heads);
  NIBBLE_CHECK(batch >= 0 && tokens >= 0 && batch <= 0x7fffffff && tokens <= 0x7fffffff,
               "batch and tokens must be in [0, 2^31)");
  NIBBLE_CHECK(max_seq >= 0 && max_seq <= 0x7fffffff, "max_seq must be in [0, 2^31), got %lld",
               (long long)max_seq);
  NIBBLE_CHECK((rope_cos == nullptr) == (rope_sin == nullptr),
               "rope_cos and rope_sin must both be given or both be null");
  NIBBLE_CHECK(rope_cos == nullptr || (rope_rows >= 1 && rope_rows <= 0x7fffffff),
               "rope tables must have between 1 and 2^31 - 1 rows, got %lld", (long long)rope_rows);
  NIBBLE_CHECK(std::isfinite(eps) && eps >= 0.0f, "eps must be finite and >= 0");
  if (batch == 0 || tokens == 0) return ok();
  const int64_t vectors_per = n_heads + 2 * n_kv_heads;
  // (a launch ends at 2^32 threads, head_dim / 16 a vector)
  NIBBLE_CHECK(batch * tokens <= ((int64_t(1) << 32) - kQkThreads) / (head_dim / 16) / vectors_per,
               "too many tokens: %lld x %lld", (long long)batch, (long long)tokens);
  for (int64_t s : {k_batch_stride, k_head_stride, k_row_stride, v_batch_stride, v_head_stride,
                    v_row_stride})
    NIBBLE_CHECK(s >= 0 && s % 8 == 0, "cache strides must be multiples of 8 elements, got %lld",
                 (long long)s);
  NIBBLE_CHECK(QKV != nullptr && K_cache != nullptr && V_cache != nullptr && Q_out != nullptr &&
                   positions != nullptr && slots != nullptr,
               "null pointer");
  NIBBLE_CHECK(aligned(QKV, 16) && aligned(K_cache, 16) && aligned(V_cache, 16) &&
                   aligned(Q_out, 16) && aligned(q_weight, 16) && aligned(k_weight, 16),
               "qkv, caches, weights and output must be 16-byte aligned");
  NIBBLE_CHECK(aligned(positions, 4) && aligned(slots, 4) && aligned(rope_cos, 4) &&
                   aligned(rope_sin, 4),
               "positions, slots and rope tables must be 4-byte aligned");
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  DeviceGuard guard;
  int dev = 0;
  NIBBLE_HIP(guard.enter(stream, &dev));
  QkArgs a;
  a.qkv = QKV;
  a.k_cache = K_cache;
  a.v_cache = V_cache;
  a.positions = static_cast<const int32_t*>(positions);
  a.slots = static_cast<const int32_t*>(slots);
  a.q_weight = q_weight;
  a.k_weight = k_weight;
  a.cos = static_cast<const float*>(rope_cos);
  a.sin = static_cast<const float*>(rope_sin);
  a.q_out = Q_out;
  a.vectors = batch * tokens * vectors_per;
  a.kb = k_batch_stride, a.kh = k_head_stride, a.ks = k_row_stride;
  a.vb = v_batch_stride, a.vh = v_head_stride, a.vs = v_row_stride;
  a.T = static_cast<int>(tokens);
  a.n_heads = static_cast<int>(n_heads);
  a.n_kv = static_cast<int>(n_kv_heads);
  a.seq = static_cast<int>(max_seq);
  a.table = rope_cos != nullptr ? static_cast<int>(rope_rows) : 0;
  a.eps = eps;
  const hipError_t e = dtype == 0 ? launch_qk<Half>(a, static_cast<int>(head_dim), stream)
                                  : launch_qk<Bfloat>(a, static_cast<int>(head_dim), stream);
  if (e != hipSuccess) return hip_fail(e, "qk_norm kernel launch");
  return ok();
}
