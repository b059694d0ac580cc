// Microscaled 4-bit floats (OCP MXFP4): quantisation, its inverse, and the
// product of two such matrices on the scaled MFMA of gfx950.
//
// A matrix [rows, K] (K a multiple of 32) is held as
//   codes   uint8 [rows, K / 2]            two a byte along K, the even k low;
//   scales  uint8 [ceil(K / 128), rows, 4]  one power of two (biased by 127) per
//                                          block of 32 k, four blocks a word;
//                                          zero behind the last block.
// A code is sign | exponent (2) | mantissa (1): 0, 0.5, 1, 1.5, 2, 3, 4, 6.
// The words of one k group lie side by side over the rows because that is how
// the matrix cores take them: a lane holds one block (16 bytes of codes) of one
// row, and the word of scales its four blocks need arrives with one load of
// adjacent lanes' words.
#include <algorithm>

#include "nibble_common.h"
#include "nibble_decode.h"
#include "nibble_reduce.h"

namespace nibble {
namespace {

constexpr int kMxF16 = 0, kMxBF16 = 1, kMxF32 = 2;
constexpr int kMxBlock = 32;   // k of one scale
constexpr int kMxGroup = 128;  // k of one word of scales
// Workgroups along a grid's first dimension, where there may be many: one dimension
// ends at 2^32 threads.
constexpr int64_t kMxGrid = 1 << 20;

typedef int i8_t __attribute__((ext_vector_type(8)));
typedef unsigned short us8_t __attribute__((ext_vector_type(8)));

template <int DT>
struct MxElem {
  using type = unsigned short;
  static __device__ __forceinline__ float get(unsigned short v) {
    return DT == kMxF16 ? static_cast<float>(__builtin_bit_cast(_Float16, v))
                        : __builtin_bit_cast(float, static_cast<uint32_t>(v) << 16);
  }
  static __device__ __forceinline__ void load8(const type* p, float (&f)[8]) {
    const us8_t v = *reinterpret_cast<const us8_t*>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = get(v[i]);
  }
};
template <>
struct MxElem<kMxF32> {
  using type = float;
  static __device__ __forceinline__ float get(float v) { return v; }
  static __device__ __forceinline__ void load8(const type* p, float (&f)[8]) {
    const f4_t a = *reinterpret_cast<const f4_t*>(p);
    const f4_t b = *(reinterpret_cast<const f4_t*>(p) + 1);
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = a[i], f[4 + i] = b[i];
  }
};

// Biased exponent of a block whose largest magnitude has these bits:
// floor(log2) - 2 (the largest code, 6, has exponent 2), never below -127.  A
// block with an infinity or a NaN gets 255 and reads as NaN.
__device__ __forceinline__ uint32_t mx_scale(uint32_t top) {
  const uint32_t e = top >> 23;
  return e == 255u ? 255u : e > 2u ? e - 2u : 0u;
}
// The power of two as a float (2^-127 is subnormal).
__device__ __forceinline__ float mx_power(uint32_t e) {
  return __builtin_bit_cast(float, e == 0u ? 0x00400000u : e << 23);
}
__device__ __forceinline__ uint32_t mag_bits(float f) {
  return __builtin_bit_cast(uint32_t, f) & 0x7fffffffu;
}

// Codes of eight values over their block's power of two, rounded half to even
// and capped at 6 by the conversion.  In a block that reads as NaN they are 0.
__device__ __forceinline__ uint32_t mx_codes8(const float (&f)[8], uint32_t e) {
  const float p = mx_power(e);
  uint32_t c = 0;
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f[0], f[1], p, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f[2], f[3], p, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f[4], f[5], p, 2);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f[6], f[7], p, 3);
  return e == 255u ? 0u : c;
}

template <int CTRL>
__device__ __forceinline__ uint32_t dpp_u32(uint32_t v) {
  return static_cast<uint32_t>(
      __builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, 0xF, 0xF, false));
}

// Rows whose k are adjacent in memory.  A workgroup takes 8 rows of 512 k;
// wave w the k group w of them, 16 lanes a row: lane j holds k 8j .. 8j + 7,
// four lanes a block.  The largest magnitude meets in the four lanes (DPP),
// the four blocks' exponents in the row's first lane, which writes the word.
// Memory bounds it: 28672 x 4096 in 53 us from fp16, 5.6 TB/s, and 91 from fp32
// (54 and 95 with 16 rows, 57 and 90 with 4; 60 and 97 with 32 rows and loads
// that pass by the caches, whose values the caches may hold).
constexpr int kMxRows = 8;
constexpr int kMxPasses = kMxRows / 4;

template <int DT, bool VEC>
__global__ __launch_bounds__(256) void mx_quantize_kernel(const typename MxElem<DT>::type* X,
                                                          int64_t ld, uint32_t* codes,
                                                          uint32_t* scales, int64_t rows, int K,
                                                          int col_tiles) {
  using E = MxElem<DT>;
  const int lane = threadIdx.x & 63;
  const uint32_t block = blockIdx.y * static_cast<uint32_t>(kMxGrid) + blockIdx.x;
  const int64_t tile = block / col_tiles;
  const int group = static_cast<int>(block % col_tiles) * 4 + (threadIdx.x >> 6);
  const int j = lane & 15;
  const int k = group * kMxGroup + 8 * j;
  const int64_t row0 = tile * kMxRows + (lane >> 4);
  if (group * kMxGroup >= K) return;
  float f[kMxPasses][8];
#pragma unroll
  for (int p = 0; p < kMxPasses; ++p) {
    const int64_t row = row0 + 4 * p;
    const bool in = row < rows && k < K;
    const typename E::type* x = X + row * ld + k;
    if (VEC) {
      if (in) {
        E::load8(x, f[p]);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[p][i] = 0.0f;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) f[p][i] = in ? E::get(x[i]) : 0.0f;
    }
  }
#pragma unroll
  for (int p = 0; p < kMxPasses; ++p) {
    const int64_t row = row0 + 4 * p;
    uint32_t top = mag_bits(f[p][0]);
#pragma unroll
    for (int i = 1; i < 8; ++i) top = max(top, mag_bits(f[p][i]));
    top = max(top, dpp_u32<kDppXor1>(top));
    top = max(top, dpp_u32<kDppXor2>(top));
    const uint32_t e = mx_scale(top);
    const uint32_t c = mx_codes8(f[p], e);
    // lanes 0, 4, 8, 12 of the row hold the four exponents; a block behind K
    // has exponent 0 (its values were taken as zeros)
    uint32_t word = e << ((j >> 2) * 8);
    word |= dpp_u32<kDppHalfMirror>(word);
    word |= dpp_u32<kDppMirror>(word);
    if (row < rows) {
      if (k < K) codes[(row * K + k) >> 3] = c;
      if (j == 0) scales[static_cast<int64_t>(group) * rows + row] = word;
    }
  }
}

// Rows that are adjacent in memory (a transposed view: element (row, k) at
// k ld + row).  A workgroup takes 128 rows of one k group; wave w its block w,
// lane l rows 2l and 2l + 1, whose 32 values it holds; the codes go through
// LDS so that a row's 64 bytes are written together.  Memory bounds it: 14336 rows
// of 4096 k from fp32 in 42 us, 6.4 TB/s, from fp16 24 us; 4102 rows of 5536 k
// from fp32 in 21 (23 with loads that pass by the caches).
constexpr int kMxCols = 128;

template <int DT, bool VEC>
__global__ __launch_bounds__(256) void mx_quantize_t_kernel(const typename MxElem<DT>::type* X,
                                                            int64_t ld, uint8_t* codes,
                                                            uint32_t* scales, int64_t rows, int K,
                                                            int groups) {
  using E = MxElem<DT>;
  typedef typename E::type pair_t __attribute__((ext_vector_type(2)));
  __shared__ u4_t buf[kMxCols][4];
  __shared__ uint8_t sbuf[kMxCols][4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int group = static_cast<int>(blockIdx.x % groups);
  const int64_t row0 = static_cast<int64_t>(blockIdx.x / groups) * kMxCols;
  const int64_t row = row0 + 2 * lane;
  const int k0 = group * kMxGroup + wave * kMxBlock;
  uint32_t e[2] = {0u, 0u};
  u4_t word[2] = {};
  if (k0 < K) {
    float f[2][kMxBlock];
    uint32_t top[2] = {0u, 0u};
#pragma unroll
    for (int i = 0; i < kMxBlock; ++i) {
      const typename E::type* x = X + (k0 + i) * ld + row;
      if (VEC) {
        const pair_t v = row < rows ? *reinterpret_cast<const pair_t*>(x)
                                    : pair_t{};
        f[0][i] = E::get(v[0]);
        f[1][i] = E::get(v[1]);
      } else {
        f[0][i] = row < rows ? E::get(x[0]) : 0.0f;
        f[1][i] = row + 1 < rows ? E::get(x[1]) : 0.0f;
      }
#pragma unroll
      for (int r = 0; r < 2; ++r) top[r] = max(top[r], mag_bits(f[r][i]));
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      e[r] = mx_scale(top[r]);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float g[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) g[i] = f[r][8 * q + i];
        word[r][q] = mx_codes8(g, e[r]);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    buf[2 * lane + r][wave] = word[r];
    sbuf[2 * lane + r][wave] = static_cast<uint8_t>(e[r]);
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int c = tid + 256 * u, r = c >> 2, b = c & 3;
    const int k = group * kMxGroup + b * kMxBlock;
    if (row0 + r < rows && k < K)
      *reinterpret_cast<u4_t*>(codes + ((row0 + r) * K + k) / 2) = buf[r][b];
  }
  if (tid < kMxCols && row0 + tid < rows)
    scales[static_cast<int64_t>(group) * rows + row0 + tid] =
        *reinterpret_cast<const uint32_t*>(sbuf[tid]);
}

template <int DT>
__device__ __forceinline__ typename MxElem<DT>::type mx_out(float v) {
  if constexpr (DT == kMxF32) {
    return v;
  } else if constexpr (DT == kMxF16) {
    return __builtin_bit_cast(unsigned short, static_cast<_Float16>(v));
  } else {
    return __builtin_bit_cast(unsigned short, static_cast<__bf16>(v));
  }
}

// Two codes' values (byte B of a word) times the block's power of two: exact in
// 32 bits (down to 2^-128; 2^126 times 4 or 6 is infinite, as it should be).
typedef float f2_t __attribute__((ext_vector_type(2)));
template <int B>
__device__ __forceinline__ f2_t mx_values2(uint32_t codes, uint32_t e) {
  const f2_t v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, mx_power(e), B);
  return e == 255u ? f2_t{__builtin_nanf(""), __builtin_nanf("")} : v;
}

// A thread expands what 16 bytes of the output hold: eight codes, or four where
// it has 32 bits.  Memory bounds it; what counts is that a wave's stores cover
// 1 KiB without a gap and pass by the caches (28672 x 4096 in bf16: 43 us against
// 60 with plain stores; in fp32 72 against 119, and 132 with 32 bytes a thread).
template <int DT>
__global__ __launch_bounds__(256) void mx_dequantize_kernel(const uint8_t* codes,
                                                            const uint8_t* scales, int64_t rows,
                                                            int K, typename MxElem<DT>::type* out) {
  typedef typename MxElem<DT>::type vec __attribute__((ext_vector_type(DT == kMxF32 ? 4 : 8)));
  constexpr int PER = DT == kMxF32 ? 4 : 8;  // values of a thread
  const uint32_t per_row = K / PER;
  const int64_t first = (static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x) * 256;
  const int64_t row0 = first / per_row;  // (of the workgroup; in 32 bits from there)
  const uint32_t at = static_cast<uint32_t>(first - row0 * per_row) + threadIdx.x;
  const int64_t row = row0 + at / per_row, i = first + threadIdx.x;
  const int k = static_cast<int>(at % per_row) * PER;
  if (row >= rows) return;
  uint32_t c;
  if constexpr (DT == kMxF32) c = reinterpret_cast<const uint16_t*>(codes)[i];
  else c = reinterpret_cast<const uint32_t*>(codes)[i];
  const uint32_t e = scales[((k / kMxGroup) * rows + row) * 4 + k / kMxBlock % 4];
  f2_t f[4];
  f[0] = mx_values2<0>(c, e), f[1] = mx_values2<1>(c, e);
  if constexpr (DT != kMxF32) f[2] = mx_values2<2>(c, e), f[3] = mx_values2<3>(c, e);
  vec v;
#pragma unroll
  for (int u = 0; u < PER; ++u) v[u] = mx_out<DT>(f[u / 2][u % 2]);
  __builtin_nontemporal_store(v, reinterpret_cast<vec*>(out) + i);
}

struct MxArgs {
  const uint8_t* xc;  // x codes [M, K / 2]
  const uint8_t* xs;  // x scales [groups, M, 4]
  const uint8_t* wc;  // w codes [N, K / 2]
  const uint8_t* ws;  // w scales [groups, N, 4]
  void* y;            // [M, N]
  int M, N, K;
  const void* x;      // dense x instead of codes: [M, K], rows ld elements apart
  int ld;
};

constexpr int kMxChunk = 512;  // k of one step of a wave: a lane's four blocks
constexpr int kMxWaves = 8;

// One 16-row operand of a step as the matrix cores take it: lane l holds row
// l % 16 and, of the step's 16 blocks, the four from 4 (l / 16) on: 64 adjacent
// bytes and one word of scales.  (The sum over k may be taken in any order, so
// the step's j-th product runs over the j-th block of every lane.)
struct MxFrag {
  u4_t c[4];
  uint32_t s;
};

// Rows r0 .. r0 + 15 of a matrix as buffer resources; a row or block that is
// not there reads as zeros (an offset no resource reaches).
struct MxRows {
  __amdgpu_buffer_rsrc_t codes, scales;
  uint32_t code0, scale0;  // this lane's offsets at k = 0
  uint32_t pitch;          // bytes between two words of scales of one row
  int blocks;              // blocks from this lane's first one on
  __device__ __forceinline__ MxRows(const uint8_t* c, const uint8_t* s, int rows, int K, int r0,
                                    int lane) {
    const int r = lane & 15, g = lane >> 4;
    const int groups = (K + kMxGroup - 1) / kMxGroup;
    const int here = min(16, rows - r0);
    codes = make_rsrc(c + static_cast<int64_t>(r0) * (K / 2),
                      static_cast<uint32_t>(max(here, 0)) * static_cast<uint32_t>(K / 2));
    scales = make_rsrc(s, static_cast<uint32_t>(groups) * static_cast<uint32_t>(rows) * 4u);
    const bool in = r < here;
    code0 = in ? static_cast<uint32_t>(r) * (K / 2) + g * 64u : kOutOfRange;
    scale0 = in ? (static_cast<uint32_t>(g) * rows + r0 + r) * 4u : kOutOfRange;
    pitch = static_cast<uint32_t>(rows) * 4u;
    blocks = K / kMxBlock - 4 * g;
  }
  __device__ __forceinline__ void load(MxFrag& f, int chunk) const {
    const int first = chunk * 16;  // of the lane's blocks, counted from its own first
#pragma unroll
    for (int j = 0; j < 4; ++j)
      f.c[j] = __builtin_bit_cast(
          u4_t, __builtin_amdgcn_raw_buffer_load_b128(
                    codes, first + j < blocks ? code0 + chunk * 256u + j * 16u : kOutOfRange, 0, 0));
    f.s = __builtin_amdgcn_raw_buffer_load_b32(
        scales, first < blocks ? scale0 + chunk * 4u * pitch : kOutOfRange, 0, 0);
  }
};

template <int J>
__device__ __forceinline__ f4_t mx_mfma16(const MxFrag& a, const MxFrag& b, f4_t c) {
  const u4_t x = a.c[J], y = b.c[J];
  const i8_t va = {(int)x[0], (int)x[1], (int)x[2], (int)x[3], 0, 0, 0, 0};
  const i8_t vb = {(int)y[0], (int)y[1], (int)y[2], (int)y[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(va, vb, c, 4, 4, J, (int)a.s, J, (int)b.s);
}

// A lane's operand from dense values: the four blocks that MxRows::load would
// read, quantised here (lane c of a 16-lane row holds row c of x).  Rows and
// blocks that are not there read as zeros.
template <int XD>
struct MxDense {
  static constexpr uint32_t kSize = XD == kMxF32 ? 4 : 2;
  __amdgpu_buffer_rsrc_t x;
  uint32_t off0;
  int blocks;
  __device__ __forceinline__ MxDense(const MxArgs& a, int lane) {
    const int r = lane & 15, g = lane >> 4;
    x = make_rsrc(a.x, (static_cast<uint32_t>(a.M - 1) * a.ld + a.K) * kSize);
    off0 = r < a.M ? (static_cast<uint32_t>(r) * a.ld + g * 128u) * kSize : kOutOfRange;
    blocks = a.K / kMxBlock - 4 * g;
  }
  __device__ __forceinline__ void load(MxFrag& f, int chunk) const {
    constexpr int PIECES = 2 * kSize;  // of 16 bytes, a block
    f.s = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t off = chunk * 16 + j < blocks
                               ? off0 + (chunk * 512u + j * kMxBlock) * kSize : kOutOfRange;
      u4_t v[PIECES];
#pragma unroll
      for (int i = 0; i < PIECES; ++i)
        v[i] = __builtin_bit_cast(u4_t, __builtin_amdgcn_raw_buffer_load_b128(x, off + 16u * i, 0, 0));
      uint32_t top = 0;
      float b[4][8];
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        float& t = b[i / 8][i % 8];
        if constexpr (XD == kMxF32) {
          const uint32_t w = v[i / 4][i % 4];
          t = __builtin_bit_cast(float, w);
        } else {
          const uint32_t w = v[i / 8][i % 8 / 2];
          t = MxElem<XD>::get(static_cast<unsigned short>(i % 2 ? w >> 16 : w));
        }
        top = max(top, mag_bits(t));
      }
      const uint32_t e = mx_scale(top);
      f.s |= e << (8 * j);
#pragma unroll
      for (int i = 0; i < 4; ++i) f.c[j][i] = mx_codes8(b[i], e);
    }
  }
};

// y = x w^T for few rows of x.  A workgroup takes 16 rows of w and 16 MT rows
// of x; its eight waves share out the k in steps of 512 and meet in LDS, in
// wave order.  Codes come straight from memory into the matrix cores' operands;
// a dense x (XD, at most 16 rows) is quantised by every workgroup on the way,
// which costs less than a launch before this one where w is small.  Latency
// bounds it: a wave's loads for a step of 512 k, the products, the meeting in LDS
// (1 x 1024 x 4096 4.0 us of kernel for 2.2 MB).
constexpr int kMxCodes = -1;
template <int MT, int XD, int DT>
__global__ __launch_bounds__(64 * kMxWaves) void mx_rows_kernel(MxArgs a) {
  static_assert(XD == kMxCodes || MT == 1, "a dense x has at most 16 rows");
  __shared__ float part[kMxWaves][MT][16][17];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 16 * MT;
  const int chunks = (a.K + kMxChunk - 1) / kMxChunk;
  const MxRows w(a.wc, a.ws, a.N, a.K, n0, lane);
  f4_t acc[MT] = {};
  for (int c = wave; c < chunks; c += kMxWaves) {
    MxFrag fw;
    w.load(fw, c);
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      MxFrag fx;
      if constexpr (XD == kMxCodes) MxRows(a.xc, a.xs, a.M, a.K, m0 + 16 * t, lane).load(fx, c);
      else MxDense<XD>(a, lane).load(fx, c);
      acc[t] = mx_mfma16<0>(fw, fx, acc[t]);
      acc[t] = mx_mfma16<1>(fw, fx, acc[t]);
      acc[t] = mx_mfma16<2>(fw, fx, acc[t]);
      acc[t] = mx_mfma16<3>(fw, fx, acc[t]);
    }
  }
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) part[wave][t][lane & 15][4 * (lane >> 4) + i] = acc[t][i];
  __syncthreads();
  auto* y = static_cast<typename MxElem<DT>::type*>(a.y);
  for (int e = threadIdx.x; e < MT * 256; e += 64 * kMxWaves) {
    const int t = e >> 8, m = e >> 4 & 15, n = e & 15;
    float s = part[0][t][m][n];
#pragma unroll
    for (int v = 1; v < kMxWaves; ++v) s += part[v][t][m][n];
    const int gm = m0 + 16 * t + m, gn = n0 + n;
    if (gm < a.M && gn < a.N) y[static_cast<int64_t>(gm) * a.N + gn] = mx_out<DT>(s);
  }
}

}  // namespace
}  // namespace nibble

#include "mx_tile.h"

namespace nibble {
namespace {

template <int XT, int WT, int WM, int WN, int RING, int OCC, int DT>
hipError_t launch_mx_tile(const MxArgs& a, hipStream_t stream) {
  using S = MxTile<XT, WT, WM, WN, RING>;
  const int tm = static_cast<int>(ceil_div(a.M, S::BM)), tn = static_cast<int>(ceil_div(a.N, S::BN));
  mx_tile_kernel<S, XT, WT, WM, WN, DT, OCC><<<dim3(tm * tn), S::THREADS, 0, stream>>>(a, tm, tn);
  return hipGetLastError();
}

// Which kernel a product runs on.  Few rows take the rows kernel while its
// workgroups (16 rows of w by up to 64 of x) are few a CU: 18 x 4136 x 5536 6.6 us
// against 10.6 with the tile kernel, 26 x 9437 x 5536 13.1 against 11.5; 65 x 2770
// x 5536 10.7 against 11.2, 128 x 4096 x 4096 12.6 against 8.6.  The tile kernel's
// forms are priced (ns): `fixed` for filling and writing a CU's tiles, and a step
// of 128 k, `alone` where a CU has one tile and `each` where it has more, the
// larger of the two.  The prices are a fit to every form's time at 94 sizes (M 17
// .. 4096, N 733 .. 28672, K 512 .. 14336), over which the form they name takes
// 1.01 of the best one's time in the mean and 1.13 at most.  us, 64 x 64 / 64 x
// 256 / 128 x 128 / 128 x 192 / 192 x 256 / 256 x 256: 512 x 4096 x 4096 10.6 /
// 13.9 / 14.3 / 16.2 / 22.1 / 27.4; 1000 x 4102 x 4096 22.7 / 25 / 22.2 / 19.4 / 25.2
// / 31.0; 2048 x 4096 x 4096 34.9 / 30 / 22.8 / 33.2 / 25.1 / 30.8; 1500 x 6144 x
// 4096 36.8 / 38 / 33.0 / 32.8 / 25.8 / 30.1; 2048 x 14336 x 4096 120 / 101 / 77 /
// 83 / 76 / 69.
enum MxForm { kMxRowsForm, kMx64x64, kMx64x256, kMx128x128, kMx128x192, kMx192x256, kMx256x256 };
MxForm mx_form(int64_t M, int64_t N, int64_t K) {
  const int64_t most = M <= 16 ? 768 : M <= 32 ? 384 : 256;
  if (ceil_div(N, 16) * ceil_div(M, 64) <= most) return kMxRowsForm;
  struct Price {
    MxForm form;
    int bm, bn, at_once;  // tiles a CU works on at once
    int fixed, alone, each;
  };
  static constexpr Price prices[] = {
      {kMx64x64, 64, 64, 2, 1400, 160, 110},     {kMx64x256, 64, 256, 1, 2630, 360, 360},
      {kMx128x128, 128, 128, 2, 3900, 310, 270}, {kMx128x192, 128, 192, 1, 4100, 370, 370},
      {kMx192x256, 192, 256, 1, 5950, 540, 540}, {kMx256x256, 256, 256, 1, 7500, 690, 690}};
  const int64_t steps = 2 * ceil_div(K, 2 * kMxGroup);
  MxForm best = kMx64x64;
  int64_t least = INT64_MAX;
  for (const Price& p : prices) {
    const int64_t tiles = ceil_div(M, p.bm) * ceil_div(N, p.bn);
    const int64_t cost = ceil_div(tiles, 256 * p.at_once) * p.fixed +
                         steps * std::max<int64_t>(p.alone, ceil_div(tiles, 256) * p.each);
    if (cost < least) least = cost, best = p.form;
  }
  return best;
}

template <int DT>
hipError_t launch_mx_matmul(const MxArgs& a, hipStream_t stream) {
  switch (mx_form(a.M, a.N, a.K)) {
    case kMx64x64: return launch_mx_tile<2, 2, 2, 2, 3, 2, DT>(a, stream);
    case kMx64x256: return launch_mx_tile<2, 4, 2, 4, 2, 2, DT>(a, stream);
    case kMx128x128: return launch_mx_tile<4, 4, 2, 2, 2, 2, DT>(a, stream);
    case kMx128x192: return launch_mx_tile<4, 3, 2, 4, 2, 2, DT>(a, stream);
    case kMx192x256: return launch_mx_tile<6, 4, 2, 4, 2, 2, DT>(a, stream);
    case kMx256x256: return launch_mx_tile<8, 4, 2, 4, 2, 2, DT>(a, stream);
    case kMxRowsForm: break;
  }
  const int mt = a.M <= 16 ? 1 : a.M <= 32 ? 2 : 4;
  const dim3 grid(static_cast<unsigned>(ceil_div(a.N, 16)),
                  static_cast<unsigned>(ceil_div(a.M, 16 * mt)));
  const int threads = 64 * kMxWaves;
  if (mt == 1) mx_rows_kernel<1, kMxCodes, DT><<<grid, threads, 0, stream>>>(a);
  else if (mt == 2) mx_rows_kernel<2, kMxCodes, DT><<<grid, threads, 0, stream>>>(a);
  else mx_rows_kernel<4, kMxCodes, DT><<<grid, threads, 0, stream>>>(a);
  return hipGetLastError();
}

template <int XD>
hipError_t launch_mx_dense(const MxArgs& a, int dtype, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(ceil_div(a.N, 16)));
  const int threads = 64 * kMxWaves;
  if (dtype == kMxF16) mx_rows_kernel<1, XD, kMxF16><<<grid, threads, 0, stream>>>(a);
  else if (dtype == kMxBF16) mx_rows_kernel<1, XD, kMxBF16><<<grid, threads, 0, stream>>>(a);
  else mx_rows_kernel<1, XD, kMxF32><<<grid, threads, 0, stream>>>(a);
  return hipGetLastError();
}

template <int DT>
hipError_t launch_mx_quantize(const void* X, int64_t rows, int64_t K, int64_t row_stride,
                              int64_t k_stride, void* codes, void* scales, hipStream_t stream) {
  using T = typename MxElem<DT>::type;
  const auto* x = static_cast<const T*>(X);
  const int64_t groups = ceil_div(K, kMxGroup);
  const int k = static_cast<int>(K);
  if (k_stride == 1) {
    const int64_t tiles = ceil_div(K, 4 * kMxGroup);
    const int64_t blocks = tiles * ceil_div(rows, kMxRows);
    const int64_t across = std::min(blocks, kMxGrid);  // (behind the last block: rows that are not there)
    const dim3 grid(static_cast<unsigned>(across), static_cast<unsigned>(ceil_div(blocks, across)));
    auto* c = static_cast<uint32_t*>(codes);
    auto* s = static_cast<uint32_t*>(scales);
    // 16-byte loads where every row starts on 16 bytes
    if (aligned(X, 16) && row_stride * sizeof(T) % 16 == 0)
      mx_quantize_kernel<DT, true><<<grid, 256, 0, stream>>>(x, row_stride, c, s, rows, k, (int)tiles);
    else
      mx_quantize_kernel<DT, false><<<grid, 256, 0, stream>>>(x, row_stride, c, s, rows, k, (int)tiles);
  } else {
    const dim3 grid(static_cast<unsigned>(groups * ceil_div(rows, kMxCols)));
    auto* c = static_cast<uint8_t*>(codes);
    auto* s = static_cast<uint32_t*>(scales);
    // two rows a load where every k starts on both
    if (aligned(X, 2 * sizeof(T)) && k_stride % 2 == 0 && rows % 2 == 0)
      mx_quantize_t_kernel<DT, true><<<grid, 256, 0, stream>>>(x, k_stride, c, s, rows, k, (int)groups);
    else
      mx_quantize_t_kernel<DT, false><<<grid, 256, 0, stream>>>(x, k_stride, c, s, rows, k, (int)groups);
  }
  return hipGetLastError();
}

int check_mx(int64_t rows, int64_t K, int64_t dtype) {
  NIBBLE_CHECK(rows >= 0 && K >= 0, "negative dimension");
  NIBBLE_CHECK(K % kMxBlock == 0, "K=%lld is not a multiple of %d", (long long)K, kMxBlock);
  // 32-bit offsets within a tile's rows of codes and within the scales
  NIBBLE_CHECK(K <= (1 << 22), "K above %d", 1 << 22);
  NIBBLE_CHECK(rows <= (1 << 28) && ceil_div(K, kMxGroup) * rows * 4 < (int64_t(1) << 31),
               "a matrix of %lld x %lld has 2^31 bytes of scales or more", (long long)rows,
               (long long)K);
  NIBBLE_CHECK(dtype == kMxF16 || dtype == kMxBF16 || dtype == kMxF32,
               "dtype must be 0 (fp16), 1 (bf16) or 2 (fp32), got %lld", (long long)dtype);
  return NIBBLE_OK;
}

}  // namespace
}  // namespace nibble

using namespace nibble;

extern "C" int nibble_mx_quantize(const void* X, int64_t rows, int64_t K, int64_t row_stride,
                                  int64_t k_stride, int64_t dtype, void* codes, void* scales,
                                  void* stream_) {
  const int rc = check_mx(rows, K, dtype);
  if (rc != NIBBLE_OK) return rc;
  if (rows == 0 || K == 0) return ok();
  NIBBLE_CHECK(row_stride > 0 && k_stride > 0 && (k_stride == 1 || row_stride == 1),
               "one of the strides must be 1 and neither below, got %lld and %lld",
               (long long)row_stride, (long long)k_stride);
  NIBBLE_CHECK(row_stride < (int64_t(1) << 40) && k_stride < (int64_t(1) << 40), "stride above 2^40");
  NIBBLE_CHECK(X != nullptr && codes != nullptr && scales != nullptr, "null pointer");
  NIBBLE_CHECK(aligned(X, dtype == kMxF32 ? 4 : 2) && aligned(codes, 16) && aligned(scales, 4),
               "misaligned pointer");
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  DeviceGuard guard;
  int dev = 0;
  NIBBLE_HIP(guard.enter(stream, &dev));
  const hipError_t e =
      dtype == kMxF16    ? launch_mx_quantize<kMxF16>(X, rows, K, row_stride, k_stride, codes, scales, stream)
      : dtype == kMxBF16 ? launch_mx_quantize<kMxBF16>(X, rows, K, row_stride, k_stride, codes, scales, stream)
                         : launch_mx_quantize<kMxF32>(X, rows, K, row_stride, k_stride, codes, scales, stream);
  if (e != hipSuccess) return hip_fail(e, "mx quantize kernel launch");
  return ok();
}

extern "C" int nibble_mx_dequantize(const void* codes, const void* scales, int64_t rows, int64_t K,
                                    int64_t dtype, void* out, void* stream_) {
  const int rc = check_mx(rows, K, dtype);
  if (rc != NIBBLE_OK) return rc;
  if (rows == 0 || K == 0) return ok();
  NIBBLE_CHECK(codes != nullptr && scales != nullptr && out != nullptr, "null pointer");
  NIBBLE_CHECK(aligned(codes, 16) && aligned(scales, 4) && aligned(out, 16), "misaligned pointer");
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  DeviceGuard guard;
  int dev = 0;
  NIBBLE_HIP(guard.enter(stream, &dev));
  const auto* c = static_cast<const uint8_t*>(codes);
  const auto* s = static_cast<const uint8_t*>(scales);
  const int64_t blocks = ceil_div(rows * (K / (dtype == kMxF32 ? 4 : 8)), 256);
  const int64_t across = std::min(blocks, kMxGrid);
  const dim3 grid(static_cast<unsigned>(across), static_cast<unsigned>(ceil_div(blocks, across)));
  if (dtype == kMxF32)
    mx_dequantize_kernel<kMxF32><<<grid, 256, 0, stream>>>(c, s, rows, (int)K, static_cast<float*>(out));
  else if (dtype == kMxF16)
    mx_dequantize_kernel<kMxF16><<<grid, 256, 0, stream>>>(c, s, rows, (int)K,
                                                         static_cast<unsigned short*>(out));
  else
    mx_dequantize_kernel<kMxBF16><<<grid, 256, 0, stream>>>(c, s, rows, (int)K,
                                                          static_cast<unsigned short*>(out));
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return hip_fail(e, "mx dequantize kernel launch");
  return ok();
}

static int check_mx_matmul(const void* x_codes, const void* x_scales, int64_t M,
                           const void* w_codes, const void* w_scales, int64_t N, int64_t K,
                           int64_t dtype, const void* Y) {
  int rc = check_mx(M, K, dtype);
  if (rc != NIBBLE_OK) return rc;
  rc = check_mx(N, K, dtype);
  if (rc != NIBBLE_OK) return rc;
  if (M == 0 || N == 0) return NIBBLE_OK;
  NIBBLE_CHECK(M <= 65535 * 64, "more than %d rows of x", 65535 * 64);
  NIBBLE_CHECK(ceil_div(M, 64) * ceil_div(N, 64) <= (1 << 30), "an output of %lld x %lld",
               (long long)M, (long long)N);
  NIBBLE_CHECK(Y != nullptr, "null pointer");
  NIBBLE_CHECK(K == 0 || (x_codes != nullptr && x_scales != nullptr && w_codes != nullptr &&
                          w_scales != nullptr),
               "null pointer");
  NIBBLE_CHECK(aligned(x_codes, 16) && aligned(w_codes, 16) && aligned(x_scales, 4) &&
                   aligned(w_scales, 4) && aligned(Y, 16),
               "misaligned pointer");
  return NIBBLE_OK;
}

extern "C" int nibble_mx_matmul(const void* x_codes, const void* x_scales, int64_t M,
                                const void* w_codes, const void* w_scales, int64_t N, int64_t K,
                                int64_t dtype, void* Y, void* stream_) {
  const int rc = check_mx_matmul(x_codes, x_scales, M, w_codes, w_scales, N, K, dtype, Y);
  if (rc != NIBBLE_OK) return rc;
  if (M == 0 || N == 0) return ok();
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  DeviceGuard guard;
  int dev = 0;
  NIBBLE_HIP(guard.enter(stream, &dev));
  const MxArgs a{static_cast<const uint8_t*>(x_codes), static_cast<const uint8_t*>(x_scales),
                 static_cast<const uint8_t*>(w_codes), static_cast<const uint8_t*>(w_scales), Y,
                 static_cast<int>(M), static_cast<int>(N), static_cast<int>(K), nullptr, 0};
  const hipError_t e = dtype == kMxF16    ? launch_mx_matmul<kMxF16>(a, stream)
                       : dtype == kMxBF16 ? launch_mx_matmul<kMxBF16>(a, stream)
                                          : launch_mx_matmul<kMxF32>(a, stream);
  if (e != hipSuccess) return hip_fail(e, "mx matmul kernel launch");
  return ok();
}

// Every workgroup quantises the whole of a dense x, so it is taken while that is
// little: at most 4096 k a CU.  us, one launch / quantised before, in a graph and
// as calls (of two launches in one call since, 11): 1 x 4096 x 1024 3.7 / 4.6, 7.5
// / 15.1; 16 x 4096 x 4096 7.5 / 6.3, 7.8 / 15.3; 16 x 12288 x 1024 7.7 / 5.8, 7.9 /
// 15.3; beyond it 1 x 12288 x 4096 10.5 / 7.8, 10.0 / 14.7; 16 x 12288 x 4096 18.7 /
// 10.0, 17.8 / 15.0; 1 x 4096 x 14336 14.2 / 8.8, 13.6 / 14.8; 16 x 12288 x 14336 64
// / 28, 64 / 27.
static bool mx_takes_dense(int64_t M, int64_t N, int64_t K) {
  return M >= 1 && M <= 16 && N >= 1 && N <= 12288 && K >= 1 &&
         ceil_div(N, 4096) * K <= 4096;  // (the rows kernel's sizes: one workgroup for 16 rows of w)
}

extern "C" size_t nibble_mx_matmul_dense_workspace_bytes(int64_t M, int64_t N, int64_t K,
                                                         int aligned) {
  if (check_mx(M, K, 0) != NIBBLE_OK || check_mx(N, K, 0) != NIBBLE_OK || M == 0 || N == 0) return 0;
  if (aligned != 0 && mx_takes_dense(M, N, K)) return 0;
  return static_cast<size_t>(M) * (K / 2) + static_cast<size_t>(ceil_div(K, kMxGroup)) * M * 4;
}

extern "C" int nibble_mx_matmul_dense(const void* X, int64_t M, int64_t row_stride, int64_t x_dtype,
                                      const void* w_codes, const void* w_scales, int64_t N,
                                      int64_t K, int64_t dtype, void* Y, void* workspace,
                                      size_t workspace_bytes, void* stream_) {
  int rc = check_mx(M, K, x_dtype);
  if (rc != NIBBLE_OK) return rc;
  rc = check_mx(N, K, dtype);
  if (rc != NIBBLE_OK) return rc;
  if (M == 0 || N == 0) return ok();
  NIBBLE_CHECK(row_stride >= 0 && row_stride < (int64_t(1) << 40), "row_stride out of range");
  const int64_t size = x_dtype == kMxF32 ? 4 : 2;
  const bool rows16 = row_stride * size % 16 == 0 && aligned(X, 16) &&
                      (M - 1) * row_stride + K < (int64_t(1) << 31) / size;
  if (!rows16 || !mx_takes_dense(M, N, K)) {
    const size_t need = nibble_mx_matmul_dense_workspace_bytes(M, N, K, 0);
    if (need > 0 && (workspace == nullptr || workspace_bytes < need))
      return fail(NIBBLE_ERR_WORKSPACE, "a dense x needs %zu bytes of workspace, got %zu", need,
                  workspace == nullptr ? size_t(0) : workspace_bytes);
    if (!aligned(workspace, 16))
      return fail(NIBBLE_ERR_WORKSPACE, "workspace must be 16-byte aligned");
    uint8_t* const codes = need > 0 ? static_cast<uint8_t*>(workspace) : nullptr;
    uint8_t* const scales = need > 0 ? codes + M * (K / 2) : nullptr;
    // (the product's arguments are looked at before anything is launched)
    rc = check_mx_matmul(codes, scales, M, w_codes, w_scales, N, K, dtype, Y);
    if (rc != NIBBLE_OK) return rc;
    rc = nibble_mx_quantize(X, M, K, row_stride, 1, x_dtype, codes, scales, stream_);
    if (rc != NIBBLE_OK) return rc;
    return nibble_mx_matmul(codes, scales, M, w_codes, w_scales, N, K, dtype, Y, stream_);
  }
  NIBBLE_CHECK(X != nullptr && Y != nullptr && w_codes != nullptr && w_scales != nullptr,
               "null pointer");
  NIBBLE_CHECK(aligned(w_codes, 16) && aligned(w_scales, 4) && aligned(Y, 16), "misaligned pointer");
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  DeviceGuard guard;
  int dev = 0;
  NIBBLE_HIP(guard.enter(stream, &dev));
  const MxArgs a{nullptr, nullptr, static_cast<const uint8_t*>(w_codes),
                 static_cast<const uint8_t*>(w_scales), Y, static_cast<int>(M), static_cast<int>(N),
                 static_cast<int>(K), X, static_cast<int>(row_stride)};
  const int d = static_cast<int>(dtype);
  const hipError_t e = x_dtype == kMxF16    ? launch_mx_dense<kMxF16>(a, d, stream)
                       : x_dtype == kMxBF16 ? launch_mx_dense<kMxBF16>(a, d, stream)
                                            : launch_mx_dense<kMxF32>(a, d, stream);
  if (e != hipSuccess) return hip_fail(e, "mx matmul kernel launch");
  return ok();
}
