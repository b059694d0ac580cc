// The tiled product of two microscaled matrices (many rows on both sides).
#pragma once

#include "nibble_common.h"
#include "nibble_copy.h"

namespace nibble {

constexpr int kMxGroupM = 8;  // row tiles of x that share a column tile of w in turn

// A tile of y = x w^T per workgroup of WM x WN waves, each XT 16-row tiles of x
// by WT of w.  A step is two k groups of 128: 128 bytes of codes (a whole line;
// rows of 64 bytes came at half the rate) and two words of scales a row, copied
// straight into a ring of RING buffers in LDS.
//
// v_mfma_scale_f32_16x16x128 takes from lane (g = l / 16, c = l % 16) block g of
// row c and its scale, byte g of the row's word.  w is the row operand: a lane
// then holds four neighbouring outputs of one row of y.  (The 32x32x64 form
// moves the same bytes; on random codes, register to register, it ran at 5.9
// PFLOP/s and this one at 6.8: the card's power sets both.)
//
// A register is read again from LDS as soon as its last product is issued, with
// the next k group's codes, so reads run under products all the time and no
// second set of registers is needed.  In a step's last k group, behind the first
// column of products, a wave waits for its own copies of the next step, by count;
// the barrier makes everybody's visible and this step's buffer free, and the
// copies of the step RING later go out.  No other memory operation is in flight
// in the loop.  2048 x 14336 x 16384 230 us against 240 with a k group's reads
// before its products.
//
// In LDS unit u (16 bytes) of row r lies at unit u ^ (r % 8): eight rows of a read
// cover 32 banks once.
//
// What bounds it: power, then the copies.  2048 x 14336 x 16384 takes 230 us, 4.2
// PFLOP/s; with codes of zero, the same instructions, 190.  Without copies it took
// 209 of then 273 us, without reads of LDS 254, without either 163, which is the
// rate of the products alone over 448 tiles in two rounds of 256 CUs.
template <int XT, int WT, int WM, int WN, int RING_>
struct MxTile {
  static constexpr int KU = 2;  // k groups of a step
  static constexpr int RING = RING_, WAVES = WM * WN, THREADS = 64 * WAVES;
  static constexpr int BM = 16 * XT * WM, BN = 16 * WT * WN;
  static constexpr int ROW = 64 * KU, UNITS = 4 * KU;   // bytes and 16-byte units of a row
  static constexpr int CODES = (BM + BN) * ROW;          // bytes of a step
  static constexpr int SCALES = (BM + BN) * 4 * KU;
  static constexpr int STEP = CODES + SCALES;
  static constexpr int XCOPIES = BM * ROW / 1024 / WAVES;  // a wave and step
  static constexpr int WCOPIES = BN * ROW / 1024 / WAVES;
  static constexpr int CHUNKS = KU * (BM + BN) / 64;       // of 64 words of scales
  static constexpr int SCOPIES = (CHUNKS + WAVES - 1) / WAVES;
  static constexpr bool SPARE = SCOPIES * WAVES > CHUNKS;  // copies that only keep the count
  static constexpr int LDS = RING * STEP + (SPARE ? 256 : 0);
  static constexpr int LOADS = XCOPIES + WCOPIES + SCOPIES;
  static_assert(XCOPIES * WAVES * 1024 == BM * ROW && WCOPIES * WAVES * 1024 == BN * ROW &&
                    BM % 64 == 0 && BN % 64 == 0, "shares");
  static_assert(LOADS * (RING - 1) <= 63, "vmcnt range");
};

template <class S, int XT, int WT, int WM, int WN, int DT, int OCC>
__global__ __launch_bounds__(S::THREADS, OCC) void mx_tile_kernel(MxArgs a, int tiles_m, int tiles_n) {
  constexpr int BM = S::BM, BN = S::BN, KU = S::KU, WAVES = S::WAVES;
  __shared__ __attribute__((aligned(16))) uint8_t lds[S::LDS];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  const int wm = wave / WN, wn = wave % WN;
  // Workgroup -> tile: XCD id % 8 takes one contiguous share of an order in
  // which 8 row tiles share each column tile's codes in its L2.
  const uint32_t total = static_cast<uint32_t>(tiles_m) * tiles_n;
  const uint32_t xcd = blockIdx.x & 7u;
  const uint32_t seq = xcd * (total >> 3) + min(xcd, total & 7u) + (blockIdx.x >> 3);
  const uint32_t block = seq / (kMxGroupM * tiles_n);
  const uint32_t in_block = seq - block * (kMxGroupM * tiles_n);
  const uint32_t rows_in = min(static_cast<uint32_t>(kMxGroupM), tiles_m - block * kMxGroupM);
  const int tile_n = static_cast<int>(in_block / rows_in);
  const int m0 = static_cast<int>(block * kMxGroupM + in_block - tile_n * rows_in) * BM;
  const int n0 = tile_n * BN;

  const int half_k = a.K / 2, blocks = a.K / kMxBlock;
  const int groups = (blocks + 3) / 4, steps = (groups + KU - 1) / KU;
  const uint8_t* const xbase = a.xc + static_cast<int64_t>(m0) * half_k;
  const uint8_t* const wbase = a.wc + static_cast<int64_t>(n0) * half_k;
  const uint32_t xbytes = static_cast<uint32_t>(min(BM, a.M - m0)) * half_k;
  const uint32_t wbytes = static_cast<uint32_t>(min(BN, a.N - n0)) * half_k;
  const uint32_t base = lds_address(lds);

  // Copy u of a wave (1 KiB, 16 / KU rows) fills rows (16 / KU) (WAVES u + wave)
  // .. of the tile's BM rows of x, then its BN of w: one lane offset for all, the
  // rows in the scalar offset.  Rows that are not there lie beyond the resource
  // and read as zeros; blocks behind K, and everything behind the last step, are
  // sent out of range lane by lane, so that the count of loads stays.
  constexpr int CROWS = 16 / KU;
  const int crow = lane / S::UNITS;
  const int unit = (lane % S::UNITS) ^ crow;  // (crow < 8, and a copy starts on a multiple of 8)
  const uint32_t voff = static_cast<uint32_t>(crow) * half_k + unit * 16u;
  const uint32_t rows_step = static_cast<uint32_t>(CROWS * WAVES) * half_k;
  const uint32_t rows_wave = static_cast<uint32_t>(CROWS * wave) * half_k;
  uint32_t soff[S::SCOPIES];  // lane offsets of the scale copies
  const uint8_t* sbase[S::SCOPIES];
  uint32_t sbytes[S::SCOPIES], sgroup[S::SCOPIES], sdst[S::SCOPIES];
  int splane[S::SCOPIES];
#pragma unroll
  for (int j = 0; j < S::SCOPIES; ++j) {
    const int c = wave + WAVES * j;  // a chunk of 64 rows; behind the last one: counts only
    const int plane = c / ((BM + BN) / 64), cc = c % ((BM + BN) / 64);
    const bool x = cc < BM / 64;
    const int gr = x ? m0 + 64 * cc + lane : n0 + 64 * cc - BM + lane;
    soff[j] = c < S::CHUNKS && gr < (x ? a.M : a.N) ? gr * 4u : kOutOfRange;
    sbase[j] = x ? a.xs : a.ws;
    sbytes[j] = static_cast<uint32_t>(groups) * (x ? a.M : a.N) * 4u;
    sgroup[j] = (x ? a.M : a.N) * 4u;
    splane[j] = plane;
    sdst[j] = c < S::CHUNKS ? base + S::CODES + c * 256u : base + S::RING * S::STEP;
  }
  struct Step {
    uint32_t v, k0, dst;
    int group;
  };
  auto prepare = [&](int step, int buf) {
    Step s;
    s.v = unit < blocks - S::UNITS * step ? voff : kOutOfRange;
    s.group = min(step, steps) * KU;
    s.k0 = s.group * 64u + rows_wave;
    s.dst = static_cast<uint32_t>(buf) * S::STEP;
    return s;
  };
  // Load u of a step: the code copies, then the scale copies.
  auto load = [&](int u, const Step& s) {
    if (u < S::XCOPIES + S::WCOPIES) {
      const bool x = u < S::XCOPIES;
      lds_copy16(x ? xbase : wbase, x ? xbytes : wbytes,
                 base + wave * 1024u + s.dst + u * (1024u * WAVES), s.v,
                 s.k0 + (x ? u : u - S::XCOPIES) * rows_step);
    } else {
      const int j = u - S::XCOPIES - S::WCOPIES, group = s.group + splane[j];
      lds_copy4(sbase[j], sbytes[j], sdst[j] + (wave + WAVES * j < S::CHUNKS ? s.dst : 0u),
                group < groups ? soff[j] : kOutOfRange, min(group, groups) * sgroup[j]);
    }
  };

  f4_t acc[XT][WT];
#pragma unroll
  for (int i = 0; i < XT; ++i)
#pragma unroll
    for (int j = 0; j < WT; ++j) acc[i][j] = f4_t{0.0f, 0.0f, 0.0f, 0.0f};

  const int c = lane & 15, g = lane >> 4;
  const int xrow = wm * 16 * XT + c, wrow = BM + wn * 16 * WT + c;
  const uint32_t at = (g ^ (c & 7)) * 16u;  // of a lane's block in k group 0; rows 16 apart agree
  u4_t x[XT], w[WT];
  uint32_t xs[XT], ws[WT];  // (a lane's block: byte g of its row's word)
  auto read_x = [&](int i, int buf, int kg) {
    const uint8_t* const p = lds + buf * S::STEP;
    xs[i] = p[S::CODES + (kg * (BM + BN) + xrow + 16 * i) * 4 + g];
    x[i] = *reinterpret_cast<const u4_t*>(p + (xrow + 16 * i) * S::ROW + (at ^ 64u * kg));
  };
  auto read_w = [&](int n, int buf, int kg) {
    const uint8_t* const p = lds + buf * S::STEP;
    ws[n] = p[S::CODES + (kg * (BM + BN) + wrow + 16 * n) * 4 + g];
    w[n] = *reinterpret_cast<const u4_t*>(p + (wrow + 16 * n) * S::ROW + (at ^ 64u * kg));
  };
#pragma unroll
  for (int t = 0; t < S::RING; ++t) {
    const Step s = prepare(t, t);
#pragma unroll
    for (int u = 0; u < S::LOADS; ++u) load(u, s);
  }
  __builtin_amdgcn_s_waitcnt(waitcnt_vm((S::RING - 1) * S::LOADS));  // (step 0)
  lds_barrier();
#pragma unroll
  for (int n = 0; n < WT; ++n) read_w(n, 0, 0);
#pragma unroll
  for (int i = 0; i < XT; ++i) read_x(i, 0, 0);
  int buf = 0;
  for (int t = 0; t < steps; ++t) {
    const int next = buf == S::RING - 1 ? 0 : buf + 1;
    const Step coming = prepare(t + S::RING, buf);
#pragma unroll
    for (int kg = 0; kg < KU; ++kg) {
      const bool last = kg == KU - 1;
      const int from = last ? next : buf, group = last ? 0 : kg + 1;
#pragma unroll
      for (int n = 0; n < WT; ++n) {
        const i8_t vw = {(int)w[n][0], (int)w[n][1], (int)w[n][2], (int)w[n][3], 0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < XT; ++i) {
          const i8_t vx = {(int)x[i][0], (int)x[i][1], (int)x[i][2], (int)x[i][3], 0, 0, 0, 0};
          acc[i][n] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
              vw, vx, acc[i][n], 4, 4, 0, (int)ws[n], 0, (int)xs[i]);
          if (n == WT - 1) {
            __builtin_amdgcn_sched_barrier(0);
            read_x(i, from, group);
            __builtin_amdgcn_sched_barrier(0);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
        if (last && n == 0) {
          __builtin_amdgcn_s_waitcnt(waitcnt_vm((S::RING - 2) * S::LOADS));
          lds_barrier();
        }
        read_w(n, from, group);
        if (last) {
#pragma unroll
          for (int u = n * S::LOADS / WT; u < (n + 1) * S::LOADS / WT; ++u) load(u, coming);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    buf = next;
  }
  // No copy may land in LDS that holds something else by then.
  __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));
  __syncthreads();

  // The outputs go through LDS, 16 rows of a wave at a time, so that a store
  // covers whole runs of a row: 16 bytes a lane where every row starts on 16,
  // else 4 or single outputs.  They pass by the caches (512 x 14336 x 4096 21.8 us
  // against 23.1).
  using T = typename MxElem<DT>::type;
  typedef T vec4 __attribute__((ext_vector_type(4)));
  constexpr int COLS = 16 * WT, PITCH = COLS + 16 / sizeof(T);
  static_assert(WAVES * 16 * PITCH * sizeof(T) <= S::RING * S::STEP, "the outputs fit");
  T* const out = reinterpret_cast<T*>(lds) + wave * 16 * PITCH;
  T* const y = static_cast<T*>(a.y);
  const int n1 = n0 + wn * COLS;
  const int cols = min(COLS, a.N - n1);
  const int row_bytes = a.N % 16 * static_cast<int>(sizeof(T)) % 16;
#pragma unroll
  for (int i = 0; i < XT; ++i) {
    const int m1 = m0 + wm * 16 * XT + 16 * i;
#pragma unroll
    for (int j = 0; j < WT; ++j) {
      vec4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = mx_out<DT>(acc[i][j][e]);
      *reinterpret_cast<vec4*>(out + c * PITCH + 16 * j + 4 * g) = v;
    }
    __builtin_amdgcn_s_waitcnt(kWaitLgkm0);
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    auto store = [&](auto piece) {
      using P = decltype(piece);
      constexpr int E = sizeof(P) / sizeof(T), PER = COLS / E;  // outputs a store, stores a row
#pragma unroll
      for (int u = 0; u < (16 * PER + 63) / 64; ++u) {
        const int r = (u * 64 + lane) / PER, n = (u * 64 + lane) % PER * E;
        if (r < 16 && m1 + r < a.M && n < cols)
          __builtin_nontemporal_store(
              *reinterpret_cast<const P*>(out + r * PITCH + n),
              reinterpret_cast<P*>(y + static_cast<int64_t>(m1 + r) * a.N + n1 + n));
      }
    };
    if (row_bytes == 0) store(u4_t{});
    else if (row_bytes % 4 == 0) store(uint32_t{});
    else store(T{});
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
  }
}

}  // namespace nibble
