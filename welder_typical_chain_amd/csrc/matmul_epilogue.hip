// matmul_epilogue.hip -- kernels of wtc_matmul_epilogue and its gradients:
//   out = round(act(A . B + bias) + residual), da = dz . B^T, db = A^T . dz
//
// One tile kernel for the three products.  An operand is either contiguous
// along the contraction (KC: A of the product, both operands of da) or strided
// along it (KS: B of the product, both operands of db); with B stored as its
// transpose the two kinds change places.  A tile's k-slab of 32 elements takes
// 64 bytes per row of the operand either way:
//   KC  [rows][4 chunks of 16 bytes], read with ds_read_b128 (a64_lds_offset)
//   KS  [32 k][128 columns] per 128 rows of the operand, read with the
//       transposing ds_read_b64_tr_b16 (btr_offset)
// 4 waves in a 2 x 2 grid, each a quarter of the tile in 32 x 32 MFMA subtiles
// (v_mfma_f32_32x32x16, D = B^T . A^T: a lane's accumulators belong to one
// output row).  Slabs go through a ring of stages filled by direct-to-LDS
// loads, all but one ahead of the one whose MFMAs run; the fragments of a slab's
// second half are read while the MFMAs of the first issue, and the next
// slab's first half under those of the second.
// bf16 8192 x 8192 x 4096: 465 us, 1180 TFLOP/s (a library product of that size
// 1270); with bias and gelu 508.  Full tiles are bound by the matrix cores at the
// clock that the power limit leaves; small ones by the tiles' count and latency.
#include <algorithm>
#include <type_traits>

#include "layer_common.h"
#include "layer_kernels.h"

namespace wtc {
namespace {

constexpr int kSlab = 64;    // bytes of k per ring stage and operand row
constexpr int kSlabK = 32;   // elements
constexpr int kThreads = 256;

// Eight consecutive values, 16-byte aligned.
template <int DT> __device__ inline void load8(const void* p, int64_t i, float (&x)[8]) {
  if constexpr (DT == DT_F32) {
    const f32x4 *q = reinterpret_cast<const f32x4*>(static_cast<const float*>(p) + i), lo = q[0], hi = q[1];
#pragma unroll
    for (int u = 0; u < 4; ++u) x[u] = lo[u], x[4 + u] = hi[u];
  } else {
    const auto v = *reinterpret_cast<const typename Elem<DT>::vec8*>(static_cast<const typename Elem<DT>::type*>(p) + i);
#pragma unroll
    for (int u = 0; u < 8; ++u) x[u] = (float)v[u];
  }
}
template <int DT> __device__ inline void store8(void* p, int64_t i, const float (&x)[8]) {
  if constexpr (DT == DT_F32) {
    f32x4* q = reinterpret_cast<f32x4*>(static_cast<float*>(p) + i);
    q[0] = f32x4{x[0], x[1], x[2], x[3]};
    q[1] = f32x4{x[4], x[5], x[6], x[7]};
  } else {
    uint32_t w[4];
    pack4<DT>(f32x4{x[0], x[1], x[2], x[3]}, &w[0], &w[1]);
    pack4<DT>(f32x4{x[4], x[5], x[6], x[7]}, &w[2], &w[3]);
    *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(p) + i) = u32x4{w[0], w[1], w[2], w[3]};
  }
}

// The epilogue of eight columns n .. n+7 of row m; z: the products.
template <int DT, int OUT_DT, int ACT>
__device__ inline void finish8(const MatmulParams& p, int64_t m, int64_t n, float (&z)[8]) {
  float y[8];
  if (p.bias) {
    if (p.bias_f32) load8<DT_F32>(p.bias, n, y);
    else load8<DT>(p.bias, n, y);
#pragma unroll
    for (int u = 0; u < 8; ++u) z[u] += y[u];
  }
  if (p.pre) store8<DT_F32>(p.pre, m * p.ldp + n, z);
#pragma unroll
  for (int u = 0; u < 8; ++u) z[u] = act_value<ACT, OUT_DT == DT_F32>(z[u]);
  if (p.residual) {
    load8<OUT_DT>(p.residual, m * p.ldr + n, y);
#pragma unroll
    for (int u = 0; u < 8; ++u) z[u] += y[u];
  }
  store8<OUT_DT>(p.out, m * p.ldo + n, z);
}

template <int DT, int OUT_DT> __device__ inline void finish(const MatmulParams& p, int64_t m, int64_t n, float (&z)[8]) {
  switch (p.act) {
    case WTC_ACT_NONE: return finish8<DT, OUT_DT, WTC_ACT_NONE>(p, m, n, z);
    case WTC_ACT_RELU: return finish8<DT, OUT_DT, WTC_ACT_RELU>(p, m, n, z);
    case WTC_ACT_GELU: return finish8<DT, OUT_DT, WTC_ACT_GELU>(p, m, n, z);
    case WTC_ACT_GELU_TANH: return finish8<DT, OUT_DT, WTC_ACT_GELU_TANH>(p, m, n, z);
    case WTC_ACT_SILU: return finish8<DT, OUT_DT, WTC_ACT_SILU>(p, m, n, z);
  }
}

// Direct-to-LDS loads of one operand: wave w fills blocks nb*w .. of 1 KiB.
// Rows (KC) and columns (KS) past the operand's end are parked at kOutOfRange,
// whose loads give zeros; so are slabs from k_end on.
template <bool KS, int ROWS> struct Loader {
  static constexpr int NB = ROWS * kSlab / 1024 / 4;  // blocks per wave: 4 or 2
  i32x4 rsrc;
  uint32_t off[NB];
  uint32_t ld, kpos, lds;
  __device__ inline void init(const uint8_t* base, uint32_t rows, uint32_t row0, uint32_t k_total, uint32_t ld_bytes,
                              int wave, int lane) {
    const uint32_t bytes = KS ? (k_total ? (k_total - 1) * ld_bytes + rows * 2 : 0) : (rows - 1) * ld_bytes + k_total * 2;
    const i32x4 r = raw_rsrc(base, bytes);
#pragma unroll
    for (int i = 0; i < 4; ++i) rsrc[i] = __builtin_amdgcn_readfirstlane(r[i]);
    ld = ld_bytes;
    if constexpr (KS) {
      // blocks of 4 k-rows x 128 columns, 8 a 128-column half
      const int half = wave * NB / 8, blk = wave * NB % 8;
      const uint32_t col = row0 + 128u * half + 8u * (uint32_t)dma_b_chunk(blk, lane);
      kpos = (uint32_t)dma_b_row(blk, lane);
#pragma unroll
      for (int q = 0; q < NB; ++q) off[q] = col < rows ? (kpos + 4u * q) * ld + col * 2u : kOutOfRange;
      lds = (uint32_t)(half * 8192 + blk * 1024);
    } else {
      kpos = 8u * (uint32_t)dma64_a_chunk(0, lane);
#pragma unroll
      for (int q = 0; q < NB; ++q) {
        const uint32_t row = row0 + (uint32_t)dma64_a_row(wave * NB + q, lane);
        off[q] = row < rows ? row * ld + kpos * 2u : kOutOfRange;
      }
      lds = (uint32_t)(wave * NB * 1024);
    }
  }
  // block q of slab kt (k from 32 kt), elements from k_end on read as zeros
  __device__ inline void issue(uint32_t stage, int kt, uint32_t k_end, int q) const {
    const uint32_t k = (uint32_t)kt * kSlabK + kpos + (KS ? 4u * q : 0u);
    const uint32_t step = KS ? (uint32_t)kt * kSlabK * ld : (uint32_t)kt * kSlab;
    dma16(rsrc, k < k_end && off[q] != kOutOfRange ? off[q] + step : kOutOfRange, stage + lds + q * 1024);
  }
};

// Fragment reads of one operand for a wave's W subtiles of 32 rows.
template <bool KS, int W> struct Frags {
  uint32_t base[KS ? W : 2];
  __device__ inline void init(uint32_t at, int row0, int lane) {
    if constexpr (KS) {
#pragma unroll
      for (int i = 0; i < W; ++i) {
        const int c = row0 + 32 * i;
        base[i] = at + (uint32_t)((c >> 7) * 8192 + btr_offset(btr_k(0, 0, lane), btr_n(c & 127, lane)));
      }
    } else {
#pragma unroll
      for (int s = 0; s < 2; ++s) base[s] = at + (uint32_t)a64_lds_offset(row0 + frag_row(lane), frag64_chunk16(lane, s));
    }
  }
  static constexpr int READS = KS ? 2 * W : W;
  __device__ inline void read(const uint8_t* st, int s, int u, u32x4 (&f)[W]) const {
    if constexpr (KS) {
      const int i = u >> 1, h = u & 1;
      const u32x2 v = tr_read(st + base[i] + (16 * s + 4 * h) * 256);
      f[i][2 * h] = v[0];
      f[i][2 * h + 1] = v[1];
    } else {
      f[u] = *reinterpret_cast<const u32x4*>(st + base[s] + u * 2048);
    }
  }
};

template <int TM, int TN, int STAGES> struct TileLds {
  static constexpr int A_STAGE = TM * kSlab, STAGE = (TM + TN) * kSlab;
  static constexpr int RING = STAGES * STAGE;
  // epilogue: a wave stages 32 rows of its quarter in f32
  static constexpr int PITCH = TN / 2 * 4 + 16;
  static constexpr int TOTAL = RING > 4 * 32 * PITCH ? RING : 4 * 32 * PITCH;
  static_assert(TOTAL <= 160 * 1024, "LDS");
};

// Grid: tiles * splits; split s takes k-slabs [s * slabs, (s + 1) * slabs) and, where
// there are several, writes f32 partial products [split][m][n] to p.partial.
template <int DT, int OUT_DT, bool AKS, bool BKS, int TM, int TN, int STAGES>
__device__ inline void matmul_tile(const MatmulParams& p, uint32_t block, uint32_t grid, uint8_t* smem) {
  using L = TileLds<TM, TN, STAGES>;
  constexpr int WM = TM / 64, WN = TN / 64;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave >> 1, wn = wave & 1;
  const uint32_t rows = (uint32_t)(p.m + TM - 1) / TM, cols = (uint32_t)(p.n + TN - 1) / TN;
  uint32_t rt, ct;  // all splits of a tile row are rows of the map
  tile_of_block(block, grid, rows * p.splits, cols, &rt, &ct);
  const uint32_t split = rt / rows;
  rt -= split * rows;
  const uint32_t row0 = rt * TM, n0 = ct * TN;
  const int kt0 = (int)split * p.slabs;
  const int nk = min(p.slabs, (p.k + kSlabK - 1) / kSlabK - kt0);
  const uint32_t k_end = (uint32_t)min((int64_t)p.k, (int64_t)(kt0 + p.slabs) * kSlabK);

  f32x16 acc[WM][WN];
#pragma unroll
  for (int i = 0; i < WM; ++i)
#pragma unroll
    for (int j = 0; j < WN; ++j)
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[i][j][v] = 0.0f;

  Loader<AKS, TM> la;
  Loader<BKS, TN> lb;
  la.init(p.a, (uint32_t)p.m, row0, (uint32_t)p.k, (uint32_t)p.lda * 2u, wave, lane);
  lb.init(p.b, (uint32_t)p.n, n0, (uint32_t)p.k, (uint32_t)p.ldb * 2u, wave, lane);
  Frags<AKS, WM> fa;
  Frags<BKS, WN> fb;
  fa.init(0, wm * (TM / 2), lane);
  fb.init(L::A_STAGE, wn * (TN / 2), lane);
  constexpr int NA = Loader<AKS, TM>::NB, NB = Loader<BKS, TN>::NB, LOADS = NA + NB, ALT = 2 * (NA < NB ? NA : NB);
  constexpr int RA = Frags<AKS, WM>::READS, R = RA + Frags<BKS, WN>::READS;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(WTC_LDS uint8_t*)smem;
  auto load = [&](uint32_t stage, int kt, int j) {
    // A and B blocks alternate, then what is left of the larger one
    const bool of_a = j < ALT ? !(j & 1) : NA > NB;
    const int q = j < ALT ? j >> 1 : j - ALT / 2;
    if (of_a) la.issue(stage, kt0 + kt, k_end, q);
    else lb.issue(stage + L::A_STAGE, kt0 + kt, k_end, q);
  };
  auto read = [&](const uint8_t* st, int s, int u, u32x4 (&a)[WM], u32x4 (&b)[WN]) {
    if (u < RA) fa.read(st, s, u, a);
    else fb.read(st, s, u - RA, b);
  };
  // Of `total` things, those that go with MFMA x of a part.
  constexpr int M = WM * WN;
  auto first = [](int total, int x) { return total * x / M; };
  if (nk > 0) {
#pragma unroll
    for (int q = 0; q < STAGES; ++q)
#pragma unroll
      for (int j = 0; j < LOADS; ++j) load(lds0 + q * L::STAGE, q, j);
    wait_loads_barrier<LOADS*(STAGES - 1)>();
    u32x4 a0[WM], b0[WN], a1[WM], b1[WN];
#pragma unroll
    for (int u = 0; u < R; ++u) read(smem, 0, u, a0, b0);
    int stage = 0;
    for (int kt = 0; kt < nk; ++kt) {
      const int next = stage + 1 == STAGES ? 0 : stage + 1;
      const uint8_t* cur = smem + stage * L::STAGE;
      const uint8_t* nxt = smem + next * L::STAGE;
      const uint32_t fill = lds0 + stage * L::STAGE;
      stage = next;
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int g = 0; g < WM; ++g) {
#pragma unroll
        for (int u = first(R, g * WN); u < first(R, (g + 1) * WN); ++u) read(cur, 1, u, a1, b1);
#pragma unroll
        for (int j = 0; j < WN; ++j) acc[g][j] = mfma32<DT>(b0[j], a0[g], acc[g][j]);
        __builtin_amdgcn_sched_barrier(0);
      }
      wait_loads_barrier<LOADS*(STAGES - 2)>();  // slab kt+1 landed; slab kt read
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int g = 0; g < WM; ++g) {
#pragma unroll
        for (int j = 0; j < WN; ++j) {
          // each load right behind an MFMA, in the first half of a group
          acc[g][j] = mfma32<DT>(b1[j], a1[g], acc[g][j]);
          constexpr int H = WN / 2;
          if (j < H) {
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int x = LOADS * (g * H + j) / (WM * H); x < LOADS * (g * H + j + 1) / (WM * H); ++x) load(fill, kt + STAGES, x);
            __builtin_amdgcn_sched_barrier(0);
          }
          if (j == H - 1) {
#pragma unroll
            for (int u = first(R, g * WN); u < first(R, (g + 1) * WN); ++u) read(nxt, 0, u, a0, b0);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    wait_loads_barrier<0>();
  }

  // ---- epilogue: each wave by itself, 32 rows at a time through its part of LDS,
  // from a row a lane to eight columns a lane.  A lane's columns are the same in
  // every step, so the bias is read once; the residual of the next 32 rows is
  // requested before the current ones are worked on (loaded where it is added,
  // its latency made up a quarter of 1500 x 3000 x 1000: 33.8 -> 26.5 us).
  constexpr int CW = TN / 2, LPR = CW / 8, RPI = 64 / LPR, ITS = 32 / RPI;
  uint8_t* stg = smem + wave * 32 * L::PITCH;
  const int c = lane % LPR * 8;
  const int64_t m0 = (int64_t)row0 + wm * (TM / 2) + lane / LPR, n = (int64_t)n0 + wn * CW + c;
  auto stage = [&](int mt) {
#pragma unroll
    for (int j = 0; j < WN; ++j)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<f32x4*>(stg + acc_j(lane) * L::PITCH + (j * 32 + acc_i(lane, 4 * g)) * 4) =
            f32x4{acc[mt][j][4 * g], acc[mt][j][4 * g + 1], acc[mt][j][4 * g + 2], acc[mt][j][4 * g + 3]};
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  };
  auto staged = [&](int it, float (&z)[8]) {
    const f32x4* src = reinterpret_cast<const f32x4*>(stg + (it * RPI + lane / LPR) * L::PITCH + c * 4);
    const f32x4 lo = src[0], hi = src[1];
#pragma unroll
    for (int u = 0; u < 4; ++u) z[u] = lo[u], z[4 + u] = hi[u];
  };
  if (p.splits > 1) {
    float* part = p.partial + (int64_t)split * p.m * p.n;
#pragma unroll
    for (int mt = 0; mt < WM; ++mt) {
      stage(mt);
#pragma unroll
      for (int it = 0; it < ITS; ++it) {
        const int64_t m = m0 + mt * 32 + it * RPI;
        float z[8];
        staged(it, z);
        if (m < p.m && n < p.n) store8<DT_F32>(part, m * p.n + n, z);
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
    return;
  }
  constexpr int RV = OUT_DT == DT_F32 ? 2 : 1;  // 16-byte words of eight values
  const int64_t n_in = n < p.n ? n : 0;
  float bias[8] = {};
  if (p.bias) {
    if (p.bias_f32) load8<DT_F32>(p.bias, n_in, bias);
    else load8<DT>(p.bias, n_in, bias);
  }
  u32x4 res[2][ITS][RV];
  auto request = [&](int mt) {
    if (!p.residual) return;
#pragma unroll
    for (int it = 0; it < ITS; ++it) {
      const int64_t m = min(m0 + mt * 32 + it * RPI, (int64_t)p.m - 1);
      const u32x4* src = reinterpret_cast<const u32x4*>(static_cast<const uint8_t*>(p.residual) + (m * p.ldr + n_in) * dtype_bytes(OUT_DT));
#pragma unroll
      for (int w = 0; w < RV; ++w) res[mt & 1][it][w] = src[w];
    }
  };
  auto epilogue = [&](auto act) {
    request(0);
#pragma unroll
    for (int mt = 0; mt < WM; ++mt) {
      if (mt + 1 < WM) request(mt + 1);
      stage(mt);
#pragma unroll
      for (int it = 0; it < ITS; ++it) {
        const int64_t m = m0 + mt * 32 + it * RPI;
        float z[8], y[8];
        staged(it, z);
#pragma unroll
        for (int u = 0; u < 8; ++u) z[u] += bias[u];
        const bool in = m < p.m && n < p.n;
        if (p.pre && in) store8<DT_F32>(p.pre, m * p.ldp + n, z);
#pragma unroll
        for (int u = 0; u < 8; ++u) z[u] = act_value<decltype(act)::value, OUT_DT == DT_F32>(z[u]);
        if (p.residual) {
          load8<OUT_DT>(res[mt & 1][it], 0, y);
#pragma unroll
          for (int u = 0; u < 8; ++u) z[u] += y[u];
        }
        if (in) store8<OUT_DT>(p.out, m * p.ldo + n, z);
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
  };
  switch (p.act) {
    case WTC_ACT_NONE: return epilogue(std::integral_constant<int, WTC_ACT_NONE>{});
    case WTC_ACT_RELU: return epilogue(std::integral_constant<int, WTC_ACT_RELU>{});
    case WTC_ACT_GELU: return epilogue(std::integral_constant<int, WTC_ACT_GELU>{});
    case WTC_ACT_GELU_TANH: return epilogue(std::integral_constant<int, WTC_ACT_GELU_TANH>{});
    case WTC_ACT_SILU: return epilogue(std::integral_constant<int, WTC_ACT_SILU>{});
  }
}

constexpr int waves_per_simd(int tm, int tn, int stages) { return (tm + tn) * kSlab * stages > 80 * 1024 ? 1 : 2; }
template <int DT, int OUT_DT, bool AKS, bool BKS, int TM, int TN, int STAGES>
__global__ void __launch_bounds__(kThreads, waves_per_simd(TM, TN, STAGES)) matmul_tile_kernel(const MatmulParams p) {
  __shared__ __attribute__((aligned(16))) uint8_t smem[TileLds<TM, TN, STAGES>::TOTAL];
  matmul_tile<DT, OUT_DT, AKS, BKS, TM, TN, STAGES>(p, blockIdx.x, gridDim.x, smem);
}

// da (x) and db (y) of a small layer in one launch: neither fills the chip alone.
// The one with more slabs a tile comes first.  The whole backward call, us: 1000 x
// 1000 x 1000 37.1 -> 24.9, 2048 x 2048 x 1024 53.7 -> 36.8, 128 x 512 x 512 17.6 ->
// 13.0; 4096 x 1024 x 1024 49.8 -> 49.0, where it ends to pay.
template <int DT, bool BKS>
__global__ void __launch_bounds__(kThreads, 2) matmul_pair_kernel(const MatmulParams x, const MatmulParams y, const uint32_t x_from, const uint32_t x_tiles, const uint32_t y_from) {
  __shared__ __attribute__((aligned(16))) uint8_t smem[TileLds<128, 128, 4>::TOTAL];
  const uint32_t b = blockIdx.x;
  if (b >= x_from && b - x_from < x_tiles) matmul_tile<DT, DT, false, BKS, 128, 128, 4>(x, b - x_from, x_tiles, smem);
  else matmul_tile<DT, DT, true, true, 128, 128, 4>(y, b - y_from, gridDim.x - x_tiles, smem);
}

// At most 16 rows against weights stored as [n][k] (decode): what counts is reading B
// once.  A workgroup takes 16 rows of B (columns of the output) and all of k: its 8
// waves take 64-element chunks of k in turn, straight from memory to registers as
// MFMA fragments (v_mfma_f32_16x16x32, D = B . A^T: a chunk is one 128-byte line
// of each row), and join their sums through LDS: one launch, and no partial
// products in memory.  Against 64-row tiles with k-splits, us: 8 x 4096 x 4096 8.8
// (10.7), 8 x 4096 x 1024 4.3 (7.7), 8 x 2048 x 2048 5.5 (8.5); what it reads of A
// grows with the workgroups and a wave's chunks come 8 at a time, so large n and
// long k go to the tiles (8 x 8192 x 8192 31.7 against 24.9).
constexpr int kRowsWaves = 8;
template <int DT> __device__ inline f32x4 mfma16(const u32x4& a, const u32x4& b, const f32x4& c) {
  if constexpr (DT == DT_F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <int DT, int OUT_DT>
__global__ void __launch_bounds__(kRowsWaves * 64, 2) matmul_rows_kernel(const MatmulParams p) {
  __shared__ __attribute__((aligned(16))) float red[kRowsWaves][16][16];  // [.][m][n]
  const int lane = threadIdx.x & 63, r = lane & 15, kq = (lane >> 4) * 8;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n0 = blockIdx.x * 16;
  // rows past the end take the last one's values; their results are not written
  const uint8_t* b = p.b + 2 * ((int64_t)min(n0 + r, p.n - 1) * p.ldb + kq);
  const uint8_t* a = p.a + 2 * ((int64_t)min(r, p.m - 1) * p.lda + kq);
  f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
  constexpr int U = 8;  // chunks requested at a time
  for (int c0 = wave; c0 * 64 < p.k; c0 += kRowsWaves * U) {
    u32x4 bf[U][2], af[U][2];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int k = (c0 + u * kRowsWaves) * 64 + s * 32;
        const bool in = k + kq < p.k;
        bf[u][s] = in ? *reinterpret_cast<const u32x4*>(b + 2 * (int64_t)k) : u32x4{0, 0, 0, 0};
        af[u][s] = in ? *reinterpret_cast<const u32x4*>(a + 2 * (int64_t)k) : u32x4{0, 0, 0, 0};
      }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int s = 0; s < 2; ++s) acc = mfma16<DT>(bf[u][s], af[u][s], acc);
  }
  *reinterpret_cast<f32x4*>(&red[wave][r][(lane >> 4) * 4]) = acc;
  __syncthreads();
  const int m = threadIdx.x >> 1, half = (threadIdx.x & 1) * 8;
  const int64_t n = n0 + half;
  if (m >= p.m || n >= p.n) return;
  float z[8] = {};
#pragma unroll
  for (int w = 0; w < kRowsWaves; ++w) {
    const f32x4* src = reinterpret_cast<const f32x4*>(&red[w][m][half]);
    const f32x4 lo = src[0], hi = src[1];
#pragma unroll
    for (int u = 0; u < 4; ++u) z[u] += lo[u], z[4 + u] += hi[u];
  }
  finish<DT, OUT_DT>(p, m, n, z);
}

// The partial products of all splits, summed in their order, and the epilogue.
template <int DT, int OUT_DT>
__global__ void __launch_bounds__(256) matmul_join_kernel(const MatmulParams p) {
  const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8, total = (int64_t)p.m * p.n;
  if (at >= total) return;
  float z[8], y[8];
  load8<DT_F32>(p.partial, at, z);
#pragma unroll 4
  for (int s = 1; s < p.splits; ++s) {
    load8<DT_F32>(p.partial, s * total + at, y);
#pragma unroll
    for (int u = 0; u < 8; ++u) z[u] += y[u];
  }
  const int64_t m = at / p.n;
  finish<DT, OUT_DT>(p, m, at - m * p.n, z);
}

// dz = dout * act'(pre), rounded for the products; the columns' sums in f32 of
// the values before rounding.  A workgroup takes 128 columns (16 threads of
// eight) of `chunk` rows, 16 rows at a time; with several row chunks the sums
// go to p.partial [chunk][n], which sum_chunks_kernel adds in order.
template <int DT>
__global__ void __launch_bounds__(256) act_backward_kernel(const ActBackwardParams p) {
  __shared__ float red[16][128 + 4];
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int cols = (int)((p.n + 127) / 128);
  const int chunk = blockIdx.x / cols;
  const int64_t n = (int64_t)(blockIdx.x % cols) * 128 + tx * 8;
  const int64_t m1 = min(p.m, (int64_t)(chunk + 1) * p.chunk_rows);
  float sum[8] = {};
  if (n < p.n)
    for (int64_t m = (int64_t)chunk * p.chunk_rows + ty; m < m1; m += 16) {
      float g[8], z[8];
      load8<DT>(p.dout, m * p.ldd + n, g);
      if (p.act != WTC_ACT_NONE) {
        load8<DT_F32>(p.pre, m * p.n + n, z);
        switch (p.act) {
          case WTC_ACT_RELU: for (int u = 0; u < 8; ++u) g[u] *= act_slope<WTC_ACT_RELU>(z[u]); break;
          case WTC_ACT_GELU: for (int u = 0; u < 8; ++u) g[u] *= act_slope<WTC_ACT_GELU>(z[u]); break;
          case WTC_ACT_GELU_TANH: for (int u = 0; u < 8; ++u) g[u] *= act_slope<WTC_ACT_GELU_TANH>(z[u]); break;
          case WTC_ACT_SILU: for (int u = 0; u < 8; ++u) g[u] *= act_slope<WTC_ACT_SILU>(z[u]); break;
        }
        if (p.dz) store8<DT>(p.dz, m * p.n + n, g);
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) sum[u] += g[u];
    }
  if (!p.dbias) return;
#pragma unroll
  for (int u = 0; u < 8; ++u) red[ty][tx * 8 + u] = sum[u];
  __syncthreads();
  const int64_t j = (int64_t)(blockIdx.x % cols) * 128 + threadIdx.x;
  if (threadIdx.x < 128 && j < p.n) {
    float s = 0.0f;
    for (int r = 0; r < 16; ++r) s += red[r][threadIdx.x];
    (p.chunks > 1 ? p.partial + chunk * p.n : p.dbias)[j] = s;
  }
}
__global__ void __launch_bounds__(256) sum_chunks_kernel(const ActBackwardParams p) {
  const int64_t j = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (j >= p.n) return;
  float s = 0.0f;
  for (int c = 0; c < p.chunks; c += 16) {  // 16 loads at a time, added in their order
    float x[16];
#pragma unroll
    for (int u = 0; u < 16; ++u) x[u] = c + u < p.chunks ? p.partial[(c + u) * p.n + j] : 0.0f;
#pragma unroll
    for (int u = 0; u < 16; ++u) s += x[u];
  }
  p.dbias[j] = s;
}

template <typename P> hipError_t run(const void* fn, int64_t grid, int threads, const P& p, hipStream_t stream) {
  P q = p;
  void* args[] = {&q};
  return hipLaunchKernel(fn, dim3((unsigned)grid), dim3(threads), args, 0, stream);
}

template <int DT, int OUT_DT, int TM, int TN, int S> const void* tile_by_kind(bool aks, bool bks) {
  if constexpr (TM > 64)
    if (aks) return (const void*)&matmul_tile_kernel<DT, DT, true, true, TM, TN, S>;  // db: out is of the input type
  return bks ? (const void*)&matmul_tile_kernel<DT, OUT_DT, false, true, TM, TN, S>
             : (const void*)&matmul_tile_kernel<DT, OUT_DT, false, false, TM, TN, S>;
}
template <int DT, int OUT_DT> const void* tile_by_size(int v, bool aks, bool bks) {
  switch (v) {
    case 0: return tile_by_kind<DT, OUT_DT, 256, 256, 4>(aks, bks);
    case 1: return tile_by_kind<DT, OUT_DT, 256, 128, 6>(aks, bks);
    case 2: return tile_by_kind<DT, OUT_DT, 128, 128, 4>(aks, bks);
  }
  return tile_by_kind<DT, OUT_DT, 64, 128, 6>(aks, bks);
}

// The tile kernels and what they take, in us (read off graph replays of 14 shapes
// from 8 x 4096 x 4096 to 8192 x 8192 x 4096, the three operand kinds, every
// tile with 1 to 16 splits): a slab of 32 k on a CU, more with every CU busy
// (the clock falls), and what a round of tiles costs besides.
//   256 x 256 is the fastest per product where its tiles fill the chip (8192 x
//   8192 x 4096: 465 us, 256 x 128 550, 128 x 128 580); 256 x 128 where those
//   are half of the chip (4096 x 2048 x 4096: 72, against 92 and 78); 128 x 128
//   for smaller products, one or two workgroups a CU (2048 x 2048 x 1024: 15,
//   against 30 and 21); 64 x 128 for few rows (8 x 4096 x 4096 in 8 splits:
//   11.2, 128 x 128 12.2).
struct Variant {
  int tm, tn;
  double slab_us, busy_us, fixed_us;
};
constexpr Variant kVariants[] = {{256, 256, 0.58, 0.34, 10.0}, {256, 128, 0.34, 0.19, 7.0}, {128, 128, 0.28, 0.0, 5.0}, {64, 128, 0.22, 0.0, 3.5}};
constexpr int kFewRows = 64;  // at most so many rows for the 64-row tile
constexpr int kRowsVariant = 4, kRowsMost = 16;  // matmul_rows_kernel

}  // namespace

// The tile and the number of k-splits with the least estimate.  Splits cost a second
// kernel (3.5 us) and their partial products' way to memory and back (6 TB/s).
MatmulPlan plan_matmul(int64_t m, int64_t n, int64_t k, bool aks, bool bks, int cu_count) {
  MatmulPlan best{};
  double best_us = 0;
  const int64_t slabs = (k + kSlabK - 1) / kSlabK;
  for (int v = 0; v < 4; ++v) {
    const Variant& t = kVariants[v];
    if (t.tm == 64 && (m > kFewRows || aks)) continue;
    const int64_t tiles = ((m + t.tm - 1) / t.tm) * ((n + t.tn - 1) / t.tn);
    for (int64_t s = 1; s <= 16 && (s == 1 || slabs / s >= 4); s *= 2) {
      const int64_t per = (slabs + s - 1) / s;
      const int64_t splits = per ? (slabs + per - 1) / per : 1;
      const int64_t groups = tiles * splits, full = groups / cu_count, rest = groups % cu_count;
      double us = t.fixed_us + (double)(full * per) * (t.slab_us + t.busy_us);
      if (rest) us += (double)per * (t.slab_us + t.busy_us * (double)rest / cu_count);
      if (splits > 1) us += 3.5 + 2.0 * (double)(splits * m * n) * 4 / 6.0e6;
      if (best_us == 0 || us < best_us) {
        best_us = us;
        best = MatmulPlan{v, (int)splits, (int)per, us};
      }
    }
  }
  // matmul_rows_kernel: a round of 16 columns a CU takes as long as k
  const double rows_us = 2.5 + (double)((n + 16 * cu_count - 1) / (16 * cu_count)) * (0.5 + 1.45e-3 * (double)k);
  if (!aks && !bks && m <= kRowsMost && rows_us < best_us) best = MatmulPlan{kRowsVariant, 1, 0, rows_us};
  return best;
}
// Both products of a backward pass as 128 x 128 tiles of one launch: the sum of their
// work over the chip, at least the longer one's tile; against one after the other
// with a launch (4 us) between.
bool pair_pays(const MatmulPlan& da, const MatmulPlan& db, int64_t m, int64_t n, int64_t k, int cu_count) {
  const Variant& t = kVariants[2];
  auto tiles = [](int64_t a, int64_t b) { return ((a + 127) / 128) * ((b + 127) / 128); };
  auto slabs = [](int64_t x) { return (x + kSlabK - 1) / kSlabK; };
  const double work = (double)(tiles(m, k) * slabs(n) + tiles(k, n) * slabs(m)) / cu_count;
  const double longest = (double)std::max(slabs(n), slabs(m));
  // (a CU takes whole tiles: on average half of one more than its share)
  return t.fixed_us + t.slab_us * (std::max(work, longest) + 0.5 * longest) < da.us + db.us + 4.0;
}
MatmulPlan pair_plan(int64_t k) { return MatmulPlan{2, 1, (int)((k + kSlabK - 1) / kSlabK), 0.0}; }
hipError_t launch_matmul_pair(const MatmulParams& da, const MatmulParams& db, int dt, bool bks, hipStream_t stream) {
  MatmulParams x = da, y = db;
  x.splits = y.splits = 1;
  x.slabs = (x.k + kSlabK - 1) / kSlabK;
  y.slabs = (y.k + kSlabK - 1) / kSlabK;
  auto tiles = [](const MatmulParams& p) { return (uint32_t)(((p.m + 127) / 128) * ((p.n + 127) / 128)); };
  uint32_t x_tiles = tiles(x), y_tiles = tiles(y);
  uint32_t x_from = x.slabs >= y.slabs ? 0 : y_tiles, y_from = x.slabs >= y.slabs ? x_tiles : 0;
  void* args[] = {&x, &y, &x_from, &x_tiles, &y_from};
  const void* fn = dt == DT_F16 ? (bks ? (const void*)&matmul_pair_kernel<DT_F16, true> : (const void*)&matmul_pair_kernel<DT_F16, false>)
                                : (bks ? (const void*)&matmul_pair_kernel<DT_BF16, true> : (const void*)&matmul_pair_kernel<DT_BF16, false>);
  return hipLaunchKernel(fn, dim3(x_tiles + y_tiles), dim3(kThreads), args, 0, stream);
}

void matmul_tile_size(const MatmulPlan& plan, int64_t* tile_m, int64_t* tile_n) {
  *tile_m = plan.variant == kRowsVariant ? kRowsMost : kVariants[plan.variant].tm;
  *tile_n = plan.variant == kRowsVariant ? 16 : kVariants[plan.variant].tn;
}

int64_t matmul_workspace(const MatmulPlan& plan, int64_t m, int64_t n) {
  return plan.splits > 1 ? plan.splits * m * n * 4 : 0;
}

hipError_t launch_matmul(const MatmulParams& params, const MatmulPlan& plan, int dt, int out_dt, bool aks, bool bks,
                         hipStream_t stream) {
  MatmulParams p = params;
  p.splits = plan.splits;
  p.slabs = plan.slabs;
  if (plan.variant == kRowsVariant) {
    const void* fn = dt == DT_F16 ? (out_dt == DT_F32 ? (const void*)&matmul_rows_kernel<DT_F16, DT_F32> : (const void*)&matmul_rows_kernel<DT_F16, DT_F16>)
                                  : (out_dt == DT_F32 ? (const void*)&matmul_rows_kernel<DT_BF16, DT_F32> : (const void*)&matmul_rows_kernel<DT_BF16, DT_BF16>);
    return run(fn, ((int64_t)p.n + 15) / 16, kRowsWaves * 64, p, stream);
  }
  const Variant& v = kVariants[plan.variant];
  const int64_t grid = ((int64_t)(p.m + v.tm - 1) / v.tm) * ((p.n + v.tn - 1) / v.tn) * p.splits;
  const bool f32 = out_dt == DT_F32;
  const void* fn = dt == DT_F16 ? (f32 ? tile_by_size<DT_F16, DT_F32>(plan.variant, aks, bks) : tile_by_size<DT_F16, DT_F16>(plan.variant, aks, bks))
                                : (f32 ? tile_by_size<DT_BF16, DT_F32>(plan.variant, aks, bks) : tile_by_size<DT_BF16, DT_BF16>(plan.variant, aks, bks));
  const hipError_t e = run(fn, grid, kThreads, p, stream);
  if (e != hipSuccess || p.splits == 1) return e;
  fn = dt == DT_F16 ? (f32 ? (const void*)&matmul_join_kernel<DT_F16, DT_F32> : (const void*)&matmul_join_kernel<DT_F16, DT_F16>)
                    : (f32 ? (const void*)&matmul_join_kernel<DT_BF16, DT_F32> : (const void*)&matmul_join_kernel<DT_BF16, DT_BF16>);
  return run(fn, ((int64_t)p.m * p.n / 8 + 255) / 256, 256, p, stream);
}

// Row chunks of the activation's gradient: enough workgroups to fill the chip, of at least 32 rows.
int64_t act_backward_chunk_rows(int64_t m, int64_t n, int cu_count) {
  const int64_t cols = (n + 127) / 128;
  const int64_t chunks = cols ? (4 * cu_count + cols - 1) / cols : 1;
  const int64_t rows = (m + chunks - 1) / chunks;
  return rows < 32 ? 32 : (rows + 15) / 16 * 16;
}

hipError_t launch_act_backward(const ActBackwardParams& p, int dt, hipStream_t stream) {
  const int64_t cols = (p.n + 127) / 128;
  const hipError_t e = run(dt == DT_F16 ? (const void*)&act_backward_kernel<DT_F16> : (const void*)&act_backward_kernel<DT_BF16>,
                           cols * p.chunks, 256, p, stream);
  if (e != hipSuccess || p.chunks == 1 || !p.dbias) return e;
  return run((const void*)&sum_chunks_kernel, (p.n + 255) / 256, 256, p, stream);
}

}  // namespace wtc
