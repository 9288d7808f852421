// window_attention.hip -- kernels of wtc_window_attention and its gradients.
#include "attention_common.h"
#include "layer_kernels.h"

#include <algorithm>

namespace wtc {
namespace {

using namespace attn;

// ---- forward -----------------------------------------------------------------
// A workgroup takes 256 / KG query rows of one sequence and key head.  The rows
// of the query heads that share the key head are packed (row r = query r / G,
// head r % G), so that a tile of keys serves all of them and the window's
// edges cost G times fewer tiles.  A wave owns 32 rows, one a lane pair:
//   S^T = K . Q^T   (32 x 32 subtiles; a lane holds 32 scores of one query)
//   online softmax  (in registers; the two lanes of a query share its maximum)
//   O^T += V^T . P^T (P^T straight from the registers, see col_frag)
// Keys come in tiles of 64 through a ring of (K, V) stages filled by
// direct-to-LDS loads; one barrier a tile.
// With one wave a SIMD a tile takes about 1.9 us whatever its loads do (deeper
// rings changed nothing): the chain from scores through maximum and exponentials
// to the values' product is serial.  So a SIMD always gets two waves: where 256
// rows a workgroup would leave CUs idle, KG = 2 gives each row to two waves that
// take every other tile and join their results through LDS at the end
// (128 tokens against 8192 keys, 32 / 8 heads of 128, window 4096: 39 -> 33 us).
// What it reaches: 4 x 4096 causal tokens, 32 / 8 heads of 128, bf16: 665 us, 829
// TFLOP/s of the pairs that see each other; 2 x 4096 with a window of 1024: 178 us,
// 680.  A large library product runs at 1270 on the same card.
constexpr int kKeys = 64;
// The running maximum is only moved when a score exceeds it by 2^8: the weights
// stay below 2^8, and the accumulators are rescaled a few times a row instead
// of once a tile.
constexpr float kSlack = 8.0f;

template <int ND, int KG> struct FwdLds {
  static constexpr int RB = row_bytes(ND), STAGES = KG == 2 ? 2 : 3;
  static constexpr int TILE = kKeys * RB, STAGE = KG * 2 * TILE;
  static constexpr int PITCH = ND * 64 + 16;    // bytes of a row staged for the output
  static constexpr int JPITCH = ND * 128 + 16;  // bytes of a row handed over (KG = 2), its maximum and sum in the last 16
  static constexpr int RING = STAGES * STAGE, OUT = 256 / KG * PITCH, JOIN = KG == 2 ? 128 * JPITCH : 0;
  static constexpr int MOST = RING > OUT ? RING : OUT;
  static constexpr int TOTAL = MOST > JOIN ? MOST : JOIN;
  static_assert(TOTAL <= 160 * 1024, "LDS");
};

template <int DT, int ND, int KG>
__global__ void __launch_bounds__(512, 2) attention_tile_kernel(const AttnParams p) {
  using L = FwdLds<ND, KG>;
  constexpr int RB = L::RB, NS = 2 * ND, ROWS = 256 / KG;
  __shared__ __attribute__((aligned(16))) uint8_t smem[L::TOTAL];
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int wave_id = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wave = wave_id % (8 / KG), group = wave_id / (8 / KG);  // rows, tiles
  const uint32_t id = xcd_remap(blockIdx.x, gridDim.x);
  const int split = (int)(id % p.splits);
  const uint32_t rest = id / p.splits;
  const int blk = p.row_blocks - 1 - (int)(rest % p.row_blocks);  // the longest rows first
  const int hk = (int)(rest / p.row_blocks % p.kv_heads), b = (int)(rest / p.row_blocks / p.kv_heads);
  const int nk = seq_keys(p, b), nq = seq_queries(p, b), shift = nk - nq;
  const int r0 = blk * ROWS;

  // this lane's row
  const int r = r0 + wave * 32 + (lane & 31), i = r / p.group, h = hk * p.group + r - i * p.group;
  const bool valid = i < nq;
  const int pos = valid ? i + shift : -1;

  // keys of the block: [0, s_end) and [lo, end)
  const int i_last = min((r0 + ROWS - 1) / p.group, nq - 1);
  const int p_lo = r0 / p.group + shift, p_hi = i_last + shift;
  const int lo = (int)max((int64_t)0, (int64_t)p_lo - p.window + 1);
  const int end = r0 / p.group < nq ? max(p_hi + 1, 0) : 0;
  const int s_end = end ? min(p.sinks, lo) : 0;
  const int t_sink = (s_end + kKeys - 1) / kKeys, t_all = end > lo ? t_sink + (end - lo + kKeys - 1) / kKeys : 0;
  const int t0 = (int)((int64_t)t_all * split / p.splits), t1 = (int)((int64_t)t_all * (split + 1) / p.splits);
  // the wave's positions: tiles that none of its rows sees are not computed
  const int w_lo = (r0 + wave * 32) / p.group + shift;
  const int w_hi = min((r0 + wave * 32 + 31) / p.group, nq - 1) + shift;
  const bool w_any = (r0 + wave * 32) / p.group < nq && w_hi >= 0;

  u32x4 qf[NS];
  load_row<NS>(p.q + 2 * (b * p.q_stride[0] + (int64_t)i * p.q_stride[1] + h * p.q_stride[2]), valid, p.dim, half, qf);
  const float c2 = positive_scale<NS>(p.scale, qf);

  f32x16 o[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int v = 0; v < 16; ++v) o[d][v] = 0.0f;
  float top = -INFINITY, total = 0.0f;  // log2 domain; total: this lane's half of the keys

  TileLoader<RB, kKeys, 8 / KG> lk, lv;
  lk.init(p.k + 2 * (b * p.k_stride[0] + hk * p.k_stride[2]), 2 * p.k_stride[1], p.dim, wave, lane);
  lv.init(p.v + 2 * (b * p.v_stride[0] + hk * p.v_stride[2]), 2 * p.v_stride[1], p.dim, wave, lane);
  constexpr int LOADS = 2 * TileLoader<RB, kKeys, 8 / KG>::NB;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(WTC_LDS uint8_t*)smem;
  auto tile_base = [&](int t) { return t < t_sink ? t * kKeys : lo + (t - t_sink) * kKeys; };
  auto tile_end = [&](int t) { return t < t_sink ? s_end : end; };
  // step x: tile t0 + x KG + group
  const int steps = (t1 - t0 + KG - 1) / KG;
  auto issue = [&](int x) {
    const int t = t0 + x * KG + group;
    const int j0 = tile_base(t), n = t < t1 ? min(kKeys, tile_end(t) - j0) : 0;
    const uint32_t st = lds0 + (uint32_t)x % L::STAGES * L::STAGE + group * 2 * L::TILE;
    lk.issue(st, j0, n);
    lv.issue(st + L::TILE, j0, n);
  };
#pragma unroll
  for (int x = 0; x < L::STAGES - 1; ++x) issue(x);

  landed(qf);
  const uint32_t k_at = row_addr<RB>(lane) + group * 2 * L::TILE, v_at = L::TILE + col_addr<RB>(lane) + group * 2 * L::TILE;
  for (int x = 0; x < steps; ++x) {
    wait_loads_barrier<LOADS*(L::STAGES - 2)>();  // the step's tiles landed; every wave is done with the last one's
    issue(x + L::STAGES - 1);
    const int t = t0 + x * KG + group;
    const int j0 = tile_base(t), j1 = tile_end(t);
    // (in the window's part the first tokens may lie below the window too)
    const bool below = t >= t_sink && (int64_t)j0 + kKeys - 1 + p.window <= w_lo && j0 >= p.sinks;
    if (t >= t1 || !w_any || j0 > w_hi || below) continue;
    const uint32_t stage = (uint32_t)x % L::STAGES * L::STAGE;
    uint32_t ka = k_at + stage, va = v_at + stage;
    fresh(ka);
    fresh(va);

    f32x16 s[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int v = 0; v < 16; ++v) s[u][v] = 0.0f;
#pragma unroll
      for (int st = 0; st < NS; ++st) s[u] = mfma32<DT>(row_frag<RB>(smem, ka, 32 * u, st), qf[st], s[u]);
    }
    __builtin_amdgcn_sched_group_barrier(0x100, 5, 0);
#pragma unroll
    for (int x = 0; x < 2 * NS - 5; ++x) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
    if (j0 + kKeys > j1 || j0 + kKeys - 1 > w_lo || (t >= t_sink && (int64_t)j0 + p.window <= w_hi)) {
      const uint64_t seen = seen_bits(j0 + 4 * half, j1, pos, p.window, p.sinks);
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int v = 0; v < 16; ++v) s[u][v] = keep_bit(s[u][v], seen, 32 * u + 8 * (v >> 2) + (v & 3));
    }
    float m = fmaxf(s[0][0], s[1][0]);
#pragma unroll
    for (int v = 1; v < 16; ++v) m = fmaxf(m, fmaxf(s[0][v], s[1][v]));
    m = xor32_max(m) * c2;
    if (__any(m > top + kSlack || (top == -INFINITY && m > top))) {
      const float next = fmaxf(top, m);
      const float keep = next == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(top - next);
      top = next;
      total *= keep;
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int v = 0; v < 16; ++v) o[d][v] *= keep;
    }
    const float ref = top == -INFINITY ? 0.0f : -top;
    u32x4 pf[4];
    float sum[2] = {0.0f, 0.0f};
    auto weights = [&](int u) {
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        f32x4 e;
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          e[v] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][4 * g + v], c2, ref));
          sum[v & 1] += e[v];
        }
        uint32_t w0, w1;
        pack4<DT>(e, &w0, &w1);
        pf[2 * u + (g >> 1)][2 * (g & 1)] = w0;
        pf[2 * u + (g >> 1)][2 * (g & 1) + 1] = w1;
      }
    };
    auto values = [&](int u) {
#pragma unroll
      for (int st = 2 * u; st < 2 * u + 2; ++st)
#pragma unroll
        for (int d = 0; d < ND; ++d) o[d] = mfma32<DT>(col_frag<RB>(smem, va, 16 * st, d), pf[st], o[d]);
    };
    weights(0);
    __builtin_amdgcn_sched_barrier(0);
    // the second half's exponentials among the first half's products
    values(0);
    weights(1);
    values(1);
    // reads run four fragments ahead of the products that take them
    __builtin_amdgcn_sched_group_barrier(0x100, 8, 0);
#pragma unroll
    for (int x = 0; x < 2 * ND; ++x) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // a product
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);  // a fragment's reads
      __builtin_amdgcn_sched_group_barrier(0x002, 9, 0);  // vector work
    }
#pragma unroll
    for (int x = 0; x < 2 * ND - 4; ++x) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
    total += sum[0] + sum[1];
  }
  wait_loads_barrier<0>();

  // ---- the rows' results
  // (a row behind the end took part in tiles that needed no mask)
  total = valid ? xor32_sum(total) : 0.0f;
  if constexpr (KG == 2) {
    uint8_t* at = smem + (wave * 32 + (lane & 31)) * L::JPITCH + half * 16;
    float2* stat = reinterpret_cast<float2*>(smem + (wave * 32 + (lane & 31)) * L::JPITCH + ND * 128);
    if (group) {
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<f32x4*>(at + (32 * d + 8 * g) * 4) = f32x4{o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]};
      if (half == 0) *stat = float2{top, total};
    }
    __syncthreads();
    if (group) return;
    const float2 other = *stat;
    const float next = fmaxf(top, other.x), base = next == -INFINITY ? 0.0f : next;
    const float f = __builtin_amdgcn_exp2f(top - base), g2 = __builtin_amdgcn_exp2f(other.x - base);
    total = total * f + other.y * g2;
    top = next;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 y = *reinterpret_cast<const f32x4*>(at + (32 * d + 8 * g) * 4);
#pragma unroll
        for (int v = 0; v < 4; ++v) o[d][4 * g + v] = o[d][4 * g + v] * f + y[v] * g2;
      }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
  const float inv = total == 0.0f ? 0.0f : 1.0f / total;
  const float lse = (top + __builtin_amdgcn_logf(total)) * kLn2;  // (v_log_f32: log2)
  if (p.slots) {
    const int64_t row = (((int64_t)b * p.lq + i) * p.heads + h) * p.slots + p.slot0 + split;
    if (valid) {
      if (half == 0) p.part_lse[row] = total == 0.0f ? -INFINITY : top + __builtin_amdgcn_logf(total);
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int c = 32 * d + 8 * g + 4 * half;
          if (c < p.dim)
            *reinterpret_cast<f32x4*>(p.part_out + row * p.dim + c) =
                f32x4{o[d][4 * g] * inv, o[d][4 * g + 1] * inv, o[d][4 * g + 2] * inv, o[d][4 * g + 3] * inv};
        }
    }
    return;
  }
  bool nan = false;
  // (with KG = 2 inside the rows that this wave alone has read)
  uint8_t* stg = smem + wave * 32 * (KG == 2 ? L::JPITCH : L::PITCH);
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      f32x4 x;
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        x[v] = valid ? o[d][4 * g + v] * inv : 0.0f;
        nan |= x[v] != x[v];
      }
      uint32_t w0, w1;
      pack4<DT>(x, &w0, &w1);
      *reinterpret_cast<u32x2*>(stg + (lane & 31) * L::PITCH + (32 * d + 8 * g + 4 * half) * 2) = u32x2{w0, w1};
    }
  if (p.lse && half == 0 && i < p.lq) p.lse[((int64_t)b * p.heads + h) * p.lq + i] = total == 0.0f ? -INFINITY : lse;
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  constexpr int CPR = ND * 4;  // chunks a row
#pragma unroll 4
  for (int x = lane; x < 32 * CPR; x += 64) {
    const int row = x / CPR, c = x % CPR;
    const int rr = r0 + wave * 32 + row, ii = rr / p.group, hh = hk * p.group + rr - ii * p.group;
    if (ii < p.lq && c * 8 < p.dim)
      *reinterpret_cast<u32x4*>(p.out + 2 * (b * p.o_stride[0] + (int64_t)ii * p.o_stride[1] + hh * p.o_stride[2]) + c * 16) =
          *reinterpret_cast<const u32x4*>(stg + row * L::PITCH + c * 16);
  }
  uint32_t redo = (uint32_t)(__ballot(nan && valid) | __ballot(nan && valid) >> 32);
  if (redo) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the rows are read back
  while (redo) {
    const int rr = r0 + wave * 32 + __builtin_ctz(redo);
    attention_row<DT, false, false>(p, b, hk * p.group + rr % p.group, rr / p.group);
    redo &= redo - 1;
  }
}

// Joins the splits of a row: half a wave a row.
template <int DT, bool FULL, bool PREFIX>
__global__ void __launch_bounds__(256) attention_join_kernel(const AttnParams p) {
  const int lane = threadIdx.x & 63, c = (lane & 31) * 4;
  const int64_t rows = (int64_t)p.batch * p.lq * p.heads, at = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int64_t row = min(at, rows - 1);
  const int h = (int)(row % p.heads), i = (int)(row / p.heads % p.lq), b = (int)(row / p.heads / p.lq);
  const bool valid = i < seq_queries(p, b);  // rows behind the end were not written
  bool nan = false;
  if (c < p.dim) {
    f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
    float lse = -INFINITY;
    if (valid) lse = join_splits(p.part_out + row * p.slots * p.dim, p.part_lse + row * p.slots, p.slots, p.dim, c, &x);
#pragma unroll
    for (int v = 0; v < 4; ++v) nan |= x[v] != x[v];
    if (at < rows) {
      uint32_t w0, w1;
      pack4<DT>(x, &w0, &w1);
      *reinterpret_cast<u32x2*>(p.out + 2 * (b * p.o_stride[0] + (int64_t)i * p.o_stride[1] + h * p.o_stride[2] + c)) = u32x2{w0, w1};
      if (p.lse && c == 0) p.lse[((int64_t)b * p.heads + h) * p.lq + i] = lse * kLn2;
    }
  }
  const uint64_t redo = __ballot(nan && at < rows);
  if (redo) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  for (int half = 0; half < 2; ++half) {
    const int64_t r = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 6) * 2 + half;
    if (redo >> (32 * half) & 0xFFFFFFFFu) attention_row<DT, FULL, PREFIX>(p, (int)(r / p.heads / p.lq), (int)(r % p.heads), (int)(r / p.heads % p.lq));
  }
}

// ---- gradients ------------------------------------------------------------------
// With P = exp(S - lse), D = sum_d dout out and dS = P (dP - D), dP = dout . V^T:
//   dq = scale dS . K      per row block, keys streamed   (attention_dq_kernel)
//   dv = P^T . dout, dk = scale dS^T . Q
//                          per key block, queries streamed (attention_dkv_kernel)
// Two kernels, each recomputing S and dP (7 products instead of 5): no dq sums
// through atomics, whose order would change the result, and no f32 dq in memory.
// The first writes each row's lse (in the log2 domain) and -D as p.row_lse and
// p.row_delta, rows packed as the tiles are: [batch][kv_heads][lq][G].
__device__ inline int64_t stats_row(const AttnParams& p, int b, int hk, int i) {
  return (((int64_t)b * p.kv_heads + hk) * p.lq + i) * p.group;
}

// float16 holds 2^-24 to 2^16, 2^-14 with all its bits.  Weights of 1 / keys, and a dS that
// goes with the gradient's size (loss-scaled ones pass 2^16 where dq and dk do not, small
// ones vanish), do not fit that range as they are.
// P: dk / dv works with P times 2^kWeightBits (row_lse is stored less by that).
template <int DT> constexpr int kWeightBits = DT == DT_F16 ? 14 : 0;
__device__ inline float power_of_2(int e) { return __builtin_amdgcn_ldexpf(1.0f, e); }
// dS: taken times 2^ex, ex of each row (dq) or key (dk) its own.  It starts higher than any
// use, short of where f32 would overflow, and is lowered, together with the sums so
// far, when a value reaches 2^15, to put that value at 2^12 or more.  What a lane packs is
// then off by 2^-11 of itself or 2^-37 of the largest so far (where none has reached 2^12,
// in dq, 2^-55 of the row's largest dout).  The factor and the test
// cost f16 2 to 5 % (forward and gradients, 4096 causal tokens, 32 / 8 heads of 128: 922 ->
// 937 us; 4 x 2048, 16 heads of 64: 329 -> 345).  bf16 has f32's range.
template <int DT> struct DsRange {
  int ex;
  // Two fragments of `ds`, which is times 2^ex already; the largest magnitude.
  __device__ inline float pack(const f32x16& ds, u32x4 (&df)[2]) const {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      uint32_t w0, w1;
      pack4<DT>(f32x4{ds[4 * q], ds[4 * q + 1], ds[4 * q + 2], ds[4 * q + 3]}, &w0, &w1);
      df[q >> 1][2 * (q & 1)] = w0;
      df[q >> 1][2 * (q & 1) + 1] = w1;
    }
    float m = 0.0f;
    if constexpr (DT == DT_F16) {
#pragma unroll
      for (int v = 0; v < 16; ++v) m = fmaxf(m, fabsf(ds[v]));
    }
    return m;
  }
  // Where that is too large: ex moves, `sums` follow, the fragments are packed again.
  template <int ND> __device__ inline void fit(float m, f32x16& ds, f32x16 (&sums)[ND], u32x4 (&df)[2]) {
    if constexpr (DT == DT_F16) {
      if (!__any(m >= 32768.0f)) return;
      m = xor32_max(m);
      const int by = m >= 32768.0f ? min(0, 13 - __builtin_amdgcn_frexp_expf(m)) : 0;  // (0 for an infinity)
      const float keep = power_of_2(by);
      ex += by;
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int v = 0; v < 16; ++v) sums[d][v] *= keep;
#pragma unroll
      for (int v = 0; v < 16; ++v) ds[v] *= keep;
      pack(ds, df);
    }
  }
  // sums without 2^(ex + bits)
  template <int ND> __device__ inline void undo(f32x16 (&sums)[ND], int bits) const {
    if constexpr (DT == DT_F16) {
      const float by = power_of_2(-ex - bits);
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int v = 0; v < 16; ++v) sums[d][v] *= by;
    }
  }
};

template <int DT, bool FULL> __device__ inline void dq_row(const AttnParams& p, int b, int h, int i) {
  using T = typename Elem<DT>::type;
  const int lane = threadIdx.x & 63;
  const T* q = (const T*)p.q + b * p.q_stride[0] + i * p.q_stride[1] + h * p.q_stride[2];
  const T* k = (const T*)p.k + b * p.k_stride[0] + h / p.group * p.k_stride[2];
  const T* v = (const T*)p.v + b * p.v_stride[0] + h / p.group * p.v_stride[2];
  const T* g = (const T*)p.dout + b * p.do_stride[0] + i * p.do_stride[1] + h * p.do_stride[2];
  const T* o = (const T*)p.o + b * p.o_stride[0] + i * p.o_stride[1] + h * p.o_stride[2];
  const float delta = dot_rows<DT>(g, o, p.dim);
  const float lse = p.lse_in[((int64_t)b * p.heads + h) * p.lq + i];
  const Seen seen(p.window, p.sinks, last_seen<FULL>(p, b, i));
  Redo<DT> dq(p.dq, (((int64_t)b * p.lq + i) * p.heads + h) * p.dim, p.dim, lane);
  for (int t0 = 0; t0 < seen.count && !dq.settled(); t0 += 64) {
    float ds = 0.0f;
    if (t0 + lane < seen.count) {
      const int j = seen.key(t0 + lane);
      const float w = __expf(p.scale * dot_rows<DT>(q, k + j * p.k_stride[1], p.dim) - lse);
      ds = p.scale * w * (dot_rows<DT>(g, v + j * p.v_stride[1], p.dim) - delta);
    }
    for (int t = 0; t < min(64, seen.count - t0); ++t) dq.add(__shfl(ds, t), k + seen.key(t0 + t) * p.k_stride[1], lane);
  }
  dq.store(1.0f, lane);
}

// dk and dv of one key.
template <int DT, bool FULL> __device__ inline void dkv_row(const AttnParams& p, int b, int hk, int j) {
  using T = typename Elem<DT>::type;
  const int lane = threadIdx.x & 63;
  const int nq = seq_queries(p, b), shift = seq_keys(p, b) - (FULL ? 1 : nq);
  const T* k = (const T*)p.k + b * p.k_stride[0] + j * p.k_stride[1] + hk * p.k_stride[2];
  const T* v = (const T*)p.v + b * p.v_stride[0] + j * p.v_stride[1] + hk * p.v_stride[2];
  // queries of positions j .. j + window - 1 (a first token: all from j on)
  const int i0 = max(0, j - shift);
  const int i1 = j < p.sinks ? nq : (int)min((int64_t)nq, j + p.window - shift);
  const float c2 = p.scale * kLog2e;
  const int64_t at = (((int64_t)b * p.lk + j) * p.kv_heads + hk) * p.dim;
  Redo<DT> dk(p.dk, at, p.dim, lane), dv(p.dv, at, p.dim, lane);
  for (int x = 0; x < p.group; ++x) {
    const int h = hk * p.group + x;
    const T* q = (const T*)p.q + b * p.q_stride[0] + h * p.q_stride[2];
    const T* g = (const T*)p.dout + b * p.do_stride[0] + h * p.do_stride[2];
    for (int t0 = i0; t0 < i1 && !(dk.settled() && dv.settled()); t0 += 64) {
      float w = 0.0f, ds = 0.0f;
      const int i = t0 + lane;
      if (i < i1) {
        const int64_t row = stats_row(p, b, hk, i) + x;
        w = __builtin_amdgcn_exp2f(c2 * dot_rows<DT>(q + i * p.q_stride[1], k, p.dim) - (p.row_lse[row] + kWeightBits<DT>));
        ds = p.scale * w * (dot_rows<DT>(g + i * p.do_stride[1], v, p.dim) + p.row_delta[row]);
      }
      for (int t = 0; t < min(64, i1 - t0); ++t) {
        dv.add(__shfl(w, t), g + (t0 + t) * p.do_stride[1], lane);
        dk.add(__shfl(ds, t), q + (t0 + t) * p.q_stride[1], lane);
      }
    }
  }
  dk.store(1.0f, lane);
  dv.store(1.0f, lane);
}

// Row blocks and key tiles as in attention_tile_kernel; keys in subtiles of 32:
//   S^T = K . Q^T, dP^T = V . dout^T, dq^T += K^T . dS^T
// 128 rows a workgroup: 4 waves, two workgroups a CU at dim 128, or with KG = 2 eight
// waves that take every other tile for a row (where the grid leaves each workgroup
// a CU of its own: 3 x 1000 causal tokens, 6 / 3 heads of 80: 36 -> 27 us).
constexpr int kDqRows = 128;
template <int ND, int KG> struct DqLds {
  static constexpr int RB = row_bytes(ND), STAGES = 2;
  static constexpr int TILE = kKeys * RB, STAGE = KG * 2 * TILE;
  static constexpr int PITCH = ND * 64 + 16, JPITCH = ND * 128 + 16;
  static constexpr int RING = STAGES * STAGE, OUT = kDqRows * (KG == 2 ? JPITCH : PITCH);
  static constexpr int TOTAL = RING > OUT ? RING : OUT;
  static_assert(TOTAL <= 160 * 1024, "LDS");
};
// What becomes of the rows' statistics: taken and written for dk / dv; no more than that, for
// sequences of few keys (FULL); or taken as they were written before.
enum class Rows { ALL, STATS, GIVEN };
constexpr int kFewTiles = 2;
__host__ __device__ inline bool few_keys(int nk) { return nk > 0 && nk <= kFewTiles * kKeys; }
// FULL: every query sees every key.
template <int DT, int ND, int KG, Rows ROWS, bool FULL>
__device__ inline void attention_dq(const AttnParams& p, uint8_t* smem, uint32_t id) {
  using L = DqLds<ND, KG>;
  constexpr int NW = 4;
  constexpr int RB = L::RB, NS = 2 * ND;
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int wave_id = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wave = wave_id % 4, group = wave_id / 4;  // rows, tiles
  const int blk = p.row_blocks - 1 - (int)(id % p.row_blocks);
  const int hk = (int)(id / p.row_blocks % p.kv_heads), b = (int)(id / p.row_blocks / p.kv_heads);
  const int nk = seq_keys(p, b), nq = seq_queries(p, b), shift = FULL ? nk - 1 : nk - nq;
  const int r0 = blk * NW * 32;
  const int r = r0 + wave * 32 + (lane & 31), i = r / p.group, x_head = r - i * p.group, h = hk * p.group + x_head;
  const bool valid = i < nq;
  const int pos = valid ? i + shift : -1;
  const int i_last = min((r0 + NW * 32 - 1) / p.group, nq - 1);
  const int p_lo = r0 / p.group + shift, p_hi = i_last + shift;
  const int lo = FULL ? 0 : (int)max((int64_t)0, (int64_t)p_lo - p.window + 1);
  const int end = r0 / p.group < nq ? min(max(p_hi + 1, 0), nk) : 0;
  const int s_end = !FULL && end ? min(p.sinks, lo) : 0;
  const int t_sink = (s_end + kKeys - 1) / kKeys, t_all = end > lo ? t_sink + (end - lo + kKeys - 1) / kKeys : 0;
  const int w_lo = (r0 + wave * 32) / p.group + shift;
  const int w_hi = min((r0 + wave * 32 + 31) / p.group, nq - 1) + shift;
  const bool w_any = (r0 + wave * 32) / p.group < nq && w_hi >= 0;
  if (ROWS == Rows::STATS && (!end || !few_keys(nk))) return;

  u32x4 qf[NS], gf[NS];
  load_row<NS>(p.q + 2 * (b * p.q_stride[0] + (int64_t)i * p.q_stride[1] + h * p.q_stride[2]), valid, p.dim, half, qf);
  load_row<NS>(p.dout + 2 * (b * p.do_stride[0] + (int64_t)i * p.do_stride[1] + h * p.do_stride[2]), valid, p.dim, half, gf);
  float delta = 0.0f, lse2 = INFINITY;  // no keys: every weight 0
  if constexpr (ROWS != Rows::GIVEN) {
    const uint8_t* orow = p.o + 2 * (b * p.o_stride[0] + (int64_t)i * p.o_stride[1] + h * p.o_stride[2]);
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      const int c = 2 * s + half;
      if (valid && c * 8 < p.dim) {
        const auto ov = *reinterpret_cast<const typename Elem<DT>::vec8*>(orow + c * 16);
        const auto gv = __builtin_bit_cast(typename Elem<DT>::vec8, gf[s]);
#pragma unroll
        for (int v = 0; v < 8; ++v) delta = __builtin_fmaf((float)gv[v], (float)ov[v], delta);
      }
    }
    delta = xor32_sum(delta);
  } else if (valid) {
    delta = -p.row_delta[stats_row(p, b, hk, i) + x_head];
  }
  if (valid) {
    const float lse = p.lse_in[((int64_t)b * p.heads + h) * p.lq + i];
    if (lse == -INFINITY) delta = 0.0f;
    else lse2 = lse * kLog2e;
  }
  const float c2 = positive_scale<NS>(p.scale, qf);
  // |P (dP - D)| is at most 2 dim max|dout| max|v|, 2^24 max|dout| for any f16 v
  DsRange<DT> range{0};
  if constexpr (DT == DT_F16) {
    float m = 0.0f;
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      const auto gv = __builtin_bit_cast(typename Elem<DT>::vec8, gf[s]);
#pragma unroll
      for (int v = 0; v < 8; ++v) m = fmaxf(m, fabsf((float)gv[v]));
    }
    range.ex = 30 - __builtin_amdgcn_frexp_expf(xor32_max(m));
  }
  float weight_off = -lse2;  // of the exponents

  TileLoader<RB, kKeys, NW> lk, lv;
  lk.init(p.k + 2 * (b * p.k_stride[0] + hk * p.k_stride[2]), 2 * p.k_stride[1], p.dim, wave, lane);
  lv.init(p.v + 2 * (b * p.v_stride[0] + hk * p.v_stride[2]), 2 * p.v_stride[1], p.dim, wave, lane);
  constexpr int LOADS = 2 * TileLoader<RB, kKeys, NW>::NB;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(WTC_LDS uint8_t*)smem;
  auto tile_base = [&](int t) { return t < t_sink ? t * kKeys : lo + (t - t_sink) * kKeys; };
  auto tile_end = [&](int t) { return t < t_sink ? s_end : end; };
  // step x: tile x KG + group
  const int steps = (t_all + KG - 1) / KG;
  auto issue = [&](int x) {
    const int t = x * KG + group;
    const int j0 = tile_base(t), n = t < t_all ? min(kKeys, tile_end(t) - j0) : 0;
    const uint32_t st = lds0 + (uint32_t)x % L::STAGES * L::STAGE + group * 2 * L::TILE;
    lk.issue(st, j0, n);
    lv.issue(st + L::TILE, j0, n);
  };
  const uint32_t k_at = row_addr<RB>(lane) + group * 2 * L::TILE, kc_at = col_addr<RB>(lane) + group * 2 * L::TILE;
  // Weights s (times 2^(weight_off + lse2)) and dP g of subtile u of step x; false: none of the wave's rows sees it.
  auto weights = [&](int x, int u, uint32_t ka, f32x16& s, f32x16& g) {
    const int t = x * KG + group;
    const int j0 = tile_base(t), j1 = tile_end(t);
    const int k0 = j0 + 32 * u;
    const bool below = !FULL && t >= t_sink && (int64_t)k0 + 31 + p.window <= w_lo && k0 >= p.sinks;
    if (t >= t_all || !w_any || (!FULL && k0 > w_hi) || k0 >= j1 || below) return false;
#pragma unroll
    for (int v = 0; v < 16; ++v) s[v] = g[v] = 0.0f;
#pragma unroll
    for (int st = 0; st < NS; ++st) s = mfma32<DT>(row_frag<RB>(smem, ka, 32 * u, st), qf[st], s);
    if (k0 + 32 > j1 || (!FULL && (k0 + 31 > w_lo || (t >= t_sink && (int64_t)k0 + p.window <= w_hi)))) {
      const uint64_t seen = FULL ? bits_below(j1 - k0 - 4 * half) : seen_bits(k0 + 4 * half, j1, pos, p.window, p.sinks);
#pragma unroll
      for (int v = 0; v < 16; ++v) s[v] = keep_bit(s[v], seen, 8 * (v >> 2) + (v & 3));
    }
    __builtin_amdgcn_sched_barrier(0);
    // the exponentials among the products of dP
#pragma unroll
    for (int st = 0; st < NS; ++st) g = mfma32<DT>(row_frag<RB>(smem, ka, 32 * u + kKeys, st), gf[st], g);
#pragma unroll
    for (int v = 0; v < 16; ++v) s[v] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[v], c2, weight_off));
    __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
#pragma unroll
    for (int x = 0; x < NS; ++x) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x002, 32 / NS, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
    return true;
  };
  auto weights_at = [&](int x) {
    uint32_t ka = k_at + (uint32_t)x % L::STAGES * L::STAGE;
    fresh(ka);
    return ka;
  };

  // D from the rounded `out` is off by that rounding times |dout|, which shows where
  // weights are large: in rows of few keys.  Blocks of at most kFewTiles tiles sum it
  // themselves first, D = sum_j P dP (dq of causal rows in f16 1.48 -> 1.42
  // roundings off 64 bits; the D of later rows changes nothing there).
  if (ROWS != Rows::GIVEN && t_all <= kFewTiles) {
#pragma unroll
    for (int x = 0; x < L::STAGES - 1; ++x) issue(x);
    float sum = 0.0f;
    for (int x = 0; x < steps; ++x) {
      wait_loads_barrier<LOADS*(L::STAGES - 2)>();
      issue(x + L::STAGES - 1);
#pragma unroll 1
      for (int u = 0; u < 2; ++u) {
        f32x16 s, g;
        if (!weights(x, u, weights_at(x), s, g)) continue;
#pragma unroll
        for (int v = 0; v < 16; ++v) sum += s[v] == 0.0f ? 0.0f : s[v] * g[v];  // (a hidden key's dP may be anything)
      }
    }
    wait_loads_barrier<0>();
    sum = xor32_sum(sum);
    if constexpr (KG == 2) {  // the other group's tiles
      float* part = reinterpret_cast<float*>(smem);
      if (half == 0) part[wave_id * 32 + (lane & 31)] = sum;
      __syncthreads();
      sum = part[wave * 32 + (lane & 31)] + part[(4 + wave) * 32 + (lane & 31)];
      __syncthreads();
    }
    delta = delta != delta ? delta : sum;  // (a NaN value that is seen, be its weight 0, is in out)
  }
  if (ROWS != Rows::GIVEN && half == 0 && group == 0 && i < (ROWS == Rows::STATS ? nq : p.lq)) {
    p.row_lse[stats_row(p, b, hk, i) + x_head] = lse2 - kWeightBits<DT>;
    p.row_delta[stats_row(p, b, hk, i) + x_head] = -delta;
  }
  if constexpr (ROWS == Rows::STATS) return;

  landed(qf);
  landed(gf);
  f32x16 dq[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int v = 0; v < 16; ++v) dq[d][v] = 0.0f;

#pragma unroll
  for (int x = 0; x < L::STAGES - 1; ++x) issue(x);
  for (int x = 0; x < steps; ++x) {
    wait_loads_barrier<LOADS*(L::STAGES - 2)>();
    issue(x + L::STAGES - 1);
    uint32_t kc = kc_at + (uint32_t)x % L::STAGES * L::STAGE;
    fresh(kc);
    const uint32_t ka = weights_at(x);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      f32x16 s, g;
      weight_off = (float)range.ex - lse2;
      if (!weights(x, u, ka, s, g)) continue;
      u32x4 df[2];
#pragma unroll
      for (int v = 0; v < 16; ++v) s[v] *= g[v] - delta;
      range.fit(range.pack(s, df), s, dq, df);
#pragma unroll
      for (int st = 0; st < 2; ++st)
#pragma unroll
        for (int d = 0; d < ND; ++d) dq[d] = mfma32<DT>(col_frag<RB>(smem, kc, 32 * u + 16 * st, d), df[st], dq[d]);
    }
  }
  wait_loads_barrier<0>();
  range.undo(dq, 0);
  if constexpr (KG == 2) {
    uint8_t* at = smem + (wave * 32 + (lane & 31)) * L::JPITCH + half * 16;
    if (group) {
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<f32x4*>(at + (32 * d + 8 * g) * 4) = f32x4{dq[d][4 * g], dq[d][4 * g + 1], dq[d][4 * g + 2], dq[d][4 * g + 3]};
    }
    __syncthreads();
    if (group) return;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 y = *reinterpret_cast<const f32x4*>(at + (32 * d + 8 * g) * 4);
#pragma unroll
        for (int v = 0; v < 4; ++v) dq[d][4 * g + v] += y[v];
      }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }

  bool nan = false;
  uint8_t* stg = smem + wave * 32 * (KG == 2 ? L::JPITCH : L::PITCH);
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      f32x4 y;
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        y[v] = valid ? dq[d][4 * g + v] * p.scale : 0.0f;
        nan |= y[v] != y[v];
      }
      uint32_t w0, w1;
      pack4<DT>(y, &w0, &w1);
      *reinterpret_cast<u32x2*>(stg + (lane & 31) * L::PITCH + (32 * d + 8 * g + 4 * half) * 2) = u32x2{w0, w1};
    }
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  constexpr int CPR = ND * 4;
#pragma unroll 4
  for (int y = lane; y < 32 * CPR; y += 64) {
    const int row = y / CPR, c = y % CPR;
    const int rr = r0 + wave * 32 + row, ii = rr / p.group, hh = hk * p.group + rr - ii * p.group;
    if (ii < p.lq && c * 8 < p.dim)
      *reinterpret_cast<u32x4*>(p.dq + 2 * ((((int64_t)b * p.lq + ii) * p.heads + hh) * p.dim) + c * 16) =
          *reinterpret_cast<const u32x4*>(stg + row * L::PITCH + c * 16);
  }
  uint32_t redo = (uint32_t)(__ballot(nan && valid) | __ballot(nan && valid) >> 32);
  if (redo) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  while (redo) {
    const int rr = r0 + wave * 32 + __builtin_ctz(redo);
    dq_row<DT, FULL>(p, b, hk * p.group + rr % p.group, rr / p.group);
    redo &= redo - 1;
  }
}
template <int DT, int ND, int KG, bool FULL>
__global__ void __launch_bounds__(KG * 256, 2) attention_dq_kernel(const AttnParams p) {
  __shared__ __attribute__((aligned(256))) uint8_t smem[DqLds<ND, KG>::TOTAL];
  attention_dq<DT, ND, KG, Rows::ALL, FULL>(p, smem, xcd_remap(blockIdx.x, gridDim.x));
}

// A workgroup takes kDkvKeys keys of one (sequence, key head) and streams the
// queries that see them in tiles of 64 packed rows: whole positions of up to 64
// query heads of the group, so that a lane's offset inside a tile is the same
// for every tile.  Wave w holds the K and V fragments of keys 32 (w % 4) .. + 31
// in registers and takes the tile's rows 32 (w / 4) .. + 31, so that a SIMD has
// two waves (one computes weights while the other's products run) and the key
// block stays at 128:
//   S = Q . K^T, dP = dout . V^T (a lane holds 16 queries of one key)
//   dV^T += dout^T . P, dK^T += Q^T . dS
// At the end the two waves of a key join their sums through LDS, one of them dk,
// the other dv.
// The first tokens are seen by every later query, more queries than see any other
// key.  A workgroup of their key block takes, like the others, the queries whose
// window reaches the block; the far queries go in p.far_chunks short chunks to
// workgroups of their own behind the key blocks.  All sums of the first tokens go
// to p.part_far in f32, and attention_sum_kernel adds them in order.  (In chunks as
// long as a block's near queries they made 280 equal workgroups on 256 CUs for
// 4096 tokens, 8 key heads, window 1024, 4 first tokens, a second round: 240 us
// against 210.)
// Where the key blocks alone leave CUs idle, the near queries go in p.near_chunks
// parts as well, and every key's sums that way (3 x 1000 causal tokens, 6 / 3 heads
// of 80: 65 -> 40 us, and 6 for the sums).
// Both kernels on 4 x 4096 causal tokens, 32 / 8 heads of 128: 1993 us, 690 TFLOP/s by
// the usual count of 5 products and 966 by the 7 that they run (f16, see DsRange: 2153).
constexpr int kDkvWaves = 8;
constexpr int kDkvKeys = 128;
constexpr int kQueries = 64;
// Rows of a tile where every query sees every key (FULL): twice as many while LDS holds them, so
// that a wave does two blocks a barrier (4 x 1024 on 1500 states, 16 heads of 64: 83 -> 77 us).
constexpr int tile_queries(int nd, bool full) { return full && nd <= 2 ? 2 * kQueries : kQueries; }

template <int ND, bool FULL> struct DkvLds {
  static constexpr int RB = row_bytes(ND), STAGES = 2;
  static constexpr int Q = tile_queries(ND, FULL), TILE = Q * RB, STATS = 2 * TILE, STAGE = 2 * TILE + 2048;
  // At dim 128 the registers do not hold all of K's and V's fragments beside the
  // sums (a spilled one is loaded through vmcnt, behind the next tile's loads):
  // the last KEPT of the k-steps of V are read from LDS, 1 KiB a wave and step.
  static constexpr int KEPT = ND == 4 ? 6 : 0, KEPT_AT = STAGES * STAGE;
  static constexpr int PITCH = ND * 128 + 16;  // bytes of a key's sums
  static constexpr int RING = KEPT_AT + 4 * KEPT * 1024, OUT = kDkvWaves * 32 * PITCH;
  static constexpr int TOTAL = (RING > OUT ? RING : OUT) + kDkvWaves * 4;
  static_assert(TOTAL <= 160 * 1024, "LDS");
};

// Sums of a part, [dk, dv][dim] of a key: part_near [batch][kv_heads][near_blocks]
// [near_chunks][kDkvKeys], part_far [batch][kv_heads][far_blocks][far_chunks][far_keys].
__device__ inline float* near_part(const AttnParams& p, int b, int hk, int kb, int slot, int key) {
  return p.part_near + (((((int64_t)b * p.kv_heads + hk) * p.near_blocks + kb) * p.near_chunks + slot) * kDkvKeys + key) * 2 * p.dim;
}
__device__ inline float* far_part(const AttnParams& p, int b, int hk, int kb, int slot, int key) {
  return p.part_far + (((((int64_t)b * p.kv_heads + hk) * p.far_blocks + kb) * p.far_chunks + slot) * p.far_keys + key) * 2 * p.dim;
}

template <int DT, int ND, bool FULL>
__device__ inline void attention_dkv(const AttnParams& p, uint8_t* smem, uint32_t id) {
  using L = DkvLds<ND, FULL>;
  constexpr int Q = L::Q, RB = L::RB, NS = 2 * ND, NB = Q * RB / 1024 / kDkvWaves;
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // workgroups of a (sequence, key head): the key blocks' near chunks, then the far ones
  const int near = p.key_blocks * p.near_chunks, per = near + p.far_blocks * p.far_chunks;
  const int w = (int)(id % per), hk = (int)(id / per % p.kv_heads), b = (int)(id / per / p.kv_heads);
  const bool far = !FULL && w >= near;
  const int parts_of = far ? p.far_chunks : p.near_chunks;
  const int kb = (far ? w - near : w) / parts_of, chunk = (far ? w - near : w) % parts_of;
  const int nk = seq_keys(p, b), nq = seq_queries(p, b), shift = FULL ? nk - 1 : nk - nq;
  const int sub = wave >> 2;  // rows of a tile
  const int j_first = kb * kDkvKeys, j_wave = j_first + (wave & 3) * 32, j = j_wave + (lane & 31);
  const bool valid = j < nk;
  // queries: the near ones are those whose window may reach a key of the block
  int i0 = FULL ? 0 : min(max(0, j_first - shift), nq);
  int i1 = FULL ? nq : (int)max((int64_t)i0, min((int64_t)nq, (int64_t)min(j_first + kDkvKeys, nk) - 1 + p.window - shift));
  if (far) {
    i0 = i1;
    i1 = nq;
  }
  if (j_first >= nk) i1 = i0;
  {
    const int first = i0, last = i1, share = (last - first + parts_of - 1) / parts_of;
    i0 = (int)min((int64_t)last, first + (int64_t)chunk * share);
    i1 = min(last, i0 + share);
  }
  const int hg = min(p.group, Q), chunks = (p.group + hg - 1) / hg;  // query heads a tile, tiles a position
  const int tp = Q / hg;                                             // positions a tile

  // loads of a tile: block q of this wave holds tile row `row[q]`, position row / hg, head row % hg
  const uint8_t* q_base = p.q + 2 * (b * p.q_stride[0] + (int64_t)hk * p.group * p.q_stride[2]);
  const uint8_t* g_base = p.dout + 2 * (b * p.do_stride[0] + (int64_t)hk * p.group * p.do_stride[2]);
  uint32_t q_off[NB], g_off[NB];
  uint32_t at_row[NB];  // position and head (high half)
#pragma unroll
  for (int q = 0; q < NB; ++q) {
    const int row = (int)block_row<RB>(wave * NB + q, lane);
    const uint32_t c = block_chunk<RB>(wave * NB + q, lane) * 16u;
    const bool in = c < (uint32_t)p.dim * 2u && row < tp * hg;
    at_row[q] = (uint32_t)(row / hg | row % hg << 16);
    q_off[q] = in ? (uint32_t)(2 * (row / hg * p.q_stride[1] + row % hg * p.q_stride[2])) + c : kOutOfRange;
    g_off[q] = in ? (uint32_t)(2 * (row / hg * p.do_stride[1] + row % hg * p.do_stride[2])) + c : kOutOfRange;
  }
  const int64_t st_row = stats_row(p, b, hk, 0);
  const uint32_t lds0 = (uint32_t)(uintptr_t)(WTC_LDS uint8_t*)smem;
  const int steps = (i1 - i0 + tp - 1) / tp, t_all = steps * chunks;
  u32x4 kf[NS], vf[NS];  // (not read where no query sees the block)
  load_row<NS>(p.k + 2 * (b * p.k_stride[0] + (int64_t)j * p.k_stride[1] + hk * p.k_stride[2]), valid && t_all, p.dim, half, kf);
  load_row<NS>(p.v + 2 * (b * p.v_stride[0] + (int64_t)j * p.v_stride[1] + hk * p.v_stride[2]), valid && t_all, p.dim, half, vf);
  const float c2 = positive_scale<NS>(p.scale, kf);
  const uint32_t kept_at = (uint32_t)(L::KEPT_AT + (wave & 3) * L::KEPT * 1024 + lane * 16);
  if (!sub) {
#pragma unroll
    for (int x = 0; x < L::KEPT; ++x) *reinterpret_cast<u32x4*>(smem + kept_at + x * 1024) = vf[NS - L::KEPT + x];
  }
  f32x16 dk[ND], dv[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int v = 0; v < 16; ++v) dk[d][v] = dv[d][v] = 0.0f;
  DsRange<DT> range{DT == DT_F16 ? 60 : 0};  // (2^14 P (dP - D) is below 2^56 for f16 inputs)

  // The next tile to load: positions from i, heads of part hc.
  struct {
    const uint8_t *q, *g;
    int64_t row;
    int i, hc;
  } next = {q_base + 2 * i0 * p.q_stride[1], g_base + 2 * i0 * p.do_stride[1], st_row + (int64_t)i0 * p.group, i0, 0};
  const int64_t q_part = 2 * hg * p.q_stride[2], q_step = 2 * tp * p.q_stride[1] - (chunks - 1) * q_part;
  const int64_t g_part = 2 * hg * p.do_stride[2], g_step = 2 * tp * p.do_stride[1] - (chunks - 1) * g_part;
  const int row_step = tp * p.group - (chunks - 1) * hg;
  auto issue = [&](int t) {
    const int npos = t < t_all ? min(tp, i1 - next.i) : 0, nhead = p.group - next.hc * hg;
    const uint32_t st = lds0 + (uint32_t)t % L::STAGES * L::STAGE + (uint32_t)(wave * NB * 1024);
    // what is in range is said by the offsets alone
    const i32x4 rq = raw_rsrc(next.q, 0x7FFFFFFFu), rg = raw_rsrc(next.g, 0x7FFFFFFFu);
    if (npos == tp && nhead >= hg) {
#pragma unroll
      for (int q = 0; q < NB; ++q) {
        dma16(rq, q_off[q], st + q * 1024);
        dma16(rg, g_off[q], st + L::TILE + q * 1024);
      }
    } else {
#pragma unroll
      for (int q = 0; q < NB; ++q) {
        const bool in = (int)(at_row[q] & 0xFFFFu) < npos && (int)(at_row[q] >> 16) < nhead;
        dma16(rq, in ? q_off[q] : kOutOfRange, st + q * 1024);
        dma16(rg, in ? g_off[q] : kOutOfRange, st + L::TILE + q * 1024);
      }
    }
    if (wave == 0) {  // the rows' lse and D: contiguous
      const int rows = min(npos * hg, hg == p.group ? Q : nhead);
      const uint32_t bytes = rows > 0 ? (uint32_t)rows * 4u : 0u, at = lds0 + (uint32_t)t % L::STAGES * L::STAGE + L::STATS;
      dma16(raw_rsrc(p.row_lse + next.row, bytes), lane * 16, at);
      dma16(raw_rsrc(p.row_delta + next.row, bytes), lane * 16, at + 1024);
    }
    const bool last = next.hc + 1 == chunks;
    next.q += last ? q_step : q_part;
    next.g += last ? g_step : g_part;
    next.row += last ? row_step : hg;
    next.i += last ? tp : 0;
    next.hc = last ? 0 : next.hc + 1;
  };
#pragma unroll
  for (int t = 0; t < L::STAGES - 1; ++t) issue(t);
  landed(kf);
  landed(vf);
  const uint32_t r_at = row_addr<RB>(lane) + (uint32_t)(32 * sub) * RB, c_at = col_addr<RB>(lane) + (uint32_t)(32 * sub) * RB;
  int i = i0, hc = 0;  // the tile's
  for (int t = 0; t < t_all; ++t, hc = hc + 1 == chunks ? 0 : hc + 1, i += hc ? 0 : tp) {
    // tile t landed; every wave is done with tile t - 1 (wave 0 has two more loads a tile)
    if (wave == 0) wait_loads_barrier<(2 * NB + 2) * (L::STAGES - 2)>();
    else wait_loads_barrier<2 * NB * (L::STAGES - 2)>();
    issue(t + L::STAGES - 1);
    const uint32_t stage = (uint32_t)t % L::STAGES * L::STAGE;
    const uint8_t* stt = smem + stage + L::STATS;
    // tile row x is a query that sees this lane's key if t_lo <= x < t_hi
    const int rows = min(min(tp, i1 - i) * hg, hg == p.group ? Q : p.group - hc * hg);
    int t_lo = 0, t_hi = rows;  // (of a key behind the end nothing is kept)
    if constexpr (!FULL) {
      const int64_t back = (int64_t)j - shift - i;
      t_lo = (int)min((int64_t)1 << 20, max((int64_t)0, back)) * hg;
      const int64_t reach = j < p.sinks ? 1 << 20 : max((int64_t)0, min((int64_t)1 << 20, back + p.window)) * hg;
      t_hi = valid ? (int)min((int64_t)rows, reach) : 0;
    }
#pragma unroll
    for (int part = 0; part < Q / 64; ++part) {
      const int row0 = 32 * sub + 64 * part;
      const bool all = __all(t_lo <= row0 && t_hi >= row0 + 32);
      if (!all && !__any(max(t_lo, row0) < min(t_hi, row0 + 32))) continue;
      uint32_t ra = r_at + stage + 64 * part * RB, ca = c_at + stage + 64 * part * RB;
      fresh(ra);
      fresh(ca);
      f32x16 s, g;
#pragma unroll
      for (int v = 0; v < 16; ++v) s[v] = 0.0f;
#pragma unroll
      for (int st = 0; st < NS; ++st) s = mfma32<DT>(row_frag<RB>(smem, ra, 0, st), kf[st], s);
      if (!all) {
        const int at = row0 + 4 * half;
        const uint64_t in = bits_below(t_hi - at) & ~bits_below(t_lo - at);
#pragma unroll
        for (int v = 0; v < 16; ++v) s[v] = keep_bit(s[v], in, 8 * (v >> 2) + (v & 3));
      }
      __builtin_amdgcn_sched_barrier(0);
      // the exponentials among the products of dP - D, which start from -D
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const f32x4 del = *reinterpret_cast<const f32x4*>(stt + 1024 + (row0 + 8 * q + 4 * half) * 4);
#pragma unroll
        for (int v = 0; v < 4; ++v) g[4 * q + v] = del[v];
      }
#pragma unroll
      for (int st = 0; st < NS; ++st) {
        const int x = st - (NS - L::KEPT);
        g = mfma32<DT>(row_frag<RB>(smem, ra, Q, st), x < 0 ? vf[st] : *reinterpret_cast<const u32x4*>(smem + kept_at + x * 1024), g);
      }
      u32x4 pf[2], df[2];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const f32x4 lse = *reinterpret_cast<const f32x4*>(stt + (row0 + 8 * q + 4 * half) * 4);
#pragma unroll
        for (int v = 0; v < 4; ++v) s[4 * q + v] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[4 * q + v], c2, -lse[v]));
        uint32_t w0, w1;
        pack4<DT>(f32x4{s[4 * q], s[4 * q + 1], s[4 * q + 2], s[4 * q + 3]}, &w0, &w1);
        pf[q >> 1][2 * (q & 1)] = w0;
        pf[q >> 1][2 * (q & 1) + 1] = w1;
      }
#pragma unroll
      for (int x = 0; x < NS; ++x) {
        __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, 40 / NS, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
      // dS among the products of dv
#pragma unroll
      for (int st = 0; st < 2; ++st)
#pragma unroll
        for (int d = 0; d < ND; ++d) dv[d] = mfma32<DT>(col_frag<RB>(smem, ca, Q + 16 * st, d), pf[st], dv[d]);
      const float by = power_of_2(range.ex);
#pragma unroll
      for (int v = 0; v < 16; ++v) s[v] = DT == DT_F16 ? s[v] * by * g[v] : s[v] * g[v];
      const float most = range.pack(s, df);
#pragma unroll
      for (int x = 0; x < 2 * ND; ++x) {
        __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, (DT == DT_F16 ? 48 : 24) / (2 * ND), 0);
      }
      __builtin_amdgcn_sched_barrier(0);
      range.fit(most, s, dk, df);
#pragma unroll
      for (int st = 0; st < 2; ++st)
#pragma unroll
        for (int d = 0; d < ND; ++d) dk[d] = mfma32<DT>(col_frag<RB>(smem, ca, 16 * st, d), df[st], dk[d]);
    }
  }
  wait_loads_barrier<0>();
  range.undo(dk, kWeightBits<DT>);
  if constexpr (kWeightBits<DT> != 0) {
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int v = 0; v < 16; ++v) dv[d][v] *= power_of_2(-kWeightBits<DT>);
  }

  // ---- join: waves 0-3 hand over dv and finish dk, waves 4-7 the other way round
  uint8_t* mine = smem + wave * 32 * L::PITCH;          // what this wave finishes
  uint8_t* other = smem + (wave ^ 4) * 32 * L::PITCH;   // what it hands over
  const uint32_t at = (uint32_t)((lane & 31) * L::PITCH + half * 16);
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const f32x16& y = sub ? dk[d] : dv[d];
      *reinterpret_cast<f32x4*>(other + at + (32 * d + 8 * q) * 4) = f32x4{y[4 * q], y[4 * q + 1], y[4 * q + 2], y[4 * q + 3]};
    }
  __syncthreads();
#pragma unroll
  for (int d = 0; d < ND; ++d) {
    f32x16& y = sub ? dv[d] : dk[d];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const f32x4 z = *reinterpret_cast<const f32x4*>(mine + at + (32 * d + 8 * q) * 4);
#pragma unroll
      for (int v = 0; v < 4; ++v) dk[d][4 * q + v] = y[4 * q + v] + z[v];  // (the result in dk from here on)
    }
  }
  // keys whose sums the last kernel adds up: all, or the first tokens'
  const int summed = p.near_chunks > 1 ? p.lk : !FULL && kb < p.far_blocks ? p.sinks : 0;
  if (summed > j_first) {
    if (j < (far ? p.sinks : summed)) {
      float* dst = (far ? far_part(p, b, hk, kb, chunk, j - j_first) : near_part(p, b, hk, kb, chunk, j - j_first)) + sub * p.dim;
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int c = 32 * d + 8 * g + 4 * half;
          if (c < p.dim) *reinterpret_cast<f32x4*>(dst + c) = f32x4{dk[d][4 * g], dk[d][4 * g + 1], dk[d][4 * g + 2], dk[d][4 * g + 3]};
        }
    }
    if (far || p.near_chunks > 1) return;
  }
  bool nan = false;
  const float scale = sub ? 1.0f : p.scale;
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      f32x4 y;
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        y[v] = valid ? dk[d][4 * g + v] * scale : 0.0f;
        nan |= y[v] != y[v];
      }
      uint32_t w0, w1;
      pack4<DT>(y, &w0, &w1);
      *reinterpret_cast<u32x2*>(mine + (lane & 31) * L::PITCH + (32 * d + 8 * g + 4 * half) * 2) = u32x2{w0, w1};
    }
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  constexpr int CPR = ND * 4;
  uint8_t* dst = sub ? p.dv : p.dk;
#pragma unroll 4
  for (int y = lane; y < 32 * CPR; y += 64) {
    const int row = y / CPR, c = y % CPR, jj = j_wave + row;
    if (jj < p.lk && c * 8 < p.dim && jj >= summed)
      *reinterpret_cast<u32x4*>(dst + 2 * ((((int64_t)b * p.lk + jj) * p.kv_heads + hk) * p.dim) + c * 16) =
          *reinterpret_cast<const u32x4*>(mine + row * L::PITCH + c * 16);
  }
  // rows that came out as NaN, once both waves' results are written
  nan = nan && j >= summed;
  uint32_t* marks = reinterpret_cast<uint32_t*>(smem + L::TOTAL - kDkvWaves * 4);
  const uint64_t ballot = __ballot(nan);
  if (lane == 0) marks[wave] = (uint32_t)(ballot | ballot >> 32);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (sub) return;
  uint32_t redo = __builtin_amdgcn_readfirstlane(marks[wave] | marks[wave + 4]);
  while (redo) {
    dkv_row<DT, FULL>(p, b, hk, j_wave + __builtin_ctz(redo));
    redo &= redo - 1;
  }
}
template <int DT, int ND, bool FULL>
__global__ void __launch_bounds__(kDkvWaves * 64, 2) attention_dkv_kernel(const AttnParams p) {
  __shared__ __attribute__((aligned(256))) uint8_t smem[DkvLds<ND, FULL>::TOTAL];
  attention_dkv<DT, ND, FULL>(p, smem, xcd_remap(blockIdx.x, gridDim.x));
}

// Both at once, where their workgroups together leave each a CU of its own: the rows'
// statistics come from a kernel before (3 x 333 on 1000 states, 6 / 3 heads of 80 in f16:
// 28 us and 21 one after the other, 4 and 31 so).
template <int DT, int ND>
__global__ void __launch_bounds__(kDkvWaves * 64, 2) attention_gradients_kernel(const AttnParams p, int dq_blocks) {
  static_assert(kDkvWaves * 64 == 2 * 256, "threads of attention_dq with KG 2");
  constexpr int MOST = DqLds<ND, 2>::TOTAL > DkvLds<ND, true>::TOTAL ? DqLds<ND, 2>::TOTAL : DkvLds<ND, true>::TOTAL;
  __shared__ __attribute__((aligned(256))) uint8_t smem[MOST];
  if ((int)blockIdx.x < dq_blocks) attention_dq<DT, ND, 2, Rows::GIVEN, true>(p, smem, blockIdx.x);
  else attention_dkv<DT, ND, true>(p, smem, blockIdx.x - (uint32_t)dq_blocks);
}
// lse in the log2 domain and -D = -sum of dout out of 16 rows, 16 lanes a row.  FEW: but
// for rows of attention_dq's Rows::STATS.
template <int DT, bool FEW>
__device__ inline void attention_stats(const AttnParams& p, int64_t block) {
  const int64_t rows = (int64_t)p.batch * p.heads * p.lq, row = block * 16 + (threadIdx.x >> 4);
  const int c = (threadIdx.x & 15) * 8;
  const int64_t at = min(row, rows - 1);
  const int h = (int)(at % p.heads), i = (int)(at / p.heads % p.lq), b = (int)(at / p.heads / p.lq);
  const bool valid = i < seq_queries(p, b);
  float delta = 0.0f;
  if (valid && c < p.dim) {
    using V = typename Elem<DT>::vec8;
    const V g = *reinterpret_cast<const V*>(p.dout + 2 * (b * p.do_stride[0] + (int64_t)i * p.do_stride[1] + h * p.do_stride[2] + c));
    const V o = *reinterpret_cast<const V*>(p.o + 2 * (b * p.o_stride[0] + (int64_t)i * p.o_stride[1] + h * p.o_stride[2] + c));
#pragma unroll
    for (int v = 0; v < 8; ++v) delta = __builtin_fmaf((float)g[v], (float)o[v], delta);
  }
#pragma unroll
  for (int x = 8; x; x >>= 1) delta += __shfl_xor(delta, x);
  if (row >= rows || c || (FEW && valid && few_keys(seq_keys(p, b)))) return;
  const float lse = valid ? p.lse_in[((int64_t)b * p.heads + h) * p.lq + i] : -INFINITY;
  const int hk = h / p.group;
  const int64_t to = stats_row(p, b, hk, i) + h - hk * p.group;
  p.row_lse[to] = (lse == -INFINITY ? INFINITY : lse * kLog2e) - kWeightBits<DT>;
  p.row_delta[to] = lse == -INFINITY ? 0.0f : -delta;
}
template <int DT> __global__ void __launch_bounds__(256) attention_stats_kernel(const AttnParams p) {
  attention_stats<DT, false>(p, blockIdx.x);
}
// The same where a padded batch may have sequences of few keys: dq and dk / dv then take
// the D that separate launches give them (3 x 333 on 1000, 128 and 40 states, 6 / 3 heads of
// 80 in f16, both gradients: 42 us, 38 with D from the rounded `out` in all).
template <int DT, int ND>
__global__ void __launch_bounds__(256, 2) attention_padded_stats_kernel(const AttnParams p, int dq_blocks) {
  __shared__ __attribute__((aligned(256))) uint8_t smem[DqLds<ND, 1>::TOTAL];
  if ((int)blockIdx.x < dq_blocks) attention_dq<DT, ND, 1, Rows::STATS, true>(p, smem, blockIdx.x);
  else attention_stats<DT, true>(p, (int64_t)blockIdx.x - dq_blocks);
}

// dk and dv of the keys whose sums came in parts, the parts in order.  One wave a
// key, four elements a lane.
template <int DT, bool FULL>
__global__ void __launch_bounds__(256) attention_sum_kernel(const AttnParams p) {
  const int lane = threadIdx.x & 63;
  const int keys = p.near_chunks > 1 ? p.lk : p.sinks;
  const int64_t at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (at >= (int64_t)p.batch * p.kv_heads * keys) return;
  const int j = (int)(at % keys), hk = (int)(at / keys % p.kv_heads), b = (int)(at / keys / p.kv_heads);
  const int kb = j / kDkvKeys, key = j % kDkvKeys, c = lane * 4;
  bool nan = false;
  if (c < 2 * p.dim) {
    f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
    auto add = [&](const float* part, int64_t step, int count) {
      for (int s = 0; s < count; s += 8) {  // 8 loads at a time, added in their order
        f32x4 x[8];
#pragma unroll
        for (int u = 0; u < 8; ++u)
          if (s + u < count) x[u] = *reinterpret_cast<const f32x4*>(part + (s + u) * step);
#pragma unroll
        for (int u = 0; u < 8; ++u)
          if (s + u < count) {
#pragma unroll
            for (int v = 0; v < 4; ++v) sum[v] += x[u][v];
          }
      }
    };
    add(near_part(p, b, hk, kb, 0, key) + c, (int64_t)kDkvKeys * 2 * p.dim, p.near_chunks);
    if (p.far_chunks && j < p.sinks) add(far_part(p, b, hk, kb, 0, key) + c, (int64_t)p.far_keys * 2 * p.dim, p.far_chunks);
    const bool is_dv = c >= p.dim, valid = j < seq_keys(p, b);
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      sum[v] = valid ? sum[v] * (is_dv ? 1.0f : p.scale) : 0.0f;
      nan |= sum[v] != sum[v];
    }
    uint32_t w0, w1;
    pack4<DT>(sum, &w0, &w1);
    uint8_t* dst = (is_dv ? p.dv : p.dk) + 2 * ((((int64_t)b * p.lk + j) * p.kv_heads + hk) * p.dim + (is_dv ? c - p.dim : c));
    *reinterpret_cast<u32x2*>(dst) = u32x2{w0, w1};
  }
  if (!__any(nan)) return;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  dkv_row<DT, FULL>(p, b, hk, j);
}

hipError_t launch(const void* fn, int64_t grid, int threads, const AttnParams& p, hipStream_t stream) {
  AttnParams q = p;
  void* args[] = {&q};
  return hipLaunchKernel(fn, dim3((unsigned)grid), dim3(threads), args, 0, stream);
}

}  // namespace

#define WTC_BY_TYPE(kernel, dt) ((dt) == DT_F16 ? (const void*)&kernel<DT_F16> : (const void*)&kernel<DT_BF16>)

namespace {
template <int DT, int KG> const void* tile_kernel(int nd) {
  switch (nd) {
    case 1: return (const void*)&attention_tile_kernel<DT, 1, KG>;
    case 2: return (const void*)&attention_tile_kernel<DT, 2, KG>;
    case 3: return (const void*)&attention_tile_kernel<DT, 3, KG>;
  }
  return (const void*)&attention_tile_kernel<DT, 4, KG>;
}
}  // namespace

// Rows a workgroup (256 / key_groups) and splits of the keys, from the sizes alone:
// splits while CUs are idle and a wave keeps 4 tiles.
AttnPlan plan_attention(const AttnParams& p, int cu_count) {
  AttnPlan plan{1, 1, AttnPlan::TILE, cu_count};
  if (p.full && p.lk) {
    if (const int splits = plan_few_rows(p, cu_count)) return AttnPlan{1, splits, AttnPlan::FEW, cu_count};
    return AttnPlan{1, plan_attention_rows(p, cu_count), AttnPlan::ROWS, cu_count};
  }
  const int64_t rows = (int64_t)p.lq * p.group, seqs = (int64_t)p.batch * p.kv_heads;
  if (seqs * ((rows + 255) / 256) < cu_count) plan.key_groups = 2;
  const int64_t block = 256 / plan.key_groups, grid = seqs * ((rows + block - 1) / block);
  // keys that a row block sees at most
  const int64_t reach = std::min<int64_t>(p.lk, p.window + (block + p.group - 1) / p.group + p.sinks);
  const int64_t tiles = (reach + kKeys - 1) / kKeys;
  while (plan.splits < 16 && grid * plan.splits < cu_count && tiles / (2 * plan.splits) >= 4 * plan.key_groups) plan.splits *= 2;
  return plan;
}
int64_t attention_workspace(const AttnParams& p, const AttnPlan& plan) {
  const int64_t rows = (int64_t)p.batch * p.lq * p.heads * plan.splits;
  return plan.splits > 1 ? rows * 4 * (p.dim + 1) : 0;
}

hipError_t launch_attention(const AttnParams& params, const AttnPlan& plan, int dt, hipStream_t stream) {
  if (plan.kernel == AttnPlan::FEW) return launch_few_rows(params, plan.splits, dt, stream);
  if (plan.kernel == AttnPlan::ROWS) return launch_attention_rows(params, plan.splits, plan.cu_count, dt, stream);
  AttnParams p = params;
  const int64_t rows = (int64_t)p.lq * p.group;
  const bool joined = p.slots;  // by the caller, with the results of other launches
  p.splits = plan.splits;
  if (!joined) {
    p.slots = plan.splits > 1 ? plan.splits : 0;
    p.part_lse = p.part_out + (int64_t)p.batch * p.lq * p.heads * p.splits * p.dim;
  }
  p.row_blocks = (int)((rows * plan.key_groups + 255) / 256);
  const int nd = (p.dim + 31) / 32;
  const void* fn = plan.key_groups == 2 ? (dt == DT_F16 ? tile_kernel<DT_F16, 2>(nd) : tile_kernel<DT_BF16, 2>(nd))
                                        : (dt == DT_F16 ? tile_kernel<DT_F16, 1>(nd) : tile_kernel<DT_BF16, 1>(nd));
  const hipError_t e = launch(fn, (int64_t)p.batch * p.kv_heads * p.row_blocks * p.splits, 512, p, stream);
  if (e != hipSuccess || p.splits == 1 || joined) return e;
  return launch_attention_join(p, dt, stream);
}

namespace {
template <int DT> const void* join_kernel(const AttnParams& p) {
  if (p.full) return (const void*)&attention_join_kernel<DT, true, false>;
  return p.prefix ? (const void*)&attention_join_kernel<DT, false, true> : (const void*)&attention_join_kernel<DT, false, false>;
}
}  // namespace

hipError_t launch_attention_join(const AttnParams& p, int dt, hipStream_t stream) {
  const void* fn = dt == DT_F16 ? join_kernel<DT_F16>(p) : join_kernel<DT_BF16>(p);
  return launch(fn, ((int64_t)p.batch * p.lq * p.heads + 7) / 8, 256, p, stream);
}

namespace {
template <int DT, int KG, bool FULL> const void* dq_kernel(int nd) {
  switch (nd) {
    case 1: return (const void*)&attention_dq_kernel<DT, 1, KG, FULL>;
    case 2: return (const void*)&attention_dq_kernel<DT, 2, KG, FULL>;
    case 3: return (const void*)&attention_dq_kernel<DT, 3, KG, FULL>;
  }
  return (const void*)&attention_dq_kernel<DT, 4, KG, FULL>;
}
template <int DT, bool FULL> const void* dq_kernel(int nd, bool pairs) {
  return pairs ? dq_kernel<DT, 2, FULL>(nd) : dq_kernel<DT, 1, FULL>(nd);
}
template <int DT> const void* gradients_kernel(int nd) {
  switch (nd) {
    case 1: return (const void*)&attention_gradients_kernel<DT, 1>;
    case 2: return (const void*)&attention_gradients_kernel<DT, 2>;
    case 3: return (const void*)&attention_gradients_kernel<DT, 3>;
  }
  return (const void*)&attention_gradients_kernel<DT, 4>;
}
const void* sum_kernel(bool full, int dt) {
  if (full) return dt == DT_F16 ? (const void*)&attention_sum_kernel<DT_F16, true> : (const void*)&attention_sum_kernel<DT_BF16, true>;
  return dt == DT_F16 ? (const void*)&attention_sum_kernel<DT_F16, false> : (const void*)&attention_sum_kernel<DT_BF16, false>;
}
template <int DT> const void* padded_stats_kernel(int nd) {
  switch (nd) {
    case 1: return (const void*)&attention_padded_stats_kernel<DT, 1>;
    case 2: return (const void*)&attention_padded_stats_kernel<DT, 2>;
    case 3: return (const void*)&attention_padded_stats_kernel<DT, 3>;
  }
  return (const void*)&attention_padded_stats_kernel<DT, 4>;
}
template <int DT, bool FULL> const void* dkv_kernel(int nd) {
  switch (nd) {
    case 1: return (const void*)&attention_dkv_kernel<DT, 1, FULL>;
    case 2: return (const void*)&attention_dkv_kernel<DT, 2, FULL>;
    case 3: return (const void*)&attention_dkv_kernel<DT, 3, FULL>;
  }
  return (const void*)&attention_dkv_kernel<DT, 4, FULL>;
}
}  // namespace

AttnBackwardPlan plan_attention_backward(const AttnParams& p, int cu_count) {
  AttnBackwardPlan plan{};
  const int64_t row_blocks = ((int64_t)p.lq * p.group + kDqRows - 1) / kDqRows;
  plan.dq_groups = (int64_t)p.batch * p.kv_heads * row_blocks <= cu_count ? 2 : 1;
  plan.key_blocks = (p.lk + kDkvKeys - 1) / kDkvKeys;
  // queries past the near ones of the first block: at most the keys past them
  const int64_t far = std::min<int64_t>(p.lq, (int64_t)p.lk - (p.window + kDkvKeys) + 1);
  if (p.sinks > 0 && far > 0) {
    plan.far_blocks = (p.sinks + kDkvKeys - 1) / kDkvKeys;
    plan.far_keys = std::min(p.sinks, kDkvKeys);
    // short ones, in the end of the key blocks' round: 256 positions or a key block's
    // share, and no more in all than there are key blocks (their sums take memory)
    plan.far_chunks = (int)std::max<int64_t>(1, std::min<int64_t>(plan.key_blocks / plan.far_blocks, far / 256));
  }
  // near chunks while CUs are idle and a chunk keeps 4 tiles of 64 rows
  const int64_t seqs = (int64_t)p.batch * p.kv_heads;
  const int64_t tiles = std::min<int64_t>(p.lq, p.window + kDkvKeys) * p.group / kQueries;
  plan.near_chunks = 1;
  while (plan.near_chunks < 16 && seqs * plan.key_blocks * plan.near_chunks * 2 <= cu_count && tiles / (2 * plan.near_chunks) >= 4) plan.near_chunks *= 2;
  // (where all sequences have few keys the statistics would take a launch like dq's own)
  plan.together = p.full && p.lq && p.lk > kFewTiles * kKeys && seqs * (row_blocks + (int64_t)plan.key_blocks * plan.near_chunks) <= cu_count;
  plan.near_blocks = plan.near_chunks > 1 ? plan.key_blocks : plan.far_blocks;
  const int64_t rows = (int64_t)p.batch * p.lq * p.heads;
  plan.part_at = (rows * 8 + 255) / 256 * 256;
  plan.far_at = plan.part_at + (seqs * plan.near_blocks * plan.near_chunks * kDkvKeys * 2 * p.dim * 4 + 255) / 256 * 256;
  plan.workspace = plan.far_at + (seqs * plan.far_blocks * plan.far_chunks * plan.far_keys * 2 * p.dim * 4 + 255) / 256 * 256;
  return plan;
}

hipError_t launch_attention_backward(const AttnParams& params, const AttnBackwardPlan& plan, int dt, hipStream_t stream) {
  AttnParams p = params;
  p.part_near = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(p.row_lse) + plan.part_at);
  p.part_far = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(p.row_lse) + plan.far_at);
  p.near_blocks = plan.near_blocks;
  p.near_chunks = plan.near_chunks;
  p.row_delta = p.row_lse + (int64_t)p.batch * p.lq * p.heads;
  p.key_blocks = plan.key_blocks;
  p.far_blocks = plan.far_blocks;
  p.far_keys = plan.far_keys;
  p.far_chunks = plan.far_chunks;
  const int nd = (p.dim + 31) / 32;
  const int64_t seqs = (int64_t)p.batch * p.kv_heads;
  if (plan.together) {
    p.row_blocks = (int)(((int64_t)p.lq * p.group + kDqRows - 1) / kDqRows);
    const int64_t stats_blocks = ((int64_t)p.batch * p.lq * p.heads + 15) / 16;
    int dq_blocks = (int)(seqs * p.row_blocks);
    void* args[] = {&p, &dq_blocks};
    hipError_t e = p.k_lens ? hipLaunchKernel(dt == DT_F16 ? padded_stats_kernel<DT_F16>(nd) : padded_stats_kernel<DT_BF16>(nd),
                                              dim3((unsigned)(dq_blocks + stats_blocks)), dim3(256), args, 0, stream)
                            : launch(WTC_BY_TYPE(attention_stats_kernel, dt), stats_blocks, 256, p, stream);
    if (e != hipSuccess) return e;
    e = hipLaunchKernel(dt == DT_F16 ? gradients_kernel<DT_F16>(nd) : gradients_kernel<DT_BF16>(nd),
                        dim3((unsigned)(dq_blocks + seqs * p.key_blocks * p.near_chunks)), dim3(kDkvWaves * 64), args, 0, stream);
    if (e != hipSuccess || p.near_chunks == 1) return e;
    return launch(sum_kernel(true, dt), (seqs * p.lk + 3) / 4, 256, p, stream);
  }
  if (p.lq) {
    p.row_blocks = (int)(((int64_t)p.lq * p.group + kDqRows - 1) / kDqRows);
    const bool pairs = plan.dq_groups == 2;
    const void* fn = p.full ? (dt == DT_F16 ? dq_kernel<DT_F16, true>(nd, pairs) : dq_kernel<DT_BF16, true>(nd, pairs))
                            : (dt == DT_F16 ? dq_kernel<DT_F16, false>(nd, pairs) : dq_kernel<DT_BF16, false>(nd, pairs));
    const hipError_t e = launch(fn, seqs * p.row_blocks, pairs ? 512 : 256, p, stream);
    if (e != hipSuccess) return e;
  }
  if (!p.lk) return hipSuccess;
  const void* dkv = p.full ? (dt == DT_F16 ? dkv_kernel<DT_F16, true>(nd) : dkv_kernel<DT_BF16, true>(nd))
                           : (dt == DT_F16 ? dkv_kernel<DT_F16, false>(nd) : dkv_kernel<DT_BF16, false>(nd));
  const hipError_t e = launch(dkv,
                              seqs * (p.key_blocks * p.near_chunks + p.far_blocks * p.far_chunks), kDkvWaves * 64, p, stream);
  if (e != hipSuccess || (p.near_chunks == 1 && !p.far_blocks)) return e;
  return launch(sum_kernel(p.full, dt), (seqs * (p.near_chunks > 1 ? p.lk : p.sinks) + 3) / 4, 256, p, stream);
}

}  // namespace wtc
