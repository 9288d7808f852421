// key_weights.hip -- kernels of wtc_window_attention_weights: what each key has
// received from the queries of its sequence,
//   w[b][g][j] = sum over the query heads h of g and the queries i that see j of
//                exp(scale q_i . k_j - lse_i).
//
// A workgroup takes 256 keys of one (sequence, key head), 64 a wave, whose fragments
// stay in registers, and streams the queries in tiles of 64 packed rows (positions
// of up to 64 query heads) through a ring of direct-to-LDS stages:
//   S^T = K . Q^T (a lane holds 32 keys of one query), w += exp2(c S - lse).
// The sums stay in the lanes, a query column each, until the end, where 31 exchanges
// add the 32 columns.  Long sequences go in chunks of queries, whose sums a second
// kernel adds in their order.
#include <algorithm>

#include "attention_common.h"
#include "layer_kernels.h"

namespace wtc {
namespace {

using namespace attn;

constexpr int kRows = 64;            // packed query rows a tile
constexpr int kWaves = 4;
constexpr int kKeys = 64 * kWaves;   // keys a workgroup

template <int ND> struct WeightsLds {
  static constexpr int RB = row_bytes(ND), STAGES = 3;
  static constexpr int TILE = kRows * RB, STAGE = TILE + 256;  // the rows, their log-sum-exps
  static constexpr int TOTAL = STAGES * STAGE;
};

// x, or 0 where bit c is clear (a hidden key's weight may be NaN)
__device__ inline float zero_bit(float x, uint64_t bits, int c) {
  const uint32_t w = c < 32 ? (uint32_t)bits : (uint32_t)(bits >> 32);
  const uint32_t in = (uint32_t)__builtin_amdgcn_sbfe((int)w, c & 31, 1);
  return __builtin_bit_cast(float, in & __builtin_bit_cast(uint32_t, x));
}

// x[0 .. N): the sums over the lanes whose numbers agree but for the bits below BIT * 2;
// afterwards x[0] of a lane is that of x[lane % N].
template <int N> __device__ inline void column_sums(float (&x)[N], int lane) {
  if constexpr (N > 1) {
    constexpr int H = N / 2;
    const bool high = lane & H;
    float y[H];
#pragma unroll
    for (int i = 0; i < H; ++i) y[i] = (high ? x[i + H] : x[i]) + __shfl_xor(high ? x[i] : x[i + H], H);
    column_sums<H>(y, lane);
    x[0] = y[0];
  }
}

template <int DT, int ND>
__global__ void __launch_bounds__(kWaves * 64, 2) key_weights_kernel(const AttnParams p, int chunk_rows) {
  using L = WeightsLds<ND>;
  constexpr int RB = L::RB, NS = 2 * ND, NB = kRows * RB / 1024 / kWaves;
  __shared__ __attribute__((aligned(256))) uint8_t smem[L::TOTAL];
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t id = xcd_remap(blockIdx.x, gridDim.x);
  const int chunk = (int)(id % p.splits), kb = (int)(id / p.splits % p.key_blocks);
  const int hk = (int)(id / p.splits / p.key_blocks % p.kv_heads), b = (int)(id / p.splits / p.key_blocks / p.kv_heads);
  const int nk = seq_keys(p, b), nq = seq_queries(p, b), shift = first_position(p, nq, nk);
  const int j_first = kb * kKeys, j_wave = j_first + wave * 64;
  // queries that may see a key of the block, and this chunk's of them
  int i0 = min(max(0, j_first - shift), nq);
  int i1 = j_first < p.sinks ? nq : (int)max((int64_t)i0, min((int64_t)nq, (int64_t)min(j_first + kKeys, nk) - 1 + p.window - shift));
  if (j_first >= nk) i1 = i0;
  i0 = (int)min((int64_t)i1, max((int64_t)i0, (int64_t)chunk * chunk_rows));
  i1 = (int)max((int64_t)i0, min((int64_t)i1, (int64_t)(chunk + 1) * chunk_rows));
  const int hg = min(p.group, kRows), groups = (p.group + hg - 1) / hg, tp = kRows / hg;  // heads, parts, positions of a tile

  u32x4 kf[2][NS];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int j = j_wave + 32 * u + (lane & 31);
    load_row<NS>(p.k + 2 * (b * p.k_stride[0] + (int64_t)j * p.k_stride[1] + hk * p.k_stride[2]), j < nk, p.dim, half, kf[u]);
  }
  const float c2 = positive_scale<NS>(p.scale, kf[0]);
  positive_scale<NS>(p.scale, kf[1]);

  const uint8_t* q_base = p.q + 2 * (b * p.q_stride[0] + (int64_t)hk * p.group * p.q_stride[2]);
  uint32_t q_off[NB], at_row[NB];  // at_row: position and head (high half)
#pragma unroll
  for (int q = 0; q < NB; ++q) {
    const int row = (int)block_row<RB>(wave * NB + q, lane);
    const uint32_t c = block_chunk<RB>(wave * NB + q, lane) * 16u;
    at_row[q] = c < (uint32_t)p.dim * 2u ? (uint32_t)(row / hg | row % hg << 16) : 0xFFFFu;
    q_off[q] = (uint32_t)(2 * (row / hg * p.q_stride[1] + row % hg * p.q_stride[2])) + c;
  }
  const uint32_t lse_row = (uint32_t)(lane / hg | lane % hg << 16), lse_off = (uint32_t)(4 * (lane % hg * (int64_t)p.lq + lane / hg));
  const float* lse_base = p.lse_in + ((int64_t)b * p.heads + hk * p.group) * p.lq;
  const int x_pos[2] = {(lane & 31) / hg, (32 + (lane & 31)) / hg};
  const int x_head[2] = {(lane & 31) % hg, (32 + (lane & 31)) % hg};
  const uint32_t lds0 = (uint32_t)(uintptr_t)(WTC_LDS uint8_t*)smem;
  const int t_all = (i1 - i0 + tp - 1) / tp * groups;
  auto issue = [&](int t) {
    const int step = t / groups, hc = t - step * groups, i = i0 + step * tp;
    const int npos = t < t_all ? min(tp, i1 - i) : 0, nhead = p.group - hc * hg;
    const uint32_t st = lds0 + (uint32_t)t % L::STAGES * L::STAGE;
    const i32x4 rq = raw_rsrc(q_base + 2 * (i * p.q_stride[1] + hc * hg * p.q_stride[2]), 0x7FFFFFFFu);
#pragma unroll
    for (int q = 0; q < NB; ++q) {
      const bool in = (int)(at_row[q] & 0xFFFFu) < npos && (int)(at_row[q] >> 16) < nhead;
      dma16(rq, in ? q_off[q] : kOutOfRange, st + wave * NB * 1024 + q * 1024);
    }
    if (wave == 0) {
      const bool in = (int)(lse_row & 0xFFFFu) < npos && (int)(lse_row >> 16) < nhead;
      dma4(raw_rsrc(lse_base + (int64_t)hc * hg * p.lq + i, 0x7FFFFFFFu), in ? lse_off : kOutOfRange, st + L::TILE);
    }
  };
  float sums[32];
#pragma unroll
  for (int v = 0; v < 32; ++v) sums[v] = 0.0f;
#pragma unroll
  for (int t = 0; t < L::STAGES - 1; ++t) issue(t);
  const uint32_t r_at = row_addr<RB>(lane);
  for (int t = 0; t < t_all; ++t) {
    if (wave == 0) wait_loads_barrier<(NB + 1) * (L::STAGES - 2)>();
    else wait_loads_barrier<NB * (L::STAGES - 2)>();
    issue(t + L::STAGES - 1);
    const int step = t / groups, hc = t - step * groups, i = i0 + step * tp;
    const int npos = min(tp, i1 - i), nhead = p.group - hc * hg;
    const uint32_t stage = (uint32_t)t % L::STAGES * L::STAGE;
    // positions of the tile's queries; keys of the wave that none of them sees, that all see
    const int64_t p_lo = (int64_t)i + shift, p_hi = p_lo + npos - 1;
    if (j_wave > p_hi || j_wave >= nk || (j_wave + 63 + p.window <= p_lo && j_wave >= p.sinks)) continue;
    const bool all = npos * hg == kRows && nhead >= hg && j_wave + 63 <= p_lo && (p_hi - j_wave < p.window || j_wave + 63 < p.sinks);
    uint32_t ra = r_at + stage;
    fresh(ra);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      f32x16 s[2];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
#pragma unroll
        for (int v = 0; v < 16; ++v) s[x][v] = 0.0f;
      }
#pragma unroll
      for (int st = 0; st < NS; ++st) {
        const u32x4 q = row_frag<RB>(smem, ra, 32 * u, st);
#pragma unroll
        for (int x = 0; x < 2; ++x) s[x] = mfma32<DT>(kf[x][st], q, s[x]);
      }
      const float lse = *reinterpret_cast<const float*>(smem + stage + L::TILE + (32 * u + (lane & 31)) * 4) * kLog2e;
      const float off = lse == -INFINITY ? lse : -lse;  // a row of scores -inf weighs nothing
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int v = 0; v < 16; ++v) s[x][v] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[x][v], c2, off));
      if (!all) {
        const int pos = i + x_pos[u] + shift;
        const bool row = x_pos[u] < npos && x_head[u] < nhead;
        const uint64_t seen = row ? seen_bits(j_wave + 4 * half, nk, pos, p.window, p.sinks) : 0;
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int v = 0; v < 16; ++v) s[x][v] = zero_bit(s[x][v], seen, 32 * x + 8 * (v >> 2) + (v & 3));
      }
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int v = 0; v < 16; ++v) sums[16 * x + v] += s[x][v];
    }
  }
  wait_loads_barrier<0>();

  column_sums<32>(sums, lane);
  const int c = lane & 31, j = j_wave + 32 * (c >> 4) + 8 * ((c >> 2) & 3) + 4 * half + (c & 3);
  if (j >= p.lk) return;
  const int64_t seq = (int64_t)b * p.kv_heads + hk;
  const float w = j < nk ? sums[0] : 0.0f;
  if (p.splits > 1) {
    p.part_out[(seq * p.splits + chunk) * p.lk + j] = w;
  } else {
    float* dst = p.weights + seq * p.lk + j;
    *dst = p.add ? *dst + w : w;
  }
}

__global__ void __launch_bounds__(256) key_weights_sum_kernel(const AttnParams p) {
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (at >= (int64_t)p.batch * p.kv_heads * p.lk) return;
  const int64_t seq = at / p.lk, j = at - seq * p.lk;
  float sum = 0.0f;
  for (int c = 0; c < p.splits; ++c) sum += p.part_out[(seq * p.splits + c) * p.lk + j];
  p.weights[at] = p.add ? p.weights[at] + sum : sum;
}

template <int DT> const void* kernel_for(int nd) {
  switch (nd) {
    case 1: return (const void*)&key_weights_kernel<DT, 1>;
    case 2: return (const void*)&key_weights_kernel<DT, 2>;
    case 3: return (const void*)&key_weights_kernel<DT, 3>;
  }
  return (const void*)&key_weights_kernel<DT, 4>;
}

}  // namespace

// Chunks of the queries: until the chip has eight workgroups a CU, while a chunk keeps
// four tiles.
KeyWeightsPlan plan_key_weights(const AttnParams& p, int cu_count) {
  KeyWeightsPlan plan{};
  plan.key_blocks = (p.lk + kKeys - 1) / kKeys;
  const int64_t seqs = (int64_t)p.batch * p.kv_heads, blocks = std::max<int64_t>(1, seqs * plan.key_blocks);
  const int64_t tiles = ((int64_t)p.lq * p.group + kRows - 1) / kRows;
  plan.chunks = (int)std::max<int64_t>(1, std::min<int64_t>(tiles / 4, 8ll * cu_count / blocks));
  plan.chunk_rows = (p.lq + plan.chunks - 1) / plan.chunks;
  plan.chunks = plan.chunk_rows ? (p.lq + plan.chunk_rows - 1) / plan.chunk_rows : 1;
  plan.workspace = plan.chunks > 1 ? seqs * plan.chunks * p.lk * 4 : 0;
  return plan;
}

hipError_t launch_key_weights(const AttnParams& params, const KeyWeightsPlan& plan, int dt, hipStream_t stream) {
  AttnParams p = params;
  p.splits = plan.chunks;
  p.key_blocks = plan.key_blocks;
  int chunk_rows = plan.chunk_rows;
  void* args[] = {&p, &chunk_rows};
  const int nd = (p.dim + 31) / 32;
  const int64_t grid = (int64_t)p.batch * p.kv_heads * p.key_blocks * p.splits;
  const hipError_t e = hipLaunchKernel(dt == DT_F16 ? kernel_for<DT_F16>(nd) : kernel_for<DT_BF16>(nd), dim3((unsigned)grid),
                                       dim3(kWaves * 64), args, 0, stream);
  if (e != hipSuccess || p.splits == 1) return e;
  return hipLaunchKernel((const void*)&key_weights_sum_kernel, dim3((unsigned)(((int64_t)p.batch * p.kv_heads * p.lk + 255) / 256)),
                         dim3(256), args, 0, stream);
}

}  // namespace wtc
