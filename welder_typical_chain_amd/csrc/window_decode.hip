// window_decode.hip -- kernels of wtc_window_attention_decode: one query row a
// sequence and head against a cache that may have wrapped.
//
// What bounds it is reading the visible rows of K and V once.  The rows stand in
// at most three runs of the cache (the first tokens, and the window's tokens,
// which may wrap); a run is cut into tiles of 32 rows, so that a tile's rows
// are consecutive and no tile needs a mask but for its length.  A workgroup
// takes the tiles of one (sequence, key head, split); its 4 waves take them in
// turn, each with a ring of its own of direct-to-LDS loads and no barrier until
// the end, so that a wave's loads are in flight while it computes.  All query
// heads of the group (up to 32) are columns of the same products:
//   S^T = K . Q^T, O^T += V^T . P^T, online softmax as in window_attention.hip.
// The waves' results are joined through LDS; splits by a second kernel.
// 64 sequences of up to 16384 tokens, 32 / 8 heads of 128, 4100 visible keys: 172 us,
// 5.5 TB/s in all and 6.2 on the CUs that still have work (sequences shorter than
// the window end early).  A CU holds 128 KiB of stages either way: two workgroups of
// one or two stages a wave, whose ends overlap, against one of two or four, are as fast here and
// 82 us against 86 with weights (32 sequences of 4096 tokens, the same heads); a
// stage's K is refilled as soon as it is read, before its V.
#include <algorithm>

#include "decode_tile.h"
#include "layer_kernels.h"

namespace wtc {
namespace {

using namespace attn;

using namespace decode;

constexpr int kGroups = 2;

template <int DT, int ND, bool SCORES>
__global__ void __launch_bounds__(kWaves * 64, kGroups) decode_kernel(const AttnParams p) {
  __shared__ __attribute__((aligned(256))) uint8_t smem[DecodeLds<ND, kGroups>::TOTAL];
  decode_tile<DT, ND, SCORES, false, kGroups>(p, smem, (int)blockIdx.x);
}
template <int DT, int ND>
__global__ void __launch_bounds__(kWaves * 64, kGroups) few_rows_kernel(const AttnParams p) {
  __shared__ __attribute__((aligned(256))) uint8_t smem[DecodeLds<ND, kGroups>::TOTAL];
  decode_tile<DT, ND, false, true, kGroups>(p, smem, (int)blockIdx.x);
}

// The splits of a head's row: half a wave a row.
template <int DT> __device__ inline void join_row(const AttnParams& p, int64_t row) {
  const int c = (threadIdx.x & 31) * 4;
  if (row >= (int64_t)p.batch * p.heads || c >= p.dim) return;
  const int h = (int)(row % p.heads), b = (int)(row / p.heads);
  f32x4 x;
  join_splits(p.part_out + row * p.slots * p.dim, p.part_lse + row * p.slots, p.slots, p.dim, c, &x);
  uint32_t w0, w1;
  pack4<DT>(x, &w0, &w1);
  *reinterpret_cast<u32x2*>(p.out + 2 * (b * p.o_stride[0] + h * p.o_stride[2] + c)) = u32x2{w0, w1};
}
template <int DT>
__global__ void __launch_bounds__(256) decode_join_kernel(const AttnParams p) {
  join_row<DT>(p, (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5));
}

// What the rows of a cache received from the token: p.weights [batch][kv_heads][lk] +=
// the sum over the key head's query heads of exp2(score - log2-sum-exp).  The newest
// token's row is set instead: nobody weighed it before.  Workgroups [0, weight_blocks)
// take 1024 tile rows of a (sequence, key head), four a thread, those behind them join the splits
// as decode_join_kernel does.  What bounds it is reading the scores (4 bytes a row and query
// head, of 512 that the caches take a row at dim 128): 8 us of the 77 for 32 sequences of 4096
// tokens, 32 / 8 heads of 128.
constexpr int kHeadsAtOnce = 64;
template <int DT>
__global__ void __launch_bounds__(256) decode_weights_kernel(const AttnParams p, int weight_blocks, int chunks) {
  if ((int)blockIdx.x >= weight_blocks) {
    join_row<DT>(p, (int64_t)((int)blockIdx.x - weight_blocks) * 8 + (threadIdx.x >> 5));
    return;
  }
  __shared__ float lse[kHeadsAtOnce];
  const int chunk = (int)blockIdx.x % chunks, seq = (int)blockIdx.x / chunks, b = seq / p.kv_heads, hk = seq % p.kv_heads;
  const Runs runs(p, max(p.k_lens[b], 0));
  const int x = (chunk * 256 + (int)threadIdx.x) * 4, t = x / kRows;
  if (chunk * 1024 / kRows >= runs.t_all) return;  // (the whole workgroup)
  int row = 0, rows = 0;
  if (t < runs.t_all) runs.tile(t, &row, &rows);
  const int in = min(4, rows - x % kRows);  // rows of this thread
  float* w = p.weights + (int64_t)seq * p.lk + row + x % kRows;
  float sum[4] = {}, before[4] = {};
#pragma unroll
  for (int v = 0; v < 4; ++v)
    if (v < in) before[v] = w[v];
  if (t == runs.t_all - 1 && in > 0 && x % kRows + in == rows) before[in - 1] = 0.0f;
  const int64_t pitch = (int64_t)most_tiles(p.lk) * kRows;
  for (int g0 = 0; g0 < p.group; g0 += kHeadsAtOnce) {
    const int heads = min(kHeadsAtOnce, p.group - g0);
    const int64_t h0 = (int64_t)b * p.heads + hk * p.group + g0;
    const float* score = p.scores + h0 * pitch + x;
    f32x4 y[4];  // of four heads, on their way while the log-sum-exps come
#pragma unroll
    for (int g = 0; g < 4; ++g)
      if (in > 0 && g < heads) y[g] = *reinterpret_cast<const f32x4*>(score + g * pitch);
    __syncthreads();
    if ((int)threadIdx.x < heads) {
      const float* part = p.part_lse + (h0 + threadIdx.x) * p.slots;
      float m = -INFINITY, total = 0.0f;
      for (int s = 0; s < p.slots; ++s) m = fmaxf(m, part[s]);
      const float ref = m == -INFINITY ? 0.0f : m;
      for (int s = 0; s < p.slots; ++s) total += __builtin_amdgcn_exp2f(part[s] - ref);
      // no weights where every score is -inf
      lse[threadIdx.x] = total == 0.0f ? INFINITY : ref + __builtin_amdgcn_logf(total);
    }
    __syncthreads();
    if (in <= 0) continue;
    for (int g4 = 0; g4 < heads; g4 += 4) {
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        if (g4 + g >= heads) continue;
        if (g4) y[g] = *reinterpret_cast<const f32x4*>(score + (g4 + g) * pitch);
#pragma unroll
        for (int v = 0; v < 4; ++v) sum[v] += __builtin_amdgcn_exp2f(y[g][v] - lse[g4 + g]);
      }
    }
  }
#pragma unroll
  for (int v = 0; v < 4; ++v)
    if (v < in) w[v] = before[v] + sum[v];
}

template <int DT> const void* few_rows_for(int nd) {
  switch (nd) {
    case 1: return (const void*)&few_rows_kernel<DT, 1>;
    case 2: return (const void*)&few_rows_kernel<DT, 2>;
    case 3: return (const void*)&few_rows_kernel<DT, 3>;
  }
  return (const void*)&few_rows_kernel<DT, 4>;
}
template <int DT, bool SCORES> const void* kernel_for(int nd) {
  switch (nd) {
    case 1: return (const void*)&decode_kernel<DT, 1, SCORES>;
    case 2: return (const void*)&decode_kernel<DT, 2, SCORES>;
    case 3: return (const void*)&decode_kernel<DT, 3, SCORES>;
  }
  return (const void*)&decode_kernel<DT, 4, SCORES>;
}

}  // namespace

// Splits of a (sequence, key head): while CUs are idle and a wave keeps at least 4 tiles.
int plan_decode(const AttnParams& p, int cu_count) {
  const int64_t grid = (int64_t)p.batch * p.kv_heads * ((p.group + kHeads - 1) / kHeads);
  const int64_t tiles = (std::min<int64_t>(p.lk, p.window + p.sinks) + kRows - 1) / kRows;
  int splits = 1;
  while (splits < 64 && grid * splits * 2 <= cu_count && tiles / (2 * splits) >= 4 * kWaves) splits *= 2;
  return splits;
}
// Sequences of unequal length leave CUs idle at the end: splits until there are `rounds`
// workgroups a CU, while a wave keeps at least 4 tiles.
int plan_decode_joined(const AttnParams& p, int rounds, int cu_count) {
  const int64_t grid = (int64_t)p.batch * p.kv_heads * ((p.group + kHeads - 1) / kHeads);
  const int64_t tiles = (std::min<int64_t>(p.lk, p.window + p.sinks) + kRows - 1) / kRows;
  int splits = 1;
  while (splits < 64 && grid * splits < (int64_t)rounds * cu_count && tiles / (2 * splits) >= 4 * kWaves) splits *= 2;
  return splits;
}
int64_t decode_workspace(const AttnParams& p, int splits) {
  return splits > 1 ? (int64_t)p.batch * p.heads * splits * (p.dim + 1) * 4 : 0;
}
int64_t decode_weights_workspace(const AttnParams& p, int splits) {
  return (int64_t)p.batch * p.heads * 4 * ((int64_t)splits * (p.dim + 1) + (int64_t)most_tiles(p.lk) * kRows);
}

namespace {
hipError_t launch(const void* fn, int64_t grid, void** args, hipStream_t stream) {
  return hipLaunchKernel(fn, dim3((unsigned)grid), dim3(kWaves * 64), args, 0, stream);
}
int64_t decode_grid(const AttnParams& p) { return (int64_t)p.batch * p.kv_heads * (((int64_t)p.lq * p.group + kHeads - 1) / kHeads) * p.splits; }
}  // namespace

// Few rows that see all of their keys: up to two blocks of 32, which both read the keys.
// Splits while CUs are idle and a wave keeps two tiles.
int plan_few_rows(const AttnParams& p, int cu_count) {
  const int64_t rows = (int64_t)p.lq * p.group;
  if (rows > 2 * kHeads) return 0;
  const int64_t grid = (int64_t)p.batch * p.kv_heads * ((rows + kHeads - 1) / kHeads), tiles = (p.lk + kRows - 1) / kRows;
  int splits = 1;
  while (splits < 64 && grid * splits * 2 <= cu_count && tiles / (2 * splits) >= 2 * kWaves) splits *= 2;
  return splits;
}
hipError_t launch_few_rows(const AttnParams& params, int splits, int dt, hipStream_t stream) {
  AttnParams p = params;
  const bool joined = p.slots;  // by the caller, with the results of other launches
  p.splits = splits;
  if (!joined) {
    p.slots = splits > 1 ? splits : 0;
    p.part_lse = p.part_out + (int64_t)p.batch * p.lq * p.heads * splits * p.dim;
  }
  void* args[] = {&p};
  const int nd = (p.dim + 31) / 32;
  const hipError_t e = launch(dt == DT_F16 ? few_rows_for<DT_F16>(nd) : few_rows_for<DT_BF16>(nd), decode_grid(p), args, stream);
  if (e != hipSuccess || splits == 1 || joined) return e;
  return launch_attention_join(p, dt, stream);
}

hipError_t launch_attention_decode(const AttnParams& params, int splits, int dt, hipStream_t stream) {
  AttnParams p = params;
  const bool joined = p.slots;  // by the caller, with the results of other launches
  p.splits = splits;
  if (!joined) {
    p.slots = splits > 1 ? splits : 0;
    p.part_lse = p.part_out + (int64_t)p.batch * p.heads * splits * p.dim;
  }
  void* args[] = {&p};
  const int nd = (p.dim + 31) / 32;
  const hipError_t e = launch(dt == DT_F16 ? kernel_for<DT_F16, false>(nd) : kernel_for<DT_BF16, false>(nd), decode_grid(p), args, stream);
  if (e != hipSuccess || splits == 1 || joined) return e;
  return launch(dt == DT_F16 ? (const void*)&decode_join_kernel<DT_F16> : (const void*)&decode_join_kernel<DT_BF16>,
                ((int64_t)p.batch * p.heads + 7) / 8, args, stream);
}

hipError_t launch_attention_decode_weights(const AttnParams& params, int splits, int dt, hipStream_t stream) {
  AttnParams p = params;
  p.splits = p.slots = splits;
  const int64_t rows = (int64_t)p.batch * p.heads;
  p.scores = p.part_out + rows * splits * p.dim;  // (both multiples of 8 elements)
  p.part_lse = p.scores + rows * most_tiles(p.lk) * kRows;
  int chunks = (most_tiles(p.lk) * kRows + 1023) / 1024, weight_blocks = p.batch * p.kv_heads * chunks;
  void* args[] = {&p, &weight_blocks, &chunks};
  const int nd = (p.dim + 31) / 32;
  const hipError_t e = launch(dt == DT_F16 ? kernel_for<DT_F16, true>(nd) : kernel_for<DT_BF16, true>(nd), decode_grid(p), args, stream);
  if (e != hipSuccess) return e;
  return launch(dt == DT_F16 ? (const void*)&decode_weights_kernel<DT_F16> : (const void*)&decode_weights_kernel<DT_BF16>,
                weight_blocks + (rows + 7) / 8, args, stream);
}

}  // namespace wtc
