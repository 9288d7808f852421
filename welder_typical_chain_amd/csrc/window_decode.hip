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
// the window end early).  Refilling a stage's K as soon as it is read, before its
// V, changed nothing.
#include <algorithm>

#include "attention_common.h"
#include "layer_kernels.h"

namespace wtc {
namespace {

using namespace attn;

constexpr int kRows = 32;   // cache rows a tile
constexpr int kWaves = 4;
constexpr int kHeads = 32;  // query heads a workgroup

template <int ND> struct DecodeLds {
  static constexpr int RB = row_bytes(ND);
  static constexpr int TILE = kRows * RB, STAGE = 2 * TILE;
  static constexpr int STAGES = RB == 256 ? 2 : 4;  // 128 KiB over the waves
  static constexpr int RING = kWaves * STAGES * STAGE;
  static constexpr int PITCH = ND * 32 + 4;          // floats of a head's result
  static constexpr int JOIN = kWaves * kHeads * PITCH * 4;
  static constexpr int TOTAL = (RING > JOIN ? RING : JOIN) + kWaves * kHeads * 8;
  static_assert(TOTAL <= 160 * 1024, "LDS");
};

// The visible rows of a sequence's cache as tiles.
struct Runs {
  int first, row_lo, len1, len2, sinks, tiles0, tiles1, t_all;
  __device__ inline Runs(const AttnParams& p, int b) {
    const int n = max(p.k_lens[b], 0), pos = n - 1, rest = p.lk - p.sinks;
    const int lo = (int)max((int64_t)0, (int64_t)pos - p.window + 1);
    sinks = p.sinks;
    first = n ? min(p.sinks, lo) : 0;
    row_lo = lo < p.lk ? lo : p.sinks + (lo - p.sinks) % rest;
    len1 = n ? min(pos - lo + 1, p.lk - row_lo) : 0;
    len2 = n ? pos - lo + 1 - len1 : 0;
    tiles0 = (first + kRows - 1) / kRows;
    tiles1 = (len1 + kRows - 1) / kRows;
    t_all = tiles0 + tiles1 + (len2 + kRows - 1) / kRows;
  }
  // First row and length of tile t; the last tile's last row is the newest token's.
  __device__ inline void tile(int t, int* row, int* rows) const {
    int at = t, base = 0, len = first;
    if (at >= tiles0) {
      at -= tiles0;
      base = row_lo;
      len = len1;
      if (at >= tiles1) {
        at -= tiles1;
        base = sinks;
        len = len2;
      }
    }
    *row = base + at * kRows;
    *rows = min(kRows, len - at * kRows);
  }
};
// Tiles that the rows of any sequence make at most: three runs end inside one.
__host__ __device__ inline int most_tiles(int lk) { return (lk + kRows - 1) / kRows + 2; }

// SCORES: the scores go to p.scores as well, in the log2 domain, [batch][heads][most_tiles][kRows].
template <int DT, int ND, bool SCORES>
__global__ void __launch_bounds__(kWaves * 64, 1) decode_kernel(const AttnParams p) {
  using L = DecodeLds<ND>;
  constexpr int RB = L::RB, NS = 2 * ND;
  using T = typename Elem<DT>::type;
  __shared__ __attribute__((aligned(16))) uint8_t smem[L::TOTAL];
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int blocks = (p.group + kHeads - 1) / kHeads;
  int id = blockIdx.x;
  const int split = id % p.splits;
  id /= p.splits;
  const int hb = id % blocks;
  id /= blocks;
  const int hk = id % p.kv_heads, b = id / p.kv_heads;
  const int h0 = hk * p.group + hb * kHeads, heads = min(kHeads, p.group - hb * kHeads);

  const Runs runs(p, b);
  const int t_all = runs.t_all;
  const int t0 = (int)((int64_t)t_all * split / p.splits), t1 = (int)((int64_t)t_all * (split + 1) / p.splits);

  u32x4 qf[NS];
  const int hq = lane & 31;
  load_row<NS>(p.q + 2 * (b * p.q_stride[0] + (int64_t)(h0 + hq) * p.q_stride[2]), hq < heads, p.dim, half, qf);
  const float c2 = positive_scale<NS>(p.scale, qf);
  f32x16 o[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int v = 0; v < 16; ++v) o[d][v] = 0.0f;
  float top = -INFINITY, total = 0.0f;

  TileLoader<RB, kRows, 1> lk, lv;
  lk.init(p.k + 2 * (b * p.k_stride[0] + hk * p.k_stride[2]), 2 * p.k_stride[1], p.dim, 0, lane);
  lv.init(p.v + 2 * (b * p.v_stride[0] + hk * p.v_stride[2]), 2 * p.v_stride[1], p.dim, 0, lane);
  constexpr int LOADS = 2 * TileLoader<RB, kRows, 1>::NB;
  uint8_t* ring = smem + wave * L::STAGES * L::STAGE;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(WTC_LDS uint8_t*)ring;
  auto issue = [&](int x) {  // this wave's x-th tile
    int row, rows;
    const int t = t0 + wave + x * kWaves;
    runs.tile(t, &row, &rows);
    if (t >= t1) rows = 0;
    const uint32_t st = lds0 + (uint32_t)x % L::STAGES * L::STAGE;
    lk.issue(st, row, rows);
    lv.issue(st + L::TILE, row, rows);
  };
#pragma unroll
  for (int x = 0; x < L::STAGES; ++x) issue(x);

  landed(qf);
  for (int x = 0; t0 + wave + x * kWaves < t1; ++x) {
    asm volatile("s_waitcnt vmcnt(%0)" : : "n"(LOADS * (L::STAGES - 1)) : "memory");
    int row, rows;
    const int t = t0 + wave + x * kWaves;
    runs.tile(t, &row, &rows);
    uint8_t* kt = ring + x % L::STAGES * L::STAGE;
    uint8_t* vt = kt + L::TILE;
    if (t == t_all - 1 && p.k_new && lane * 8 < p.dim) {  // the new token: over what the cache held in its row
      const u32x4 kn = *reinterpret_cast<const u32x4*>(p.k_new + 2 * (b * p.kn_stride[0] + hk * p.kn_stride[1]) + lane * 16);
      const u32x4 vn = *reinterpret_cast<const u32x4*>(p.v_new + 2 * (b * p.vn_stride[0] + hk * p.vn_stride[1]) + lane * 16);
      *reinterpret_cast<u32x4*>(kt + tile_offset<RB>(rows - 1, lane)) = kn;
      *reinterpret_cast<u32x4*>(vt + tile_offset<RB>(rows - 1, lane)) = vn;
      if (hb == 0) {
        const int64_t to = row + rows - 1;
        *reinterpret_cast<u32x4*>(const_cast<uint8_t*>(p.k) + 2 * (b * p.k_stride[0] + to * p.k_stride[1] + hk * p.k_stride[2]) + lane * 16) = kn;
        *reinterpret_cast<u32x4*>(const_cast<uint8_t*>(p.v) + 2 * (b * p.v_stride[0] + to * p.v_stride[1] + hk * p.v_stride[2]) + lane * 16) = vn;
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    uint32_t ka = row_addr<RB>(lane) + (uint32_t)(kt - smem), va = col_addr<RB>(lane) + (uint32_t)(vt - smem);
    fresh(ka);
    fresh(va);
    f32x16 s;
#pragma unroll
    for (int v = 0; v < 16; ++v) s[v] = 0.0f;
#pragma unroll
    for (int st = 0; st < NS; ++st) s = mfma32<DT>(row_frag<RB>(smem, ka, 0, st), qf[st], s);
    float m = -INFINITY;
#pragma unroll
    for (int v = 0; v < 16; ++v) {
      if (8 * (v >> 2) + (v & 3) + 4 * half >= rows) s[v] = -INFINITY;
      m = fmaxf(m, s[v]);
    }
    if constexpr (SCORES) {
      if (hq < heads) {
        float* dst = p.scores + (((int64_t)b * p.heads + h0 + hq) * most_tiles(p.lk) + t) * kRows + 4 * half;
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<f32x4*>(dst + 8 * g) = f32x4{s[4 * g] * c2, s[4 * g + 1] * c2, s[4 * g + 2] * c2, s[4 * g + 3] * c2};
      }
    }
    m = xor32_max(m) * c2;
    const float next = fmaxf(top, m);
    const float keep = next == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(top - next);
    if (__any(next > top)) {
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int v = 0; v < 16; ++v) o[d][v] *= keep;
    }
    top = next;
    const float ref = top == -INFINITY ? 0.0f : -top;
    u32x4 pf[2];
    float sum = 0.0f;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      f32x4 e;
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        e[v] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[4 * g + v], c2, ref));
        sum += e[v];
      }
      uint32_t w0, w1;
      pack4<DT>(e, &w0, &w1);
      pf[g >> 1][2 * (g & 1)] = w0;
      pf[g >> 1][2 * (g & 1) + 1] = w1;
    }
    total = __builtin_fmaf(total, keep, sum);
#pragma unroll
    for (int st = 0; st < 2; ++st)
#pragma unroll
      for (int d = 0; d < ND; ++d) o[d] = mfma32<DT>(col_frag<RB>(smem, va, 16 * st, d), pf[st], o[d]);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the tile is read: its stage may be filled again
    issue(x + L::STAGES);
  }
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __syncthreads();

  // ---- join the waves: head q's result at [wave][q][PITCH], its (maximum, sum) behind them
  total = xor32_sum(total);
  float* res = reinterpret_cast<float*>(smem);
  float2* stat = reinterpret_cast<float2*>(smem + L::TOTAL - kWaves * kHeads * 8);
  if (hq < heads) {
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<f32x4*>(res + (wave * kHeads + hq) * L::PITCH + 32 * d + 8 * g + 4 * half) =
            f32x4{o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]};
    if (half == 0) stat[wave * kHeads + hq] = float2{top, total};
  }
  __syncthreads();
  const int per = p.dim / 8;  // 8 elements a thread
  for (int x = threadIdx.x; x < heads * per; x += kWaves * 64) {
    const int q = x / per, c = x % per * 8;
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) m = fmaxf(m, stat[w * kHeads + q].x);
    const float ref = m == -INFINITY ? 0.0f : m;
    float sum = 0.0f, y[8] = {};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      // (a wave without keys has a maximum of -inf and zeros; one whose scores are all NaN
      // has that maximum too, which leaves NaN out, and its sum says so)
      const float2 st = stat[w * kHeads + q];
      const float f = __builtin_amdgcn_exp2f(st.x - ref);
      sum = __builtin_fmaf(st.y, f, sum);
      const float* src = res + (w * kHeads + q) * L::PITCH + c;
#pragma unroll
      for (int u = 0; u < 8; ++u) y[u] = __builtin_fmaf(src[u], f, y[u]);
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int u = 0; u < 8; ++u) y[u] *= inv;
    if (p.slots) {
      const int64_t row = ((int64_t)b * p.heads + h0 + q) * p.slots + p.slot0 + split;
      f32x4* dst = reinterpret_cast<f32x4*>(p.part_out + row * p.dim + c);
      dst[0] = f32x4{y[0], y[1], y[2], y[3]};
      dst[1] = f32x4{y[4], y[5], y[6], y[7]};
      if (c == 0) p.part_lse[row] = sum == 0.0f ? -INFINITY : m + __builtin_amdgcn_logf(sum);
    } else {
      uint32_t w[4];
      pack4<DT>(f32x4{y[0], y[1], y[2], y[3]}, &w[0], &w[1]);
      pack4<DT>(f32x4{y[4], y[5], y[6], y[7]}, &w[2], &w[3]);
      *reinterpret_cast<u32x4*>(p.out + 2 * (b * p.o_stride[0] + (int64_t)(h0 + q) * p.o_stride[2] + c)) = u32x4{w[0], w[1], w[2], w[3]};
    }
  }
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
// take 256 tile rows of a (sequence, key head), those behind them join the splits
// as decode_join_kernel does.
constexpr int kHeadsAtOnce = 64;
template <int DT>
__global__ void __launch_bounds__(256) decode_weights_kernel(const AttnParams p, int weight_blocks, int chunks) {
  if ((int)blockIdx.x >= weight_blocks) {
    join_row<DT>(p, (int64_t)((int)blockIdx.x - weight_blocks) * 8 + (threadIdx.x >> 5));
    return;
  }
  __shared__ float lse[kHeadsAtOnce];
  const int chunk = (int)blockIdx.x % chunks, seq = (int)blockIdx.x / chunks, b = seq / p.kv_heads, hk = seq % p.kv_heads;
  const Runs runs(p, b);
  const int x = chunk * 256 + threadIdx.x, t = x / kRows;
  if (chunk * 256 / kRows >= runs.t_all) return;  // (the whole workgroup)
  int row = 0, rows = 0;
  if (t < runs.t_all) runs.tile(t, &row, &rows);
  const bool in = x % kRows < rows;
  float sum = 0.0f;
  for (int g0 = 0; g0 < p.group; g0 += kHeadsAtOnce) {
    const int heads = min(kHeadsAtOnce, p.group - g0);
    const int64_t h0 = (int64_t)b * p.heads + hk * p.group + g0;
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
    if (in) {
      const float* score = p.scores + h0 * most_tiles(p.lk) * kRows + x;
      for (int g = 0; g < heads; ++g) sum += __builtin_amdgcn_exp2f(score[(int64_t)g * most_tiles(p.lk) * kRows] - lse[g]);
    }
  }
  if (!in) return;
  float* w = p.weights + (int64_t)seq * p.lk + row + x % kRows;
  *w = t == runs.t_all - 1 && x % kRows == rows - 1 ? sum : *w + sum;
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
// Sequences of unequal length leave CUs idle at the end: splits until the chip has two
// workgroups a CU, one after another, while a wave keeps at least 4 tiles.
int plan_decode_joined(const AttnParams& p, int cu_count) {
  const int64_t grid = (int64_t)p.batch * p.kv_heads * ((p.group + kHeads - 1) / kHeads);
  const int64_t tiles = (std::min<int64_t>(p.lk, p.window + p.sinks) + kRows - 1) / kRows;
  int splits = 1;
  while (splits < 64 && grid * splits < 2 * cu_count && tiles / (2 * splits) >= 4 * kWaves) splits *= 2;
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
int64_t decode_grid(const AttnParams& p) { return (int64_t)p.batch * p.kv_heads * ((p.group + kHeads - 1) / kHeads) * p.splits; }
}  // namespace

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
  int chunks = (most_tiles(p.lk) * kRows + 255) / 256, weight_blocks = p.batch * p.kv_heads * chunks;
  void* args[] = {&p, &weight_blocks, &chunks};
  const int nd = (p.dim + 31) / 32;
  const hipError_t e = launch(dt == DT_F16 ? kernel_for<DT_F16, true>(nd) : kernel_for<DT_BF16, true>(nd), decode_grid(p), args, stream);
  if (e != hipSuccess) return e;
  return launch(dt == DT_F16 ? (const void*)&decode_weights_kernel<DT_F16> : (const void*)&decode_weights_kernel<DT_BF16>,
                weight_blocks + (rows + 7) / 8, args, stream);
}

}  // namespace wtc
