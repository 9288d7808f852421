// decode_tile.h -- a workgroup's part of attention of few rows against many keys; what
// bounds it and why it is as it is stands in window_decode.hip.
#pragma once
#include "attention_common.h"

namespace wtc {
namespace decode {

using namespace attn;

constexpr int kRows = 32;   // cache rows a tile
constexpr int kWaves = 4;
constexpr int kHeads = 32;  // query heads a workgroup

// GROUPS: workgroups a CU.
template <int ND, int GROUPS> struct DecodeLds {
  static constexpr int RB = row_bytes(ND);
  static constexpr int TILE = kRows * RB, STAGE = 2 * TILE;
  static constexpr int STAGES = (RB == 256 ? 2 : 4) / GROUPS;  // 128 KiB a CU
  static constexpr int RING = kWaves * STAGES * STAGE;
  static constexpr int PITCH = ND * 32 + 4;          // floats of a head's result
  static constexpr int JOIN = kWaves * kHeads * PITCH * 4;
  static constexpr int TOTAL = (RING > JOIN ? RING : JOIN) + kWaves * kHeads * 8;
  static_assert(TOTAL * GROUPS <= 160 * 1024, "LDS");
};

// The visible rows of a sequence's cache as tiles.
struct Runs {
  int first, row_lo, len1, len2, sinks, tiles0, tiles1, t_all;
  __device__ inline Runs(const AttnParams& p, int n) {  // n tokens
    const int pos = n - 1, rest = p.lk - p.sinks;
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

// ROWS: the rows are those of p.lq queries, each of which sees every key, instead of one
// query's heads; a batch's queries may be one sequence's (p.seq_rows).
// SCORES: the scores go to p.scores as well, in the log2 domain, [batch][heads][most_tiles][kRows].
template <int DT, int ND, bool SCORES, bool ROWS, int GROUPS>
__device__ inline void decode_tile(const AttnParams& p, uint8_t* smem, int id) {
  using L = DecodeLds<ND, GROUPS>;
  constexpr int RB = L::RB, NS = 2 * ND;
  using T = typename Elem<DT>::type;
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int all_rows = ROWS ? p.lq * p.group : p.group, blocks = (all_rows + kHeads - 1) / kHeads;
  const int split = id % p.splits;
  id /= p.splits;
  const int hb = id % blocks;
  id /= blocks;
  const int hk = id % p.kv_heads, b = id / p.kv_heads;
  // rows (ROWS) or query heads of the workgroup
  const int h0 = hk * p.group + hb * kHeads, heads = min(kHeads, all_rows - hb * kHeads);
  auto row_query = [&](int q) { return ROWS ? (hb * kHeads + q) / p.group : 0; };
  auto row_head = [&](int q, int i) { return ROWS ? hk * p.group + hb * kHeads + q - i * p.group : h0 + q; };
  const int nq = ROWS ? seq_queries(p, b) : 1;

  const Runs runs(p, ROWS ? seq_keys(p, b) : max(p.k_lens[b], 0));
  const int t_all = runs.t_all;
  const int t0 = (int)((int64_t)t_all * split / p.splits), t1 = (int)((int64_t)t_all * (split + 1) / p.splits);

  u32x4 qf[NS];
  const int hq = lane & 31;
  {
    const int i = row_query(hq), seq = ROWS && p.seq_rows ? i / p.seq_rows : b, row = ROWS && p.seq_rows ? i % p.seq_rows : i;
    load_row<NS>(p.q + 2 * (seq * p.q_stride[0] + row * p.q_stride[1] + (int64_t)row_head(hq, i) * p.q_stride[2]),
                 hq < heads && i < nq, p.dim, half, qf);
  }
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
  // The loads, stores too, count in their order: those that may be in flight when a tile's keys,
  // or its values, have landed (of each tensor STAGES tiles are under way, and from the
  // second tile on the scores of the one before).
  constexpr int BEHIND = TileLoader<RB, kRows, 1>::NB * (2 * L::STAGES - 1), STORES = SCORES ? 4 : 0;
  auto wait = [](bool first) __attribute__((always_inline)) {
    if (first) asm volatile("s_waitcnt vmcnt(%0)" : : "n"(BEHIND) : "memory");
    else asm volatile("s_waitcnt vmcnt(%0)" : : "n"(BEHIND + STORES) : "memory");
  };
  uint8_t* ring = smem + wave * L::STAGES * L::STAGE;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(WTC_LDS uint8_t*)ring;
  auto issue = [&](auto& of, int x, int at) __attribute__((always_inline)) {  // this wave's x-th tile
    int row, rows;
    const int t = t0 + wave + x * kWaves;
    runs.tile(t, &row, &rows);
    of.issue(lds0 + (uint32_t)x % L::STAGES * L::STAGE + at, row, t < t1 ? rows : 0);
  };
#pragma unroll
  for (int x = 0; x < L::STAGES; ++x) {
    issue(lk, x, 0);
    issue(lv, x, L::TILE);
  }

  landed(qf);
  for (int x = 0; t0 + wave + x * kWaves < t1; ++x) {
    int row, rows;
    const int t = t0 + wave + x * kWaves;
    runs.tile(t, &row, &rows);
    wait(x == 0);
    uint8_t* kt = ring + x % L::STAGES * L::STAGE;
    uint8_t* vt = kt + L::TILE;
    if (!ROWS && t == t_all - 1 && p.k_new && lane * 8 < p.dim) {  // the new token: over what the cache held in its row
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
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
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the keys are read: their place may be filled again
    issue(lk, x + L::STAGES, 0);
    float m = -INFINITY;
#pragma unroll
    for (int v = 0; v < 16; ++v) {
      if (8 * (v >> 2) + (v & 3) + 4 * half >= rows) s[v] = -INFINITY;
      m = fmaxf(m, s[v]);
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
    wait(x == 0);
#pragma unroll
    for (int st = 0; st < 2; ++st)
#pragma unroll
      for (int d = 0; d < ND; ++d) o[d] = mfma32<DT>(col_frag<RB>(smem, va, 16 * st, d), pf[st], o[d]);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    issue(lv, x + L::STAGES, L::TILE);
    if constexpr (SCORES) {
      if (hq < heads) {
        float* dst = p.scores + (((int64_t)b * p.heads + h0 + hq) * most_tiles(p.lk) + t) * kRows + 4 * half;
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<f32x4*>(dst + 8 * g) = f32x4{s[4 * g] * c2, s[4 * g + 1] * c2, s[4 * g + 2] * c2, s[4 * g + 3] * c2};
      }
    }
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
    const int i = row_query(q), h = row_head(q, i);
    const float lse = sum == 0.0f ? -INFINITY : m + __builtin_amdgcn_logf(sum);
    if (p.slots) {
      const int64_t row = (((int64_t)b * (ROWS ? p.lq : 1) + i) * p.heads + h) * p.slots + p.slot0 + split;
      f32x4* dst = reinterpret_cast<f32x4*>(p.part_out + row * p.dim + c);
      dst[0] = f32x4{y[0], y[1], y[2], y[3]};
      dst[1] = f32x4{y[4], y[5], y[6], y[7]};
      if (c == 0) p.part_lse[row] = lse;
    } else {
      const bool valid = !ROWS || i < nq;
      uint32_t w[4];
#pragma unroll
      for (int u = 0; u < 8; ++u) y[u] = valid ? y[u] : 0.0f;
      if (ROWS && p.lse && c == 0) p.lse[((int64_t)b * p.heads + h) * p.lq + i] = valid ? lse * kLn2 : -INFINITY;
      pack4<DT>(f32x4{y[0], y[1], y[2], y[3]}, &w[0], &w[1]);
      pack4<DT>(f32x4{y[4], y[5], y[6], y[7]}, &w[2], &w[3]);
      *reinterpret_cast<u32x4*>(p.out + 2 * (b * p.o_stride[0] + i * p.o_stride[1] + (int64_t)h * p.o_stride[2] + c)) = u32x4{w[0], w[1], w[2], w[3]};
    }
  }
}

}  // namespace decode
}  // namespace wtc
