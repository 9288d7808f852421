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
// add the 32 columns.  A score costs a lane 24 cycles of its SIMD (16 of them the
// exponential) and 16 of the matrix cores: so 32 rows' exponentials against 32
// keys run among the products of the next ones, and the loop is kept short of scalar work,
// which a wave issues like any other instruction.
// Long sequences go in chunks of queries, whose sums a second kernel adds in their order.
// 4096 causal tokens, 32 / 8 heads of 128, bf16: 101 us, 680 TFLOP/s of the visible half
// (exponentials after their products instead of among the next ones: 127); eight such
// sequences 79 each.  Alone, its workgroups with queries are 488, of up to 40 tiles where 34
// would be equal shares of one round.
#include <algorithm>
#include <cmath>

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

// x[0 .. N) of the 2 N lanes whose numbers agree above bit log2(N) are summed over the lanes
// of each half of 32; a lane's x[0] is then the sum of x[lane % N].
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

// Queries i0 .. i1 - 1 of a chunk that may see a key of block kb: the block's queries in as
// many equal chunks as keep within chunk_rows.
struct Chunk {
  int i0, i1;
  __device__ inline Chunk(const AttnParams& p, int nq, int nk, int kb, int chunk, int chunk_rows, int tile_rows) {
    const int shift = first_position(p, nq, nk), j_first = kb * kKeys;
    const int lo = min(max(0, j_first - shift), nq);
    int hi = j_first < p.sinks ? nq : (int)max((int64_t)lo, min((int64_t)nq, (int64_t)min(j_first + kKeys, nk) - 1 + p.window - shift));
    if (j_first >= nk) hi = lo;
    const int chunks = (hi - lo + chunk_rows - 1) / chunk_rows, tiles = (hi - lo + tile_rows - 1) / tile_rows;
    const int share = chunks ? (tiles + chunks - 1) / chunks * tile_rows : 0;
    i0 = (int)min((int64_t)hi, lo + (int64_t)chunk * share);
    i1 = min(hi, i0 + share);
  }
};
__device__ inline int clamp32(int64_t x) { return (int)min((int64_t)INT32_MAX, max((int64_t)INT32_MIN, x)); }

template <int DT, int ND>
__global__ void __launch_bounds__(kWaves * 64, 2) key_weights_kernel(const AttnParams p, int chunk_rows) {
  using L = WeightsLds<ND>;
  constexpr int RB = L::RB, NS = 2 * ND, NB = kRows * RB / 1024 / kWaves;
  __shared__ __attribute__((aligned(256))) uint8_t smem[L::TOTAL];
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t id = xcd_remap(blockIdx.x, gridDim.x);
  // (the chunks that a causal sequence's last blocks do not have come last)
  const int kb = (int)(id % p.key_blocks), chunk = (int)(id / p.key_blocks % p.splits);
  const int hk = (int)(id / p.splits / p.key_blocks % p.kv_heads), b = (int)(id / p.splits / p.key_blocks / p.kv_heads);
  const int nk = seq_keys(p, b), nq = seq_queries(p, b), shift = first_position(p, nq, nk);
  const int j_wave = kb * kKeys + wave * 64;
  const int hg = min(p.group, kRows), groups = (p.group + hg - 1) / hg, tp = kRows / hg;  // heads, parts, positions of a tile
  const auto [i0, i1] = Chunk(p, nq, nk, kb, chunk, chunk_rows, tp);
  if (p.splits > 1 && i0 == i1) return;  // (nothing to add: the second kernel knows)

  const uint8_t* q_base = p.q + 2 * (b * p.q_stride[0] + (int64_t)hk * p.group * p.q_stride[2]);
  uint32_t q_off[NB], at_row[NB];  // at_row: position and head (high half)
#pragma unroll
  for (int q = 0; q < NB; ++q) {
    const int row = (int)block_row<RB>(wave * NB + q, lane);
    const uint32_t c = block_chunk<RB>(wave * NB + q, lane) * 16u;
    at_row[q] = (uint32_t)(row / hg | row % hg << 16);
    q_off[q] = c < (uint32_t)p.dim * 2u && row < tp * hg ? (uint32_t)(2 * (row / hg * p.q_stride[1] + row % hg * p.q_stride[2])) + c : kOutOfRange;
  }
  const uint32_t lse_row = (uint32_t)(lane / hg | lane % hg << 16), lse_off = lane < tp * hg ? (uint32_t)(4 * (lane % hg * (int64_t)p.lq + lane / hg)) : kOutOfRange;
  const uint32_t x_row[2] = {(uint32_t)((lane & 31) / hg | (lane & 31) % hg << 16), (uint32_t)((32 + (lane & 31)) / hg | (32 + (lane & 31)) % hg << 16)};
  const uint32_t lds0 = (uint32_t)(uintptr_t)(WTC_LDS uint8_t*)smem;
  // The next tile to load: its positions from `i`, its heads from head part `part` (of `groups`).
  struct {
    const uint8_t *q, *lse;
    uint32_t at;
    int i, part;
  } next = {q_base + 2 * i0 * p.q_stride[1], reinterpret_cast<const uint8_t*>(p.lse_in + ((int64_t)b * p.heads + hk * p.group) * p.lq + i0), 0, i0, 0};
  const int64_t q_part = 2 * hg * p.q_stride[2], q_step = 2 * tp * p.q_stride[1] - (groups - 1) * q_part;
  const int64_t lse_part = 4 * (int64_t)hg * p.lq, lse_step = 4 * tp - (groups - 1) * lse_part;
  auto issue = [&]() __attribute__((always_inline)) {
    const int npos = i1 - next.i, nhead = p.group - next.part * hg;
    const i32x4 rq = raw_rsrc(next.q, 0x7FFFFFFFu), rl = raw_rsrc(next.lse, 0x7FFFFFFFu);
    if (npos >= tp && nhead >= hg) {
#pragma unroll
      for (int q = 0; q < NB; ++q) dma16(rq, q_off[q], lds0 + next.at + wave * NB * 1024 + q * 1024);
      if (wave == 0) dma4(rl, lse_off, lds0 + next.at + L::TILE);
    } else {
#pragma unroll
      for (int q = 0; q < NB; ++q) {
        const bool in = (int)(at_row[q] & 0xFFFFu) < npos && (int)(at_row[q] >> 16) < nhead;
        dma16(rq, in ? q_off[q] : kOutOfRange, lds0 + next.at + wave * NB * 1024 + q * 1024);
      }
      const bool in = (int)(lse_row & 0xFFFFu) < npos && (int)(lse_row >> 16) < nhead;
      if (wave == 0) dma4(rl, in ? lse_off : kOutOfRange, lds0 + next.at + L::TILE);
    }
    const bool last = next.part + 1 == groups;
    next.q += last ? q_step : q_part;
    next.lse += last ? lse_step : lse_part;
    next.i += last ? tp : 0;
    next.part = last ? 0 : next.part + 1;
    next.at = next.at + L::STAGE == L::TOTAL ? 0 : next.at + L::STAGE;
  };
#pragma unroll
  for (int t = 0; t < L::STAGES - 1; ++t) issue();

  u32x4 kf[2][NS];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int j = j_wave + 32 * u + (lane & 31);
    load_row<NS>(p.k + 2 * (b * p.k_stride[0] + (int64_t)j * p.k_stride[1] + hk * p.k_stride[2]), j < nk, p.dim, half, kf[u]);
  }
  const float c2 = positive_scale<NS>(p.scale, kf[0]);
  positive_scale<NS>(p.scale, kf[1]);
  landed(kf[0]);
  landed(kf[1]);

  // Tiles whose first position is i: [see0, see1) has rows that see keys of the wave, and in
  // [all0, all1) every row of a whole tile sees all of them.
  const bool sink = j_wave < p.sinks, sinks = j_wave + 63 < p.sinks;
  const int see0 = j_wave < nk ? clamp32((int64_t)j_wave - shift - tp + 1) : INT32_MAX;
  const int see1 = sink ? INT32_MAX : clamp32((int64_t)j_wave + 63 + p.window - shift);
  const int all0 = clamp32((int64_t)j_wave + 63 - shift);
  const int all1 = min(i1 - tp + 1, sinks ? INT32_MAX : clamp32((int64_t)j_wave + p.window - shift - tp + 1));
  const bool whole = tp * hg == kRows && groups * hg == p.group && j_wave + 64 <= nk;

  // Weights of 32 rows by 32 keys, whose scores are in one of s, while the matrix cores take
  // the next ones into the other; a tile's last ones in the next tile that the wave
  // computes.  (With 64 keys at a time half of the fragment reads would do, but the
  // registers of two waves a SIMD do not hold their scores twice.)
  float sums[32];
#pragma unroll
  for (int v = 0; v < 32; ++v) sums[v] = 0.0f;
  f32x16 s[2];
#pragma unroll
  for (int v = 0; v < 16; ++v) s[1][v] = 0.0f;
  float off = -INFINITY;  // minus the log-sum-exp of the lane's row, log2 domain
  uint64_t seen = 0;
  const uint32_t r_at = row_addr<RB>(lane);
  constexpr int AHEAD = NS < 3 ? NS : 3;
  u32x4 frag[NS + AHEAD];  // the first AHEAD ones of a phase were read in the one before
  // Scores in groups of 16 / NS: exponents, exponentials and sums of a group in three steps,
  // one after another, so that none waits for the one before.
  auto weigh = [&](auto mask, f32x16& of, int x, int y, int what) __attribute__((always_inline)) {  // keys 32 x ..
#pragma unroll
    for (int v = 0; v < 16; ++v) {
      if (v * NS / 16 != y) continue;
      if (what == 0) of[v] = __builtin_fmaf(of[v], c2, off);
      if (what == 1) of[v] = __builtin_amdgcn_exp2f(of[v]);
      if (what == 2) {
        if constexpr (decltype(mask)::value) of[v] = zero_bit(of[v], seen, 32 * x + 8 * (v >> 2) + (v & 3));
        sums[16 * x + v] += of[v];
      }
    }
  };
  auto phase = [&](auto mask, uint32_t ra, int u, int x) __attribute__((always_inline)) {
    weigh(mask, s[x ^ 1], x ^ 1, 0, 0);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int y = 0; y < NS; ++y) {
      if (y + AHEAD < NS) frag[y + AHEAD] = row_frag<RB>(smem, ra, 32 * u, y + AHEAD);
      else if (!(u == 1 && x == 1)) frag[y + AHEAD] = row_frag<RB>(smem, ra, 32 * (u + x), y + AHEAD - NS);
      const f32x16 zero = {};
      s[x] = mfma32<DT>(kf[x][y], frag[y], y == 0 ? zero : s[x]);
      weigh(mask, s[x ^ 1], x ^ 1, y + 1, 0);
      weigh(mask, s[x ^ 1], x ^ 1, y, 1);
      weigh(mask, s[x ^ 1], x ^ 1, y - 1, 2);
      __builtin_amdgcn_sched_barrier(0);
    }
    weigh(mask, s[x ^ 1], x ^ 1, NS - 1, 2);
#pragma unroll
    for (int y = 0; y < AHEAD; ++y) frag[y] = frag[NS + y];
  };
  uint32_t stage = 0;
  int i = i0, part = 0;
  auto tile = [&](auto mask) __attribute__((always_inline)) {
    // the tile landed; every wave is done with the last one (wave 0 has one load more a tile)
    if (wave == 0) wait_loads_barrier<(NB + 1) * (L::STAGES - 2)>();
    else wait_loads_barrier<NB * (L::STAGES - 2)>();
    issue();
    if (!decltype(mask)::value || (i >= see0 && i < see1)) {
      uint32_t ra = r_at + stage;
      fresh(ra);
#pragma unroll
      for (int y = 0; y < AHEAD; ++y) frag[y] = row_frag<RB>(smem, ra, 0, y);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const float lse = *reinterpret_cast<const float*>(smem + stage + L::TILE + (32 * u + (lane & 31)) * 4) * -kLog2e;
        phase(mask, ra, u, 0);
        off = lse == INFINITY ? -INFINITY : lse;  // a row of scores -inf weighs nothing
        if constexpr (decltype(mask)::value) {
          const int pos = (int)(x_row[u] & 0xFFFFu);
          const bool row = pos < min(tp, i1 - i) && (int)(x_row[u] >> 16) < p.group - part * hg;
          seen = row ? seen_bits(j_wave + 4 * half, nk, (int64_t)i + pos + shift, p.window, p.sinks) : 0;
        }
        phase(mask, ra, u, 1);
      }
    }
    part = part + 1 == groups ? 0 : part + 1;
    i += part ? 0 : tp;
    stage = stage + L::STAGE == L::TOTAL ? 0 : stage + L::STAGE;
  };
  auto finish = [&](auto mask) __attribute__((always_inline)) {  // the scores that wait
#pragma unroll
    for (int z = 0; z < 3 * NS; ++z) weigh(mask, s[1], 1, z / 3, z % 3);
#pragma unroll
    for (int v = 0; v < 16; ++v) s[1][v] = 0.0f;
    off = -INFINITY;
  };
  // (loops of their own: a tile that asks inside for its mask has both sides' common work,
  // exponents and sums, moved before and behind its products)
  const int fast0 = whole ? all0 : INT32_MAX;
  while (i < i1) {
    while (i < i1 && !(i >= fast0 && i < all1)) tile(std::true_type{});
    finish(std::true_type{});
    while (i >= fast0 && i < all1) tile(std::false_type{});
    finish(std::false_type{});
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

// One key a thread, the chunks that see its block in their order.
__global__ void __launch_bounds__(256) key_weights_sum_kernel(const AttnParams p, int chunk_rows) {
  const int blocks = (p.lk + kKeys - 1) / kKeys, kb = (int)(blockIdx.x % blocks);
  const int64_t seq = blockIdx.x / blocks;
  const int b = (int)(seq / p.kv_heads), j = kb * kKeys + (int)threadIdx.x;
  const int nk = seq_keys(p, b), nq = seq_queries(p, b);
  if (j >= p.lk) return;
  float sum = 0.0f;
  if (j < nk) {
    for (int c0 = 0; c0 < p.splits; c0 += 8) {  // 8 loads at a time
      float x[8];
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        x[c] = 0.0f;
        if (c0 + c >= p.splits) continue;
        const Chunk of(p, nq, nk, kb, c0 + c, chunk_rows, kRows / min(p.group, kRows));
        if (of.i0 < of.i1) x[c] = p.part_out[(seq * p.splits + c0 + c) * p.lk + j];
      }
#pragma unroll
      for (int c = 0; c < 8; ++c) sum += x[c];
    }
  }
  float* dst = p.weights + seq * p.lk + j;
  *dst = p.add ? *dst + sum : sum;
}
static_assert(kKeys == 256, "a key block is a workgroup of the sum kernel");

template <int DT> const void* kernel_for(int nd) {
  switch (nd) {
    case 1: return (const void*)&key_weights_kernel<DT, 1>;
    case 2: return (const void*)&key_weights_kernel<DT, 2>;
    case 3: return (const void*)&key_weights_kernel<DT, 3>;
  }
  return (const void*)&key_weights_kernel<DT, 4>;
}

}  // namespace

// Chunks of the queries, so that the rounds of workgroups (two a CU) times what each
// takes are least: its tiles and about eight tiles' time for its start and end.
KeyWeightsPlan plan_key_weights(const AttnParams& p, int cu_count) {
  KeyWeightsPlan plan{};
  plan.key_blocks = (p.lk + kKeys - 1) / kKeys;
  const int64_t seqs = (int64_t)p.batch * p.kv_heads;
  const int hg = std::min(p.group, kRows), parts = (p.group + hg - 1) / hg, tp = kRows / hg;
  // positions that see a key of the first, middle, ... block
  constexpr int SAMPLES = 16;
  int64_t seen[SAMPLES];
  for (int i = 0; i < SAMPLES; ++i) {
    const int64_t j = (2 * i + 1) * (int64_t)p.lk / (2 * SAMPLES) / kKeys * kKeys, lo = std::max<int64_t>(0, j - (p.lk - p.lq));
    const int64_t hi = j < p.sinks ? p.lq : std::min<int64_t>(p.lq, j + kKeys - 1 + p.window - (p.lk - p.lq));
    seen[i] = std::max<int64_t>(0, hi - lo);
  }
  double least = 1e30;
  for (int64_t tiles = 4, end = (p.lq + tp - 1) / tp;; tiles += std::max<int64_t>(1, tiles / 16)) {  // positions' tiles a chunk
    tiles = std::min(tiles, std::max<int64_t>(1, end));
    int64_t chunks = 0;
    for (int i = 0; i < SAMPLES; ++i) chunks += std::max<int64_t>(1, (seen[i] + tiles * tp - 1) / (tiles * tp));
    const double groups = (double)seqs * plan.key_blocks * chunks / SAMPLES;
    const double us = std::ceil(groups / (2 * cu_count)) * (tiles * parts + 8) + (tiles < end ? 4 : 0);
    if (us < least) {
      least = us;
      plan.chunk_rows = (int)(tiles * tp);
    }
    if (tiles >= end) break;
  }
  plan.chunks = std::max(1, (p.lq + plan.chunk_rows - 1) / plan.chunk_rows);
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
  return hipLaunchKernel((const void*)&key_weights_sum_kernel, dim3((unsigned)((int64_t)p.batch * p.kv_heads * p.key_blocks)),
                         dim3(kKeys), args, 0, stream);
}

}  // namespace wtc
