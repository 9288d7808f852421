// rows_tile.h -- a workgroup's part of forward attention of many query rows that see
// (nearly) all of their keys:
//   S^T = K . Q^T,  W = exp2(c S - ref),  O^T += V^T . W^T,  total += sum W,
// and at the end O / total and ref + log2 total.
//
// What bounds it: a unit of 32 keys against 32 rows is 8 ND products of 8 passes (at
// ND = 4, 256 cycles of a SIMD's matrix core) beside 16 exponentials, 16 multiply-adds,
// 16 additions and 8 conversions a lane, about 300 cycles of its vector unit, and a
// fragment read from LDS feeds one product a row block.  So
// - a wave owns two row blocks (64 rows, whose queries stay in registers) and reads each
//   key and value fragment once for both: one a wave needs the whole of LDS's bandwidth;
// - unit n's weights are taken among the products of unit n + 1's scores and n - 1's
//   values, in steps of one fragment each: the two pipes work at once, and no
//   product waits for a weight;
// - no running maximum is kept.  The weights' own sum, needed anyway, says whether a row
//   has outgrown its reference (kMostSum), which happens once or twice a row;
// - keys and values go straight to LDS through a ring of three stages of two units, one
//   barrier a stage.
// 4 x 2048 rows on 4096 keys, 32 / 8 heads of 128, bf16: 475 us, 1160 TFLOP/s, in which the
// matrix cores are busy 57 % of the cycles; the clock is held at 1.89 GHz by the power
// that this takes.  Tiles of 32 rows a wave with a maximum a tile: 680 us.
#pragma once
#include "attention_common.h"
#include "rows_schedule.h"

namespace wtc {
namespace rows {

using namespace attn;

constexpr int kRows = 256;  // query rows a workgroup
// A: the row blocks of 32 that a wave owns.
constexpr int waves(int a) { return kRows / 32 / a; }
constexpr int kUnit = 32;           // keys
// The reference that a row's exponentials are taken against is only moved when 16 of
// them pass this in sum (weights then stay below it, and sums far from f16's and f32's
// ends): no maximum is taken of the other scores.
constexpr float kMostSum = 1024.0f;

template <int ND, int A> struct RowsLds {
  static constexpr int RB = row_bytes(ND), STAGES = RowsSchedule<ND, false, A>::STAGES;
  static constexpr int HALF = kUnit * RB, STAGE = 4 * HALF;
  static constexpr int PITCH = ND * 64 + 16;  // bytes of a row staged for the output
  static constexpr int RING = STAGES * STAGE, OUT = waves(A) * 32 * PITCH;
  static constexpr int TOTAL = RING > OUT ? RING : OUT;
  static_assert(TOTAL <= 160 * 1024, "LDS");
};

// Loads of two units by four waves, of which each loads part of both.
template <int RB> struct UnitLoader {
  static constexpr int NB = kUnit * RB / 1024 / 4;
  const uint8_t* base;
  uint32_t stride;  // bytes
  uint32_t off[2 * NB];
  __device__ inline void init(const uint8_t* base_, int64_t stride_bytes, int dim, int wave, int lane) {
    base = base_;
    stride = (uint32_t)stride_bytes;
#pragma unroll
    for (int q = 0; q < 2 * NB; ++q) {
      const int block = wave * NB + q % NB;
      const uint32_t c = block_chunk<RB>(block, lane) * 16u;
      off[q] = c < (uint32_t)dim * 2u ? (block_row<RB>(block, lane) + kUnit * (q / NB)) * stride + c : kOutOfRange;
    }
  }
  __device__ inline i32x4 rows(const uint8_t* at, int n, uint32_t dim_bytes) const {
    return raw_rsrc(at, n > 0 ? (uint32_t)(n - 1) * stride + dim_bytes : 0u);
  }
  // rows row0 .. row0 + n - 1 (0: zeros) of one unit
  __device__ inline void issue(uint32_t to, int row0, int n, uint32_t dim_bytes) const {
    const i32x4 r = rows(base + (uint64_t)(uint32_t)row0 * stride, n, dim_bytes);
#pragma unroll
    for (int q = 0; q < NB; ++q) dma16(r, off[q], to + q * 1024);
  }
  // of two
  __device__ inline void issue2(uint32_t to, const uint8_t* at, int n, uint32_t dim_bytes) const {
    const i32x4 r = rows(at, min(n, 2 * kUnit), dim_bytes);
#pragma unroll
    for (int q = 0; q < 2 * NB; ++q) dma16(r, off[q], to + (q / NB) * (kUnit * RB) + q % NB * 1024);
  }
};

template <int DT> __device__ inline uint32_t pack2(float a, float b) {
  if constexpr (DT == DT_F16) return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, f16x2));
  else return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, bf16x2));
}

// PREFIX: p.prefix keys before the own ones, of which a row sees those up to its own position.
template <int DT, int ND, bool PREFIX, int A>
__device__ inline void attention_rows(const AttnParams& p, uint8_t* smem, uint32_t id) {
  using L = RowsLds<ND, A>;
  using Order = RowsSchedule<ND, PREFIX, A>;
  constexpr int RB = L::RB, NS = Order::FRAGS;
  using Loader = UnitLoader<RB>;
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int split = (int)(id % p.splits);
  const uint32_t rest = id / p.splits;
  const int blk = p.row_blocks - 1 - (int)(rest % p.row_blocks);
  const int hk = (int)(rest / p.row_blocks % p.kv_heads), b = (int)(rest / p.row_blocks / p.kv_heads);
  const int nk = seq_keys(p, b), nq = seq_queries(p, b), shift = first_position(p, nq, nk);
  const int r0 = blk * kRows;

  // this lane's rows; `sees`: own keys that a row sees
  int i[A], h[A], sees[A];
  bool valid[A];
  u32x4 qf[A][NS];
  float c2 = 0.0f;
#pragma unroll
  for (int a = 0; a < A; ++a) {
    const int r = r0 + wave * 32 * A + 32 * a + (lane & 31);
    i[a] = r / p.group;
    h[a] = hk * p.group + r - i[a] * p.group;
    valid[a] = i[a] < nq;
    sees[a] = valid[a] ? min(max(i[a] + shift + 1, 0), nk) : 0;
    const int q_seq = p.seq_rows ? i[a] / p.seq_rows : b, q_row = p.seq_rows ? i[a] % p.seq_rows : i[a];
    load_row<NS>(p.q + 2 * (q_seq * p.q_stride[0] + (int64_t)q_row * p.q_stride[1] + h[a] * p.q_stride[2]), valid[a], p.dim, half, qf[a]);
    c2 = positive_scale<NS>(p.scale, qf[a]);
    if constexpr (A == 2 && ND >= 3) {  // (one wave a SIMD) the products read them in the accumulation registers
#pragma unroll
      for (int st = 0; st < NS; ++st) asm volatile("" : "+a"(qf[a][st]));
    } else {
      landed(qf[a]);
    }
  }
  // units: the prefix's, then the own keys' up to the last one that a row of the block sees
  const bool any = r0 / p.group < nq;
  const int prefix = PREFIX ? p.prefix : 0, prefix_units = (prefix + kUnit - 1) / kUnit;
  const int end = any ? min(max(min((r0 + kRows - 1) / p.group, nq - 1) + shift + 1, 0), nk) : 0;
  const int all = any ? prefix_units + (end + kUnit - 1) / kUnit : 0;
  // those that need no mask
  const int whole = PREFIX && prefix % kUnit ? prefix / kUnit : prefix_units + min(max(r0 / p.group + shift + 1, 0), end) / kUnit;
  const int n0 = (int)((int64_t)all * split / p.splits), n1 = (int)((int64_t)all * (split + 1) / p.splits);
  const int steps = (n1 - n0 + 1) / 2, plain = max(0, min(whole, n1) - n0) / 2;

  // Of eight waves the first four load keys, the others values; four load both.
  constexpr int TENSORS = Order::TENSORS, LOADS = TENSORS * 2 * Loader::NB;
  const int loader = wave & 3, other = A == 2 ? 0 : wave >> 2;  // other: 1 for values
  const uint32_t lds0 = (uint32_t)(uintptr_t)(WTC_LDS uint8_t*)smem + (uint32_t)(loader * Loader::NB * 1024);
  const uint32_t dim_bytes = (uint32_t)p.dim * 2u;
  Loader own[TENSORS], pre[TENSORS];
#pragma unroll
  for (int y = 0; y < TENSORS; ++y) {
    const bool values = y + other;
    own[y].init(values ? p.v + 2 * (b * p.v_stride[0] + hk * p.v_stride[2]) : p.k + 2 * (b * p.k_stride[0] + hk * p.k_stride[2]),
                2 * (values ? p.v_stride[1] : p.k_stride[1]), p.dim, loader, lane);
    if constexpr (PREFIX)
      pre[y].init(values ? p.vp + 2 * hk * p.vp_stride[1] : p.kp + 2 * hk * p.kp_stride[1],
                  2 * (values ? p.vp_stride[0] : p.kp_stride[0]), p.dim, loader, lane);
  }
  auto load = [&](const Loader& of_own, const Loader& of_prefix, int n, uint32_t to) __attribute__((always_inline)) {
    const int g = n0 + n;
    const bool in = n >= 0 && g < n1;
    if (PREFIX && g < prefix_units) of_prefix.issue(to, in ? g * kUnit : 0, in ? min(kUnit, prefix - g * kUnit) : 0, dim_bytes);
    else of_own.issue(to, in ? (g - prefix_units) * kUnit : 0, in ? min(kUnit, end - (g - prefix_units) * kUnit) : 0, dim_bytes);
  };
  // stage s: keys of units 2 s + 1 and 2 s + 2, values of units 2 s - 1 and 2 s, in parts of one
  auto issue = [&](int s, uint32_t at, int part) __attribute__((always_inline)) {
    const int x = part & 1, y = part >> 1, values = y + other;
    if (y < TENSORS) load(own[y], pre[y], 2 * s + 1 - 2 * values + x, lds0 + at + (2 * values + x) * L::HALF);
  };
  auto after = [&](uint32_t at) { return at + L::STAGE == L::RING ? 0u : at + L::STAGE; };
  // The same in parts of two from stage STAGES - 1 on, one after another, where there is one
  // kind of keys: pointers go on by 64 rows, and the rows that are left count down.
  const int first = L::STAGES - 1, limit = min(end, n1 * kUnit);
  const uint8_t* next_rows[TENSORS];
#pragma unroll
  for (int y = 0; y < TENSORS; ++y)
    next_rows[y] = own[y].base + (uint64_t)(uint32_t)((n0 + 2 * first + 1 - 2 * (y + other)) * kUnit) * own[y].stride;
  int left = limit - (n0 + 2 * first + 1) * kUnit;  // of the keys
  auto issue_pair = [&](uint32_t at, int y) __attribute__((always_inline)) {
    const int values = y + other;
    own[y].issue2(lds0 + at + 2 * values * L::HALF, next_rows[y], left + 2 * values * kUnit, dim_bytes);
    next_rows[y] += (uint64_t)(2 * kUnit) * own[y].stride;
    if (y == TENSORS - 1) left -= 2 * kUnit;
  };

  f32x16 o[A][ND], s[2][A];  // s: of two units in turn
#pragma unroll
  for (int a = 0; a < A; ++a)
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int v = 0; v < 16; ++v) o[a][d][v] = 0.0f;
  u32x4 pf[A][2];
  // ref: minus the reference (log2 domain); +inf where there is none yet, which makes any
  // exponential pass kMostSum or be NaN.  total: this lane's half of the keys.
  float ref[A], total[A];
#pragma unroll
  for (int a = 0; a < A; ++a) {
    ref[a] = INFINITY;
    total[a] = 0.0f;
    pf[a][0] = pf[a][1] = u32x4{0, 0, 0, 0};
  }

  const uint32_t k_at = row_addr<RB>(lane), v_at = 2 * L::HALF + col_addr<RB>(lane);
  // Fragment y of half x of a stage: NS of keys, then NS of values.
  constexpr int STEPS = Order::STEPS, AHEAD = Order::AHEAD;
  auto read = [&](uint32_t stage, int x, int y) __attribute__((always_inline)) {
    if (y < NS) return row_frag<RB>(smem, k_at + stage, kUnit * x, y);
    return col_frag<RB>(smem, v_at + stage, kUnit * x + 16 * ((y - NS) / ND), (y - NS) % ND);
  };
  u32x4 frag[STEPS + AHEAD];  // the first AHEAD ones were read before
  // Unit n (its scores in cur): weights, while the matrix cores take unit n + 1's scores
  // (into next) and unit n - 1's values.  In steps of one fragment, two products and a
  // share of the weights, each fragment read AHEAD steps before its products; the
  // compiler moves nothing from one step to another.
  auto phase = [&](auto masked, int t, int x, uint32_t& stage, uint32_t fill, f32x16 (&cur)[A], f32x16 (&next)[A]) __attribute__((always_inline)) {
    u32x4 w[A][2];
    float sum[A];
#pragma unroll
    for (int a = 0; a < A; ++a) sum[a] = 0.0f;
    if constexpr (decltype(masked)::value) {
      const int g = n0 + 2 * t + x;
      const bool common = PREFIX && g < prefix_units;
      const int j0 = (common ? g : g - prefix_units) * kUnit + 4 * half;
#pragma unroll
      for (int a = 0; a < A; ++a) {
        const uint64_t seen = g < n1 ? bits_below((common ? prefix : sees[a]) - j0) : 0;
#pragma unroll
        for (int v = 0; v < 16; ++v) cur[a][v] = keep_bit(cur[a][v], seen, 8 * (v >> 2) + (v & 3));
      }
    }
    uint32_t from = stage;
    fresh(from);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int y = 0; y < STEPS; ++y) {
      if (x == 1 && y == Order::BARRIER) {
        // all of the stage is read: the next one landed, every wave is done with this one
        wait_loads_barrier<LOADS*Order::LOADING>();
        stage = from = after(stage);
        fresh(from);
      }
      frag[y + AHEAD] = y + AHEAD < STEPS ? read(from, x, y + AHEAD) : read(from, x ^ 1, y + AHEAD - STEPS);
#pragma unroll
      for (int a = 0; a < A; ++a) {
        if (y < NS) {
          const f32x16 zero = {};
          next[a] = mfma32<DT>(frag[y], qf[a][y], y == 0 ? zero : next[a]);
        } else {
          o[a][(y - NS) % ND] = mfma32<DT>(frag[y], pf[a][(y - NS) / ND], o[a][(y - NS) % ND]);
        }
      }
      // the stage that every wave has left takes units of the iteration after the next
      // (all of them before the barrier, which counts loads)
      if constexpr (PREFIX) {
        if (y == Order::FIRST) issue(t + L::STAGES - 1, fill, x);
        if (y == Order::SECOND) issue(t + L::STAGES - 1, fill, 2 + x);
      } else if (y == (x ? Order::SECOND : Order::FIRST) && x < TENSORS) {
        issue_pair(fill, x);
      }
#pragma unroll
      for (int z = 0; z < 8 * A; ++z) {  // pairs of scores
        if (z * STEPS / (8 * A) != y) continue;
        const int a = z / 8, v = z % 8 * 2;
        const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(cur[a][v], c2, ref[a]));
        const float e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(cur[a][v + 1], c2, ref[a]));
        sum[a] += e0;
        sum[a] += e1;
        w[a][v / 8][v / 2 % 4] = pack2<DT>(e0, e1);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if (__any(!(sum[0] < kMostSum && sum[A - 1] < kMostSum))) {
#pragma unroll
      for (int a = 0; a < A; ++a) {
        float m = cur[a][0];
#pragma unroll
        for (int v = 1; v < 16; ++v) m = fmaxf(m, cur[a][v]);
        m = xor32_max(m) * c2;
        // (of the rows that passed it: a row's result does not depend on its neighbours)
        const bool mine = xor32_max(sum[a] < kMostSum ? 0.0f : 1.0f) != 0.0f;
        const float before = -ref[a], now = mine ? fmaxf(before, m) : before;  // (-inf: none)
        const float by = now == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(before - now), off = now == -INFINITY ? 0.0f : -now;
        ref[a] = -now;
        sum[a] = 0.0f;
#pragma unroll
        for (int v = 0; v < 16; v += 2) {
          const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(cur[a][v], c2, off));
          const float e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(cur[a][v + 1], c2, off));
          sum[a] += e0;
          sum[a] += e1;
          w[a][v / 8][v / 2 % 4] = pack2<DT>(e0, e1);
        }
        total[a] *= by;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
          for (int v = 0; v < 16; ++v) o[a][d][v] *= by;
      }
    }
#pragma unroll
    for (int y = 0; y < AHEAD; ++y) frag[y] = frag[STEPS + y];
#pragma unroll
    for (int a = 0; a < A; ++a) {
      total[a] += sum[a];
      pf[a][0] = w[a][0];
      pf[a][1] = w[a][1];
    }
  };

  // stages -1 and up; unit 0's scores
#pragma unroll
  for (int x = 0; x < L::STAGES; ++x) {
    if (x == L::STAGES - 1) wait_loads_barrier<LOADS*Order::LOADING>();
#pragma unroll
    for (int part = 0; part < 4; ++part) issue(x - 1, x * L::STAGE, part);
  }
#pragma unroll
  for (int a = 0; a < A; ++a)
#pragma unroll
    for (int v = 0; v < 16; ++v) s[0][a][v] = 0.0f;
#pragma unroll
  for (int st = 0; st < NS; ++st) {
    const u32x4 k = read(0, 1, st);
#pragma unroll
    for (int a = 0; a < A; ++a) s[0][a] = mfma32<DT>(k, qf[a][st], s[0][a]);
  }
  uint32_t stage = L::STAGE, fill = 0;  // read, and left by every wave
  wait_loads_barrier<LOADS*Order::LOADING>();
#pragma unroll
  for (int y = 0; y < AHEAD; ++y) frag[y] = read(stage, 0, y);
  auto step = [&](auto masked, int t) __attribute__((always_inline)) {
    phase(masked, t, 0, stage, fill, s[0], s[1]);
    phase(masked, t, 1, stage, fill, s[1], s[0]);
    fill = after(fill);
  };
  int t = 0;
  for (; t < plain; ++t) step(std::false_type{}, t);
  for (; t < steps; ++t) step(std::true_type{}, t);
  // the last unit's values
#pragma unroll
  for (int y = NS; y < STEPS; ++y) {
    const u32x4 v = read(stage, 0, y);
#pragma unroll
    for (int a = 0; a < A; ++a) o[a][(y - NS) % ND] = mfma32<DT>(v, pf[a][(y - NS) / ND], o[a][(y - NS) % ND]);
  }
  wait_loads_barrier<0>();

  // ---- the rows' results
#pragma unroll
  for (int a = 0; a < A; ++a) {
    total[a] = valid[a] ? xor32_sum(total[a]) : 0.0f;
    const float inv = total[a] == 0.0f ? 0.0f : 1.0f / total[a];
    const float lse = total[a] == 0.0f ? -INFINITY : __builtin_amdgcn_logf(total[a]) - ref[a];
    if (p.slots) {
      const int64_t row = (((int64_t)b * p.lq + i[a]) * p.heads + h[a]) * p.slots + p.slot0 + split;
      if (valid[a]) {
        if (half == 0) p.part_lse[row] = lse;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const int c = 32 * d + 8 * g + 4 * half;
            if (c < p.dim)
              *reinterpret_cast<f32x4*>(p.part_out + row * p.dim + c) =
                  f32x4{o[a][d][4 * g] * inv, o[a][d][4 * g + 1] * inv, o[a][d][4 * g + 2] * inv, o[a][d][4 * g + 3] * inv};
          }
      }
      continue;
    }
    bool nan = false;
    uint8_t* stg = smem + wave * 32 * L::PITCH;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        f32x4 x;
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          x[v] = valid[a] ? o[a][d][4 * g + v] * inv : 0.0f;
          nan |= x[v] != x[v];
        }
        uint32_t w0, w1;
        pack4<DT>(x, &w0, &w1);
        *reinterpret_cast<u32x2*>(stg + (lane & 31) * L::PITCH + (32 * d + 8 * g + 4 * half) * 2) = u32x2{w0, w1};
      }
    if (p.lse && half == 0 && i[a] < p.lq) p.lse[((int64_t)b * p.heads + h[a]) * p.lq + i[a]] = lse * kLn2;
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    constexpr int CPR = ND * 4;  // chunks a row
    const int first = r0 + wave * 32 * A + 32 * a;
#pragma unroll 4
    for (int x = lane; x < 32 * CPR; x += 64) {
      const int row = x / CPR, c = x % CPR;
      const int rr = first + row, ii = rr / p.group, hh = hk * p.group + rr - ii * p.group;
      if (ii < p.lq && c * 8 < p.dim)
        *reinterpret_cast<u32x4*>(p.out + 2 * (b * p.o_stride[0] + (int64_t)ii * p.o_stride[1] + hh * p.o_stride[2]) + c * 16) =
            *reinterpret_cast<const u32x4*>(stg + row * L::PITCH + c * 16);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if constexpr (PREFIX) {  // (without a causal part nothing is hidden)
      uint32_t redo = (uint32_t)(__ballot(nan && valid[a]) | __ballot(nan && valid[a]) >> 32);
      if (redo) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the rows are read back
      while (redo) {
        const int rr = first + __builtin_ctz(redo);
        attention_row<DT, false, true>(p, b, hk * p.group + rr % p.group, rr / p.group);
        redo &= redo - 1;
      }
    }
  }
}

}  // namespace rows
}  // namespace wtc
