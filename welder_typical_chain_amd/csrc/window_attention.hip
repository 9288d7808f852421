// window_attention.hip -- kernels of wtc_window_attention and its gradients.
#include "attention_common.h"
#include "layer_kernels.h"

#include <algorithm>

namespace wtc {
namespace {

using namespace attn;

// One query row by a whole wave, 64 keys at a time, with nothing but the keys it
// sees: what the tile kernel's rows fall back on that come out as NaN (a NaN or an
// infinity in a key or value that the mask hides would reach them through the
// tile's products, as 0 * NaN).
template <int DT> __device__ inline void attention_row(const AttnParams& p, int b, int h, int i) {
  using T = typename Elem<DT>::type;
  const int lane = threadIdx.x & 63;
  const int pos = i + seq_keys(p, b) - seq_queries(p, b);
  const T* q = (const T*)p.q + b * p.q_stride[0] + i * p.q_stride[1] + h * p.q_stride[2];
  const T* k = (const T*)p.k + b * p.k_stride[0] + h / p.group * p.k_stride[2];
  const T* v = (const T*)p.v + b * p.v_stride[0] + h / p.group * p.v_stride[2];
  const Seen seen(p.window, p.sinks, pos);
  float top = -INFINITY, total = 0.0f, acc[2] = {0.0f, 0.0f};
  for (int t0 = 0; t0 < seen.count; t0 += 64) {
    const bool in = t0 + lane < seen.count;
    const float s = in ? p.scale * dot_rows<DT>(q, k + seen.key(t0 + lane) * p.k_stride[1], p.dim) : -INFINITY;
    const float next = fmaxf(top, wave_max(s));
    const float keep = next == -INFINITY ? 1.0f : __expf(top - next);
    const float e = in ? (next == -INFINITY ? (s != s ? s : 0.0f) : __expf(s - next)) : 0.0f;
    total = total * keep + wave_sum(e);
    acc[0] *= keep;
    acc[1] *= keep;
    top = next;
    for (int t = 0; t < min(64, seen.count - t0); ++t) {
      const float w = __shfl(e, t);
      const T* row = v + seen.key(t0 + t) * p.v_stride[1];
      for (int c = 0; c < 2; ++c)
        if (lane + 64 * c < p.dim) acc[c] = __builtin_fmaf(w, (float)row[lane + 64 * c], acc[c]);
    }
  }
  T* out = (T*)p.out + b * p.o_stride[0] + i * p.o_stride[1] + h * p.o_stride[2];
  const float r = total == 0.0f ? 0.0f : 1.0f / total;
  for (int c = 0; c < 2; ++c)
    if (lane + 64 * c < p.dim) out[lane + 64 * c] = (T)(acc[c] * r);
  if (p.lse && lane == 0) p.lse[((int64_t)b * p.heads + h) * p.lq + i] = top + __logf(total);
}

// ---- forward -----------------------------------------------------------------
// A workgroup takes NW * 32 query rows of one sequence and key head.  The rows
// of the query heads that share the key head are packed (row r = query r / G,
// head r % G), so that a tile of keys serves all of them and the window's
// edges cost G times fewer tiles.  A wave owns 32 rows, one a lane pair:
//   S^T = K . Q^T   (32 x 32 subtiles; a lane holds 32 scores of one query)
//   online softmax  (in registers; the two lanes of a query share its maximum)
//   O^T += V^T . P^T (P^T straight from the registers, see col_frag)
// Keys come in tiles of 64 through a ring of (K, V) stages filled by
// direct-to-LDS loads; one barrier a tile.  Workgroups of 8 waves have 3 stages
// (one workgroup a CU at dim 128), those of 4 waves 2 (two a CU).
constexpr int kKeys = 64;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
// The running maximum is only moved when a score exceeds it by 2^8: the weights
// stay below 2^8, and the accumulators are rescaled a few times a row instead
// of once a tile.
constexpr float kSlack = 8.0f;

template <int ND, int NW> struct FwdLds {
  static constexpr int RB = row_bytes(ND), STAGES = NW == 8 ? 3 : 2;
  static constexpr int TILE = kKeys * RB, STAGE = 2 * TILE;
  static constexpr int PITCH = ND * 64 + 16;  // bytes of a row staged for the output
  static constexpr int RING = STAGES * STAGE, OUT = NW * 32 * PITCH;
  static constexpr int TOTAL = RING > OUT ? RING : OUT;
  static_assert(TOTAL <= 160 * 1024, "LDS");
};

template <int DT, int ND, int NW>
__global__ void __launch_bounds__(NW * 64, 2) attention_tile_kernel(const AttnParams p) {
  using L = FwdLds<ND, NW>;
  constexpr int RB = L::RB, NS = 2 * ND;
  __shared__ __attribute__((aligned(16))) uint8_t smem[L::TOTAL];
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t id = xcd_remap(blockIdx.x, gridDim.x);
  const int split = (int)(id % p.splits);
  const uint32_t rest = id / p.splits;
  const int blk = p.row_blocks - 1 - (int)(rest % p.row_blocks);  // the longest rows first
  const int hk = (int)(rest / p.row_blocks % p.kv_heads), b = (int)(rest / p.row_blocks / p.kv_heads);
  const int nk = seq_keys(p, b), nq = seq_queries(p, b), shift = nk - nq;
  const int r0 = blk * NW * 32;

  // this lane's row
  const int r = r0 + wave * 32 + (lane & 31), i = r / p.group, h = hk * p.group + r - i * p.group;
  const bool valid = i < nq;
  const int pos = valid ? i + shift : -1;

  // keys of the block: [0, s_end) and [lo, end)
  const int i_last = min((r0 + NW * 32 - 1) / p.group, nq - 1);
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
  float c2 = p.scale * kLog2e;
  if (c2 < 0.0f) {  // then the largest score is the smallest product: negate the queries instead
    c2 = -c2;
#pragma unroll
    for (int s = 0; s < NS; ++s) qf[s] ^= 0x80008000u;
  }

  f32x16 o[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int v = 0; v < 16; ++v) o[d][v] = 0.0f;
  float top = -INFINITY, total = 0.0f;  // log2 domain; total: this lane's half of the keys

  TileLoader<RB, kKeys, NW> lk, lv;
  lk.init(p.k + 2 * (b * p.k_stride[0] + hk * p.k_stride[2]), 2 * p.k_stride[1], p.dim, wave, lane);
  lv.init(p.v + 2 * (b * p.v_stride[0] + hk * p.v_stride[2]), 2 * p.v_stride[1], p.dim, wave, lane);
  constexpr int LOADS = 2 * TileLoader<RB, kKeys, NW>::NB;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(WTC_LDS uint8_t*)smem;
  auto tile_base = [&](int t) { return t < t_sink ? t * kKeys : lo + (t - t_sink) * kKeys; };
  auto tile_end = [&](int t) { return t < t_sink ? s_end : end; };
  auto issue = [&](int t) {
    const int j0 = tile_base(t), n = t < t1 ? min(kKeys, tile_end(t) - j0) : 0;
    const uint32_t st = lds0 + (uint32_t)(t - t0) % L::STAGES * L::STAGE;
    lk.issue(st, j0, n);
    lv.issue(st + L::TILE, j0, n);
  };
#pragma unroll
  for (int t = 0; t < L::STAGES - 1; ++t) issue(t0 + t);

  for (int t = t0; t < t1; ++t) {
    wait_loads_barrier<LOADS*(L::STAGES - 2)>();  // tile t landed; every wave is done with tile t - 1
    issue(t + L::STAGES - 1);
    const int j0 = tile_base(t), j1 = tile_end(t);
    // (in the window's part the first tokens may lie below the window too)
    const bool below = t >= t_sink && (int64_t)j0 + kKeys - 1 + p.window <= w_lo && j0 >= p.sinks;
    if (!w_any || j0 > w_hi || below) continue;
    const uint8_t* kt = smem + (t - t0) % L::STAGES * L::STAGE;
    const uint8_t* vt = kt + L::TILE;

    f32x16 s[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int v = 0; v < 16; ++v) s[u][v] = 0.0f;
#pragma unroll
      for (int st = 0; st < NS; ++st) s[u] = mfma32<DT>(row_frag<RB>(kt, 32 * u, st, lane), qf[st], s[u]);
    }
    if (j0 + kKeys > j1 || j0 + kKeys - 1 > w_lo || (t >= t_sink && (int64_t)j0 + p.window <= w_hi)) {
      // key j0 + 4 half + c is seen if c <= top_c and (c > low_c or c < sink_c)
      const int at = j0 + 4 * half;
      const int top_c = min(pos, j1 - 1) - at;
      const int low_c = (int)max((int64_t)pos - p.window - at, (int64_t)-1);
      const int sink_c = p.sinks - at;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          const int c = 32 * u + 8 * (v >> 2) + (v & 3);
          s[u][v] = c <= top_c && (c > low_c || c < sink_c) ? s[u][v] : -INFINITY;
        }
    }
    float m = s[0][0];
#pragma unroll
    for (int v = 1; v < 16; ++v) m = fmaxf(m, s[0][v]);
#pragma unroll
    for (int v = 0; v < 16; ++v) m = fmaxf(m, s[1][v]);
    m = xor32_max(m);
    m = m == -INFINITY ? m : m * c2;  // (a scale of 0 times -inf)
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
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        f32x4 e;
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const float x = s[u][4 * g + v];
          e[v] = __builtin_amdgcn_exp2f(__builtin_fmaf(x, c2, ref));
          if (c2 == 0.0f) e[v] = x == -INFINITY ? 0.0f : e[v];  // a scale of 0 keeps the mask
          sum[v & 1] += e[v];
        }
        uint32_t w0, w1;
        pack4<DT>(e, &w0, &w1);
        pf[2 * u + (g >> 1)][2 * (g & 1)] = w0;
        pf[2 * u + (g >> 1)][2 * (g & 1) + 1] = w1;
      }
    total += sum[0] + sum[1];
#pragma unroll
    for (int st = 0; st < 4; ++st)
#pragma unroll
      for (int d = 0; d < ND; ++d) o[d] = mfma32<DT>(col_frag<RB>(vt, 16 * st, 32 * d, lane), pf[st], o[d]);
  }
  wait_loads_barrier<0>();

  // ---- the rows' results
  // (a row behind the end took part in tiles that needed no mask)
  total = valid ? xor32_sum(total) : 0.0f;
  const float inv = total == 0.0f ? 0.0f : 1.0f / total;
  const float lse = (top + __builtin_amdgcn_logf(total)) * kLn2;  // (v_log_f32: log2)
  if (p.splits > 1) {
    const int64_t row = (((int64_t)b * p.lq + i) * p.heads + h) * p.splits + split;
    if (valid) {
      if (half == 0) p.part_lse[row] = total == 0.0f ? -INFINITY : lse;
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
  bool nan = lse != lse && total != 0.0f;
  uint8_t* stg = smem + wave * 32 * L::PITCH;
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
  while (redo) {
    const int rr = r0 + wave * 32 + __builtin_ctz(redo);
    attention_row<DT>(p, b, hk * p.group + rr % p.group, rr / p.group);
    redo &= redo - 1;
  }
}

// Joins the splits of a row: one wave a row.
template <int DT>
__global__ void __launch_bounds__(256) attention_join_kernel(const AttnParams p) {
  using T = typename Elem<DT>::type;
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= (int64_t)p.batch * p.lq * p.heads) return;
  const int h = (int)(row % p.heads), i = (int)(row / p.heads % p.lq), b = (int)(row / p.heads / p.lq);
  const float* part = p.part_lse + row * p.splits;
  const int splits = i < seq_queries(p, b) ? p.splits : 0;  // rows behind the end were not written
  float top = -INFINITY;
  for (int s = 0; s < splits; ++s) top = fmaxf(top, part[s]);
  const float ref = top == -INFINITY ? 0.0f : top;
  float total = 0.0f, acc[2] = {0.0f, 0.0f};
  for (int s = 0; s < splits; ++s) {
    const float w = __expf(part[s] - ref);
    total += w;
    for (int c = 0; c < 2; ++c)
      if (lane + 64 * c < p.dim) acc[c] = __builtin_fmaf(w, p.part_out[(row * p.splits + s) * p.dim + lane + 64 * c], acc[c]);
  }
  const float inv = total == 0.0f ? 0.0f : 1.0f / total;
  T* out = (T*)p.out + b * p.o_stride[0] + i * p.o_stride[1] + h * p.o_stride[2];
  bool nan = total != total;
  for (int c = 0; c < 2; ++c)
    if (lane + 64 * c < p.dim) {
      const float x = acc[c] * inv;
      nan |= x != x;
      out[lane + 64 * c] = (T)x;
    }
  if (p.lse && lane == 0) p.lse[((int64_t)b * p.heads + h) * p.lq + i] = top + __logf(total);
  if (__any(nan) && i < seq_queries(p, b)) attention_row<DT>(p, b, h, i);
}

// ---- gradients ------------------------------------------------------------------
// delta = sum_d dout * out of a row, and the row's dq.  One wave a row.
template <int DT>
__global__ void __launch_bounds__(64) attention_dq_rows_kernel(const AttnParams p) {
  using T = typename Elem<DT>::type;
  const int lane = threadIdx.x;
  const int h = blockIdx.x % p.heads;
  const int i = blockIdx.x / p.heads % p.lq, b = blockIdx.x / p.heads / p.lq;
  const int nq = seq_queries(p, b), pos = i + seq_keys(p, b) - nq;
  const T* q = (const T*)p.q + b * p.q_stride[0] + i * p.q_stride[1] + h * p.q_stride[2];
  const T* k = (const T*)p.k + b * p.k_stride[0] + h / p.group * p.k_stride[2];
  const T* v = (const T*)p.v + b * p.v_stride[0] + h / p.group * p.v_stride[2];
  const T* g = (const T*)p.dout + b * p.do_stride[0] + i * p.do_stride[1] + h * p.do_stride[2];
  const T* o = (const T*)p.o + b * p.o_stride[0] + i * p.o_stride[1] + h * p.o_stride[2];
  const int64_t row_id = ((int64_t)b * p.heads + h) * p.lq + i;
  Seen seen(p.window, p.sinks, pos);
  if (i >= nq) seen.count = 0;
  float acc[2] = {0.0f, 0.0f}, delta = 0.0f;
  if (seen.count) {
    for (int d = lane; d < p.dim; d += 64) delta = __builtin_fmaf((float)g[d], (float)o[d], delta);
    delta = wave_sum(delta);
  }
  if (lane == 0) p.delta[row_id] = delta;
  const float lse = p.lse_in[row_id];
  for (int t0 = 0; t0 < seen.count; t0 += 64) {
    float ds = 0.0f;
    if (t0 + lane < seen.count) {
      const int j = seen.key(t0 + lane);
      const float w = __expf(p.scale * dot_rows<DT>(q, k + j * p.k_stride[1], p.dim) - lse);
      ds = p.scale * w * (dot_rows<DT>(g, v + j * p.v_stride[1], p.dim) - delta);
    }
    for (int t = 0; t < min(64, seen.count - t0); ++t) {
      const float w = __shfl(ds, t);
      const T* row = k + seen.key(t0 + t) * p.k_stride[1];
      for (int c = 0; c < 2; ++c)
        if (lane + 64 * c < p.dim) acc[c] = __builtin_fmaf(w, (float)row[lane + 64 * c], acc[c]);
    }
  }
  T* dq = (T*)p.dq + (((int64_t)b * p.lq + i) * p.heads + h) * p.dim;
  for (int c = 0; c < 2; ++c)
    if (lane + 64 * c < p.dim) dq[lane + 64 * c] = (T)acc[c];
}

// dk and dv of one key row: over the query heads that share it, 64 queries at a time.
template <int DT>
__global__ void __launch_bounds__(64) attention_dkv_rows_kernel(const AttnParams p) {
  using T = typename Elem<DT>::type;
  const int lane = threadIdx.x;
  const int hk = blockIdx.x % p.kv_heads;
  const int j = blockIdx.x / p.kv_heads % p.lk, b = blockIdx.x / p.kv_heads / p.lk;
  const int nq = seq_queries(p, b), nk = seq_keys(p, b), shift = nk - nq;
  const T* k = (const T*)p.k + b * p.k_stride[0] + j * p.k_stride[1] + hk * p.k_stride[2];
  const T* v = (const T*)p.v + b * p.v_stride[0] + j * p.v_stride[1] + hk * p.v_stride[2];
  // queries of positions j .. j + window - 1 (a first token: all from j on)
  const int i0 = max(0, j - shift);
  int i1 = j < nk ? nq : 0;
  if (j >= p.sinks) i1 = (int)min((int64_t)i1, j + p.window - shift);
  float ak[2] = {0.0f, 0.0f}, av[2] = {0.0f, 0.0f};
  for (int h = hk * p.group; h < (hk + 1) * p.group; ++h) {
    const T* q = (const T*)p.q + b * p.q_stride[0] + h * p.q_stride[2];
    const T* g = (const T*)p.dout + b * p.do_stride[0] + h * p.do_stride[2];
    const int64_t row0 = ((int64_t)b * p.heads + h) * p.lq;
    for (int t0 = i0; t0 < i1; t0 += 64) {
      float w = 0.0f, ds = 0.0f;
      const int i = t0 + lane;
      if (i < i1) {
        w = __expf(p.scale * dot_rows<DT>(q + i * p.q_stride[1], k, p.dim) - p.lse_in[row0 + i]);
        ds = p.scale * w * (dot_rows<DT>(g + i * p.do_stride[1], v, p.dim) - p.delta[row0 + i]);
      }
      for (int t = 0; t < min(64, i1 - t0); ++t) {
        const float wt = __shfl(w, t), dt = __shfl(ds, t);
        for (int c = 0; c < 2; ++c)
          if (lane + 64 * c < p.dim) {
            av[c] = __builtin_fmaf(wt, (float)g[(t0 + t) * p.do_stride[1] + lane + 64 * c], av[c]);
            ak[c] = __builtin_fmaf(dt, (float)q[(t0 + t) * p.q_stride[1] + lane + 64 * c], ak[c]);
          }
      }
    }
  }
  const int64_t at = (((int64_t)b * p.lk + j) * p.kv_heads + hk) * p.dim;
  for (int c = 0; c < 2; ++c)
    if (lane + 64 * c < p.dim) {
      ((T*)p.dk)[at + lane + 64 * c] = (T)ak[c];
      ((T*)p.dv)[at + lane + 64 * c] = (T)av[c];
    }
}

hipError_t launch(const void* fn, int64_t grid, int threads, const AttnParams& p, hipStream_t stream) {
  AttnParams q = p;
  void* args[] = {&q};
  return hipLaunchKernel(fn, dim3((unsigned)grid), dim3(threads), args, 0, stream);
}

}  // namespace

#define WTC_BY_TYPE(kernel, dt) ((dt) == DT_F16 ? (const void*)&kernel<DT_F16> : (const void*)&kernel<DT_BF16>)

namespace {
template <int DT, int NW> const void* tile_kernel(int nd) {
  switch (nd) {
    case 1: return (const void*)&attention_tile_kernel<DT, 1, NW>;
    case 2: return (const void*)&attention_tile_kernel<DT, 2, NW>;
    case 3: return (const void*)&attention_tile_kernel<DT, 3, NW>;
  }
  return (const void*)&attention_tile_kernel<DT, 4, NW>;
}
}  // namespace

// Waves a workgroup (32 rows each) and splits of the keys, from the sizes alone.
AttnPlan plan_attention(const AttnParams& p, int cu_count) {
  AttnPlan plan{8, 1};
  const int64_t rows = (int64_t)p.lq * p.group, seqs = (int64_t)p.batch * p.kv_heads;
  if (seqs * ((rows + 255) / 256) < cu_count) plan.waves = 4;
  const int64_t grid = seqs * ((rows + plan.waves * 32 - 1) / (plan.waves * 32));
  // keys that a row block sees at most
  const int64_t reach = std::min<int64_t>(p.lk, p.window + (plan.waves * 32 + p.group - 1) / p.group + p.sinks);
  const int64_t tiles = (reach + kKeys - 1) / kKeys;
  while (plan.splits < 16 && grid * plan.splits < cu_count && tiles / (2 * plan.splits) >= 4) plan.splits *= 2;
  return plan;
}
int64_t attention_workspace(const AttnParams& p, const AttnPlan& plan) {
  const int64_t rows = (int64_t)p.batch * p.lq * p.heads * plan.splits;
  return plan.splits > 1 ? rows * 4 * (p.dim + 1) : 0;
}

hipError_t launch_attention(const AttnParams& params, const AttnPlan& plan, int dt, hipStream_t stream) {
  AttnParams p = params;
  const int64_t rows = (int64_t)p.lq * p.group;
  p.splits = plan.splits;
  p.row_blocks = (int)((rows + plan.waves * 32 - 1) / (plan.waves * 32));
  p.part_lse = p.part_out + (int64_t)p.batch * p.lq * p.heads * p.splits * p.dim;
  const int nd = (p.dim + 31) / 32;
  const void* fn = plan.waves == 8 ? (dt == DT_F16 ? tile_kernel<DT_F16, 8>(nd) : tile_kernel<DT_BF16, 8>(nd))
                                   : (dt == DT_F16 ? tile_kernel<DT_F16, 4>(nd) : tile_kernel<DT_BF16, 4>(nd));
  const hipError_t e = launch(fn, (int64_t)p.batch * p.kv_heads * p.row_blocks * p.splits, plan.waves * 64, p, stream);
  if (e != hipSuccess || p.splits == 1) return e;
  return launch(WTC_BY_TYPE(attention_join_kernel, dt), ((int64_t)p.batch * p.lq * p.heads + 3) / 4, 256, p, stream);
}

hipError_t launch_attention_backward(const AttnParams& p, int dt, hipStream_t stream) {
  if (p.lq) {
    const hipError_t e = launch(WTC_BY_TYPE(attention_dq_rows_kernel, dt), (int64_t)p.batch * p.lq * p.heads, 64, p, stream);
    if (e != hipSuccess) return e;
  }
  if (!p.lk) return hipSuccess;
  return launch(WTC_BY_TYPE(attention_dkv_rows_kernel, dt), (int64_t)p.batch * p.lk * p.kv_heads, 64, p, stream);
}

}  // namespace wtc
