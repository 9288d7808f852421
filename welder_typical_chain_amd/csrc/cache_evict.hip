// cache_evict.hip -- the kernels of wtc_cache_evict: the rows of a cache that stay, and
// the smaller cache that holds them.
//
// A sequence of n > keep rows keeps its first `sinks`, its last `recent` and, of those
// between, the ones of greatest weight (of equal ones the lowest), in their order.
// The weight of the last one that stays is found digit by digit, 11, 11 and 10 bits
// from the top, from counts of the rows' digits in LDS (11 bits: the sign, the exponent
// and two bits of the mantissa, so that the lanes of a wave seldom meet in one count);
// a row stays if its weight is greater, or equal and among the first that are.
//
// One workgroup finds the rows of a (sequence, key head), with up to kHeld weights kept
// in LDS; a second launch copies them, 16 bytes a thread, neighbours in the new cache
// by neighbours, which bounds the call while the weights fit.  (In one launch, with as many
// workgroups a sequence as fill the chip, each finding all rows for itself: 72 us for 16
// caches of 8192 rows of 8 heads of 128 cut to 2048, against 57.)  More weights than kHeld are
// read from memory once a digit and once for the rows, which then bounds it: one cache of
// 65536 rows, 8 heads of 128, cut to 4096 takes 98 us so and 8 for the copy; of 8200 rows 20,
// of 8192 rows 14.
#include "layer_kernels.h"

namespace wtc {
namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kHeld = 8 * kThreads;  // weights kept in LDS
constexpr int kDigits = 2048;

// Weights as integers in the same order; -0 as 0, NaN above everything.
__device__ inline uint32_t ordered(float w) {
  const uint32_t u = __builtin_bit_cast(uint32_t, w + 0.0f);
  if (w != w) return 0xFFFFFFFFu;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ inline float unordered(uint32_t u) {  // (some NaN for 0xFFFFFFFF)
  return __builtin_bit_cast(float, u & 0x80000000u ? u ^ 0x80000000u : ~u);
}

template <bool HELD>
__global__ void __launch_bounds__(kThreads) evict_select_kernel(const EvictParams p) {
  __shared__ int count[kDigits];
  __shared__ int wave_sum[kWaves];
  __shared__ int2 table[kHeld / 64], all;
  __shared__ ulonglong2 found_here[kHeld / 64];
  __shared__ uint32_t held[HELD ? kHeld : 1];
  __shared__ uint32_t found;
  __shared__ int left;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t seq = blockIdx.x;
  const int b = (int)(seq / p.kv_heads), g = (int)(seq % p.kv_heads);
  const int n = min(max(p.lengths[b], 0), p.rows), kept = min(n, p.keep);
  const float* w = p.weights + seq * p.rows;
  int32_t* rows = p.kept + seq * p.keep;
  float* w_out = p.weights_out + seq * p.out_rows;
  // row r of the old cache is row `to` of the new one
  auto keep = [&](int to, int r, float x) {
    rows[to] = r;
    w_out[to] = x;
  };
  for (int to = kept + tid; to < p.out_rows; to += kThreads) {
    if (to < p.keep) rows[to] = -1;
    w_out[to] = 0.0f;
  }
  if (tid == 0 && g == 0) p.lengths_out[b] = kept;
  if (n <= p.keep) {
    for (int r = tid; r < n; r += kThreads) keep(r, r, w[r]);
  } else {
    // rows [first, last) are weighed, `take` of them stay
    const int first = p.sinks, last = n - p.recent, take = p.keep - p.sinks - p.recent;
    if constexpr (HELD) {
      float x[kHeld / kThreads];  // all loads before the first use
#pragma unroll
      for (int k = 0; k < kHeld / kThreads; ++k) x[k] = w[min(k * kThreads + tid, n - 1)];
#pragma unroll
      for (int k = 0; k < kHeld / kThreads; ++k) held[k * kThreads + tid] = ordered(x[k]);  // (each thread reads its own)
    }
    auto key = [&](int r) {
      if constexpr (HELD) return held[r];
      else return ordered(w[r]);
    };
    uint32_t top = 0;  // digits found so far
    int rest = take;   // rows to take of those that begin with them
    if (take) {
#pragma unroll 1
      for (int step = 0; step < 3; ++step) {
        const int shift = step == 0 ? 21 : step == 1 ? 10 : 0, above = step == 0 ? 31 : step == 1 ? 21 : 10;
        const uint32_t mask = step == 2 ? kDigits / 2 - 1 : kDigits - 1;
        count[tid] = count[kThreads + tid] = 0;
        __syncthreads();
        for (int r = tid; r < last; r += kThreads) {
          const uint32_t u = key(r);
          if (r >= first && (step == 0 || u >> above == top >> above)) atomicAdd(&count[u >> shift & mask], 1);
        }
        __syncthreads();
        // two digits a thread, from the greatest down
        const int c0 = count[kDigits - 1 - 2 * tid], c1 = count[kDigits - 2 - 2 * tid];
        int before = c0 + c1;
        for (int o = 1; o < 64; o <<= 1) {
          const int y = __shfl_up(before, o);
          if (lane >= o) before += y;
        }
        if (lane == 63) wave_sum[wave] = before;
        __syncthreads();
        before -= c0 + c1;
#pragma unroll
        for (int v = 0; v < kWaves; ++v) before += v < wave ? wave_sum[v] : 0;
        if (before < rest && rest <= before + c0 + c1) {
          const bool second = rest > before + c0;
          found = top | (uint32_t)(kDigits - 1 - 2 * tid - second) << shift;
          left = rest - before - (second ? c0 : 0);
        }
        __syncthreads();
        top = found;
        rest = left;
      }
    }
    // In order: `rest` of the rows equal to `top`, all above it, and those that are not
    // weighed.  kHeld rows at a time: what each wave has of them, the sums before, then the rows.
    auto marks = [&](int r, uint64_t* above, uint64_t* same) {
      const bool in = r < n, between = r >= first && r < last;
      const uint32_t u = in ? key(r) : 0u;
      *above = __ballot(in && (!between || (take && u > top)));
      *same = __ballot(in && take && between && u == top);
    };
    const uint64_t me = 1ull << lane, below = me - 1;
    int2 done = {0, 0};
#pragma unroll 1
    for (int r0 = 0; r0 < n; r0 += kHeld) {
      const int chunks = min(kHeld, n - r0 + kThreads - 1) / kThreads;
      for (int k = 0; k < kHeld / kThreads; ++k) {
        uint64_t a = 0, e = 0;
        if (k < chunks) marks(r0 + k * kThreads + tid, &a, &e);
        if (lane == 0) {
          table[k * kWaves + wave] = int2{__popcll(a), __popcll(e)};
          found_here[k * kWaves + wave] = ulonglong2{a, e};
        }
      }
      __syncthreads();
      if (wave == 0) {
        constexpr int EACH = kHeld / 64 / 64;
        int2 c[EACH], sum = {0, 0};
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
          c[i] = table[EACH * lane + i];
          sum.x += c[i].x;
          sum.y += c[i].y;
        }
        int2 before = sum;
        for (int o = 1; o < 64; o <<= 1) {
          const int x = __shfl_up(before.x, o), y = __shfl_up(before.y, o);
          if (lane >= o) before.x += x, before.y += y;
        }
        if (lane == 63) all = before;
        before.x -= sum.x;
        before.y -= sum.y;
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
          table[EACH * lane + i] = before;
          before.x += c[i].x;
          before.y += c[i].y;
        }
      }
      __syncthreads();
      for (int k = 0; k < chunks; ++k) {
        const int r = r0 + k * kThreads + tid;
        const uint64_t a = found_here[k * kWaves + wave].x, e = found_here[k * kWaves + wave].y;
        const int2 t = table[k * kWaves + wave];
        const int na = done.x + t.x + __popcll(a & below), ne = done.y + t.y + __popcll(e & below);
        if (a & me || (e & me && ne < rest)) keep(na + min(ne, rest), r, unordered(key(r)));
      }
      done.x += all.x;
      done.y += all.y;
      __syncthreads();
    }
  }
}

// 16 bytes a thread of a row of k and of v.
__global__ void __launch_bounds__(256) evict_copy_kernel(const EvictParams p) {
  const int chunks = p.row_bytes / 16;
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x, row = at / chunks;
  const int c = (int)(at - row * chunks) * 16;
  const int g = (int)(row % p.kv_heads);
  const int64_t rest = row / p.kv_heads;
  const int to = (int)(rest % p.keep), b = (int)(rest / p.keep);
  if (b >= p.batch) return;
  const int from = p.kept[((int64_t)b * p.kv_heads + g) * p.keep + to];
  u32x4 k = {0, 0, 0, 0}, v = {0, 0, 0, 0};
  if (from >= 0) {
    k = *reinterpret_cast<const u32x4*>(p.k + b * p.k_stride[0] + from * p.k_stride[1] + g * p.k_stride[2] + c);
    v = *reinterpret_cast<const u32x4*>(p.v + b * p.v_stride[0] + from * p.v_stride[1] + g * p.v_stride[2] + c);
  }
  *reinterpret_cast<u32x4*>(p.k_out + b * p.ko_stride[0] + to * p.ko_stride[1] + g * p.ko_stride[2] + c) = k;
  *reinterpret_cast<u32x4*>(p.v_out + b * p.vo_stride[0] + to * p.vo_stride[1] + g * p.vo_stride[2] + c) = v;
}

}  // namespace

hipError_t launch_cache_evict(const EvictParams& params, hipStream_t stream) {
  EvictParams p = params;
  void* args[] = {&p};
  const void* select = p.rows <= kHeld ? (const void*)&evict_select_kernel<true> : (const void*)&evict_select_kernel<false>;
  const hipError_t e = hipLaunchKernel(select, dim3((unsigned)(p.batch * p.kv_heads)), dim3(kThreads), args, 0, stream);
  if (e != hipSuccess) return e;
  const int64_t threads = (int64_t)p.batch * p.keep * p.kv_heads * (p.row_bytes / 16);
  return hipLaunchKernel((const void*)&evict_copy_kernel, dim3((unsigned)((threads + 255) / 256)), dim3(256), args, 0, stream);
}

}  // namespace wtc
