// cache_evict.hip -- kernels of wtc_cache_evict: the rows of a cache that stay, and
// the smaller cache that holds them.
//
// A sequence of n > keep rows keeps its first `sinks`, its last `recent` and, of those
// between, the ones of greatest weight (of equal ones the lowest), in their order.
// The weight of the last one that stays is found digit by digit, eight bits a pass
// from the top, from counts of the rows' digits in LDS; a row stays if its weight is
// greater, or equal and among the first rows that are.  One workgroup finds the rows
// of a (sequence, key head); a second kernel copies them, 16 bytes a lane.
#include "layer_kernels.h"

namespace wtc {
namespace {

constexpr int kThreads = 1024;

// Weights as integers in the same order; -0 as 0, NaN above everything.
__device__ inline uint32_t ordered(float w) {
  const uint32_t u = __builtin_bit_cast(uint32_t, w + 0.0f);
  if (w != w) return 0xFFFFFFFFu;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ inline int evict_rows(const EvictParams& p, int b) { return min(max(p.lengths[b], 0), p.rows); }

__global__ void __launch_bounds__(kThreads) evict_select_kernel(const EvictParams p) {
  __shared__ int count[256];
  __shared__ int2 wave_count[kThreads / 64];
  __shared__ uint32_t found;
  __shared__ int left;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t seq = blockIdx.x;
  const int b = (int)(seq / p.kv_heads), n = evict_rows(p, b), kept = min(n, p.keep);
  const float* w = p.weights + seq * p.rows;
  int32_t* out = p.kept + seq * p.keep;
  float* w_out = p.weights_out + seq * p.out_rows;
  for (int r = kept + tid; r < p.out_rows; r += kThreads) w_out[r] = 0.0f;
  for (int r = kept + tid; r < p.keep; r += kThreads) out[r] = -1;
  if (tid == 0 && seq % p.kv_heads == 0) p.lengths_out[b] = kept;
  if (n <= p.keep) {
    for (int r = tid; r < n; r += kThreads) {
      out[r] = r;
      w_out[r] = w[r];
    }
    return;
  }
  // rows [first, last) are weighed, `take` of them stay
  const int first = p.sinks, last = n - p.recent, take = p.keep - p.sinks - p.recent;
  uint32_t top = 0;  // digits found so far
  int rest = take;   // rows to take of those that begin with them
  if (take) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) count[tid] = 0;
      __syncthreads();
      for (int r = first + tid; r < last; r += kThreads) {
        const uint32_t u = ordered(w[r]);
        if (shift == 24 || u >> (shift + 8) == top >> (shift + 8)) atomicAdd(&count[u >> shift & 255], 1);
      }
      __syncthreads();
      if (wave == 0) {  // four digits a lane, from the greatest down
        int c[4], sum = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) sum += c[i] = count[255 - 4 * lane - i];
        int before = sum;
        for (int o = 1; o < 64; o <<= 1) {
          const int y = __shfl_up(before, o);
          if (lane >= o) before += y;
        }
        before -= sum;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (before < rest && rest <= before + c[i]) {
            found = top | (uint32_t)(255 - 4 * lane - i) << shift;
            left = rest - before;
          }
          before += c[i];
        }
      }
      __syncthreads();
      top = found;
      rest = left;
    }
  }
  // in order: `rest` of the rows equal to `top`, all above it
  int at = 0, equal = 0;
  for (int r0 = 0; r0 < n; r0 += kThreads) {
    const int r = r0 + tid;
    const float x = r < n ? w[r] : 0.0f;
    const bool between = r >= first && r < last, fixed = r < n && !between;
    const uint32_t u = ordered(x);
    const bool above = fixed || (take && between && u > top), same = take && between && u == top;
    const uint64_t a = __ballot(above), e = __ballot(same), below = (1ull << lane) - 1;
    if (lane == 0) wave_count[wave] = int2{__popcll(a), __popcll(e)};
    __syncthreads();
    int na = at, ne = equal, all_a = 0, all_e = 0;
    for (int v = 0; v < kThreads / 64; ++v) {
      const int2 c = wave_count[v];
      if (v < wave) na += c.x, ne += c.y;
      all_a += c.x, all_e += c.y;
    }
    na += __popcll(a & below);
    ne += __popcll(e & below);
    if (above || (same && ne < rest)) {
      const int to = na + min(ne, rest);
      out[to] = r;
      w_out[to] = x;
    }
    at += all_a;
    equal += all_e;
    __syncthreads();
  }
}

// 16 bytes a thread: of a row of k, then of v.
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
  const hipError_t e = hipLaunchKernel((const void*)&evict_select_kernel, dim3((unsigned)(p.batch * p.kv_heads)), dim3(kThreads), args, 0, stream);
  if (e != hipSuccess) return e;
  const int64_t threads = (int64_t)p.batch * p.keep * p.kv_heads * (p.row_bytes / 16);
  return hipLaunchKernel((const void*)&evict_copy_kernel, dim3((unsigned)((threads + 255) / 256)), dim3(256), args, 0, stream);
}

}  // namespace wtc
