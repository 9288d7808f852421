// window_attention.hip -- kernels of wtc_window_attention and its gradients.
#include "layer_common.h"
#include "layer_kernels.h"

namespace wtc {
namespace {

// Keys that the query at position `pos` sees: the first `first` ones and then lo .. pos.
struct Seen {
  int lo, first, count;
  __device__ inline Seen(const AttnParams& p, int pos) {
    lo = (int)max((int64_t)0, (int64_t)pos - p.window + 1);
    first = min(p.sinks, lo);
    count = pos < 0 ? 0 : first + pos - lo + 1;
  }
  __device__ inline int key(int t) const { return t < first ? t : lo + t - first; }
};

template <int DT>
__device__ inline float dot_rows(const typename Elem<DT>::type* x, const typename Elem<DT>::type* y, int dim) {
  float s = 0.0f;
  for (int d = 0; d < dim; ++d) s = __builtin_fmaf((float)x[d], (float)y[d], s);
  return s;
}
__device__ inline float wave_max(float x) {
  for (int o = 32; o; o >>= 1) x = fmaxf(x, __shfl_xor(x, o));
  return x;
}
__device__ inline float wave_sum(float x) {
  for (int o = 32; o; o >>= 1) x += __shfl_xor(x, o);
  return x;
}

// One wave a query row: 64 keys at a time, a running maximum and sum.
template <int DT>
__global__ void __launch_bounds__(64) attention_rows_kernel(const AttnParams p) {
  using T = typename Elem<DT>::type;
  const int lane = threadIdx.x;
  const int h = blockIdx.x % p.heads;
  const int i = blockIdx.x / p.heads % p.lq, b = blockIdx.x / p.heads / p.lq;
  const int nq = seq_queries(p, b), pos = i + seq_keys(p, b) - nq;
  const T* q = (const T*)p.q + b * p.q_stride[0] + i * p.q_stride[1] + h * p.q_stride[2];
  const T* k = (const T*)p.k + b * p.k_stride[0] + h / p.group * p.k_stride[2];
  const T* v = (const T*)p.v + b * p.v_stride[0] + h / p.group * p.v_stride[2];
  Seen seen(p, pos);
  if (i >= nq) seen.count = 0;
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
  Seen seen(p, pos);
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

hipError_t launch_attention(const AttnParams& p, int dt, hipStream_t stream) {
  return launch(WTC_BY_TYPE(attention_rows_kernel, dt), (int64_t)p.batch * p.lq * p.heads, 64, p, stream);
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
