// window_decode.hip -- kernels of wtc_window_attention_decode.
#include "layer_common.h"
#include "layer_kernels.h"

namespace wtc {
namespace {

// One wave a query head: 64 keys at a time.  The wave of a key head's first
// query head writes the new row; the others read it from k_new / v_new, and
// no wave reads the row it replaces.
template <int DT>
__global__ void __launch_bounds__(64) decode_rows_kernel(const AttnParams p) {
  using T = typename Elem<DT>::type;
  const int lane = threadIdx.x;
  const int h = blockIdx.x % p.heads, b = blockIdx.x / p.heads, hk = h / p.group;
  const int rest = p.lk - p.sinks;
  const int n = max(p.k_lens[b], 0), pos = n - 1;
  const T* q = (const T*)p.q + b * p.q_stride[0] + h * p.q_stride[2];
  T* k = (T*)p.k + b * p.k_stride[0] + hk * p.k_stride[2];
  T* v = (T*)p.v + b * p.v_stride[0] + hk * p.v_stride[2];
  const T* kn = p.k_new ? (const T*)p.k_new + b * p.kn_stride[0] + hk * p.kn_stride[1] : nullptr;
  const T* vn = p.v_new ? (const T*)p.v_new + b * p.vn_stride[0] + hk * p.vn_stride[1] : nullptr;
  const int lo = (int)max((int64_t)0, (int64_t)pos - p.window + 1);
  const int first = min(p.sinks, lo), count = n == 0 ? 0 : first + pos - lo + 1;
  auto key = [&](int t) { return t < first ? t : lo + t - first; };
  auto row = [&](int j) { return (int64_t)(j < p.lk ? j : p.sinks + (j - p.sinks) % rest); };
  float top = -INFINITY, total = 0.0f, acc[2] = {0.0f, 0.0f};
  for (int t0 = 0; t0 < count; t0 += 64) {
    const bool in = t0 + lane < count;
    float s = -INFINITY;
    if (in) {
      const int j = key(t0 + lane);
      const T* kr = j == pos && kn ? kn : k + row(j) * p.k_stride[1];
      s = 0.0f;
      for (int d = 0; d < p.dim; ++d) s = __builtin_fmaf((float)q[d], (float)kr[d], s);
      s *= p.scale;
    }
    float next = s;
    for (int o = 32; o; o >>= 1) next = fmaxf(next, __shfl_xor(next, o));
    next = fmaxf(top, next);
    const float keep = next == -INFINITY ? 1.0f : __expf(top - next);
    const float e = in ? (next == -INFINITY ? (s != s ? s : 0.0f) : __expf(s - next)) : 0.0f;
    float sum = e;
    for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
    total = total * keep + sum;
    acc[0] *= keep;
    acc[1] *= keep;
    top = next;
    for (int t = 0; t < min(64, count - t0); ++t) {
      const float w = __shfl(e, t);
      const int j = key(t0 + t);
      const T* vr = j == pos && vn ? vn : v + row(j) * p.v_stride[1];
      for (int c = 0; c < 2; ++c)
        if (lane + 64 * c < p.dim) acc[c] = __builtin_fmaf(w, (float)vr[lane + 64 * c], acc[c]);
    }
  }
  T* out = (T*)p.out + b * p.o_stride[0] + h * p.o_stride[2];
  const float r = total == 0.0f ? 0.0f : 1.0f / total;
  for (int c = 0; c < 2; ++c)
    if (lane + 64 * c < p.dim) {
      out[lane + 64 * c] = (T)(acc[c] * r);
      if (kn && n && h % p.group == 0) {
        k[row(pos) * p.k_stride[1] + lane + 64 * c] = kn[lane + 64 * c];
        v[row(pos) * p.v_stride[1] + lane + 64 * c] = vn[lane + 64 * c];
      }
    }
}

}  // namespace

hipError_t launch_attention_decode(const AttnParams& p, int dt, hipStream_t stream) {
  AttnParams q = p;
  void* args[] = {&q};
  const void* fn = dt == DT_F16 ? (const void*)&decode_rows_kernel<DT_F16> : (const void*)&decode_rows_kernel<DT_BF16>;
  return hipLaunchKernel(fn, dim3((unsigned)(p.batch * p.heads)), dim3(64), args, 0, stream);
}

}  // namespace wtc
