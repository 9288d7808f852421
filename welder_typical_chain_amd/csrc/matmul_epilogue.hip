// matmul_epilogue.hip -- kernels of wtc_matmul_epilogue and its gradients.
#include "layer_common.h"
#include "layer_kernels.h"

namespace wtc {
namespace {

__device__ inline float load_elem(const void* p, int64_t i, int dt) {
  if (dt == DT_F32) return static_cast<const float*>(p)[i];
  if (dt == DT_F16) return (float)static_cast<const _Float16*>(p)[i];
  return (float)static_cast<const __bf16*>(p)[i];
}
template <int DT> __device__ inline void store_elem(void* p, int64_t i, float x) {
  static_cast<typename Elem<DT>::type*>(p)[i] = (typename Elem<DT>::type)x;
}

constexpr int kT = 16;

// One output element a thread, operands staged 16 x 16 at a time.
template <int DT, int OUT_DT>
__global__ void __launch_bounds__(kT* kT) matmul_simple_kernel(const MatmulParams p) {
  __shared__ float sa[kT][kT + 1], sb[kT][kT + 1];
  const int tx = threadIdx.x % kT, ty = threadIdx.x / kT;
  const int nt = (p.n + kT - 1) / kT;
  const int64_t i = (int64_t)(blockIdx.x / nt) * kT + ty, j = (int64_t)(blockIdx.x % nt) * kT + tx;
  const int64_t i_b = j - tx + ty;  // column of b this thread stages
  float acc = 0.0f;
  for (int k0 = 0; k0 < p.k; k0 += kT) {
    const int ka = k0 + tx;
    sa[ty][tx] = i < p.m && ka < p.k ? load_elem(p.a, i * p.a_row + ka * p.a_col, DT) : 0.0f;
    sb[tx][ty] = i_b < p.n && ka < p.k ? load_elem(p.b, ka * p.b_row + i_b * p.b_col, DT) : 0.0f;
    __syncthreads();
    for (int kk = 0; kk < kT; ++kk) acc = __builtin_fmaf(sa[ty][kk], sb[kk][tx], acc);
    __syncthreads();
  }
  if (i >= p.m || j >= p.n) return;
  if (p.bias) acc += load_elem(p.bias, j, p.bias_f32 ? DT_F32 : DT);
  if (p.pre) store_elem<DT>(p.pre, i * p.ldp + j, acc);
  acc = act_value(acc, p.act);
  if (p.residual) acc += load_elem(p.residual, i * p.ldr + j, OUT_DT);
  store_elem<OUT_DT>(p.out, i * p.ldo + j, acc);
}

// dz = dout * act'(pre), rounded for the products; a column's sum in f32 of the
// values before rounding.  One thread a column, rows in their order.
template <int DT>
__global__ void __launch_bounds__(256) act_backward_kernel(const ActBackwardParams p) {
  const int64_t j = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (j >= p.n) return;
  float sum = 0.0f;
  for (int64_t i = 0; i < p.m; ++i) {
    float g = load_elem(p.dout, i * p.ldd + j, DT);
    if (p.act != WTC_ACT_NONE) g *= act_slope(load_elem(p.pre, i * p.n + j, DT), p.act);
    sum += g;
    if (p.dz) store_elem<DT>(p.dz, i * p.n + j, g);
  }
  if (p.dbias) p.dbias[j] = sum;
}

}  // namespace

hipError_t launch_matmul(const MatmulParams& p, int dt, int out_dt, hipStream_t stream) {
  const int64_t grid = ((int64_t)(p.m + kT - 1) / kT) * ((p.n + kT - 1) / kT);
  const void* fn =
      dt == DT_F16 ? (out_dt == DT_F32 ? (const void*)&matmul_simple_kernel<DT_F16, DT_F32> : (const void*)&matmul_simple_kernel<DT_F16, DT_F16>)
                   : (out_dt == DT_F32 ? (const void*)&matmul_simple_kernel<DT_BF16, DT_F32> : (const void*)&matmul_simple_kernel<DT_BF16, DT_BF16>);
  MatmulParams q = p;
  void* args[] = {&q};
  return hipLaunchKernel(fn, dim3((unsigned)grid), dim3(kT * kT), args, 0, stream);
}

hipError_t launch_act_backward(const ActBackwardParams& p, int dt, hipStream_t stream) {
  const void* fn = dt == DT_F16 ? (const void*)&act_backward_kernel<DT_F16> : (const void*)&act_backward_kernel<DT_BF16>;
  ActBackwardParams q = p;
  void* args[] = {&q};
  return hipLaunchKernel(fn, dim3((unsigned)((p.n + 255) / 256)), dim3(256), args, 0, stream);
}

}  // namespace wtc
