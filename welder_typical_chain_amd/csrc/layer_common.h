// layer_common.h -- arguments and device helpers shared by the kernels of
// include/wtc/wtc_layer.h (matmul_epilogue.hip, window_attention.hip,
// window_decode.hip) and their launcher (layer_launch.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <string>

#include "device_common.h"
#include "wtc/wtc_layer.h"

namespace wtc {

// Sets the calling thread's wtc_last_error() text (launch.hip) and returns code.
int report(int code, const std::string& msg);

template <int DT> struct Elem;
template <> struct Elem<DT_F16> {
  typedef _Float16 type;
  typedef f16x8 vec8;
};
template <> struct Elem<DT_BF16> {
  typedef __bf16 type;
  typedef bf16x8 vec8;
};
template <> struct Elem<DT_F32> {
  typedef float type;
};

template <int DT>
__device__ inline f32x16 mfma32(const u32x4& a, const u32x4& b, const f32x16& c) {
  if constexpr (DT == DT_F16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// ---- activations -----------------------------------------------------------
// erfc(|x|) by Abramowitz & Stegun 7.1.26 (|error| <= 1.5e-7): t = 1 / (1 + p |x|),
// (a1 t + .. + a5 t^5) exp(-x^2).  Taken as erfc so that the tail of the normal
// distribution keeps its relative size.
__device__ inline float erfc_abs(float x) {
  const float ax = fabsf(x);
  const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.3275911f, ax, 1.0f));
  float y = 1.061405429f;
  y = __builtin_fmaf(y, t, -1.453152027f);
  y = __builtin_fmaf(y, t, 1.421413741f);
  y = __builtin_fmaf(y, t, -0.284496736f);
  y = __builtin_fmaf(y, t, 0.254829592f);
  return y * t * __builtin_amdgcn_exp2f(-1.4426950408889634f * ax * ax);
}
__device__ inline float normal_cdf(float z) {  // Phi(z) = erfc(-z / sqrt 2) / 2
  const float half = 0.5f * erfc_abs(z * 0.70710678118654752f);
  return z < 0.0f ? half : 1.0f - half;
}
__device__ inline float sigmoid(float z) {
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * z));
}
constexpr float kTanhC = 1.5957691216057308f;   // 2 sqrt(2 / pi): tanh(u) = 2 sigmoid(2u) - 1
constexpr float kTanhC3 = 0.044715f;

template <int ACT> __device__ inline float act_value(float z) {
  if constexpr (ACT == WTC_ACT_RELU) return z < 0.0f ? 0.0f : z;  // NaN stays NaN
  // z of -inf: Phi and the sigmoid are 0 there, and so is the product's limit
  if constexpr (ACT == WTC_ACT_GELU) return z == -INFINITY ? 0.0f : z * normal_cdf(z);
  if constexpr (ACT == WTC_ACT_GELU_TANH)
    return z == -INFINITY ? 0.0f : z * sigmoid(kTanhC * z * __builtin_fmaf(kTanhC3 * z, z, 1.0f));
  if constexpr (ACT == WTC_ACT_SILU) return z == -INFINITY ? 0.0f : z * sigmoid(z);
  return z;
}
// Far out the slopes are 0 or 1 to the last bit of f32 (and the formulas would meet inf * 0).
template <int ACT> __device__ inline float act_slope(float z) {
  if constexpr (ACT == WTC_ACT_RELU) return z > 0.0f ? 1.0f : (z <= 0.0f ? 0.0f : z);
  if constexpr (ACT == WTC_ACT_GELU) {
    if (fabsf(z) > 16.0f) return z < 0.0f ? 0.0f : 1.0f;
    return __builtin_fmaf(z * 0.3989422804014327f, __builtin_amdgcn_exp2f(-0.7213475204444817f * z * z), normal_cdf(z));
  }
  if constexpr (ACT == WTC_ACT_GELU_TANH) {
    if (fabsf(z) > 16.0f) return z < 0.0f ? 0.0f : 1.0f;
    const float y = sigmoid(kTanhC * z * __builtin_fmaf(kTanhC3 * z, z, 1.0f));
    return __builtin_fmaf(z * y * (1.0f - y) * kTanhC, __builtin_fmaf(3.0f * kTanhC3 * z, z, 1.0f), y);
  }
  if constexpr (ACT == WTC_ACT_SILU) {
    if (fabsf(z) > 128.0f) return z < 0.0f ? 0.0f : 1.0f;
    const float y = sigmoid(z);
    return y * __builtin_fmaf(z, 1.0f - y, 1.0f);
  }
  return 1.0f;
}

// ---- kernel arguments --------------------------------------------------------
struct MatmulParams {
  const uint8_t *a, *b;
  const void *bias, *residual;
  void *out, *pre;
  float* partial;        // [splits][m][n], if splits > 1
  int64_t lda, ldb;      // elements between rows (KC) or between k (KS)
  int64_t ldr, ldo, ldp;
  int32_t m, n, k;
  int32_t bias_f32, act;
  int32_t splits, slabs;  // k-slabs per split
};

struct AttnParams {
  const uint8_t *q, *k, *v, *dout, *o;
  uint8_t *out, *dq, *dk, *dv;
  const float* lse_in;
  float* lse;
  float *row_lse, *row_delta;  // backward: a row's lse in the log2 domain, sum of dout * out
  const int32_t *q_lens, *k_lens;
  const uint8_t *k_new, *v_new;
  int64_t q_stride[3], k_stride[3], v_stride[3], o_stride[3], do_stride[3];  // elements
  int64_t kn_stride[2], vn_stride[2];
  int64_t window;  // INT32_MAX at most (no limit)
  float *part_out, *part_lse;  // of a row's splits: normalised results and log-sum-exp
  float *part_near, *part_far;
  int32_t splits, row_blocks;
  int32_t key_blocks, near_blocks, near_chunks, far_blocks, far_chunks, far_keys;
  int32_t batch, heads, kv_heads, group, lq, lk, dim, sinks;
  float scale;
};

// Tokens of sequence b: queries and keys (clamped to what the tensors hold).
__device__ inline int seq_queries(const AttnParams& p, int b) {
  return p.q_lens ? min(max(p.q_lens[b], 0), p.lq) : p.lq;
}
__device__ inline int seq_keys(const AttnParams& p, int b) {
  return p.k_lens ? min(max(p.k_lens[b], 0), p.lk) : p.lk;
}

}  // namespace wtc
