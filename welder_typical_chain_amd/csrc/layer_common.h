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
// EXACT: to a few steps of f32 relative to the result, tails included (f32 outputs,
// slopes).  Otherwise to 2e-5, enough below a rounding to 16 bits: a tile's epilogue
// has its SIMD to itself, and what EXACT adds shows in full (4096 x 4096 x 1024 with gelu
// and f32 outputs 52 -> 60 us; bf16 outputs 8192 x 8192 x 4096 513 either way).
constexpr float kLn2Act = 0.6931471805599453f;

// exp(x), x <= 0.  A product with log2 e alone is off by |x| 2^-24 relative to the
// exponential: what it lost goes to first order into the result.
template <bool EXACT> __device__ inline float exp_neg(float x) {
  constexpr float kL = 1.4426950216293335f, kLow = 1.9259629911e-8f;  // log2 e in two parts
  if constexpr (!EXACT) return __builtin_amdgcn_exp2f(kL * x);
  x = fmaxf(x, -200.0f);  // (0 from -104 on; an infinity would give inf - inf below)
  const float a = kL * x;
  const float low = __builtin_fmaf(kLow, x, __builtin_fmaf(kL, x, -a));
  const float e = __builtin_amdgcn_exp2f(a);
  return __builtin_fmaf(e, low * kLn2Act, e);
}

// Phi(-u) for u >= 0 and e = exp(-u^2 / 2).  Phi(-u) / e falls off like 1 / u; in t =
// 1 / (1 + p u) it is t times a polynomial, fitted here for the least relative error over
// u in [0, 15] (beyond, e is 0 in f32): 1.1e-6 with seven terms, 3.2e-9 with ten.
template <bool EXACT> __device__ inline float normal_tail(float u, float* e) {
  if constexpr (EXACT) {
    u = fminf(u, 20.0f);
    constexpr float kC = -0.72134751081466675f, kLow = -9.6298149556e-9f;  // -log2(e) / 2 in two parts
    const float sq = u * u, sq_low = __builtin_fmaf(u, u, -sq), a = kC * sq;
    const float low = __builtin_fmaf(kC, sq_low, __builtin_fmaf(kLow, sq, __builtin_fmaf(kC, sq, -a)));
    const float x = __builtin_amdgcn_exp2f(a);
    *e = __builtin_fmaf(x, low * kLn2Act, x);
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.24f, u, 1.0f));
    float y = 0.025550249885556375f;
    y = __builtin_fmaf(y, t, -0.1247736784746638f);
    y = __builtin_fmaf(y, t, 0.20581449505106691f);
    y = __builtin_fmaf(y, t, -0.1447380430190452f);
    y = __builtin_fmaf(y, t, 0.1418602120985404f);
    y = __builtin_fmaf(y, t, 0.027922579540306077f);
    y = __builtin_fmaf(y, t, 0.08784785440251673f);
    y = __builtin_fmaf(y, t, 0.08891451431208887f);
    y = __builtin_fmaf(y, t, 0.09585989701536322f);
    y = __builtin_fmaf(y, t, 0.09574192077833424f);
    return y * t * *e;
  } else {
    *e = __builtin_amdgcn_exp2f(-0.72134752044448170f * u * u);
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.36f, u, 1.0f));
    float y = 0.0465226344455747f;
    y = __builtin_fmaf(y, t, -0.17793573815964808f);
    y = __builtin_fmaf(y, t, 0.17846623471992618f);
    y = __builtin_fmaf(y, t, 0.028257545930096425f);
    y = __builtin_fmaf(y, t, 0.13909894153507807f);
    y = __builtin_fmaf(y, t, 0.14188468341772179f);
    y = __builtin_fmaf(y, t, 0.14370518277156705f);
    return y * t * *e;
  }
}
template <bool EXACT> __device__ inline float normal_cdf(float z, float* e) {
  const float tail = normal_tail<EXACT>(fabsf(z), e);
  return z < 0.0f ? tail : 1.0f - tail;
}
// *rest: 1 - sigmoid(z), as exactly as the sigmoid itself
__device__ inline float sigmoid_exact(float z, float* rest) {
  const float e = exp_neg<true>(-fabsf(z)), big = __builtin_amdgcn_rcpf(1.0f + e), small = e * big;
  *rest = z < 0.0f ? big : small;
  return z < 0.0f ? small : big;
}
template <bool EXACT> __device__ inline float sigmoid(float z) {
  float rest;
  if constexpr (EXACT) return sigmoid_exact(z, &rest);
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * z));
}
constexpr float kTanhC = 1.5957691216057308f;   // 2 sqrt(2 / pi): tanh(u) = 2 sigmoid(2u) - 1
constexpr float kTanhC3 = 0.044715f;

template <int ACT, bool EXACT> __device__ inline float act_value(float z) {
  if constexpr (ACT == WTC_ACT_RELU) return z < 0.0f ? 0.0f : z;  // NaN stays NaN
  // z of -inf: Phi and the sigmoid are 0 there, and so is the product's limit
  if constexpr (ACT == WTC_ACT_GELU) {
    float e;
    return z == -INFINITY ? 0.0f : z * normal_cdf<EXACT>(z, &e);
  }
  if constexpr (ACT == WTC_ACT_GELU_TANH)
    return z == -INFINITY ? 0.0f : z * sigmoid<EXACT>(kTanhC * z * __builtin_fmaf(kTanhC3 * z, z, 1.0f));
  if constexpr (ACT == WTC_ACT_SILU) return z == -INFINITY ? 0.0f : z * sigmoid<EXACT>(z);
  return z;
}
// Far out the slopes are 0 or 1 to the last bit of f32 (and the formulas would meet inf * 0).
template <int ACT> __device__ inline float act_slope(float z) {
  if constexpr (ACT == WTC_ACT_RELU) return z > 0.0f ? 1.0f : (z <= 0.0f ? 0.0f : z);
  if constexpr (ACT == WTC_ACT_GELU) {
    if (fabsf(z) > 16.0f) return z < 0.0f ? 0.0f : 1.0f;
    float e;
    const float y = normal_cdf<true>(z, &e);
    return __builtin_fmaf(z * 0.3989422804014327f, e, y);
  }
  if constexpr (ACT == WTC_ACT_GELU_TANH) {
    if (fabsf(z) > 16.0f) return z < 0.0f ? 0.0f : 1.0f;
    float rest;
    const float y = sigmoid_exact(kTanhC * z * __builtin_fmaf(kTanhC3 * z, z, 1.0f), &rest);
    return y * __builtin_fmaf(z * rest * kTanhC, __builtin_fmaf(3.0f * kTanhC3 * z, z, 1.0f), 1.0f);
  }
  if constexpr (ACT == WTC_ACT_SILU) {
    if (fabsf(z) > 128.0f) return z < 0.0f ? 0.0f : 1.0f;
    float rest;
    const float y = sigmoid_exact(z, &rest);
    return y * __builtin_fmaf(z, rest, 1.0f);
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
  float *row_lse, *row_delta;  // backward: a row's lse in the log2 domain, less its weights' bits; -sum of dout * out
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
  int32_t full;       // every query sees every key: it stands behind the last one
  int32_t seq_rows;   // a batch's queries as one sequence: tokens of each in q (0: they are not)
  int32_t slots, slot0;  // partial results of a row, and this launch's first (slots 0: it writes results)
  const uint8_t *kp, *vp;  // keys that a batch shares, [prefix][kv_heads][dim]
  int64_t kp_stride[2], vp_stride[2];
  int32_t prefix;
  float *weights, *scores;  // [batch][kv_heads][lk]; of a decode step, see window_decode.hip
  int32_t add;              // weights: added to what is there
};

// Tokens of sequence b: queries and keys (clamped to what the tensors hold).
__device__ inline int seq_queries(const AttnParams& p, int b) {
  return p.q_lens ? min(max(p.q_lens[b], 0), p.lq) : p.lq;
}
__device__ inline int seq_keys(const AttnParams& p, int b) {
  return p.k_lens ? min(max(p.k_lens[b], 0), p.lk) : p.lk;
}
// Position of a sequence's query 0 among its nk keys, of which a query sees those up to its own.
__device__ inline int first_position(const AttnParams& p, int nq, int nk) { return p.full ? nk - 1 : nk - nq; }

}  // namespace wtc
