/*
 * wtc_layer.h -- C-ABI of the operators around the fused Matmul->row-Softmax
 * chain that a transformer layer needs, on device pointers and a HIP stream:
 *
 *   wtc_matmul_epilogue            out = round(act(A . B + bias) + residual)
 *   wtc_matmul_epilogue_backward   dA, dB, dbias of it
 *   wtc_window_attention           causal attention with a sliding window and
 *                                  a few first tokens that stay visible
 *   wtc_window_attention_backward  dQ, dK, dV of it
 *   wtc_window_attention_decode    the same for one token a sequence against
 *                                  a cache, which it also appends to
 *   wtc_cross_attention            attention to another sequence: no order, every
 *                                  query sees every key
 *   wtc_cross_attention_backward   dQ, dK, dV of it
 *   wtc_prefix_attention           causal attention of a batch behind a prefix that
 *                                  its sequences share
 *   wtc_prefix_attention_decode    the same for one token a sequence
 *   wtc_window_attention_weights   what each key has received from the queries
 *   wtc_window_attention_decode_weights  decode that adds up what its rows receive
 *   wtc_cache_evict                a smaller cache of the rows of most weight
 *   wtc_*_plan                     what such a call runs
 *
 * Status codes, wtc_last_error() and element type codes are wtc_hip.h's.
 * Every call is asynchronous on `stream` (a hipStream_t, or NULL) and may be
 * captured into a graph: nothing is allocated, synchronised or kept.  All
 * buffers are the caller's.  Where a *_workspace_size function says that a
 * call needs scratch memory, the caller passes it (256-byte aligned,
 * uninitialised; calls that may overlap must not share one); too little of it
 * is WTC_ERR_WORKSPACE.  Outputs may not overlap inputs, but for the residual,
 * which may be the output itself, and the caches and weights that decode and
 * wtc_window_attention_weights add to.  Calls
 * may come from any host thread.  Results do not depend on timing: nothing is
 * summed by atomics.
 */
#ifndef WTC_LAYER_H
#define WTC_LAYER_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define WTC_ACT_NONE 0
#define WTC_ACT_RELU 1
#define WTC_ACT_GELU 2      /* z * Phi(z) */
#define WTC_ACT_GELU_TANH 3 /* its tanh form */
#define WTC_ACT_SILU 4

/*
 * A matrix product with an epilogue.  A [m][k] row-major; B [k][n] row-major,
 * or with b_trans its transpose stored as [n][k]; out, residual and pre [m][n].
 * The ld* are row strides in elements.  dtype (WTC_DTYPE_F16 / BF16): A and B;
 * out_dtype (dtype or WTC_DTYPE_F32): out and residual; bias_dtype
 * (dtype or WTC_DTYPE_F32): bias.  Every pointer, bias, residual and the
 * gradients too, is 16-byte aligned and every ld* a multiple of 8, and so are n and k
 * (k may be 0: then A . B is 0).  m and n may be 0.  No operand spans 2 GiB.
 * Activations and their slopes keep their relative accuracy out to both tails: to
 * a few roundings with f32 outputs, below the output's rounding with 16-bit ones.
 */
typedef struct wtc_matmul_args {
  int64_t m, n, k;
  int64_t lda, ldb, ldr, ldo;
  int64_t b_trans;
  int64_t dtype, out_dtype, bias_dtype;
  int64_t activation;
  int64_t ldd; /* dout (backward) */
} wtc_matmul_args;

int64_t wtc_matmul_epilogue_workspace_size(const wtc_matmul_args* p);
/* bias, residual and pre may be NULL.  pre: z = A . B + bias in f32 (dense
 * [m][n]), what the backward pass of an activation needs. */
int wtc_matmul_epilogue(const wtc_matmul_args* p, const void* a, const void* b, const void* bias,
                        const void* residual, void* out, float* pre, void* workspace, size_t workspace_bytes,
                        void* stream);

int64_t wtc_matmul_epilogue_backward_workspace_size(const wtc_matmul_args* p);
/* dz = dout * act'(pre); da = dz . B^T (dense [m][k]), db = A^T . dz (dense, in
 * B's layout), both of `dtype`, and dbias = the column sums of dz in f32.  Each
 * of the three may be NULL (not computed).  dout is of `dtype`.  pre may be
 * NULL with WTC_ACT_NONE.  The residual's gradient is dout itself.  The products
 * take dz rounded to `dtype`: in f16, dout is best scaled to well above 6e-5 and
 * below 5e4. */
int wtc_matmul_epilogue_backward(const wtc_matmul_args* p, const void* dout, const void* a, const void* b,
                                 const float* pre, void* da, void* db, float* dbias, void* workspace,
                                 size_t workspace_bytes, void* stream);

/* The kernel that a product of these sizes runs on a device of `cu_count` compute
 * units (0: the current one's): its output tile and the parts that k is split
 * into.  part: 0 the forward product, 1 da, 2 db.  16 x 16: the kernel for few
 * rows, which has no tiles. */
int wtc_matmul_epilogue_plan(const wtc_matmul_args* p, int part, int cu_count, int64_t* tile_m, int64_t* tile_n,
                             int64_t* splits);

/*
 * Attention.  q, out and dout [batch][lq][heads][dim]; k and v
 * [batch][lk][kv_heads][dim]; heads a multiple of kv_heads, query head h
 * reads key head h / (heads / kv_heads).  Strides (elements) of sequence,
 * token and head; dim is contiguous, a multiple of 8 up to 128.  All starts
 * and strides are 16-byte aligned.  dtype: WTC_DTYPE_F16 or BF16.
 *
 * q_lens / k_lens: int32 [batch] on the device, the tokens of each sequence
 * (clamped to lq / lk), or NULL (all).  The queries are the last tokens: query
 * i of a sequence stands at position p = i + k_len - q_len and sees the keys
 * j <= p with p - j < window or j < sinks (window 0: no limit).  A query that
 * sees no key, or stands behind its sequence's end, gives zeros (log-sum-exp
 * -inf, gradient 0); keys behind the end are not read (gradient 0).  A NaN or an
 * infinity that the mask hides from a row does not reach it; a NaN that the row
 * sees does, whatever its weight.
 *
 * Sums and statistics are f32; the products take the softmax weights, and in the
 * backward pass their gradients, rounded to dtype (f16: times powers of two that
 * keep them in its range).
 */
typedef struct wtc_attention_args {
  int64_t batch, heads, kv_heads, lq, lk, dim;
  int64_t window, sinks;
  int64_t dtype;
  int64_t q_stride[3], k_stride[3], v_stride[3], o_stride[3];
  int64_t do_stride[3];            /* backward: dout */
  int64_t kn_stride[2], vn_stride[2]; /* decode: sequence and head of k_new, v_new */
  const int32_t* q_lens;
  const int32_t* k_lens;
  double scale;
} wtc_attention_args;

int64_t wtc_window_attention_workspace_size(const wtc_attention_args* p);
/* lse: f32 [batch][heads][lq], the rows' log-sum-exp of scale * q . k (NULL: not written) */
int wtc_window_attention(const wtc_attention_args* p, const void* q, const void* k, const void* v, void* out,
                         float* lse, void* workspace, size_t workspace_bytes, void* stream);

int64_t wtc_window_attention_backward_workspace_size(const wtc_attention_args* p);
/* out and lse: of the forward call.  dq, dk, dv: dense, in the layouts of q, k, v. */
int wtc_window_attention_backward(const wtc_attention_args* p, const void* dout, const void* q, const void* k,
                                  const void* v, const void* out, const float* lse, void* dq, void* dk, void* dv,
                                  void* workspace, size_t workspace_bytes, void* stream);

/* What the two calls above run on a device of `cu_count` compute units (0: the
 * current one's), five numbers: waves that share a query row and key splits of
 * the forward pass; waves that share a row in dq; parts of a key block's queries
 * in dk / dv, and workgroups for the first tokens' far queries. */
int wtc_window_attention_plan(const wtc_attention_args* p, int cu_count, int64_t* plan);

int64_t wtc_window_attention_decode_workspace_size(const wtc_attention_args* p);
/* One token a sequence (lq = 1).  k and v are caches of lk rows a sequence, lk
 * > sinks: token j stands in row j if j < sinks, else in row sinks + (j -
 * sinks) % (lk - sinks), so that a cache that is full keeps the first `sinks`
 * and the newest lk - sinks tokens (the window is at most that).  k_lens:
 * tokens of each sequence with the new one, any number (0: an idle sequence;
 * its out is 0 and its cache is left alone).  k_new, v_new
 * [batch][kv_heads][dim]: the new token's key and value, written to the
 * caches and attended to (the caches are two then); both NULL: the caches hold
 * them already.  A cache's rows do not overlap; stride 0, one row for all tokens,
 * is for caches that are only read. */
int wtc_window_attention_decode(const wtc_attention_args* p, const void* q, void* k, void* v, const void* k_new,
                                const void* v_new, void* out, void* workspace, size_t workspace_bytes,
                                void* stream);

/*
 * Attention to another sequence: as wtc_window_attention, but query i < q_len sees
 * every key j < k_len.  window and sinks are 0; lq + lk is at most 2^30.
 * The rows of a sequence of k, and of v, do not overlap.
 */
int64_t wtc_cross_attention_workspace_size(const wtc_attention_args* p);
int wtc_cross_attention(const wtc_attention_args* p, const void* q, const void* k, const void* v, void* out,
                        float* lse, void* workspace, size_t workspace_bytes, void* stream);
int64_t wtc_cross_attention_backward_workspace_size(const wtc_attention_args* p);
int wtc_cross_attention_backward(const wtc_attention_args* p, const void* dout, const void* q, const void* k,
                                 const void* v, const void* out, const float* lse, void* dq, void* dk, void* dv,
                                 void* workspace, size_t workspace_bytes, void* stream);

/* What the two calls above run on a device of `cu_count` compute units (0: the
 * current one's), five numbers: whether the kernel for few rows takes the forward
 * pass; row blocks of 32 that a wave holds; key splits; whether the gradients are
 * one launch behind the rows' statistics; parts of a key block's queries in dk / dv. */
int wtc_cross_attention_plan(const wtc_attention_args* p, int cu_count, int64_t* plan);

/*
 * A prefix that all sequences of a batch share, [prefix][kv_heads][dim], strides of
 * token and head.  A query i < q_len sees every prefix key and, of its sequence's
 * own keys, those that it sees in wtc_window_attention without a window (window and
 * sinks are 0).  prefix and lk may be 0; the prefix's rows do not overlap.
 */
typedef struct wtc_prefix_args {
  int64_t prefix;
  int64_t kp_stride[2], vp_stride[2];
} wtc_prefix_args;

int64_t wtc_prefix_attention_workspace_size(const wtc_attention_args* p, const wtc_prefix_args* x);
/* lse: as in wtc_window_attention, over prefix and own keys (NULL: not written) */
int wtc_prefix_attention(const wtc_attention_args* p, const wtc_prefix_args* x, const void* q, const void* k_prefix,
                         const void* v_prefix, const void* k, const void* v, void* out, float* lse, void* workspace,
                         size_t workspace_bytes, void* stream);

/* What it runs on a device of `cu_count` compute units (0: the current one's), four
 * numbers: whether one launch takes prefix and own keys; key splits of the prefix's
 * own launch (0: there is none) and of the launch for the own keys or for both (0:
 * none); row blocks of 32 that a wave holds where the prefix is read. */
int wtc_prefix_attention_plan(const wtc_attention_args* p, const wtc_prefix_args* x, int cu_count, int64_t* plan);

int64_t wtc_prefix_attention_decode_workspace_size(const wtc_attention_args* p, const wtc_prefix_args* x);
/* One token a sequence.  The own caches, their lengths (without the prefix) and the
 * new token as in wtc_window_attention_decode without sinks: token j stands in row
 * j % lk.  A sequence of length 0 is idle: its out is 0. */
int wtc_prefix_attention_decode(const wtc_attention_args* p, const wtc_prefix_args* x, const void* q,
                                const void* k_prefix, const void* v_prefix, void* k, void* v, const void* k_new,
                                const void* v_new, void* out, void* workspace, size_t workspace_bytes, void* stream);

/*
 * What each key receives, f32 [batch][kv_heads][lk]: the sum over the query heads of
 * its key head and the queries that see it of exp(scale q . k - lse), lse f32
 * [batch][heads][lq] as wtc_window_attention gave it for the same arguments.  With
 * add, it is added to what `weights` holds; otherwise it replaces it (keys behind
 * their sequence's end: 0).
 */
int64_t wtc_window_attention_weights_workspace_size(const wtc_attention_args* p);
int wtc_window_attention_weights(const wtc_attention_args* p, const void* q, const void* k, const float* lse,
                                 float* weights, int add, void* workspace, size_t workspace_bytes, void* stream);

/* wtc_window_attention_decode that also adds what each visible row of the cache
 * receives from the token to `weights`, f32 [batch][kv_heads][lk].  The newest
 * token's row is set to it: what it held was another token's. */
int64_t wtc_window_attention_decode_weights_workspace_size(const wtc_attention_args* p);
int wtc_window_attention_decode_weights(const wtc_attention_args* p, const void* q, void* k, void* v,
                                        const void* k_new, const void* v_new, void* out, float* weights,
                                        void* workspace, size_t workspace_bytes, void* stream);

/*
 * The rows of a cache that stay, in a smaller one.  k, v [batch][rows][kv_heads][dim],
 * weights [batch][kv_heads][rows] f32 (dense), lengths int32 [batch] (clamped to 0 ..
 * rows).  A sequence of up to `keep` rows keeps them all; of a longer one each key head
 * keeps the first `sinks`, the last `recent` and, of those between, the ones of
 * greatest weight (of equal ones the lowest rows; a NaN is the greatest).  They go,
 * in their order, to k_out, v_out [batch][out_rows][kv_heads][dim] and weights_out
 * [batch][kv_heads][out_rows], out_rows >= keep; rows [batch][kv_heads][keep] says
 * which they were (-1 behind the last one), lengths_out how many.  Behind a sequence's
 * last row, k_out and v_out are 0 up to row keep and left alone from there on;
 * weights_out is 0 to its end.  recent + sinks <= keep.  Strides (elements,
 * multiples of 8) of sequence, row and head; dtype f16 or bf16.
 */
typedef struct wtc_evict_args {
  int64_t batch, kv_heads, rows, out_rows, dim, dtype;
  int64_t keep, recent, sinks;
  int64_t k_stride[3], v_stride[3], ko_stride[3], vo_stride[3];
} wtc_evict_args;

int wtc_cache_evict(const wtc_evict_args* p, const void* k, const void* v, const float* weights,
                    const int32_t* lengths, void* k_out, void* v_out, float* weights_out, int32_t* rows,
                    int32_t* lengths_out, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* WTC_LAYER_H */
