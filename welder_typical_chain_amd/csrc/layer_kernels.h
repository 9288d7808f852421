// layer_kernels.h -- host-side launch functions of the kernels behind
// include/wtc/wtc_layer.h.  Arguments are checked by the callers
// (layer_launch.hip).
#pragma once
#include "layer_common.h"

namespace wtc {

struct MatmulPlan {
  int variant, splits, slabs;
  double us;  // estimate
};
MatmulPlan plan_matmul(int64_t m, int64_t n, int64_t k, bool aks, bool bks, int cu_count);
int64_t matmul_workspace(const MatmulPlan& plan, int64_t m, int64_t n);
void matmul_tile_size(const MatmulPlan& plan, int64_t* tile_m, int64_t* tile_n);
// aks / bks: the operand is strided along k (element (row, k) at k * ld + row) instead
// of contiguous (row * ld + k); aks only with bks and out_dt == dt.
hipError_t launch_matmul(const MatmulParams& p, const MatmulPlan& plan, int dt, int out_dt, bool aks, bool bks,
                         hipStream_t stream);

// da = x . y and db of an [m][k] . [k][n] product, whether one launch for both is
// faster; bks: of da's second operand.
bool pair_pays(const MatmulPlan& da, const MatmulPlan& db, int64_t m, int64_t n, int64_t k, int cu_count);
MatmulPlan pair_plan(int64_t k);  // of one of them alone, k elements summed
hipError_t launch_matmul_pair(const MatmulParams& da, const MatmulParams& db, int dt, bool bks, hipStream_t stream);

struct ActBackwardParams {
  const void* dout;
  const float* pre;  // dense [m][n]
  void* dz;          // dense [m][n]; NULL: not written
  float* dbias;      // [n]; NULL: not computed
  float* partial;    // [chunks][n], if chunks > 1
  int64_t m, n, ldd, chunk_rows;
  int32_t chunks, act;
};
int64_t act_backward_chunk_rows(int64_t m, int64_t n, int cu_count);
hipError_t launch_act_backward(const ActBackwardParams& p, int dt, hipStream_t stream);

struct AttnPlan {
  int key_groups, splits;
  enum { TILE, ROWS, FEW } kernel;  // attention_tile_kernel, launch_attention_rows, launch_few_rows
  int cu_count;
};
AttnPlan plan_attention(const AttnParams& p, int cu_count);
int64_t attention_workspace(const AttnParams& p, const AttnPlan& plan);
// p.part_out: attention_workspace() bytes
hipError_t launch_attention(const AttnParams& p, const AttnPlan& plan, int dt, hipStream_t stream);
// Many rows that see nearly all of their keys (p.full, or behind p.prefix).
// Splits; p.part_out of launch_attention_rows: attention_workspace() bytes.
int plan_attention_rows(const AttnParams& p, int cu_count);
int attention_rows_blocks(const AttnParams& p, int splits, int cu_count);  // of 32 rows a wave
double attention_rows_us(const AttnParams& p, int splits, int slots, int cu_count);
hipError_t launch_attention_rows(const AttnParams& p, int splits, int cu_count, int dt, hipStream_t stream);
// Few rows (p.full) against many keys; splits, 0: too many rows.  p.part_out: as above.
int plan_few_rows(const AttnParams& p, int cu_count);
hipError_t launch_few_rows(const AttnParams& p, int splits, int dt, hipStream_t stream);
// One token a sequence: the batch's queries as one sequence's against a prefix, and own caches,
// into p.slots partial results, and their join; splits of both.
struct PrefixTokenPlan {
  int common, own;
  bool many;  // attention_rows for the prefix
};
PrefixTokenPlan plan_prefix_token(const AttnParams& common, const AttnParams& own, int cu_count);
hipError_t launch_prefix_token(const AttnParams& common, const AttnParams& own, const PrefixTokenPlan& plan, int dt, hipStream_t stream);
// Results of the rows from p.slots partial ones, p.part_out [batch][lq][heads][slots][dim] and p.part_lse without dim.
hipError_t launch_attention_join(const AttnParams& p, int dt, hipStream_t stream);
struct AttnBackwardPlan {
  int dq_groups;  // waves that share a query row
  bool together;  // dq and dk / dv in one launch
  int key_blocks, near_blocks, near_chunks, far_blocks, far_chunks, far_keys;
  int64_t part_at, far_at, workspace;  // bytes
};
AttnBackwardPlan plan_attention_backward(const AttnParams& p, int cu_count);
// p.row_lse: plan.workspace bytes
hipError_t launch_attention_backward(const AttnParams& p, const AttnBackwardPlan& plan, int dt, hipStream_t stream);
int plan_decode(const AttnParams& p, int cu_count);  // splits
int plan_decode_joined(const AttnParams& p, int rounds, int cu_count);  // the same where a second launch is there anyway
int64_t decode_workspace(const AttnParams& p, int splits);
// p.part_out: decode_workspace() bytes; p.window: at most p.lk - p.sinks
hipError_t launch_attention_decode(const AttnParams& p, int splits, int dt, hipStream_t stream);
// The same with p.weights; p.part_out: decode_weights_workspace() bytes
int64_t decode_weights_workspace(const AttnParams& p, int splits);
hipError_t launch_attention_decode_weights(const AttnParams& p, int splits, int dt, hipStream_t stream);

struct KeyWeightsPlan {
  int key_blocks, chunks, chunk_rows;  // chunks of the queries, positions of each
  int64_t workspace;
};
KeyWeightsPlan plan_key_weights(const AttnParams& p, int cu_count);
// p.lse_in, p.weights, p.add; p.part_out: plan.workspace bytes
hipError_t launch_key_weights(const AttnParams& p, const KeyWeightsPlan& plan, int dt, hipStream_t stream);

struct EvictParams {
  const uint8_t *k, *v;
  uint8_t *k_out, *v_out;
  const float* weights;  // [batch][kv_heads][rows]
  float* weights_out;    // [batch][kv_heads][out_rows]
  const int32_t* lengths;
  int32_t *kept, *lengths_out;  // [batch][kv_heads][keep]: source rows
  int64_t k_stride[3], v_stride[3], ko_stride[3], vo_stride[3];  // bytes
  int32_t batch, kv_heads, rows, out_rows, keep, recent, sinks, row_bytes;
};
hipError_t launch_cache_evict(const EvictParams& p, hipStream_t stream);

}  // namespace wtc
