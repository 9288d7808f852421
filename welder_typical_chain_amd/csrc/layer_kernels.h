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
};
AttnPlan plan_attention(const AttnParams& p, int cu_count);
int64_t attention_workspace(const AttnParams& p, const AttnPlan& plan);
// p.part_out: attention_workspace() bytes
hipError_t launch_attention(const AttnParams& p, const AttnPlan& plan, int dt, hipStream_t stream);
struct AttnBackwardPlan {
  int dq_groups;  // waves that share a query row
  int key_blocks, near_blocks, near_chunks, far_blocks, far_chunks, far_keys;
  int64_t part_at, far_at, workspace;  // bytes
};
AttnBackwardPlan plan_attention_backward(const AttnParams& p, int cu_count);
// p.row_lse: plan.workspace bytes
hipError_t launch_attention_backward(const AttnParams& p, const AttnBackwardPlan& plan, int dt, hipStream_t stream);
int plan_decode(const AttnParams& p, int cu_count);  // splits
int64_t decode_workspace(const AttnParams& p, int splits);
// p.part_out: decode_workspace() bytes; p.window: at most p.lk - p.sinks
hipError_t launch_attention_decode(const AttnParams& p, int splits, int dt, hipStream_t stream);

}  // namespace wtc
