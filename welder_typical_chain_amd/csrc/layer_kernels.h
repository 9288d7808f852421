// layer_kernels.h -- host-side launch functions of the kernels behind
// include/wtc/wtc_layer.h.  Arguments are checked by the callers
// (layer_launch.hip).
#pragma once
#include "layer_common.h"

namespace wtc {

struct ActBackwardParams {
  const void *dout, *pre;
  void* dz;      // dense [m][n]; NULL: not written
  float* dbias;  // [n]; NULL: not computed
  int64_t m, n, ldd;
  int32_t act;
};

hipError_t launch_matmul(const MatmulParams& p, int dt, int out_dt, hipStream_t stream);
hipError_t launch_act_backward(const ActBackwardParams& p, int dt, hipStream_t stream);

hipError_t launch_attention(const AttnParams& p, int dt, hipStream_t stream);
hipError_t launch_attention_backward(const AttnParams& p, int dt, hipStream_t stream);
hipError_t launch_attention_decode(const AttnParams& p, int dt, hipStream_t stream);

}  // namespace wtc
