// cross_attention.hip -- forward attention of many query rows that see (nearly) all
// of their keys: wtc_cross_attention, and both parts of wtc_prefix_attention.
#include "decode_tile.h"
#include "layer_kernels.h"
#include "rows_tile.h"

#include <algorithm>

namespace wtc {
namespace {

using namespace attn;

using namespace rows;

// A row block of 32 or two a wave (up to dim 64: two, and two workgroups a CU).  One a wave
// makes two waves a SIMD, between which issue slots and the two pipes are shared, but
// reads each key fragment twice as often.  On a full chip the clock then falls from 1.89
// to 1.65 GHz and two a wave are faster (4 x 2048 x 4096, 32 / 8 heads of 128: 465 us
// against 488); where workgroups are few, one (8 x 200 behind 4096: 121 against 126).
template <int DT, int ND, bool PREFIX, int A>
__global__ void __launch_bounds__(waves(A) * 64, A == 1 || ND <= 2 ? 2 : 1) attention_rows_kernel(const AttnParams p) {
  __shared__ __attribute__((aligned(256))) uint8_t smem[RowsLds<ND, A>::TOTAL];
  attention_rows<DT, ND, PREFIX, A>(p, smem, xcd_remap(blockIdx.x, gridDim.x));
}

template <int DT, bool PREFIX> const void* kernel_for(int nd, int a) {
  if (a == 1) {
    switch (nd) {
      case 1: return (const void*)&attention_rows_kernel<DT, 1, PREFIX, 1>;
      case 2: return (const void*)&attention_rows_kernel<DT, 2, PREFIX, 1>;
      case 3: return (const void*)&attention_rows_kernel<DT, 3, PREFIX, 1>;
    }
    return (const void*)&attention_rows_kernel<DT, 4, PREFIX, 1>;
  }
  switch (nd) {
    case 1: return (const void*)&attention_rows_kernel<DT, 1, PREFIX, 2>;
    case 2: return (const void*)&attention_rows_kernel<DT, 2, PREFIX, 2>;
    case 3: return (const void*)&attention_rows_kernel<DT, 3, PREFIX, 2>;
  }
  return (const void*)&attention_rows_kernel<DT, 4, PREFIX, 2>;
}

}  // namespace

int attention_rows_blocks(const AttnParams& p, int splits, int cu_count) {
  const int64_t blocks = ((int64_t)p.lq * p.group + kRows - 1) / kRows;
  return (int64_t)p.batch * p.kv_heads * blocks * splits <= cu_count ? 1 : 2;
}

// What a launch of so many splits takes about, with the join of `slots` partial results a row
// (0: none): the rounds of workgroups (two a CU up to dim 64), each of some six units' time
// for its start and end.  An estimate to choose by: a unit is given 0.6 us, what one takes
// where a round does not fill the chip and splits are chosen (0.9 on a full chip, where the
// clock is held down, which weighs on all choices alike); every unit counts as seen, and
// a workgroup as full.
double attention_rows_us(const AttnParams& p, int splits, int slots, int cu_count) {
  constexpr double kUnitUs = 0.6, kJoinUs = 4, kJoinBytesUs = 4e6;
  const int64_t rows = (int64_t)p.lq * p.group, blocks = (rows + kRows - 1) / kRows;
  const int64_t grid = (int64_t)p.batch * p.kv_heads * blocks * splits, at_once = (int64_t)cu_count * (p.dim <= 64 ? 2 : 1);
  const int64_t units = ((int64_t)p.prefix + kUnit - 1) / kUnit + (p.lk + kUnit - 1) / kUnit;
  const double row_bytes = 8.0 * p.dim * p.batch * p.lq * p.heads;  // written and read a partial result
  const int64_t rounds = (grid + at_once - 1) / at_once;
  return rounds * ((units + splits - 1) / splits + 6) * kUnitUs + (slots ? kJoinUs + row_bytes * slots / kJoinBytesUs : 0);
}

// The splits of the keys for which that is least, while each keeps four units.
int plan_attention_rows(const AttnParams& p, int cu_count) {
  const int64_t units = ((int64_t)p.prefix + kUnit - 1) / kUnit + (p.lk + kUnit - 1) / kUnit;
  int best = 1;
  double least = 1e30;
  for (int s = 1; s <= 32 && (s == 1 || units / s >= 4); ++s) {
    const double us = attention_rows_us(p, s, s > 1 ? s : 0, cu_count);
    if (us < least) least = us, best = s;
  }
  return best;
}

hipError_t launch_attention_rows(const AttnParams& params, int splits, int cu_count, int dt, hipStream_t stream) {
  AttnParams p = params;
  const bool joined = p.slots;  // by the caller, with the results of other launches
  p.splits = splits;
  if (!joined) {
    p.slots = splits > 1 ? splits : 0;
    p.part_lse = p.part_out + (int64_t)p.batch * p.lq * p.heads * splits * p.dim;
  }
  p.row_blocks = (int)(((int64_t)p.lq * p.group + kRows - 1) / kRows);
  const int nd = (p.dim + 31) / 32;
  const int64_t grid = (int64_t)p.batch * p.kv_heads * p.row_blocks * splits;
  const int a = attention_rows_blocks(p, splits, cu_count);
  const void* fn = p.prefix ? (dt == DT_F16 ? kernel_for<DT_F16, true>(nd, a) : kernel_for<DT_BF16, true>(nd, a))
                            : (dt == DT_F16 ? kernel_for<DT_F16, false>(nd, a) : kernel_for<DT_BF16, false>(nd, a));
  void* args[] = {&p};
  const hipError_t e = hipLaunchKernel(fn, dim3((unsigned)grid), dim3(waves(a) * 64), args, 0, stream);
  if (e != hipSuccess || splits == 1 || joined) return e;
  return launch_attention_join(p, dt, stream);
}

// ---- one token a sequence behind a shared prefix ------------------------------------
// Workgroups [0, common_blocks) take the batch's queries as one sequence's against the
// prefix, the others each sequence's own cache, in one launch: the first are bound by the
// matrix cores (from some 100 rows a key head on), the second by memory.  A prefix is read
// once for all sequences (MANY: over 64 rows a key head; fewer take the memory-bound tiles of
// decode_tile.h).  64 tokens behind 8192, own caches of up to 1024, 32 / 8 heads of 128, bf16:
// 53 us with the caches cold (44 warm), of which the join takes 5; the prefix and the caches
// in two launches one after another took 63 warm.  The prefix's 64 workgroups alone take 37 and
// the caches' alone 33 (a CU holds one workgroup of either), both together 46.
namespace {

template <int DT, int ND, bool MANY>
__global__ void __launch_bounds__(256, 1) prefix_token_kernel(const AttnParams common, const AttnParams own, int common_blocks) {
  constexpr int MOST = decode::DecodeLds<ND, 1>::TOTAL > RowsLds<ND, 2>::TOTAL ? decode::DecodeLds<ND, 1>::TOTAL : RowsLds<ND, 2>::TOTAL;
  __shared__ __attribute__((aligned(256))) uint8_t smem[MOST];
  if ((int)blockIdx.x >= common_blocks) decode::decode_tile<DT, ND, false, false, 1>(own, smem, (int)blockIdx.x - common_blocks);
  else if constexpr (MANY) attention_rows<DT, ND, false, 2>(common, smem, xcd_remap(blockIdx.x, (uint32_t)common_blocks));
  else decode::decode_tile<DT, ND, false, true, 1>(common, smem, (int)blockIdx.x);
}
template <int DT, bool MANY> const void* token_kernel_for(int nd) {
  switch (nd) {
    case 1: return (const void*)&prefix_token_kernel<DT, 1, MANY>;
    case 2: return (const void*)&prefix_token_kernel<DT, 2, MANY>;
    case 3: return (const void*)&prefix_token_kernel<DT, 3, MANY>;
  }
  return (const void*)&prefix_token_kernel<DT, 4, MANY>;
}

}  // namespace

// Splits of the prefix: a quarter of the CUs' worth of workgroups (the own caches have the
// others' time; half of them: 48 us for the above against 44, each split more to join), while
// each keeps 8 units.
PrefixTokenPlan plan_prefix_token(const AttnParams& common, const AttnParams& own, int cu_count) {
  PrefixTokenPlan plan{};
  const int64_t rows = (int64_t)common.lq * common.group;
  plan.many = rows > 2 * decode::kHeads;
  const int64_t grid = common.kv_heads * (plan.many ? (rows + kRows - 1) / kRows : (rows + decode::kHeads - 1) / decode::kHeads);
  const int64_t units = ((int64_t)common.lk + kUnit - 1) / kUnit;
  plan.common = common.lk ? 1 : 0;
  while (plan.common && plan.common < 64 && grid * plan.common * 2 <= cu_count / 4 && units / (2 * plan.common) >= 8) plan.common *= 2;
  plan.own = plan_decode_joined(own, 2, cu_count);
  return plan;
}

hipError_t launch_prefix_token(const AttnParams& common, const AttnParams& own, const PrefixTokenPlan& plan, int dt, hipStream_t stream) {
  AttnParams c = common, o = own;
  c.splits = plan.common;
  o.splits = plan.own;
  const int64_t rows = (int64_t)c.lq * c.group;
  c.row_blocks = (int)((rows + kRows - 1) / kRows);
  int common_blocks = (int)(c.kv_heads * (plan.many ? c.row_blocks : (rows + decode::kHeads - 1) / decode::kHeads) * plan.common);
  const int64_t grid = common_blocks + (int64_t)o.batch * o.kv_heads * ((o.group + decode::kHeads - 1) / decode::kHeads) * plan.own;
  const int nd = (c.dim + 31) / 32;
  const void* fn = plan.many ? (dt == DT_F16 ? token_kernel_for<DT_F16, true>(nd) : token_kernel_for<DT_BF16, true>(nd))
                             : (dt == DT_F16 ? token_kernel_for<DT_F16, false>(nd) : token_kernel_for<DT_BF16, false>(nd));
  void* args[] = {&c, &o, &common_blocks};
  const hipError_t e = hipLaunchKernel(fn, dim3((unsigned)grid), dim3(256), args, 0, stream);
  return e != hipSuccess ? e : launch_attention_join(o, dt, stream);
}

}  // namespace wtc
