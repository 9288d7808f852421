// layer_launch.hip -- host side of include/wtc/wtc_layer.h: argument checks,
// workspace layouts and the launches.
#include <algorithm>
#include <cmath>
#include <exception>

#include "layer_common.h"
#include "layer_kernels.h"
#include "wtc/wtc_hip.h"

namespace {

using namespace wtc;

constexpr int64_t kMost = 1ll << 30;          // rows, tokens, heads, ...
constexpr int64_t kSpan = 0x7FFFFFFFll;       // bytes of an operand of a product
constexpr int64_t kTokenStride = 1ll << 23;   // elements: a tile's rows stay within 32-bit offsets
constexpr int64_t kMaxDim = 128;
constexpr int64_t kThreads = 1ll << 32;       // a launch takes fewer

int64_t align256(int64_t x) { return (x + 255) / 256 * 256; }
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
int bad(const std::string& msg) { return report(WTC_ERR_ARG, msg); }

// No C++ exception leaves a C entry point.
template <typename F> int guarded(F f) {
  try {
    return f();
  } catch (const std::exception& e) {
    return report(WTC_ERR_HIP, e.what());
  }
}
int launched(hipError_t e, const char* what) {
  return e == hipSuccess ? WTC_OK : report(WTC_ERR_HIP, std::string(what) + ": " + hipGetErrorString(e));
}
int check_workspace(const void* ws, size_t bytes, int64_t need) {
  if (need == 0) return WTC_OK;
  if (!ws || (int64_t)bytes < need)
    return report(WTC_ERR_WORKSPACE, "workspace of " + std::to_string(need) + " bytes needed");
  if (reinterpret_cast<uintptr_t>(ws) & 255) return bad("the workspace must be 256-byte aligned");
  return WTC_OK;
}

// ---- matrix products ---------------------------------------------------------
int check_matmul(const wtc_matmul_args& p, bool backward) {
  if (p.dtype != WTC_DTYPE_F16 && p.dtype != WTC_DTYPE_BF16) return bad("dtype must be f16 or bf16");
  if (p.out_dtype != p.dtype && p.out_dtype != WTC_DTYPE_F32) return bad("out_dtype must be the input type or f32");
  if (p.bias_dtype != p.dtype && p.bias_dtype != WTC_DTYPE_F32) return bad("bias_dtype must be the input type or f32");
  if (p.activation < WTC_ACT_NONE || p.activation > WTC_ACT_SILU) return bad("unknown activation");
  if (p.m < 0 || p.n < 0 || p.k < 0) return bad("negative extent");
  if (p.m > kMost || p.n > kMost || p.k > kMost) return report(WTC_ERR_UNSUPPORTED, "extent above 2^30");
  if (p.n % 8 || p.k % 8) return bad("n and k must be multiples of 8");
  // workgroups of the forward product and of the gradients (splits are for few of them)
  const int64_t mt = (p.m + 127) / 128, nt = (p.n + 127) / 128, kt = (p.k + 127) / 128;
  if (std::max({mt * nt, mt * kt, kt * nt}) >= kThreads / 256) return report(WTC_ERR_UNSUPPORTED, "too many tiles");
  const int64_t b_cols = p.b_trans ? p.k : p.n, b_rows = p.b_trans ? p.n : p.k;
  if (p.lda < p.k || p.ldb < b_cols || p.lda % 8 || p.ldb % 8)
    return bad("lda and ldb must be multiples of 8 that hold a row");
  if (p.lda > kMost || p.ldb > kMost || p.m * p.lda * 2 > kSpan || b_rows * p.ldb * 2 > kSpan)
    return report(WTC_ERR_UNSUPPORTED, "an operand spans more than 2 GiB");
  if (backward) {
    if (p.ldd < p.n || p.ldd % 8) return bad("ldd must be a multiple of 8 that holds a row");
    if (p.ldd > kMost || p.m * p.ldd * 2 > kSpan || p.m * p.n * 2 > kSpan)
      return report(WTC_ERR_UNSUPPORTED, "dout spans more than 2 GiB");
  } else if (p.ldo < p.n || p.ldr < p.n || p.ldo % 8 || p.ldr % 8 || p.ldo > kMost || p.ldr > kMost) {
    return bad("ldo and ldr must be multiples of 8 that hold a row");
  }
  return WTC_OK;
}

// Compute units of the current device (256 where none is visible).
int cu_count() {
  static thread_local int dev = -1, count = 256;
  int now = -1;
  if (hipGetDevice(&now) != hipSuccess) return 256;
  if (now != dev) {
    int n = 0;
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, now) != hipSuccess || n <= 0) n = 256;
    dev = now;
    count = n;
  }
  return count;
}

// Scratch of a backward call: dz (where an activation makes one), the columns'
// sums of row chunks, the partial products of da, then of db (one after the
// other in the same place).
struct MatmulBackwardPlan {
  int64_t chunk_rows, chunks;
  MatmulPlan da, db;
  bool pair;
  int64_t sums_at, partial_at, total;
};
MatmulBackwardPlan plan_backward(const wtc_matmul_args& p, int cus) {
  MatmulBackwardPlan q{};
  q.chunk_rows = act_backward_chunk_rows(p.m, p.n, cus);
  q.chunks = std::max<int64_t>(1, (p.m + q.chunk_rows - 1) / q.chunk_rows);
  q.da = plan_matmul(p.m, p.k, p.n, false, p.b_trans, cus);
  q.db = p.b_trans ? plan_matmul(p.n, p.k, p.m, true, true, cus) : plan_matmul(p.k, p.n, p.m, true, true, cus);
  q.pair = pair_pays(q.da, q.db, p.m, p.n, p.k, cus);
  if (q.pair) {  // da or db alone: the same tiles, so the same bits
    q.da = pair_plan(p.n);
    q.db = pair_plan(p.m);
  }
  q.sums_at = p.activation == WTC_ACT_NONE ? 0 : align256(p.m * p.n * 2);
  q.partial_at = q.sums_at + (q.chunks > 1 ? align256(q.chunks * p.n * 4) : 0);
  q.total = q.partial_at + align256(std::max(matmul_workspace(q.da, p.m, p.k), matmul_workspace(q.db, p.k, p.n)));
  return q;
}

// ---- attention ----------------------------------------------------------------
int check_strides(const int64_t* s, int count, int64_t tokens, const char* what) {
  for (int i = 0; i < count; ++i)
    if (s[i] < 0 || s[i] % 8) return bad(std::string(what) + ": strides must be multiples of 8");
  if (count == 3 && tokens > 1 && s[1] > kTokenStride)
    return report(WTC_ERR_UNSUPPORTED, std::string(what) + ": token stride above 2^23 elements");
  return WTC_OK;
}
// Rows of a tensor that is written may not overlap.
int check_distinct(const int64_t* s, int64_t n0, int64_t n1, int64_t n2, int64_t dim, const char* what) {
  std::pair<int64_t, int64_t> d[3] = {{s[0], n0}, {s[1], n1}, {s[2], n2}};
  std::sort(d, d + 3);
  int64_t span = dim;
  for (auto& x : d) {
    if (x.second <= 1) continue;
    if (x.first < span) return bad(std::string(what) + ": rows overlap");
    span += x.first * (x.second - 1);
  }
  return WTC_OK;
}

int too_many() { return report(WTC_ERR_UNSUPPORTED, "more sequences, heads and tokens than one launch takes"); }

int check_attention(const wtc_attention_args& p, bool decode) {
  if (p.dtype != WTC_DTYPE_F16 && p.dtype != WTC_DTYPE_BF16) return bad("dtype must be f16 or bf16");
  if (p.batch < 0 || p.lq < 0 || p.lk < 0 || p.window < 0 || p.sinks < 0) return bad("negative extent");
  if (p.heads <= 0 || p.kv_heads <= 0 || p.heads % p.kv_heads) return bad("heads must be a multiple of kv_heads");
  if (p.dim < 8 || p.dim > kMaxDim || p.dim % 8) return bad("dim must be a multiple of 8 up to 128");
  if (p.batch > kMost || p.lq > kMost || p.lk > kMost || p.heads > (1 << 16) ||
      p.batch * p.heads > kMost || p.batch * p.heads * p.lq > kMost || p.batch * p.kv_heads > kMost / std::max<int64_t>(p.lk, 1))
    return report(WTC_ERR_UNSUPPORTED, "extent above 2^30");
  // row blocks of 128 (splits are for few of them), query heads by 32 in decode
  const int64_t group = p.heads / p.kv_heads, seqs = p.batch * p.kv_heads;
  const int64_t groups = seqs * (decode ? (group + 31) / 32 : (p.lq * group + 127) / 128);
  if (groups >= kThreads / (decode ? 256 : 512)) return too_many();
  if (!std::isfinite((float)p.scale)) return bad("scale must be finite in float32");
  int rc;
  if ((rc = check_strides(p.q_stride, 3, p.lq, "q"))) return rc;
  if ((rc = check_strides(p.k_stride, 3, p.lk, "k"))) return rc;
  if ((rc = check_strides(p.v_stride, 3, p.lk, "v"))) return rc;
  if ((rc = check_strides(p.o_stride, 3, p.lq, "out"))) return rc;
  if (decode) {
    if (p.lq != 1) return bad("decode takes one token a sequence");
    if (p.lk <= p.sinks) return bad("the cache must have more rows than sinks");
    if (!p.k_lens && p.batch) return bad("decode needs k_lens");
    // (a tile's rows behind the last one would be parts of it, not zeros)
    for (const int64_t s : {p.k_stride[1], p.v_stride[1]})
      if (p.lk > 1 && s > 0 && s < p.dim) return bad("a cache's rows overlap");
    if ((rc = check_strides(p.kn_stride, 2, 0, "k_new"))) return rc;
    if ((rc = check_strides(p.vn_stride, 2, 0, "v_new"))) return rc;
  }
  return WTC_OK;
}

AttnParams attention_params(const wtc_attention_args& p) {
  AttnParams q{};
  for (int i = 0; i < 3; ++i) {
    q.q_stride[i] = p.q_stride[i];
    q.k_stride[i] = p.k_stride[i];
    q.v_stride[i] = p.v_stride[i];
    q.o_stride[i] = p.o_stride[i];
    q.do_stride[i] = p.do_stride[i];
  }
  // The stride of a single token counts for nothing.  A tile's rows behind a single key lie
  // outside what its loads may read, and give zeros, only if they are apart from it.
  if (p.lq <= 1) q.q_stride[1] = q.o_stride[1] = q.do_stride[1] = 0;
  if (p.lk <= 1) q.k_stride[1] = q.v_stride[1] = p.dim;
  for (int i = 0; i < 2; ++i) {
    q.kn_stride[i] = p.kn_stride[i];
    q.vn_stride[i] = p.vn_stride[i];
  }
  q.q_lens = p.q_lens;
  q.k_lens = p.k_lens;
  q.window = p.window == 0 ? INT32_MAX : std::min<int64_t>(p.window, INT32_MAX);
  q.batch = (int)p.batch;
  q.heads = (int)p.heads;
  q.kv_heads = (int)p.kv_heads;
  q.group = (int)(p.heads / p.kv_heads);
  q.lq = (int)p.lq;
  q.lk = (int)p.lk;
  q.dim = (int)p.dim;
  q.sinks = (int)std::min<int64_t>(p.sinks, p.lk);
  q.scale = (float)p.scale;
  return q;
}

// The cache keeps lk - sinks tokens behind the first ones: the window is at most that.
AttnParams decode_params(const wtc_attention_args& p) {
  AttnParams q = attention_params(p);
  q.window = std::min<int64_t>(q.window, p.lk - p.sinks);
  return q;
}

// The gradient addresses a tile's query rows (64 positions or one group of query
// heads) with 32-bit offsets.
int check_group_span(const wtc_attention_args& p, const int64_t* s, const char* what) {
  const int64_t heads = std::min<int64_t>(p.heads / p.kv_heads, 64), most = kSpan / 2;
  if (p.heads > 1 && s[2] > most / heads) return report(WTC_ERR_UNSUPPORTED, std::string(what) + ": a key head's query heads span more than 2 GiB");
  if (p.lq > 1 && (heads - 1) * s[2] + 64 / heads * s[1] + p.dim > most)
    return report(WTC_ERR_UNSUPPORTED, std::string(what) + ": a tile of query rows spans more than 2 GiB");
  return WTC_OK;
}
int check_attention_backward(const wtc_attention_args& p) {
  if (int rc = check_attention(p, false)) return rc;
  if (int rc = check_strides(p.do_stride, 3, p.lq, "dout")) return rc;
  if (int rc = check_group_span(p, p.q_stride, "q")) return rc;
  if (int rc = check_group_span(p, p.do_stride, "dout")) return rc;
  const AttnParams a = attention_params(p);
  const AttnBackwardPlan plan = plan_attention_backward(a, cu_count());
  const int64_t seqs = p.batch * p.kv_heads;
  const int64_t groups = seqs * ((int64_t)plan.key_blocks * plan.near_chunks + (int64_t)plan.far_blocks * plan.far_chunks);
  if (groups >= kThreads / 512 || (plan.far_blocks && seqs * a.sinks >= kThreads / 64)) return too_many();
  return WTC_OK;
}

}  // namespace

extern "C" {

int64_t wtc_matmul_epilogue_workspace_size(const wtc_matmul_args* p) {
  if (!p) return bad("NULL arguments"), -1;
  if (guarded([&] { return check_matmul(*p, false); })) return -1;
  return align256(matmul_workspace(plan_matmul(p->m, p->n, p->k, false, !p->b_trans, cu_count()), p->m, p->n));
}

int wtc_matmul_epilogue(const wtc_matmul_args* p, const void* a, const void* b, const void* bias,
                        const void* residual, void* out, float* pre, void* workspace, size_t workspace_bytes,
                        void* stream) {
  return guarded([&]() -> int {
    if (!p) return bad("NULL arguments");
    if (int rc = check_matmul(*p, false)) return rc;
    if (p->m == 0 || p->n == 0) return WTC_OK;
    if (!out || (p->k && (!a || !b))) return bad("NULL operand");
    if (!aligned16(a) || !aligned16(b) || !aligned16(out) || !aligned16(pre) || !aligned16(residual) || !aligned16(bias))
      return bad("pointers must be 16-byte aligned");
    const MatmulPlan plan = plan_matmul(p->m, p->n, p->k, false, !p->b_trans, cu_count());
    if (int rc = check_workspace(workspace, workspace_bytes, align256(matmul_workspace(plan, p->m, p->n)))) return rc;
    MatmulParams q{};
    q.a = static_cast<const uint8_t*>(a);
    q.b = static_cast<const uint8_t*>(b);
    q.bias = bias;
    q.residual = residual;
    q.out = out;
    q.pre = pre;
    q.partial = static_cast<float*>(workspace);
    q.lda = p->lda;
    q.ldb = p->ldb;
    q.ldr = p->ldr;
    q.ldo = p->ldo;
    q.ldp = p->n;
    q.m = (int)p->m;
    q.n = (int)p->n;
    q.k = (int)p->k;
    q.bias_f32 = p->bias_dtype == WTC_DTYPE_F32;
    q.act = (int)p->activation;
    return launched(launch_matmul(q, plan, (int)p->dtype, (int)p->out_dtype, false, !p->b_trans,
                                  static_cast<hipStream_t>(stream)),
                    "matmul_epilogue");
  });
}

int64_t wtc_matmul_epilogue_backward_workspace_size(const wtc_matmul_args* p) {
  if (!p) return bad("NULL arguments"), -1;
  if (guarded([&] { return check_matmul(*p, true); })) return -1;
  return plan_backward(*p, cu_count()).total;
}

int wtc_matmul_epilogue_backward(const wtc_matmul_args* p, const void* dout, const void* a, const void* b,
                                 const float* pre, void* da, void* db, float* dbias, void* workspace,
                                 size_t workspace_bytes, void* stream_) {
  return guarded([&]() -> int {
    if (!p) return bad("NULL arguments");
    if (int rc = check_matmul(*p, true)) return rc;
    const hipStream_t stream = static_cast<hipStream_t>(stream_);
    const bool act = p->activation != WTC_ACT_NONE;
    if ((p->m && p->n) && (!dout || (act && !pre) || (db && p->k && !a) || (da && p->k && !b)))
      return bad("NULL operand");
    if (!aligned16(dout) || !aligned16(a) || !aligned16(b) || !aligned16(pre) || !aligned16(da) || !aligned16(db) ||
        !aligned16(dbias))
      return bad("pointers must be 16-byte aligned");
    const MatmulBackwardPlan plan = plan_backward(*p, cu_count());
    if (int rc = check_workspace(workspace, workspace_bytes, plan.total)) return rc;
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    uint8_t* dz = act ? ws : static_cast<uint8_t*>(const_cast<void*>(dout));
    const int64_t ldz = act ? p->n : p->ldd;
    const int dt = (int)p->dtype;
    if (p->n && ((act && (da || db)) || dbias)) {
      ActBackwardParams q{};
      q.dout = dout;
      q.pre = pre;
      q.dz = act && (da || db) ? dz : nullptr;
      q.dbias = dbias;
      q.partial = reinterpret_cast<float*>(ws + plan.sums_at);
      q.m = p->m;
      q.n = p->n;
      q.ldd = p->ldd;
      q.chunk_rows = plan.chunk_rows;
      q.chunks = (int)plan.chunks;
      q.act = (int)p->activation;
      if (int rc = launched(launch_act_backward(q, dt, stream), "activation gradient")) return rc;
    }
    const bool want_da = da && p->m && p->k, want_db = db && p->n && p->k;
    MatmulParams x{}, y{};
    x.partial = y.partial = reinterpret_cast<float*>(ws + plan.partial_at);
    // dz [m][n] . B^T: B stored by rows is contiguous along n
    x.a = dz;
    x.b = static_cast<const uint8_t*>(b);
    x.lda = ldz;
    x.ldb = p->ldb;
    x.out = da;
    x.ldo = p->k;
    x.m = (int)p->m;
    x.n = (int)p->k;
    x.k = (int)p->n;
    // A^T . dz, or its transpose dz^T . A: both strided along m
    const uint8_t* rows = static_cast<const uint8_t*>(a);
    y.a = p->b_trans ? dz : rows;
    y.b = p->b_trans ? rows : dz;
    y.lda = p->b_trans ? ldz : p->lda;
    y.ldb = p->b_trans ? p->lda : ldz;
    y.out = db;
    y.m = (int)(p->b_trans ? p->n : p->k);
    y.n = (int)(p->b_trans ? p->k : p->n);
    y.ldo = y.n;
    y.k = (int)p->m;
    if (want_da && want_db && plan.pair) return launched(launch_matmul_pair(x, y, dt, p->b_trans, stream), "da and db");
    if (want_da)
      if (int rc = launched(launch_matmul(x, plan.da, dt, dt, false, p->b_trans, stream), "da")) return rc;
    if (want_db)
      if (int rc = launched(launch_matmul(y, plan.db, dt, dt, true, true, stream), "db")) return rc;
    return WTC_OK;
  });
}

int wtc_matmul_epilogue_plan(const wtc_matmul_args* p, int part, int cus, int64_t* tile_m, int64_t* tile_n,
                             int64_t* splits) {
  return guarded([&]() -> int {
    if (!p || !tile_m || !tile_n || !splits) return bad("NULL argument");
    if (part < 0 || part > 2) return bad("part must be 0 (forward), 1 (da) or 2 (db)");
    if (int rc = check_matmul(*p, part > 0)) return rc;
    if (cus <= 0) cus = cu_count();
    MatmulPlan plan;
    if (part == 0) {
      plan = plan_matmul(p->m, p->n, p->k, false, !p->b_trans, cus);
    } else {
      const MatmulBackwardPlan both = plan_backward(*p, cus);
      plan = part == 1 ? both.da : both.db;
    }
    matmul_tile_size(plan, tile_m, tile_n);
    *splits = plan.splits;
    return WTC_OK;
  });
}

int64_t wtc_window_attention_workspace_size(const wtc_attention_args* p) {
  if (!p) return bad("NULL arguments"), -1;
  if (guarded([&] { return check_attention(*p, false); })) return -1;
  const AttnParams a = attention_params(*p);
  return align256(attention_workspace(a, plan_attention(a, cu_count())));
}

int wtc_window_attention(const wtc_attention_args* p, const void* q, const void* k, const void* v, void* out,
                         float* lse, void* workspace, size_t workspace_bytes, void* stream) {
  return guarded([&]() -> int {
    if (!p) return bad("NULL arguments");
    if (int rc = check_attention(*p, false)) return rc;
    if (int rc = check_distinct(p->o_stride, p->batch, p->lq, p->heads, p->dim, "out")) return rc;
    if (p->batch == 0 || p->lq == 0) return WTC_OK;
    if (!q || !out || (p->lk && (!k || !v))) return bad("NULL operand");
    if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out)) return bad("pointers must be 16-byte aligned");
    AttnParams a = attention_params(*p);
    a.q = static_cast<const uint8_t*>(q);
    a.k = static_cast<const uint8_t*>(k);
    a.v = static_cast<const uint8_t*>(v);
    a.out = static_cast<uint8_t*>(out);
    a.lse = lse;
    const AttnPlan plan = plan_attention(a, cu_count());
    if (int rc = check_workspace(workspace, workspace_bytes, align256(attention_workspace(a, plan)))) return rc;
    a.part_out = static_cast<float*>(workspace);
    return launched(launch_attention(a, plan, (int)p->dtype, static_cast<hipStream_t>(stream)), "window_attention");
  });
}

int64_t wtc_window_attention_backward_workspace_size(const wtc_attention_args* p) {
  if (!p) return bad("NULL arguments"), -1;
  if (guarded([&] { return check_attention_backward(*p); })) return -1;
  return plan_attention_backward(attention_params(*p), cu_count()).workspace;
}

int wtc_window_attention_backward(const wtc_attention_args* p, const void* dout, const void* q, const void* k,
                                  const void* v, const void* out, const float* lse, void* dq, void* dk, void* dv,
                                  void* workspace, size_t workspace_bytes, void* stream) {
  return guarded([&]() -> int {
    if (!p) return bad("NULL arguments");
    if (int rc = check_attention_backward(*p)) return rc;
    if (p->batch == 0) return WTC_OK;
    if ((p->lq && (!dout || !q || !out || !lse || !dq)) || (p->lk && (!k || !v || !dk || !dv)))
      return bad("NULL operand");
    if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out) || !aligned16(dout) || !aligned16(dq) ||
        !aligned16(dk) || !aligned16(dv))
      return bad("pointers must be 16-byte aligned");
    AttnParams a = attention_params(*p);
    const AttnBackwardPlan plan = plan_attention_backward(a, cu_count());
    if (int rc = check_workspace(workspace, workspace_bytes, plan.workspace)) return rc;
    a.q = static_cast<const uint8_t*>(q);
    a.k = static_cast<const uint8_t*>(k);
    a.v = static_cast<const uint8_t*>(v);
    a.o = static_cast<const uint8_t*>(out);
    a.dout = static_cast<const uint8_t*>(dout);
    a.lse_in = lse;
    a.row_lse = static_cast<float*>(workspace);
    a.dq = static_cast<uint8_t*>(dq);
    a.dk = static_cast<uint8_t*>(dk);
    a.dv = static_cast<uint8_t*>(dv);
    return launched(launch_attention_backward(a, plan, (int)p->dtype, static_cast<hipStream_t>(stream)),
                    "window_attention_backward");
  });
}

int wtc_window_attention_plan(const wtc_attention_args* p, int cus, int64_t* plan) {
  return guarded([&]() -> int {
    if (!p || !plan) return bad("NULL argument");
    if (int rc = check_attention_backward(*p)) return rc;
    if (cus <= 0) cus = cu_count();
    const AttnParams a = attention_params(*p);
    const AttnPlan forward = plan_attention(a, cus);
    const AttnBackwardPlan backward = plan_attention_backward(a, cus);
    plan[0] = forward.key_groups;
    plan[1] = forward.splits;
    plan[2] = backward.dq_groups;
    plan[3] = backward.near_chunks;
    plan[4] = (int64_t)backward.far_blocks * backward.far_chunks;
    return WTC_OK;
  });
}

int64_t wtc_window_attention_decode_workspace_size(const wtc_attention_args* p) {
  if (!p) return bad("NULL arguments"), -1;
  if (guarded([&] { return check_attention(*p, true); })) return -1;
  const AttnParams a = decode_params(*p);
  return align256(decode_workspace(a, plan_decode(a, cu_count())));
}

int wtc_window_attention_decode(const wtc_attention_args* p, const void* q, void* k, void* v, const void* k_new,
                                const void* v_new, void* out, void* workspace, size_t workspace_bytes,
                                void* stream) {
  return guarded([&]() -> int {
    if (!p) return bad("NULL arguments");
    if (int rc = check_attention(*p, true)) return rc;
    if (int rc = check_distinct(p->o_stride, p->batch, 1, p->heads, p->dim, "out")) return rc;
    if (!k_new != !v_new) return bad("k_new and v_new go together");
    if (k_new) {
      if (k && k == v) return bad("k and v are the same cache: it cannot take both k_new and v_new");
      if (int rc = check_distinct(p->k_stride, p->batch, p->lk, p->kv_heads, p->dim, "k")) return rc;
      if (int rc = check_distinct(p->v_stride, p->batch, p->lk, p->kv_heads, p->dim, "v")) return rc;
    }
    if (p->batch == 0) return WTC_OK;
    if (!q || !k || !v || !out) return bad("NULL operand");
    if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out) || !aligned16(k_new) || !aligned16(v_new))
      return bad("pointers must be 16-byte aligned");
    AttnParams a = decode_params(*p);
    const int splits = plan_decode(a, cu_count());
    if (int rc = check_workspace(workspace, workspace_bytes, align256(decode_workspace(a, splits)))) return rc;
    a.part_out = static_cast<float*>(workspace);
    a.q = static_cast<const uint8_t*>(q);
    a.k = static_cast<const uint8_t*>(k);
    a.v = static_cast<const uint8_t*>(v);
    a.k_new = static_cast<const uint8_t*>(k_new);
    a.v_new = static_cast<const uint8_t*>(v_new);
    a.out = static_cast<uint8_t*>(out);
    return launched(launch_attention_decode(a, splits, (int)p->dtype, static_cast<hipStream_t>(stream)),
                    "window_attention_decode");
  });
}

}  // extern "C"
