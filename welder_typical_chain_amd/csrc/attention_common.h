// attention_common.h -- index maps and device helpers shared by the kernels of
// window_attention (forward, gradients) and its decode form.
#pragma once
#include "layer_common.h"

namespace wtc {
namespace attn {

// Compute width: dim rounded up to ND 32-column subtiles.  LDS rows hold 64 or
// 128 elements.
constexpr int row_bytes(int nd) { return nd <= 2 ? 128 : 256; }

// LDS layout of a tile of token rows ([row][16-byte chunk], chunks swizzled by
// the row), made for both kinds of read: 16 consecutive rows at one chunk
// (ds_read_b128, a row an MFMA row) and 4 consecutive rows at 4 chunks (the
// transposing ds_read_b64_tr_b16, a column an MFMA row) each fall in distinct
// 16-byte bank groups.
template <int RB> __device__ inline uint32_t row_swizzle(uint32_t row) {
  return RB == 256 ? ((row & 3) << 2) | ((row >> 2) & 3) : (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
}
template <int RB> __device__ inline uint32_t tile_offset(uint32_t row, uint32_t chunk) {
  return row * RB + ((chunk ^ row_swizzle<RB>(row)) << 4);
}

// A direct-to-LDS block (1 KiB) holds 1024 / RB rows; lane l of block b lands in
// row b * (1024 / RB) + l / (RB / 16), slot l % (RB / 16).
template <int RB> __device__ inline uint32_t block_row(int b, int lane) { return (uint32_t)(b * (1024 / RB) + lane / (RB / 16)); }
template <int RB> __device__ inline uint32_t block_chunk(int b, int lane) {
  return (uint32_t)(lane % (RB / 16)) ^ row_swizzle<RB>(block_row<RB>(b, lane));
}

// Loads of a tile of ROWS token rows by NW waves.  Rows past the descriptor's
// range and chunks past dim read as zeros.
template <int RB, int ROWS, int NW> struct TileLoader {
  static constexpr int BLOCKS = ROWS * RB / 1024;
  static constexpr int NB = BLOCKS / NW;
  static_assert(NB * NW == BLOCKS, "blocks over waves");
  const uint8_t* base;  // row 0 of the (sequence, head)
  uint32_t stride;      // bytes
  uint32_t dim_bytes;
  uint32_t off[NB];
  uint32_t lds;
  __device__ inline void init(const uint8_t* base_, int64_t stride_bytes, int dim, int wave, int lane) {
    base = base_;
    stride = (uint32_t)stride_bytes;
    dim_bytes = (uint32_t)dim * 2u;
    lds = (uint32_t)(wave * NB * 1024);
#pragma unroll
    for (int q = 0; q < NB; ++q) {
      const uint32_t c = block_chunk<RB>(wave * NB + q, lane) * 16u;
      off[q] = c < dim_bytes ? block_row<RB>(wave * NB + q, lane) * stride + c : kOutOfRange;
    }
  }
  // rows row0 .. row0 + rows - 1 (rows <= ROWS; none: zeros)
  __device__ inline void issue(uint32_t stage, int row0, int rows) const {
    const i32x4 r = raw_rsrc(base + (uint64_t)(uint32_t)max(rows > 0 ? row0 : 0, 0) * stride, rows > 0 ? (uint32_t)(rows - 1) * stride + dim_bytes : 0u);
#pragma unroll
    for (int q = 0; q < NB; ++q) dma16(r, off[q], stage + lds + q * 1024);
  }
};

// Where a lane reads its fragments in a tile.  The swizzle makes every other
// address of the tile an exclusive or of these with a constant (the tile starts
// 256-byte aligned, so that this holds for the address in LDS too), plus an
// offset that the instruction takes: one register for a tile instead of one a
// fragment.  fresh() keeps the compiler from holding the results over the loop,
// where they cost registers (and, in the dk/dv kernel, spills).
__device__ inline void fresh(uint32_t& x) { asm volatile("" : "+v"(x)); }
template <int RB> __device__ inline uint32_t row_addr(int lane) {
  const uint32_t row = (uint32_t)(lane & 31);
  return row * RB + (((uint32_t)(lane >> 5) ^ row_swizzle<RB>(row)) << 4);
}
template <int RB> __device__ inline uint32_t col_addr(int lane) {
  const uint32_t row = (uint32_t)(4 * (lane >> 5) + ((lane & 15) >> 2)), chunk = (uint32_t)(2 * ((lane >> 4) & 1) + ((lane & 3) >> 1));
  return row * RB + ((chunk ^ row_swizzle<RB>(row)) << 4) + (uint32_t)(lane & 1) * 8;
}
// 32 token rows as MFMA rows, k-step s (16 elements of dim): lane l reads row
// l % 32, chunk 2 s + l / 32.  `at`: row_addr + the tile; row0 a multiple of 32.
template <int RB> __device__ inline u32x4 row_frag(const uint8_t* lds, uint32_t at, int row0, int s) {
  return *reinterpret_cast<const u32x4*>(lds + (at ^ (uint32_t)(s << 5)) + row0 * RB);
}
// 32 columns (elements 32 d .. of dim) as MFMA rows, the 16 token rows from row0 (a
// multiple of 16) as its k.  A 32 x 32 accumulator holds, in registers 4 g .. 4 g + 3
// of lane half h, its rows 8 g + 4 h ..; packed to 16 bits, registers 8 s .. 8 s + 7
// are the other operand of k-step s with k in that order, so this reads token
// rows row0 + 4 h .. + 3, then row0 + 8 + 4 h .. + 3.  `at`: col_addr + the tile.
template <int RB> __device__ inline u32x4 col_frag(const uint8_t* lds, uint32_t at, int row0, int d) {
  const u32x2 lo = tr_read(lds + (at ^ (uint32_t)(d << 6)) + row0 * RB);
  const u32x2 hi = tr_read(lds + (at ^ (uint32_t)((d << 6) | 32)) + (row0 + 8) * RB);
  return u32x4{lo[0], lo[1], hi[0], hi[1]};
}

// A lane's fragments of one row in global memory (16-byte chunks 2 s + half).
template <int NS> __device__ inline void load_row(const uint8_t* row, bool valid, int dim, int half, u32x4 (&f)[NS]) {
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    const int c = 2 * s + half;
    f[s] = valid && c * 8 < dim ? *reinterpret_cast<const u32x4*>(row + c * 16) : u32x4{0, 0, 0, 0};
  }
}

// Has the loads of f arrive here.  The compiler waits for a load where its result is first
// used; in a loop it would do so in every turn, for all loads in flight, the
// direct-to-LDS ones (which it does not know of) too.
template <int NS> __device__ inline void landed(u32x4 (&f)[NS]) {
#pragma unroll
  for (int s = 0; s < NS; ++s) asm volatile("" : "+v"(f[s]));
}

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// Scores in the log2 domain are c2 times the products, c2 > 0: with a negative scale
// one operand's fragments are negated, with a scale of 0 they are zero.
template <int NS> __device__ inline float positive_scale(float scale, u32x4 (&f)[NS]) {
  const float c2 = scale * kLog2e;
  if (c2 > 0.0f) return c2;
#pragma unroll
  for (int s = 0; s < NS; ++s) f[s] = c2 < 0.0f ? f[s] ^ 0x80008000u : f[s] & 0u;
  return c2 < 0.0f ? -c2 : 1.0f;
}

// Masks as bits, a lane's own: bit c of bits_below(n) is set for c < n.  One bit
// then costs an element two vector instructions; compares would go through scalar
// masks, three to an element and each waiting for the last.
__device__ inline uint64_t bits_below(int64_t n) {
  return n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1;
}
__device__ inline float keep_bit(float x, uint64_t bits, int c) {  // x, or -inf where bit c is clear
  const uint32_t w = c < 32 ? (uint32_t)bits : (uint32_t)(bits >> 32);
  const uint32_t in = (uint32_t)__builtin_amdgcn_sbfe((int)w, c & 31, 1);
  return __builtin_bit_cast(float, (in & __builtin_bit_cast(uint32_t, x)) | (~in & 0xFF800000u));
}
// Of the 64 keys from j on, those below `end` that a query at `pos` sees.
__device__ inline uint64_t seen_bits(int64_t j, int64_t end, int64_t pos, int64_t window, int64_t sinks) {
  return bits_below(min(pos + 1, end) - j) & (~bits_below(pos - window + 1 - j) | bits_below(sinks - j));
}

// Keys that the query at position `pos` sees: the first `first` ones and then lo .. pos.
struct Seen {
  int lo, first, count;
  __device__ inline Seen(int64_t window, int sinks, int pos) {
    lo = (int)max((int64_t)0, (int64_t)pos - window + 1);
    first = min(sinks, lo);
    count = pos < 0 ? 0 : first + pos - lo + 1;
  }
  __device__ inline int key(int t) const { return t < first ? t : lo + t - first; }
};

template <int DT>
__device__ inline float dot_rows(const typename Elem<DT>::type* x, const typename Elem<DT>::type* y, int dim) {
  float s = 0.0f;
  for (int d = 0; d < dim; ++d) s = __builtin_fmaf((float)x[d], (float)y[d], s);
  return s;
}
__device__ inline float wave_max(float x) {
  for (int o = 32; o; o >>= 1) x = fmaxf(x, __shfl_xor(x, o));
  return x;
}
__device__ inline float wave_sum(float x) {
  for (int o = 32; o; o >>= 1) x += __shfl_xor(x, o);
  return x;
}

// Where the mask hides a NaN or an infinity.  The tiles' products meet it as 0 * NaN,
// so an output element that comes out as NaN is computed again by a whole wave
// from the keys (queries) that it sees, 64 at a time.  Only those elements are,
// and only until each of them is NaN again, which an element that sees the bad
// value is as soon as it is met: an input full of NaN costs one step a row.
constexpr int kCols = 2;  // columns a lane: lane, lane + 64
template <int DT> struct Redo {
  using T = typename Elem<DT>::type;
  T* row;
  bool bad[kCols];
  float acc[kCols];
  __device__ inline Redo(void* base, int64_t at, int dim, int lane) : row(static_cast<T*>(base) + at) {
#pragma unroll
    for (int c = 0; c < kCols; ++c) {
      const float x = lane + 64 * c < dim ? (float)row[lane + 64 * c] : 0.0f;
      bad[c] = x != x;
      acc[c] = 0.0f;
    }
  }
  __device__ inline void add(float w, const T* x, int lane) {
#pragma unroll
    for (int c = 0; c < kCols; ++c)
      if (bad[c]) acc[c] = __builtin_fmaf(w, (float)x[lane + 64 * c], acc[c]);
  }
  __device__ inline bool settled() const {  // every one of them is NaN for good
    return __all((!bad[0] || acc[0] != acc[0]) && (!bad[1] || acc[1] != acc[1]));
  }
  __device__ inline void store(float by, int lane) {
#pragma unroll
    for (int c = 0; c < kCols; ++c)
      if (bad[c]) row[lane + 64 * c] = (T)(acc[c] * by);
  }
};

// The last key that query i of sequence b sees.  FULL: every one.  (Known when compiled: code
// for other masks, though it is not run, took 0.6 us of every causal forward call at dim 128.)
template <bool FULL> __device__ inline int last_seen(const AttnParams& p, int b, int i) {
  const int nk = seq_keys(p, b);
  return FULL ? nk - 1 : i + nk - seq_queries(p, b);
}

// PREFIX: p.prefix keys before the own ones.
template <int DT, bool FULL, bool PREFIX> __device__ inline void attention_row(const AttnParams& p, int b, int h, int i) {
  using T = typename Elem<DT>::type;
  const int lane = threadIdx.x & 63;
  const T* q = (const T*)p.q + b * p.q_stride[0] + i * p.q_stride[1] + h * p.q_stride[2];
  const T* k = (const T*)p.k + b * p.k_stride[0] + h / p.group * p.k_stride[2];
  const T* v = (const T*)p.v + b * p.v_stride[0] + h / p.group * p.v_stride[2];
  const Seen seen(p.window, p.sinks, last_seen<FULL>(p, b, i));
  const int prefix = PREFIX ? p.prefix : 0, count = prefix + seen.count;
  auto key = [&](int t) {
    if (PREFIX && t < prefix) return (const T*)p.kp + h / p.group * p.kp_stride[1] + t * p.kp_stride[0];
    return k + seen.key(t - prefix) * p.k_stride[1];
  };
  auto value = [&](int t) {
    if (PREFIX && t < prefix) return (const T*)p.vp + h / p.group * p.vp_stride[1] + t * p.vp_stride[0];
    return v + seen.key(t - prefix) * p.v_stride[1];
  };
  Redo<DT> out(p.out, b * p.o_stride[0] + i * p.o_stride[1] + h * p.o_stride[2], p.dim, lane);
  float top = -INFINITY, total = 0.0f;
  for (int t0 = 0; t0 < count && !out.settled(); t0 += 64) {
    const bool in = t0 + lane < count;
    const float s = in ? p.scale * dot_rows<DT>(q, key(t0 + lane), p.dim) : -INFINITY;
    const float next = fmaxf(top, wave_max(s));
    const float keep = next == -INFINITY ? 1.0f : __expf(top - next);
    const float e = in ? (next == -INFINITY ? (s != s ? s : 0.0f) : __expf(s - next)) : 0.0f;
    total = total * keep + wave_sum(e);
    for (int c = 0; c < kCols; ++c) out.acc[c] *= keep;
    top = next;
    for (int t = 0; t < min(64, count - t0); ++t) out.add(__shfl(e, t), value(t0 + t), lane);
  }
  out.store(total == 0.0f ? 0.0f : 1.0f / total, lane);
}

// Joins the normalised results of a row's splits, [splits][dim] at `part` with their
// log2-sum-exps at `lse`, in their order: a lane takes elements c .. c + 3.  Returns
// the row's log2-sum-exp (-inf: no split has keys).  Four splits are read at a
// time, so that a row costs a few trips to memory and not one a split.
__device__ inline float join_splits(const float* part, const float* lse, int splits, int dim, int c, f32x4* out) {
  float m = -INFINITY;
  for (int s = 0; s < splits; ++s) m = fmaxf(m, lse[s]);
  const float ref = m == -INFINITY ? 0.0f : m;
  float total = 0.0f;
  f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int s0 = 0; s0 < splits; s0 += 4) {
    f32x4 x[4];
    float l[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int s = min(s0 + u, splits - 1);
      x[u] = *reinterpret_cast<const f32x4*>(part + (int64_t)s * dim + c);
      l[u] = s0 + u < splits ? lse[s] : -INFINITY;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      // No keys there: whatever it holds does not count.  Where there are keys a NaN
      // counts, also if their weight beside the others' is 0, as it does inside a tile.
      if (l[u] == -INFINITY) continue;
      const float w = __builtin_amdgcn_exp2f(l[u] - ref);
      total += w;
#pragma unroll
      for (int v = 0; v < 4; ++v) acc[v] = __builtin_fmaf(w, x[u][v], acc[v]);
    }
  }
  const float inv = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
  for (int v = 0; v < 4; ++v) (*out)[v] = acc[v] * inv;
  return total == 0.0f ? -INFINITY : m + __builtin_amdgcn_logf(total);
}

}  // namespace attn
}  // namespace wtc
