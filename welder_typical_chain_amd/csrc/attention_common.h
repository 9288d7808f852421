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
  int64_t stride;       // bytes
  uint32_t dim_bytes;
  uint32_t off[NB];
  uint32_t lds;
  __device__ inline void init(const uint8_t* base_, int64_t stride_bytes, int dim, int wave, int lane) {
    base = base_;
    stride = stride_bytes;
    dim_bytes = (uint32_t)dim * 2u;
    lds = (uint32_t)(wave * NB * 1024);
#pragma unroll
    for (int q = 0; q < NB; ++q) {
      const uint32_t c = block_chunk<RB>(wave * NB + q, lane) * 16u;
      off[q] = c < dim_bytes ? block_row<RB>(wave * NB + q, lane) * (uint32_t)stride + c : kOutOfRange;
    }
  }
  // rows row0 .. row0 + rows - 1 (rows <= ROWS; none: zeros)
  __device__ inline void issue(uint32_t stage, int row0, int rows) const {
    const i32x4 r = raw_rsrc(base + (rows > 0 ? (int64_t)row0 * stride : 0), rows > 0 ? (uint32_t)(rows - 1) * (uint32_t)stride + dim_bytes : 0u);
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

}  // namespace attn
}  // namespace wtc
