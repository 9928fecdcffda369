// Block quantisation to e4m3 (gfx950): scale = amax / 448 and q = e4m3(x * (448 / amax)) for each 1 x 128
// run of a row or each 128 x 128 block, amax = max(max|x|, 2^-96).
//
// One pass: a lane takes 8 consecutive elements, 16 lanes one row's 128 columns, everything stays in
// registers between the maximum and the conversion.  Bound by HBM: 2 or 4 bytes read and 1 written per
// element.  The maximum is taken over bit patterns, where a NaN is the largest: a block that holds a NaN
// or an infinity comes back as NaN instead of losing it.  16384 rows of 7168 in bf16: 57 us, 6.2 TB/s read and written;
// 32 weights of [4096, 7168] in 128 x 128 blocks: 451 us, 6.3 TB/s.
#pragma once

#include "fp8_gemm.h"

namespace moegemm {

struct QuantizeParams {
  const void* x;
  uint8_t* q;
  float* scale;
  int64_t sxb, sxr, sqb, sqr, ssb, ssr, ssk;  // batch and row strides in elements; scale strides
  int32_t rows, k;
  int32_t col_tiles;  // column tiles of a launch (blocks / kQuantBlocks, or blocks)
};

constexpr int kQuantRows = 16;   // rows and blocks of columns of a workgroup in the 1 x 128 kernel
constexpr int kQuantBlocks = 4;

// fp32 rows in vectors: a lane's 8 elements are two runs of 4, half a block apart, so that each load of 16 lanes covers
// 256 bytes in a row; with 8 elements in a row it covers every other 16 bytes of 512 (8 x [5760, 2880]: 127 us, not 108).
__device__ __forceinline__ int first_run(int col) { return (col & ~(kScaleBlock - 1)) + ((col & (kScaleBlock - 1)) >> 1); }

// Elements [col, col + 8) of a row (fp32 in vectors: first_run(col) and 64 further on, 4 each), zeros past k.  VEC: the row
// is 16-byte aligned and k a multiple of 8.
template <class E, bool VEC>
__device__ __forceinline__ void load8(const typename E::raw* row, int col, int k, float (&v)[8]) {
  using raw = typename E::raw;
  raw r[8];
  if constexpr (VEC) {
    constexpr int N = sizeof(raw) * 8 / 16;
    u32x4_t c[N] = {};
    if constexpr (N == 1) {
      if (col < k) c[0] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(row + col));
    } else {
      const int first = first_run(col);
      if (first < k) c[0] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(row + first));
      if (first + 64 < k) c[1] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(row + first + 64));
    }
    __builtin_memcpy(r, c, sizeof(r));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = col + i < k ? row[col + i] : (raw)0;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if constexpr (E::dtype == DT_F32) v[i] = __builtin_bit_cast(float, r[i]);
    else if constexpr (E::dtype == DT_BF16) v[i] = __builtin_bit_cast(float, (uint32_t)r[i] << 16);
    else v[i] = (float)__builtin_bit_cast(_Float16, r[i]);
  }
}

// The 8 values of load8 scaled and converted; vector stores where the row allows.
template <class E, bool VEC>
__device__ __forceinline__ void store8(uint8_t* row, int col, int k, const float (&v)[8], float inverse) {
  f32x4_t lo, hi;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    lo[i] = v[i] * inverse;
    hi[i] = v[i + 4] * inverse;
  }
  const int32_t a = pack_e4m3(lo), b = pack_e4m3(hi);
  if constexpr (VEC && E::is_f32) {
    const int first = first_run(col);
    if (first < k) *reinterpret_cast<int32_t*>(row + first) = a;
    if (first + 64 < k) *reinterpret_cast<int32_t*>(row + first + 64) = b;
  } else if (col >= k) {
    return;
  } else if (VEC || col + 8 <= k) {
    *reinterpret_cast<u32x2_t*>(row + col) = u32x2_t{(uint32_t)a, (uint32_t)b};
  } else {
    for (int i = 0; i < k - col; ++i) row[col + i] = (uint8_t)((i < 4 ? a >> (8 * i) : b >> (8 * (i - 4))) & 0xff);
  }
}

__device__ __forceinline__ uint32_t top8(const float (&v)[8]) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, abs_bits(v[i]));
  return top;
}

template <class E, bool VEC>
__global__ void __launch_bounds__(256) quantize_rows_kernel(QuantizeParams p) {
  __shared__ float s_scale[kQuantBlocks][kQuantRows];
  const int tile_r = (int)(blockIdx.x / (unsigned)p.col_tiles), tile_c = (int)(blockIdx.x % (unsigned)p.col_tiles);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int blk = lane >> 4;  // a wave reads one row's 512 columns at a time
  const int col = tile_c * kQuantBlocks * kScaleBlock + lane * 8;
  const int batch = blockIdx.y;
  const typename E::raw* x = static_cast<const typename E::raw*>(p.x) + (int64_t)batch * p.sxb;
  uint8_t* q = p.q + (int64_t)batch * p.sqb;
  constexpr int PER = kQuantRows / 4;
  float v[PER][8];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int row = tile_r * kQuantRows + wave * PER + i;
    load8<E, VEC>(x + (int64_t)min(row, p.rows - 1) * p.sxr, col, p.k, v[i]);
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int row = tile_r * kQuantRows + wave * PER + i;
    uint32_t top = top8(v[i]);
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, d));
    const float amax = floored(top);
    if ((lane & 15) == 0) s_scale[blk][wave * PER + i] = amax / kE4m3Max;
    if (row < p.rows) store8<E, VEC>(q + (int64_t)row * p.sqr, col, p.k, v[i], kE4m3Max / amax);
  }
  __syncthreads();
  // Scales leave block by block, 16 consecutive rows each.
  const int sb = threadIdx.x / kQuantRows, sr = threadIdx.x % kQuantRows;
  const int block = tile_c * kQuantBlocks + sb, row = tile_r * kQuantRows + sr;
  if (sb < kQuantBlocks && block * kScaleBlock < p.k && row < p.rows)
    p.scale[(int64_t)batch * p.ssb + (int64_t)row * p.ssr + (int64_t)block * p.ssk] = s_scale[sb][sr];
}

template <class E, bool VEC>
__global__ void __launch_bounds__(256) quantize_blocks_kernel(QuantizeParams p) {
  __shared__ uint32_t s_top[4];
  const int tile_r = (int)(blockIdx.x / (unsigned)p.col_tiles), tile_c = (int)(blockIdx.x % (unsigned)p.col_tiles);
  const int col = tile_c * kScaleBlock + (threadIdx.x & 15) * 8;
  const int batch = blockIdx.y;
  const typename E::raw* x = static_cast<const typename E::raw*>(p.x) + (int64_t)batch * p.sxb;
  uint8_t* q = p.q + (int64_t)batch * p.sqb;
  constexpr int PER = kScaleBlock / 16;
  float v[PER][8];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int row = tile_r * kScaleBlock + i * 16 + (threadIdx.x >> 4);
    // Rows past the end repeat the last one: it is in the block already.
    load8<E, VEC>(x + (int64_t)min(row, p.rows - 1) * p.sxr, col, p.k, v[i]);
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) top = max(top, top8(v[i]));
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, d));
  if ((threadIdx.x & 63) == 0) s_top[threadIdx.x >> 6] = top;
  __syncthreads();
  const float amax = floored(max(max(s_top[0], s_top[1]), max(s_top[2], s_top[3])));
  const float inverse = kE4m3Max / amax;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int row = tile_r * kScaleBlock + i * 16 + (threadIdx.x >> 4);
    if (row < p.rows) store8<E, VEC>(q + (int64_t)row * p.sqr, col, p.k, v[i], inverse);
  }
  if (threadIdx.x == 0)
    p.scale[(int64_t)batch * p.ssb + (int64_t)tile_r * p.ssr + (int64_t)tile_c * p.ssk] = amax / kE4m3Max;
}

}  // namespace moegemm
