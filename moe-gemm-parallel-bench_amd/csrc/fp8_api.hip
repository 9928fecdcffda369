// C ABI of the block-scaled fp8 operators: argument checks, the choice of a variant, the launches: one a call, and
// another for every further 2^24 workgroups (quantisation), 768 groups or 192 rounds of tiles (products on tiles).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstring>

#include "../../include/moegemm.h"
#include "error.h"
#include "fp8_menu.h"
#include "quantize_fp8.h"

using namespace moegemm;

namespace {

constexpr int64_t kPitchLimit = int64_t(1) << 23;  // 256 rows of a panel under 2 GiB

// Workgroups of 256 threads that one launch takes: it counts threads in 32 bits and drops what is past them without
// an error (2^28 + 37 rows of 16 columns wrote nothing in one launch).
constexpr int64_t kLaunchTiles = (int64_t(1) << 24) - 1;

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
bool aligned(const void* p, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

template <class E>
hipError_t launch_quantize(const QuantizeParams& p, int block_rows, bool vec, dim3 grid, hipStream_t stream) {
  if (block_rows == 1) {
    if (vec) hipLaunchKernelGGL((quantize_rows_kernel<E, true>), grid, dim3(256), 0, stream, p);
    else hipLaunchKernelGGL((quantize_rows_kernel<E, false>), grid, dim3(256), 0, stream, p);
  } else {
    if (vec) hipLaunchKernelGGL((quantize_blocks_kernel<E, true>), grid, dim3(256), 0, stream, p);
    else hipLaunchKernelGGL((quantize_blocks_kernel<E, false>), grid, dim3(256), 0, stream, p);
  }
  return hipGetLastError();
}

// What both fp8 products check; `out_cols` columns of output.
int check_operands(const void* a, const float* scale_a, const void* w, const float* scale_w, const void* out,
                   const int32_t* offs, int32_t group_count, int32_t rows, int32_t n, int32_t k, int64_t stride_am,
                   int64_t stride_wg, int64_t stride_wn, int64_t stride_om, int64_t out_cols) {
  if (group_count <= 0) return report(MOEGEMM_ERR_INVALID, "group_count must be positive (got %d)", group_count);
  if (!offs && group_count != 1)
    return report(MOEGEMM_ERR_INVALID, "without offsets there is one group (got %d)", group_count);
  if (rows < 0 || n <= 0 || k <= 0)
    return report(MOEGEMM_ERR_INVALID, "bad shape (rows=%d n=%d k=%d)", rows, n, k);
  if (!a || !scale_a || !w || !scale_w || !out)
    return report(MOEGEMM_ERR_INVALID, "operands, scales and output must be non-null");
  if (!aligned(a, 16) || !aligned(w, 16) || stride_am % 16 || stride_wn % 16 || stride_wg % 16)
    return report(MOEGEMM_ERR_INVALID, "fp8 rows must start at multiples of 16 bytes");
  if (stride_am < k || stride_wn < k || stride_om < out_cols)
    return report(MOEGEMM_ERR_INVALID, "row pitches must cover a row");
  if (stride_am >= kPitchLimit || stride_wn >= kPitchLimit)
    return report(MOEGEMM_ERR_INVALID, "fp8 row pitches must be under %lld bytes", (long long)kPitchLimit);
  return MOEGEMM_OK;
}

// The row scales of a tile are addressed by 32-bit byte offsets from its first row, the weight's from its group.
int check_scales(int64_t stride_sam, int64_t stride_ssn, int32_t n) {
  if (stride_sam < 0 || stride_ssn < 0 || stride_sam * 256 * 4 >= (int64_t(1) << 31) ||
      stride_ssn * cdiv(n, kScaleBlock) * 4 >= (int64_t(1) << 31))
    return report(MOEGEMM_ERR_INVALID, "scale strides must be non-negative and address 2 GiB at most");
  return MOEGEMM_OK;
}

// Variant for `rows` rows over `groups` groups.
//
// Up to about 32 rows a group (20 with fast sums, whose tiles are faster) a call is bound by reading the weights, and
// the stream kernels read them once where a group's rows fit their 16 or 32; routed groups are taken to hold up to
// 1.6 times the mean (a group of more rows than a unit holds has its row tiles run one after another and reads its
// weights again for each: 256 rows over 32 experts of [4096, 7168] 140 us even, 485 with half of them on one expert,
// 791 with all).  32 experts of [4096, 7168], us: 8 rows each stream 142, tile 194; 32 rows stream 155, exact
// tile 196; 64 rows stream 314, exact tile 209, fast tile 198.
// Among stream kernels: units run in rounds of one per CU, at a cost of their weights and about 200 rows of one
// block for the join and the stores.  [7168, 2048] x 32: 256 columns 86, 128 columns 80 (7 whole rounds), 64
// columns 102; one group of [4096, 7168]: 256 columns 55, 16 columns 12.8.
// Among tiles: rounds by the time of a slice, in units of 10 ns (1000 rows of [4096, 4096]: 256x256 50 us, 128x256 35,
// 128x128 31; 16384 rows of 32 x [4096, 7168]: 515, 621, 840; exact 128x256 57 and 868, 128x128 47 and 1069).
int choose(const Fp8Variant* table, int count, int64_t rows, int64_t groups, int64_t cols, int64_t k, int fast,
           int cus) {
  const int64_t active = std::min(groups, rows), mean = cdiv(rows, active);
  const int64_t high = active == 1 ? rows : cdiv(mean * 8, 5);
  const bool stream = active == 1 ? rows <= 32 : mean <= (fast ? 20 : 32);
  const int64_t blocks = cdiv(k, kScaleBlock);
  int best = -1;
  int64_t least = 0;
  for (int i = 0; i < count; ++i) {
    const Fp8Variant& v = table[i];
    if ((v.stream != 0) != stream || (!stream && v.fast != fast)) continue;
    const int64_t n_tiles = cdiv(cols, v.block_n);
    int64_t cost;
    if (stream) {
      if (v.block_m != (high <= 16 ? 16 : 32)) continue;
      const int64_t padded = cdiv(blocks, v.waves_k) * v.waves_k;
      cost = cdiv(active * n_tiles, cus) * (v.block_n * padded + 200);
    } else {
      const int64_t row_tiles = rows / v.block_m + active / 2 + (active == 1 && rows % v.block_m != 0);
      const int64_t tiles = std::max(active, row_tiles) * n_tiles;
      const int slice = v.block_m == 256 ? 170 : v.block_n == 256 ? (v.fast ? 115 : 190) : (v.fast ? 90 : 115);
      cost = cdiv(tiles, cus) * slice;
    }
    if (best < 0 || cost < least) {
      best = i;
      least = cost;
    }
  }
  return best;
}

int launch_product(const Fp8Variant* table, int count, Fp8Params& p, int64_t out_cols, int gated, int fast,
                   int32_t variant, int32_t grid_size, void* stream) {
  if (fast != 0 && fast != 1) return report(MOEGEMM_ERR_INVALID, "fast_accum must be 0 or 1 (got %d)", fast);
  if (variant < -1 || variant >= count)
    return report(MOEGEMM_ERR_NO_KERNEL, "fp8 variant %d is not compiled (0 to %d, or -1)", variant, count - 1);
  if (p.rows == 0) return MOEGEMM_OK;
  const int cus = grid_size > 0 ? grid_size : 256;
  const int64_t cols = gated ? cdiv(out_cols, 128) * 256 : p.n;
  if (variant < 0) variant = choose(table, count, p.rows, p.groups, cols, p.k, fast, cus);
  if (variant < 0) return report(MOEGEMM_ERR_NO_KERNEL, "no fp8 variant for this shape");
  const Fp8Variant& v = table[variant];
  const int64_t n_tiles = cdiv(p.n, v.block_n);  // gated: n = 2F weight rows in tiles of 128 + 128
  const int64_t col_tiles = gated ? cdiv(out_cols, v.block_n / 2) : n_tiles;
  p.n_tiles = (int32_t)col_tiles;
  const int64_t bound = (v.stream ? (int64_t)p.groups  // units, or tiles at most
                                  : std::min(p.rows / v.block_m + (int64_t)p.groups, p.groups * cdiv(p.rows, v.block_m))) *
                        col_tiles;
  if (bound > INT32_MAX / 2) return report(MOEGEMM_ERR_INVALID, "tile count exceeds int32");
  const int64_t grid = std::min<int64_t>(bound, cus);
  const int32_t groups = p.groups, most = v.stream ? groups : kTableGroups;
  for (; p.first < groups; p.first += most) {
    p.groups = std::min(groups - p.first, most);
    for (p.round = 0; p.round * grid < bound; p.round += kListTiles) {
      const hipError_t err = v.launch(p, (int)grid, reinterpret_cast<hipStream_t>(stream));
      if (err != hipSuccess) return report(MOEGEMM_ERR_LAUNCH, "kernel launch failed: %s", hipGetErrorString(err));
      if (v.stream) break;  // goes on to its last unit
    }
  }
  return MOEGEMM_OK;
}

}  // namespace

extern "C" {

int moegemm_quantize_fp8(const void* x, void* q, float* scale, int32_t batch, int32_t rows, int32_t k,
                         int64_t stride_xb, int64_t stride_xr, int64_t stride_qb, int64_t stride_qr, int64_t stride_sb,
                         int64_t stride_sr, int64_t stride_sk, int32_t dtype, int32_t block_rows, void* stream) {
  if (dtype != DT_F16 && dtype != DT_BF16 && dtype != DT_F32)
    return report(MOEGEMM_ERR_INVALID, "unsupported dtype code %d", dtype);
  if (block_rows != 1 && block_rows != kScaleBlock)
    return report(MOEGEMM_ERR_INVALID, "block_rows must be 1 or 128 (got %d)", block_rows);
  if (batch < 0 || rows < 0 || k <= 0)
    return report(MOEGEMM_ERR_INVALID, "bad shape (batch=%d rows=%d k=%d)", batch, rows, k);
  if (batch == 0 || rows == 0) return MOEGEMM_OK;
  if (!x || !q || !scale) return report(MOEGEMM_ERR_INVALID, "x, q and scale must be non-null");
  if (!aligned(q, 8) || stride_qr % 8 || stride_qb % 8 || stride_qr < k)
    return report(MOEGEMM_ERR_INVALID, "q rows must cover k and start at multiples of 8 bytes");
  if (batch > 65535) return report(MOEGEMM_ERR_INVALID, "batch must be at most 65535 (got %d)", batch);
  const int64_t es = dtype == DT_F32 ? 4 : 2;
  if (!aligned(x, es)) return report(MOEGEMM_ERR_INVALID, "x must be aligned to its element size");
  QuantizeParams p{x, static_cast<uint8_t*>(q), scale, stride_xb, stride_xr, stride_qb, stride_qr,
                   stride_sb, stride_sr, stride_sk, rows, k, 0};
  const int64_t blocks = cdiv(k, kScaleBlock);
  const int64_t col_tiles = block_rows == 1 ? cdiv(blocks, kQuantBlocks) : blocks;
  if (col_tiles > kLaunchTiles) return report(MOEGEMM_ERR_INVALID, "k must be at most 2^31 - 128 (got %d)", k);
  p.col_tiles = (int32_t)col_tiles;
  const bool vec = k % 8 == 0 && aligned(x, 16) && stride_xr * es % 16 == 0 && stride_xb * es % 16 == 0;
  const auto s = reinterpret_cast<hipStream_t>(stream);
  const int64_t tile_rows = block_rows == 1 ? kQuantRows : kScaleBlock;
  const int64_t step = kLaunchTiles / col_tiles * tile_rows;  // rows of a launch
  for (int64_t row = 0; row < rows; row += step) {
    p.x = static_cast<const char*>(x) + row * stride_xr * es;
    p.q = static_cast<uint8_t*>(q) + row * stride_qr;
    p.scale = scale + row / block_rows * stride_sr;
    p.rows = (int32_t)std::min(rows - row, step);
    const dim3 grid((unsigned)(cdiv(p.rows, tile_rows) * col_tiles), (unsigned)batch);
    const hipError_t err = dtype == DT_F32    ? launch_quantize<EF32>(p, block_rows, vec, grid, s)
                           : dtype == DT_BF16 ? launch_quantize<EBf16>(p, block_rows, vec, grid, s)
                                              : launch_quantize<EF16>(p, block_rows, vec, grid, s);
    if (err != hipSuccess) return report(MOEGEMM_ERR_LAUNCH, "kernel launch failed: %s", hipGetErrorString(err));
  }
  return MOEGEMM_OK;
}

int moegemm_fp8_variant_count(int32_t gated) { return gated ? kNumFp8Gated : kNumFp8; }

int moegemm_fp8_variant_fast(int32_t gated, int32_t variant) {
  if (variant < 0 || variant >= moegemm_fp8_variant_count(gated))
    return report(MOEGEMM_ERR_INVALID, "fp8 variant %d is not compiled", variant);
  return (gated ? kFp8Gated : kFp8Bf16)[variant].fast;
}

int moegemm_grouped_mm_fp8(const void* a, const float* scale_a, const void* w, const float* scale_w, void* out,
                           const int32_t* offs, int32_t group_count, int32_t rows, int32_t n, int32_t k,
                           int64_t stride_am, int64_t stride_sam, int64_t stride_sak, int64_t stride_wg,
                           int64_t stride_wn, int64_t stride_swg, int64_t stride_swn, int64_t stride_swk,
                           int64_t stride_om, int32_t out_dtype, int32_t fast_accum, int32_t variant,
                           int32_t grid_size, void* stream) {
  if (out_dtype != DT_F16 && out_dtype != DT_BF16 && out_dtype != DT_F32)
    return report(MOEGEMM_ERR_INVALID, "unsupported dtype code %d", out_dtype);
  int rc = check_operands(a, scale_a, w, scale_w, out, offs, group_count, rows, n, k, stride_am, stride_wg, stride_wn,
                          stride_om, n);
  if (rc == MOEGEMM_OK) rc = check_scales(stride_sam, stride_swn, n);
  if (rc != MOEGEMM_OK) return rc;
  if (!aligned(out, out_dtype == DT_F32 ? 4 : 2))
    return report(MOEGEMM_ERR_INVALID, "out must be aligned to its element size");
  Fp8Params p{static_cast<const uint8_t*>(a), scale_a, static_cast<const uint8_t*>(w), scale_w, out, nullptr, offs,
              stride_am, stride_sam, stride_sak, stride_wg, stride_wn, stride_swg, stride_swn, stride_swk,
              stride_om, 0, 0, group_count, rows, n, k, 0};
  const Fp8Variant* table = out_dtype == DT_F32 ? kFp8F32 : out_dtype == DT_BF16 ? kFp8Bf16 : kFp8F16;
  return launch_product(table, kNumFp8, p, n, 0, fast_accum, variant, grid_size, stream);
}

int moegemm_grouped_mm_fp8_swiglu(const void* a, const float* scale_a, const void* w, const float* scale_w, void* out,
                                  float* out_scale, const int32_t* offs, int32_t group_count, int32_t rows, int32_t n,
                                  int32_t k, int64_t stride_am, int64_t stride_sam, int64_t stride_sak,
                                  int64_t stride_wg, int64_t stride_wn, int64_t stride_swg, int64_t stride_swn,
                                  int64_t stride_swk, int64_t stride_om, int64_t stride_osm, int64_t stride_osk,
                                  int32_t fast_accum, int32_t variant, int32_t grid_size, void* stream) {
  int rc = check_operands(a, scale_a, w, scale_w, out, offs, group_count, rows, n, k, stride_am, stride_wg, stride_wn,
                          stride_om, n / 2);
  if (rc == MOEGEMM_OK) rc = check_scales(stride_sam, stride_swn, n);
  if (rc != MOEGEMM_OK) return rc;
  if (n % 16) return report(MOEGEMM_ERR_INVALID, "packed Gate+Up width must be a multiple of 16 (got %d)", n);
  if (!out_scale) return report(MOEGEMM_ERR_INVALID, "out_scale must be non-null");
  if (!aligned(out, 8) || stride_om % 8)
    return report(MOEGEMM_ERR_INVALID, "out rows must start at multiples of 8 bytes");
  Fp8Params p{static_cast<const uint8_t*>(a), scale_a, static_cast<const uint8_t*>(w), scale_w, out, out_scale, offs,
              stride_am, stride_sam, stride_sak, stride_wg, stride_wn, stride_swg, stride_swn, stride_swk,
              stride_om, stride_osm, stride_osk, group_count, rows, n, k, 0};
  return launch_product(kFp8Gated, kNumFp8Gated, p, n / 2, 1, fast_accum, variant, grid_size, stream);
}

}  // extern "C"
