// C ABI of the 4-bit (MXFP4) operators: argument checks, the choice of a variant, the launches: one a call, and another
// for every further 1024 groups of a product.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "../../include/moegemm.h"
#include "error.h"
#include "mxfp4_menu.h"

using namespace moegemm;

namespace {

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
bool aligned(const void* p, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

int checked(hipError_t err) {
  return err == hipSuccess ? MOEGEMM_OK
                           : report(MOEGEMM_ERR_LAUNCH, "kernel launch failed: %s", hipGetErrorString(err));
}

bool is_dtype(int32_t dtype) { return dtype == DT_F16 || dtype == DT_BF16 || dtype == DT_F32; }

constexpr int64_t kPitchLimit = int64_t(1) << 23;  // a unit's rows lie within 2 GiB

constexpr int64_t kMaxBlocks = 1 << 16;  // workgroups of a conversion, which go on to what is past them

int check_conversion(int64_t rows, int32_t k, const void* x, const uint8_t* q, const uint8_t* scale, int64_t stride_q,
                     int32_t dtype) {
  if (!is_dtype(dtype)) return report(MOEGEMM_ERR_INVALID, "unsupported dtype code %d", dtype);
  if (rows < 0 || k <= 0 || k % kMxGroup)
    return report(MOEGEMM_ERR_INVALID, "bad shape (rows=%lld k=%d, k a multiple of 32)", (long long)rows, k);
  if (rows && (!x || !q || !scale)) return report(MOEGEMM_ERR_INVALID, "values, q and scale must be non-null");
  if (!aligned(q, 4) || stride_q % 4) return report(MOEGEMM_ERR_INVALID, "q rows must start at multiples of 4 bytes");
  if (!aligned(x, dtype == DT_F32 ? 4 : 2))
    return report(MOEGEMM_ERR_INVALID, "values must be aligned to their element size");
  return MOEGEMM_OK;
}

template <class E>
dim3 conversion_grid(const MxConvertParams& p) {
  return dim3((unsigned)std::min(cdiv(p.rows * (p.k / MxItem<E>::VALUES), 256 * kMxItems), kMaxBlocks));
}
// Rows that follow on one another are one long row: no division by a row's length.
MxConvertParams flat(MxConvertParams p, bool dense) {
  if (dense) {
    p.k *= p.rows;
    p.rows = 1;
  }
  return p;
}

template <class E>
hipError_t launch_quantize(const MxConvertParams& p, bool vec, hipStream_t s) {
  if (vec) hipLaunchKernelGGL((mx_quantize_kernel<E, true>), conversion_grid<E>(p), dim3(256), 0, s, p);
  else hipLaunchKernelGGL((mx_quantize_kernel<E, false>), conversion_grid<E>(p), dim3(256), 0, s, p);
  return hipGetLastError();
}
template <class E>
hipError_t launch_dequantize(const MxConvertParams& p, hipStream_t s) {
  hipLaunchKernelGGL((mx_dequantize_kernel<E>), conversion_grid<E>(p), dim3(256), 0, s, p);
  return hipGetLastError();
}

// Variant of the least estimated time for `rows` rows over `groups` groups of `cols` output columns.  Routed groups are
// taken to hold 0.4 to 1.6 times the mean; a group of more rows than a unit has its weights read again for each unit's
// rows.  A CU works on two units at a time: it takes half of its units' number, at least 0.65, times what a unit of the
// variant takes for 256 of K (us, from launches of many units, in the tables' order; rows of one part, of two, of three):
constexpr double kUnitTime[3][kNumMx] = {
    {1.15, 1.36, 1.72, 0.46, 0.67, 2.55}, {1.57, 1.66, 2.90, 0.72, 0.95, 2.90}, {1.76, 1.94, 3.80, 0.80, 1.15, 3.80}};
// Of 207 calls (10 weights, 1 to 1024 rows, three types) the chosen one took 1.01 times the best one's time in the
// mean, at most 1.32; of 144 calls of three parts (11 weights, 1 to 2048 rows) 1.01 times, at most 1.19.  What the
// variants take, in the same order (us, bf16): 32 experts of [4096, 7168] by 256 rows 122, 88, 99, 161, 135, 131; by
// 1024 rows 340, 204, 162, 467, 369, 151; one weight of [4096, 7168] by 16 rows 22, 25, 31, 11, 13, 46; by 32 rows 23,
// 24, 31, 18, 14, 47.
int choose(int parts, const MxVariant* table, int64_t rows, int64_t groups, int64_t cols, int cus) {
  const int64_t active = std::min(groups, rows);
  const double mean = (double)rows / active;
  int best = 0;
  double least = 0;
  for (int i = 0; i < kNumMx; ++i) {
    double tiles = 0;
    for (int j = 0; j < 7; ++j)
      tiles += std::ceil(std::max(active == 1 ? mean : mean * (0.4 + 0.2 * j), 1.0) / table[i].rows - 1e-9) / 7;
    const double units = std::ceil(active * tiles * cdiv(cols, table[i].cols) / cus - 1e-9);  // of a CU
    const double time = std::max(units / 2, 0.65) * kUnitTime[parts - 1][i];
    if (i == 0 || time < least) {
      best = i;
      least = time;
    }
  }
  return best;
}

int launch_product(const void* a, const uint8_t* w, const uint8_t* scale, void* out, const int32_t* offs, int32_t group_count,
                   int32_t rows, int32_t n, int32_t k, int64_t stride_am, int64_t stride_wg, int64_t stride_wn,
                   int64_t stride_sg, int64_t stride_sn, int64_t stride_om, int32_t dtype, int32_t out_dtype, bool gated,
                   int32_t variant, int32_t grid_size, void* stream) {
  if (!is_dtype(dtype) || !is_dtype(out_dtype))
    return report(MOEGEMM_ERR_INVALID, "unsupported dtype code %d or %d", dtype, out_dtype);
  if (group_count <= 0) return report(MOEGEMM_ERR_INVALID, "group_count must be positive (got %d)", group_count);
  if (!offs && group_count != 1)
    return report(MOEGEMM_ERR_INVALID, "without offsets there is one group (got %d)", group_count);
  if (rows < 0 || rows >= 1 << 30 || n <= 0 || n >= 1 << 30 || k <= 0 || k % kMxGroup)
    return report(MOEGEMM_ERR_INVALID, "bad shape (rows=%d n=%d k=%d, k a multiple of 32)", rows, n, k);
  if (gated && n % 2) return report(MOEGEMM_ERR_INVALID, "packed Gate+Up width must be even (got %d)", n);
  if (variant < -1 || variant >= kNumMx)
    return report(MOEGEMM_ERR_NO_KERNEL, "4-bit variant %d is not compiled (0 to %d, or -1)", variant, kNumMx - 1);
  if (rows == 0) return MOEGEMM_OK;
  const int64_t cols = gated ? n / 2 : n;
  if (!a || !w || !scale || !out) return report(MOEGEMM_ERR_INVALID, "operands, scales and output must be non-null");
  if (!aligned(a, 16) || stride_am % (dtype == DT_F32 ? 4 : 8) || !aligned(w, 16) || stride_wn % 16 || stride_wg % 16)
    return report(MOEGEMM_ERR_INVALID, "rows of a and weight must start at multiples of 16 bytes");
  if (stride_am < 0 || stride_wn < k / 2 || stride_sn < k / kMxGroup || (rows > 1 && stride_om < cols))
    return report(MOEGEMM_ERR_INVALID, "row pitches must cover a row");
  const int64_t es = dtype == DT_F32 ? 4 : 2;
  if (stride_am * es >= kPitchLimit || k * es >= kPitchLimit || stride_wn >= kPitchLimit || stride_sn >= kPitchLimit)
    return report(MOEGEMM_ERR_INVALID, "rows of a, weight and scale must be less than %lld bytes apart", (long long)kPitchLimit);
  if (!aligned(out, out_dtype == DT_F32 ? 4 : 2))
    return report(MOEGEMM_ERR_INVALID, "out must be aligned to its element size");
  const int cus = grid_size > 0 ? grid_size : 256;
  const MxVariant* table = dtype == DT_BF16  ? (gated ? kMxGatedBf16 : kMxBf16)
                           : dtype == DT_F16 ? (gated ? kMxGatedF16 : kMxF16)
                                             : (gated ? kMxGatedF32 : kMxF32);
  if (variant < 0) variant = choose(dtype == DT_BF16 ? 1 : dtype == DT_F16 ? 2 : 3, table, rows, group_count, cols, cus);
  const MxVariant& v = table[variant];
  MxParams p{a, w, scale, out, offs, stride_am, stride_wg, stride_wn, stride_sg, stride_sn,
             stride_om, group_count, rows, n, k, (int32_t)cdiv(cols, v.cols), out_dtype};
  const int64_t row_tiles = std::min({rows / v.rows + (int64_t)group_count, group_count * cdiv(rows, v.rows), (int64_t)rows});
  const int64_t bound = row_tiles * p.n_tiles;
  if (bound > INT32_MAX / 2) return report(MOEGEMM_ERR_INVALID, "tile count exceeds int32");
  const int grid = (int)std::min<int64_t>(bound, (int64_t)cus * v.per_cu);
  const bool once = stride_wn % 128 == 0 && aligned(w, 128) && cdiv(rows, group_count) <= v.rows;
  for (; p.first < group_count; p.first += kMxTable) {
    p.groups = std::min(group_count - p.first, kMxTable);
    const int rc = checked(v.launch(p, grid, once, reinterpret_cast<hipStream_t>(stream)));
    if (rc != MOEGEMM_OK) return rc;
  }
  return MOEGEMM_OK;
}

}  // namespace

extern "C" {

int moegemm_quantize_mxfp4(const void* x, uint8_t* q, uint8_t* scale, int64_t rows, int32_t k, int64_t stride_xr,
                           int64_t stride_qr, int64_t stride_sr, int32_t dtype, void* stream) {
  const int rc = check_conversion(rows, k, x, q, scale, stride_qr, dtype);
  if (rc != MOEGEMM_OK || rows == 0) return rc;
  const MxConvertParams p = flat({x, q, scale, nullptr, stride_xr, stride_qr, stride_sr, rows, k},
                                 stride_xr == k && stride_qr == k / 2 && stride_sr == k / kMxGroup);
  const bool vec = aligned(x, 16) && stride_xr * (dtype == DT_F32 ? 4 : 2) % 16 == 0;
  const auto s = reinterpret_cast<hipStream_t>(stream);
  return checked(dtype == DT_F32    ? launch_quantize<EF32>(p, vec, s)
                 : dtype == DT_BF16 ? launch_quantize<EBf16>(p, vec, s)
                                    : launch_quantize<EF16>(p, vec, s));
}

int moegemm_dequantize_mxfp4(const uint8_t* q, const uint8_t* scale, void* out, int64_t rows, int32_t k, int64_t stride_qr,
                             int64_t stride_sr, int32_t dtype, void* stream) {
  const int rc = check_conversion(rows, k, out, q, scale, stride_qr, dtype);
  if (rc != MOEGEMM_OK || rows == 0) return rc;
  if (!aligned(out, 16)) return report(MOEGEMM_ERR_INVALID, "out must be 16-byte aligned");
  const MxConvertParams p = flat({q, nullptr, const_cast<uint8_t*>(scale), out, 0, stride_qr, stride_sr, rows, k},
                                 stride_qr == k / 2 && stride_sr == k / kMxGroup);
  const auto s = reinterpret_cast<hipStream_t>(stream);
  return checked(dtype == DT_F32    ? launch_dequantize<EF32>(p, s)
                 : dtype == DT_BF16 ? launch_dequantize<EBf16>(p, s)
                                    : launch_dequantize<EF16>(p, s));
}

int moegemm_mxfp4_variant_count(void) { return kNumMx; }

int moegemm_grouped_mm_mxfp4(const void* a, const uint8_t* w, const uint8_t* scale, void* out, const int32_t* offs,
                             int32_t group_count, int32_t rows, int32_t n, int32_t k, int64_t stride_am, int64_t stride_wg,
                             int64_t stride_wn, int64_t stride_sg, int64_t stride_sn, int64_t stride_om, int32_t dtype,
                             int32_t out_dtype, int32_t variant, int32_t grid_size, void* stream) {
  return launch_product(a, w, scale, out, offs, group_count, rows, n, k, stride_am, stride_wg, stride_wn, stride_sg, stride_sn,
                        stride_om, dtype, out_dtype, false, variant, grid_size, stream);
}

int moegemm_grouped_mm_mxfp4_swiglu(const void* a, const uint8_t* w, const uint8_t* scale, void* out, const int32_t* offs,
                                    int32_t group_count, int32_t rows, int32_t n, int32_t k, int64_t stride_am,
                                    int64_t stride_wg, int64_t stride_wn, int64_t stride_sg, int64_t stride_sn,
                                    int64_t stride_om, int32_t dtype, int32_t out_dtype, int32_t variant, int32_t grid_size,
                                    void* stream) {
  return launch_product(a, w, scale, out, offs, group_count, rows, n, k, stride_am, stride_wg, stride_wn, stride_sg, stride_sn,
                        stride_om, dtype, out_dtype, true, variant, grid_size, stream);
}

}  // extern "C"
