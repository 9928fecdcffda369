// C ABI of the 4-bit (MXFP4) operators: argument checks, the choice of a variant, the launches: one a call, and another for
// every further 1024 groups of a product.
#include <hip/hip_runtime.h>

#include <algorithm>

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

// Variant for `rows` rows over `groups` groups of `cols` output columns.  Routed groups are taken to hold up to 1.6 times the mean;
// a group of more rows than a unit has its weights read again for each unit's rows.  Wide units, Gate+Up (us): 256 rows over
// 128 experts of [5760, 2880] 8 rows a unit 234, 16 rows 244; 256 rows over 32 of [4096, 7168] 124 and 102; 768 rows over them 16
// rows 177, 32 rows 128.
// Narrow units, whose waves split K, where the wide ones would not fill two workgroups a CU: one row of [5760, 2880] 5.7, wide 12.6,
// four experts' rows of 128 x [2880, 2880] 8.3 and 13.3, 32 rows of [4096, 7168] 13.0 and 23.2; but 256 rows over 32
// experts of [4096, 7168] 171 and 86.  Sixteen rows a narrow unit where that leaves no CU idle: 32 rows of [4096, 7168], 256 units, 13.0
// and by eight rows 16.9, but 16 rows, 128 units, 12.6 and by eight 10.0.
int choose(const MxVariant* table, int64_t rows, int64_t groups, int64_t cols, int cus) {
  const int64_t active = std::min(groups, rows), mean = cdiv(rows, active);
  const int64_t high = active == 1 ? rows : cdiv(mean * 8, 5);
  auto find = [&](int wanted_rows, bool wide) {
    int i = 0;
    while (table[i].rows != wanted_rows || (table[i].waves_k == 1) != wide) ++i;
    return i;
  };
  auto units = [&](int i) { return active * cdiv(mean, table[i].rows) * cdiv(cols, table[i].cols); };
  const int wide = find(high <= 8 ? 8 : high <= 16 ? 16 : 32, true);
  if (units(wide) >= 2 * cus) return wide;
  const int narrow = find(16, false);
  return high <= 8 || units(narrow) < cus ? find(8, false) : narrow;
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
  if (variant < 0) variant = choose(table, rows, group_count, cols, cus);
  const MxVariant& v = table[variant];
  MxParams p{a, w, scale, out, offs, stride_am, stride_wg, stride_wn, stride_sg, stride_sn,
             stride_om, group_count, rows, n, k, (int32_t)cdiv(cols, v.cols), out_dtype};
  const int64_t row_tiles = std::min({rows / v.rows + (int64_t)group_count, group_count * cdiv(rows, v.rows), (int64_t)rows});
  const int64_t bound = row_tiles * p.n_tiles;
  if (bound > INT32_MAX / 2) return report(MOEGEMM_ERR_INVALID, "tile count exceeds int32");
  const int grid = (int)std::min<int64_t>(bound, (int64_t)cus * v.per_cu);
  for (; p.first < group_count; p.first += kMxTable) {
    p.groups = std::min(group_count - p.first, kMxTable);
    const int rc = checked(v.launch(p, grid, reinterpret_cast<hipStream_t>(stream)));
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
