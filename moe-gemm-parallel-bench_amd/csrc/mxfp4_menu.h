// Compiled variants of the 4-bit products, one table per type of the rows (inst_mxfp4_*.hip).
#pragma once

#include "mxfp4.h"

namespace moegemm {

typedef hipError_t (*MxLaunchFn)(const MxParams&, int grid, bool once, hipStream_t stream);

struct MxVariant {
  int rows, cols;  // of a unit: output rows, and output columns
  int waves_k;     // waves that have a part of K each; 1: waves that share the rows
  int per_cu;      // workgroups a CU
  MxLaunchFn launch;
};

template <class T>
hipError_t launch_mx(const MxParams& p, int grid, bool once, hipStream_t stream) {
  const size_t lds = MxTable::bytes(p.groups);
  // Few units' weights are small: kept.
  if (T::SHARED && once) hipLaunchKernelGGL((mx_stream_kernel<T, T::SHARED>), dim3(grid), dim3(T::NT), lds, stream, p);
  else hipLaunchKernelGGL((mx_stream_kernel<T, false>), dim3(grid), dim3(T::NT), lds, stream, p);
  return hipGetLastError();
}

// X(A, ROWS, FN, WAVES_N, WAVES_K, GATED): 8, 16 or 32 rows by 128 weight rows for many units, 8 or 16 rows by 32
// weight rows with K split over the waves for few.  A table ends with the unit of the most rows: 64 for bf16; of two
// parts 64 would leave LDS for one workgroup a CU (2048 rows over 32 experts of [4096, 7168] 594 us, 32 rows a unit
// 446), of three for none, so there it is the 32 again.
#define MOEGEMM_MENU_MX(X, A, GATED)                                        \
  X(A, 8, 4, 4, 1, GATED) X(A, 16, 4, 4, 1, GATED) X(A, 32, 4, 4, 1, GATED) \
  X(A, 8, 4, 1, 4, GATED) X(A, 16, 4, 1, 4, GATED)

#define MOEGEMM_MX_X(A, ROWS, FN, WN, WK, GATED)                                                                \
  MxVariant{ROWS, 8 * FN * WN / (GATED ? 2 : 1), WK, MxStream<A, ROWS, FN, WN, WK, GATED>::PER_CU, \
            &launch_mx<MxStream<A, ROWS, FN, WN, WK, GATED>>},
// The kernels of a menu, for the device pass.
#define MOEGEMM_MX_XK(A, ROWS, FN, WN, WK, GATED)                                                   \
  template __global__ void mx_stream_kernel<MxStream<A, ROWS, FN, WN, WK, GATED>, false>(MxParams); \
  MOEGEMM_MX_ONCE_##WK(A, ROWS, FN, WN, WK, GATED)
#define MOEGEMM_MX_ONCE_1(A, ROWS, FN, WN, WK, GATED) \
  template __global__ void mx_stream_kernel<MxStream<A, ROWS, FN, WN, WK, GATED>, true>(MxParams);
#define MOEGEMM_MX_ONCE_4(A, ROWS, FN, WN, WK, GATED)

#define MOEGEMM_MX_COUNT(...) +1
constexpr int kNumMx = 1 MOEGEMM_MENU_MX(MOEGEMM_MX_COUNT, , false);  // and the most rows

extern const MxVariant kMxBf16[], kMxF16[], kMxF32[], kMxGatedBf16[], kMxGatedF16[], kMxGatedF32[];

}  // namespace moegemm
