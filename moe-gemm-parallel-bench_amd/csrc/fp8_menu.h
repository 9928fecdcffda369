// Compiled variants of the block-scaled fp8 products, one table per output type (inst_fp8_*.hip).
#pragma once

#include "fp8_gemm.h"

namespace moegemm {

typedef hipError_t (*Fp8LaunchFn)(const Fp8Params&, int grid, hipStream_t stream);

struct Fp8Variant {
  int block_m, block_n;  // rows and weight rows of a tile
  int stream;            // 1: units of (group, column tile); 0: tiles of each group's rows and columns
  int waves_k;           // stream: waves that share K
  int fast;              // sums on the 8-bit matrix instructions
  Fp8LaunchFn launch;
};

template <class T>
hipError_t launch_fp8_tile(const Fp8Params& p, int grid, hipStream_t stream) {
  hipLaunchKernelGGL((fp8_tile_kernel<T>), dim3(grid), dim3(T::NT), 0, stream, p);
  return hipGetLastError();
}
template <class T, class E>
hipError_t launch_fp8_stream(const Fp8Params& p, int grid, hipStream_t stream) {
  hipLaunchKernelGGL((fp8_stream_kernel<T, E>), dim3(grid), dim3(T::NT), 0, stream, p);
  return hipGetLastError();
}

// X(E, BM, BN, WAVES_M, WAVES_N, STAGES, FAST) and Y(E, FM, FN, WAVES_N, WAVES_K, STAGES).  Stream tiles are
// 16 or 32 rows by 256 to 16 columns: wide ones for many units, narrow ones with K split over the waves for few.
#define MOEGEMM_MENU_FP8(X, Y, E)                                                               \
  X(E, 256, 256, 2, 4, 2, true) X(E, 128, 256, 2, 4, 2, true) X(E, 128, 128, 2, 2, 2, true)     \
  X(E, 128, 256, 2, 4, 2, false) X(E, 128, 128, 2, 2, 2, false)                                 \
  Y(E, 1, 4, 4, 1, 3) Y(E, 1, 2, 4, 2, 2) Y(E, 1, 4, 1, 4, 3) Y(E, 1, 1, 1, 8, 4)   \
  Y(E, 2, 4, 4, 1, 2) Y(E, 2, 1, 1, 8, 2)
#define MOEGEMM_MENU_FP8_GATED(X, Y, E)                                                         \
  X(E, 256, 256, 2, 4, 2, true) X(E, 128, 256, 2, 4, 2, true) X(E, 128, 256, 2, 4, 2, false)    \
  Y(E, 1, 4, 4, 1, 3) Y(E, 2, 4, 4, 1, 3)

#define MOEGEMM_FP8_X(E, BM, BN, WM, WN, S, FAST) \
  Fp8Variant{BM, BN, 0, 1, FAST, &launch_fp8_tile<Fp8Tile<E, BM, BN, WM, WN, S, false, FAST>>},
#define MOEGEMM_FP8_Y(E, FM, FN, WN, WK, S) \
  Fp8Variant{16 * FM, 16 * FN * WN, 1, WK, 0, &launch_fp8_stream<Fp8Stream<E, FM, FN, WN, WK, S, false>, E>},
#define MOEGEMM_FP8_GX(E, BM, BN, WM, WN, S, FAST) \
  Fp8Variant{BM, BN, 0, 1, FAST, &launch_fp8_tile<Fp8Tile<E, BM, BN, WM, WN, S, true, FAST>>},
#define MOEGEMM_FP8_GY(E, FM, FN, WN, WK, S) \
  Fp8Variant{16 * FM, 16 * FN * WN, 1, WK, 0, &launch_fp8_stream<Fp8Stream<E, FM, FN, WN, WK, S, true>, E>},

// The kernels of a menu, for the device pass.
#define MOEGEMM_FP8_XK(E, BM, BN, WM, WN, S, FAST) \
  template __global__ void fp8_tile_kernel<Fp8Tile<E, BM, BN, WM, WN, S, false, FAST>>(Fp8Params);
#define MOEGEMM_FP8_YK(E, FM, FN, WN, WK, S) \
  template __global__ void fp8_stream_kernel<Fp8Stream<E, FM, FN, WN, WK, S, false>, E>(Fp8Params);
#define MOEGEMM_FP8_GXK(E, BM, BN, WM, WN, S, FAST) \
  template __global__ void fp8_tile_kernel<Fp8Tile<E, BM, BN, WM, WN, S, true, FAST>>(Fp8Params);
#define MOEGEMM_FP8_GYK(E, FM, FN, WN, WK, S) \
  template __global__ void fp8_stream_kernel<Fp8Stream<E, FM, FN, WN, WK, S, true>, E>(Fp8Params);

#define MOEGEMM_FP8_COUNT(...) +1
constexpr int kNumFp8 = 0 MOEGEMM_MENU_FP8(MOEGEMM_FP8_COUNT, MOEGEMM_FP8_COUNT, );
constexpr int kNumFp8Gated = 0 MOEGEMM_MENU_FP8_GATED(MOEGEMM_FP8_COUNT, MOEGEMM_FP8_COUNT, );

extern const Fp8Variant kFp8Bf16[], kFp8F16[], kFp8F32[], kFp8Gated[];

}  // namespace moegemm
