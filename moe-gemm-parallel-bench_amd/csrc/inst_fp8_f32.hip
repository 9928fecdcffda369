// Compiled fp8 products with fp32 output.
#include "fp8_menu.h"
namespace moegemm {
MOEGEMM_MENU_FP8(MOEGEMM_FP8_XK, MOEGEMM_FP8_YK, EF32)
#if !defined(__HIP_DEVICE_COMPILE__)
const Fp8Variant kFp8F32[] = {MOEGEMM_MENU_FP8(MOEGEMM_FP8_X, MOEGEMM_FP8_Y, EF32)};
#endif
}  // namespace moegemm
