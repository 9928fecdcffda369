// Compiled fp8 products with bf16 output.
#include "fp8_menu.h"
namespace moegemm {
MOEGEMM_MENU_FP8(MOEGEMM_FP8_XK, MOEGEMM_FP8_YK, EBf16)
#if !defined(__HIP_DEVICE_COMPILE__)
const Fp8Variant kFp8Bf16[] = {MOEGEMM_MENU_FP8(MOEGEMM_FP8_X, MOEGEMM_FP8_Y, EBf16)};
#endif
}  // namespace moegemm
