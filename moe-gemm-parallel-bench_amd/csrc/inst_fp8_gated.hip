// Compiled fp8 Gate+Up products with SwiGLU and e4m3 output.
#include "fp8_menu.h"
namespace moegemm {
MOEGEMM_MENU_FP8_GATED(MOEGEMM_FP8_GXK, MOEGEMM_FP8_GYK, EBf16)
#if !defined(__HIP_DEVICE_COMPILE__)
const Fp8Variant kFp8Gated[] = {MOEGEMM_MENU_FP8_GATED(MOEGEMM_FP8_GX, MOEGEMM_FP8_GY, EBf16)};
#endif
}  // namespace moegemm
