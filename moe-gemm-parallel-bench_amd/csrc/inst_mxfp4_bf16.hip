// Compiled 4-bit products of bf16 rows.
#include "mxfp4_menu.h"
namespace moegemm {
MOEGEMM_MENU_MX(MOEGEMM_MX_XK, EBf16, false) MOEGEMM_MX_XK(EBf16, 64, 4, 4, 1, false)
MOEGEMM_MENU_MX(MOEGEMM_MX_XK, EBf16, true) MOEGEMM_MX_XK(EBf16, 64, 4, 4, 1, true)
#if !defined(__HIP_DEVICE_COMPILE__)
const MxVariant kMxBf16[] = {MOEGEMM_MENU_MX(MOEGEMM_MX_X, EBf16, false) MOEGEMM_MX_X(EBf16, 64, 4, 4, 1, false)};
const MxVariant kMxGatedBf16[] = {MOEGEMM_MENU_MX(MOEGEMM_MX_X, EBf16, true) MOEGEMM_MX_X(EBf16, 64, 4, 4, 1, true)};
#endif
}  // namespace moegemm
