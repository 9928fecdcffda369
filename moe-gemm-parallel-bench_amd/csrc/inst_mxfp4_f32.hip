// Compiled 4-bit products of fp32 rows.
#include "mxfp4_menu.h"
namespace moegemm {
MOEGEMM_MENU_MX(MOEGEMM_MX_XK, EF32, false)
MOEGEMM_MENU_MX(MOEGEMM_MX_XK, EF32, true)
#if !defined(__HIP_DEVICE_COMPILE__)
const MxVariant kMxF32[] = {MOEGEMM_MENU_MX(MOEGEMM_MX_X, EF32, false) MOEGEMM_MX_X(EF32, 32, 4, 4, 1, false)};
const MxVariant kMxGatedF32[] = {MOEGEMM_MENU_MX(MOEGEMM_MX_X, EF32, true) MOEGEMM_MX_X(EF32, 32, 4, 4, 1, true)};
#endif
}  // namespace moegemm
