// Compiled 4-bit products of fp16 rows.
#include "mxfp4_menu.h"
namespace moegemm {
MOEGEMM_MENU_MX(MOEGEMM_MX_XK, EF16, false)
MOEGEMM_MENU_MX(MOEGEMM_MX_XK, EF16, true)
#if !defined(__HIP_DEVICE_COMPILE__)
const MxVariant kMxF16[] = {MOEGEMM_MENU_MX(MOEGEMM_MX_X, EF16, false) MOEGEMM_MX_X(EF16, 32, 4, 4, 1, false)};
const MxVariant kMxGatedF16[] = {MOEGEMM_MENU_MX(MOEGEMM_MX_X, EF16, true) MOEGEMM_MX_X(EF16, 32, 4, 4, 1, true)};
#endif
}  // namespace moegemm
