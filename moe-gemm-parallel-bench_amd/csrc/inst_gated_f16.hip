// Compiled kernels of the Gate+Up training form, fp16 operands.
#include "gated_train.h"
namespace moegemm {
MOEGEMM_MENU_GATED(MOEGEMM_GATED_KERNEL, EF16)
MOEGEMM_MENU_DX(MOEGEMM_GATED_KERNEL, EF16)
MOEGEMM_MENU_DW(MOEGEMM_GATED_KERNEL, EF16)
template __global__ void gate_up_gradient_kernel<EF16>(GatedParams, const void*, int64_t, void*);
#if !defined(__HIP_DEVICE_COMPILE__)
namespace {
const GatedVariant kForward[] = {MOEGEMM_MENU_GATED(MOEGEMM_GATED_ENTRY, EF16){}};
const GatedVariant kDx[] = {MOEGEMM_MENU_DX(MOEGEMM_GATED_ENTRY, EF16){}};
const GatedVariant kDw[] = {MOEGEMM_MENU_DW(MOEGEMM_GATED_ENTRY, EF16){}};
}  // namespace
const GatedTable kGatedF16 = {{kForward, kDx, kDw}, &launch_gradient<EF16>};
#endif
}  // namespace moegemm
