// Compiled kernels of the Gate+Up training form, bf16 operands.
#include "gated_train.h"
namespace moegemm {
MOEGEMM_MENU_GATED(MOEGEMM_GATED_KERNEL, EBf16)
MOEGEMM_MENU_DX(MOEGEMM_GATED_KERNEL, EBf16)
MOEGEMM_MENU_DW(MOEGEMM_GATED_KERNEL, EBf16)
template __global__ void gate_up_gradient_kernel<EBf16>(GatedParams, const void*, int64_t, void*);
#if !defined(__HIP_DEVICE_COMPILE__)
namespace {
const GatedVariant kForward[] = {MOEGEMM_MENU_GATED(MOEGEMM_GATED_ENTRY, EBf16){}};
const GatedVariant kDx[] = {MOEGEMM_MENU_DX(MOEGEMM_GATED_ENTRY, EBf16){}};
const GatedVariant kDw[] = {MOEGEMM_MENU_DW(MOEGEMM_GATED_ENTRY, EBf16){}};
}  // namespace
const GatedTable kGatedBf16 = {{kForward, kDx, kDw}, &launch_gradient<EBf16>};
#endif
}  // namespace moegemm
