// w4_bf16_half.hip -- the 4-bit linear kernels (w4.h) for bfloat16 activations whose rows begin in the middle of a dword.
#define W4_KERNELS
#include "w4.h"

hipError_t w4_launch_bf16_half(const W4Params& p, int scale_type, bool grad, hipStream_t st) {
    return launch_any<GR_DT_BF16, true>(p, scale_type, grad, st);
}
