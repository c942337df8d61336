// w4_bf16.hip -- the 4-bit linear kernels (w4.h) for bfloat16 activations.
#define W4_KERNELS
#include "w4.h"

hipError_t w4_launch_bf16(const W4Params& p, int scale_type, bool grad, hipStream_t st) {
    return launch_any<GR_DT_BF16, false>(p, scale_type, grad, st);
}
