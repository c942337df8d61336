// w4_f32.hip -- the 4-bit linear kernels (w4.h) for float32 activations.
#define W4_KERNELS
#include "w4.h"

hipError_t w4_launch_f32(const W4Params& p, int scale_type, bool grad, hipStream_t st) {
    return launch_any<GR_DT_F32, false>(p, scale_type, grad, st);
}
