// The radix-4 step of the ConvRot rotation, shared by the int4 / int8 quantizers
// and the MX4 kernels: every rotation is a sequence of these steps, so all of
// them sum in the same order.
#pragma once

#include <cuda_runtime.h>

namespace convrot {

// Regular Hadamard H4 = J - 2R (ones, minus twice the anti-diagonal):
// out_i = (v0+v1)+(v2+v3) - 2*v_(3-i), each output rounded once.
__device__ __forceinline__ void h4(float& v0, float& v1, float& v2, float& v3) {
    const float s = __fadd_rn(__fadd_rn(v0, v1), __fadd_rn(v2, v3));
    const float o0 = __fmaf_rn(-2.0f, v3, s);
    const float o1 = __fmaf_rn(-2.0f, v2, s);
    const float o2 = __fmaf_rn(-2.0f, v1, s);
    const float o3 = __fmaf_rn(-2.0f, v0, s);
    v0 = o0; v1 = o1; v2 = o2; v3 = o3;
}

}  // namespace convrot
