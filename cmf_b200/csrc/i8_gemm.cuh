// Shared by the 8-bit product's kernels: the scaling of an integer sum.
#pragma once
#include "text_ops.cuh"

namespace cmfc {

constexpr int64_t I8_MAX_K = 131071;  // 128 * 128 * K stays below 2^31

int launch_i8_pair(const I8Params& p, int num_sms, cudaStream_t s);  // 16-byte aligned rows

#ifdef __CUDACC__
// The product of the scales is taken first in every kernel, so that all of them round alike.
__device__ __forceinline__ float i8_scaled(int acc, float x_scale, float w_scale) {
    return __fmul_rn(__int2float_rn(acc), __fmul_rn(x_scale, w_scale));
}
#endif

}  // namespace cmfc
