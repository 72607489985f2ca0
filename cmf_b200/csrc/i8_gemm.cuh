// Shared by the 8-bit product's kernels: the scaling of an integer sum.
#pragma once
#include "text_ops.cuh"

namespace cmfc {

constexpr int64_t I8_MAX_K = 131071;  // 128 * 128 * K stays below 2^31

int launch_i8_pair(const I8Params& p, int num_sms, cudaStream_t s);  // 16-byte aligned rows

// rounding of the activations inside the product (few short tokens)
bool i8_fused_fits(int64_t M, int64_t K);
bool i8_fused_supported(const I8Params& p, const void* act, int elem, int64_t ld_act);
int launch_i8_fused(const I8Params& p, const void* act, int elem, int64_t ld_act, cudaStream_t s);

#ifdef __CUDACC__
// A row's scale and levels from the largest bit pattern of its |x| (NaN above infinity above every number):
// scale = max |x| / 127, level = rint(x / scale) (ties to even), both quotients IEEE f32.  Zeros, or a scale
// that underflows to zero: scale 0, levels 0; an infinity or a NaN: scale NaN, levels 0.
struct RowScale {
    float scale;
    bool zero;
    __device__ __forceinline__ explicit RowScale(unsigned top) {
        const bool finite = top < 0x7f800000u;
        scale = finite ? __fdiv_rn(__uint_as_float(top), 127.0f) : __int_as_float(0x7fc00000);
        zero = !finite || scale == 0.0f;
    }
    // a scale rounded down among the subnormals could let the largest quotient pass 127
    __device__ __forceinline__ int level(float f) const { return zero ? 0 : max(-127, min(127, __float2int_rn(__fdiv_rn(f, scale)))); }
    // V (1, 4 or 8) levels to an address aligned to V
    template <int V>
    __device__ __forceinline__ void store(int8_t* dst, const float* v) const {
        if constexpr (V == 1) {
            *dst = (int8_t)level(v[0]);
        } else {
            uint32_t w[V / 4];
#pragma unroll
            for (int e = 0; e < V; e += 4)
                w[e / 4] = (uint32_t)(uint8_t)level(v[e]) | (uint32_t)(uint8_t)level(v[e + 1]) << 8 | (uint32_t)(uint8_t)level(v[e + 2]) << 16 |
                           (uint32_t)(uint8_t)level(v[e + 3]) << 24;
            if constexpr (V == 8) *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
            else *reinterpret_cast<uint32_t*>(dst) = w[0];
        }
    }
};
// The product of the scales is taken first in every kernel, so that all of them round alike.
__device__ __forceinline__ float i8_scaled(int acc, float x_scale, float w_scale) {
    return __fmul_rn(__int2float_rn(acc), __fmul_rn(x_scale, w_scale));
}
#endif

}  // namespace cmfc
