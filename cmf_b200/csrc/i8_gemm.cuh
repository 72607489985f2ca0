// Shared by the 8-bit product's kernels: the scaling of an integer sum.
#pragma once
#include "text_ops.cuh"

namespace cmfc {

constexpr int64_t I8_MAX_K = 131071;  // 128 * 128 * K stays below 2^31

int launch_i8_pair(const I8Params& p, int num_sms, cudaStream_t s);  // 16-byte aligned rows

// rounding of the activations inside the product (few short tokens)
bool i8_fused_supported(const I8Params& p, const void* act, int elem, int64_t ld_act);
int launch_i8_fused(const I8Params& p, const void* act, int elem, int64_t ld_act, cudaStream_t s);

#ifdef __CUDACC__
// A row's scale and levels from the largest bit pattern of its |x| (NaN above infinity above every number):
// scale = max |x| / 127, level = rint(x / scale) (ties to even), both quotients IEEE f32.  Zeros, or a scale
// that underflows to zero: scale 0, levels 0; an infinity or a NaN: scale NaN, levels 0.
struct RowScale {
    float scale, inv;
    bool zero, slow;
    __device__ __forceinline__ explicit RowScale(unsigned top) {
        const bool finite = top < 0x7f800000u;
        scale = finite ? __fdiv_rn(__uint_as_float(top), 127.0f) : __int_as_float(0x7fc00000);
        zero = !finite || scale == 0.0f;
        slow = !(scale >= 1e-30f && scale <= 1e30f);  // the reciprocal could leave the normal numbers
        inv = __frcp_rn(scale);
    }
    // the definition; a scale rounded down among the subnormals could let the largest quotient pass 127
    __device__ __forceinline__ int exact(float f) const { return zero ? 0 : max(-127, min(127, __float2int_rn(__fdiv_rn(f, scale)))); }
    // Levels without a division each: t = f * (1 / scale) is off f / scale by at most 127 x 2 x 2^-24 = 1.6e-5 (two
    // roundings of a number up to 127), and the rounded quotient by at most 127 x 2^-24 = 7.6e-6, so both round to the same
    // integer unless t lies within 2.4e-5 of a half.  Values that do (one in some thousands) take the definition.
    // Rounding to an integer is the addition of 1.5 x 2^23; its low byte is the level.
    template <int V>
    __device__ __forceinline__ void levels(const float* v, uint32_t* bits) const {
        constexpr float MAGIC = 12582912.0f;
        float far = 0.0f;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float t = v[e] * inv, u = t + MAGIC;
            bits[e] = __float_as_uint(u);
            far = fmaxf(far, fabsf(t - (u - MAGIC)));
        }
        if (slow || zero || far > 0.49997f) {
#pragma unroll
            for (int e = 0; e < V; ++e) bits[e] = (uint32_t)exact(v[e]);
        }
    }
    // V (1, 4 or 8) levels to an address aligned to V
    template <int V>
    __device__ __forceinline__ void store(int8_t* dst, const float* v) const {
        uint32_t b[V];
        levels<V>(v, b);
        if constexpr (V == 1) {
            *dst = (int8_t)b[0];
        } else {
            uint32_t w[V / 4];
#pragma unroll
            for (int e = 0; e < V; e += 4)
                w[e / 4] = __byte_perm(__byte_perm(b[e], b[e + 1], 0x0040), __byte_perm(b[e + 2], b[e + 3], 0x0040), 0x5410);
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
