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
// The product is launched while the quantizer in front of it still runs (programmatic stream serialization): it sets
// itself up and then waits here until the quantizer is through.  Without that attribute the wait is over at once.
__device__ __forceinline__ void wait_for_quantizer() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_product_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// A row's scale and levels from the largest bit pattern of its |x| (NaN above infinity above every number):
// scale = max |x| * (1 / 127), the constant and the product each rounded to f32; level = rint(x / scale) (ties to
// even), an IEEE f32 quotient.  The product is what torch computes for `x.abs().amax(1) / 127` on a CUDA tensor: x = max / 2
// and every odd multiple of max / 254 that the type holds lie on a tie, so that a scale one unit off the caller's would
// move their levels.  Zeros, or a scale that underflows to zero: scale 0, levels 0; an infinity or a NaN: scale NaN, levels 0.
struct RowScale {
    float scale, inv;
    bool zero, slow;
    __device__ __forceinline__ explicit RowScale(unsigned top) {
        const bool finite = top < 0x7f800000u;
        scale = finite ? __fmul_rn(__uint_as_float(top), 1.0f / 127.0f) : __int_as_float(0x7fc00000);
        zero = !finite || scale == 0.0f;
        slow = !(scale >= 1e-30f && scale <= 1e30f);  // the reciprocal could leave the normal numbers
        inv = __frcp_rn(scale);
    }
    // the definition; a scale rounded down among the subnormals could let the largest quotient pass 127
    static __device__ __forceinline__ int exact(float f, float scale, bool zero) {
        return zero ? 0 : max(-127, min(127, __float2int_rn(__fdiv_rn(f, scale))));
    }
    __device__ __forceinline__ int8_t level(float f) const { return (int8_t)exact(f, scale, zero); }
    // a 16-byte chunk of T -> its levels, one byte each (.y stays 0 for the four of f32)
    template <typename T>
    static __device__ __noinline__ uint2 exact_chunk(uint4 raw, float scale, bool zero) {
        constexpr int V = 16 / (int)sizeof(T);
        float v[V];
        unpack16<T>(raw, v);
        uint32_t w[2] = {0u, 0u};
#pragma unroll
        for (int e = 0; e < V; ++e) w[e / 4] |= (uint32_t)(uint8_t)exact(v[e], scale, zero) << (8 * (e & 3));
        return make_uint2(w[0], w[1]);
    }
    // The same without a division each.  t = RN(f * inv) is off f / scale by at most 127 x 2 x 2^-24 = 1.6e-5 (two roundings
    // of a number up to 127), and the rounded quotient by at most 127 x 2^-24 = 7.6e-6, so both round to the same integer
    // unless t lies within 2.4e-5 of a half h (bf16 values over a bf16 maximum do in 0.3 % of all cases).  There the
    // remainder e = f - h scale is exact: h has 8 bits, so e is a multiple of half a unit in the last place of scale and
    // smaller than 2^10 of them.  f / scale = h + e / scale, and only the side of h on which its f32 rounding falls
    // matters: |e / scale| against half a unit of h, two numbers that differ by 2^-23 of them at least (integers over
    // 2^17 parts of the 24-bit scale; equality would make the quotient a tie between two f32 numbers, which a
    // quotient of f32 numbers never is), while e * inv is off by 2^-24.  So RN(h + e * inv) falls on the right side.
    // Rounding to an integer, ties to even, is the addition of 1.5 x 2^23; its low byte is the level.
    template <typename T>
    __device__ __forceinline__ uint2 chunk(const uint4& raw) const {
        constexpr int V = 16 / (int)sizeof(T);
        constexpr float MAGIC = 12582912.0f;
        float v[V], far = 0.0f;
        uint32_t b[V];
        unpack16<T>(raw, v);
        const uint64_t inv2 = pack_f32x2(inv, inv), up = pack_f32x2(MAGIC, MAGIC), down = pack_f32x2(-MAGIC, -MAGIC), neg = pack_f32x2(-1.0f, -1.0f);
#pragma unroll
        for (int e = 0; e < V; e += 2) {  // two at a time: t, t + magic, (t + magic) - magic, t minus that
            const uint64_t t = mul_f32x2(pack_f32x2(v[e], v[e + 1]), inv2), u = add_f32x2(t, up);
            float u0, u1, d0, d1;
            unpack_f32x2(u, u0, u1);
            unpack_f32x2(fma_f32x2(add_f32x2(u, down), neg, t), d0, d1);
            b[e] = __float_as_uint(u0);
            b[e + 1] = __float_as_uint(u1);
            far = fmaxf(far, fmaxf(fabsf(d0), fabsf(d1)));
        }
        if (far > 0.49997f) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float t = v[e] * inv, n = __uint_as_float(b[e]) - MAGIC, d = t - n;
                if (fabsf(d) > 0.49997f) {
                    const float h = n + copysignf(0.5f, d);
                    b[e] = __float_as_uint(fmaf(fmaf(-h, scale, v[e]), inv, h) + MAGIC);
                }
            }
        }
        uint32_t w[2] = {0u, 0u};
#pragma unroll
        for (int e = 0; e < V; e += 4)
            w[e / 4] = __byte_perm(__byte_perm(b[e], b[e + 1], 0x0040), __byte_perm(b[e + 2], b[e + 3], 0x0040), 0x5410);
        uint2 r = make_uint2(w[0], w[1]);
        if (slow || zero) r = exact_chunk<T>(raw, scale, zero);
        return r;
    }
    template <typename T>
    __device__ __forceinline__ void store(int8_t* dst, const uint4& raw) const {  // dst aligned to the chunk's levels
        const uint2 r = chunk<T>(raw);
        if constexpr (sizeof(T) == 2) *reinterpret_cast<uint2*>(dst) = r;
        else *reinterpret_cast<uint32_t*>(dst) = r.x;
    }
};
// The product of the scales is taken first in every kernel, so that all of them round alike.
__device__ __forceinline__ float i8_scaled(int acc, float x_scale, float w_scale) {
    return __fmul_rn(__int2float_rn(acc), __fmul_rn(x_scale, w_scale));
}
#endif

}  // namespace cmfc
