// What the text-layer operators share: element types of the caller's device tensors, strided head
// views, parameter blocks and their launchers.
#pragma once
#include <cuda_fp16.h>

#include "common.cuh"

namespace cmfc {

enum : int { ET_F32 = 0, ET_F16 = 1, ET_BF16 = 2 };
inline size_t elem_bytes(int elem) { return elem == ET_F32 ? 4 : 2; }

// [rows, heads, hd] with unit stride inside a head; strides in elements
struct HeadView {
    const void* p;
    int64_t row, head;
};

struct NormRopeParams {
    HeadView q, k, q_out, k_out;
    const float *norm_q, *norm_k;   // [hd]
    const float *cos_t, *sin_t;     // [table_rows, rot / 2]
    const void* positions;          // null: token t is at position t; else int32 or int64 [n]
    int64_t n, table_rows;
    int nh, nkv, hd, rot;
    int pos64;
    float eps;
};
int launch_norm_rope(const NormRopeParams& p, int elem, bool half_split, cudaStream_t s);

int launch_quantize_rows(const void* x, int elem, int64_t rows, int64_t cols, int64_t ldx, int8_t* q, int64_t ldq, float* scale,
                         cudaStream_t s);

// y[m, n] = (sum_k x[m, k] w[n, k]) * x_scale[m] * w_scale[n]
struct I8Params {
    const int8_t *x, *w;
    const float *x_scale, *w_scale;
    void* y;
    int64_t ldx, ldw, ldy;
    int64_t M, N, K;
    int out_elem;
    uint32_t* status;
    int behind_quantizer;  // the launch before this one on the stream is the quantizer of x: set up while it runs
};
int launch_i8_matmat(const I8Params& p, int num_sms, cudaStream_t s);

// Causal attention over packed sequences or caches; see cmfc_window_attention_args
struct WindowAttnParams {
    HeadView q, k, v, out;
    const int32_t *q_start, *k_start, *k_len;  // device, or all null: one sequence of all rows
    int64_t q_rows, k_rows;
    int seqs, nh, nkv, hd;
    int window;   // keys a query reaches back over, itself included; INT_MAX: all
    int sinks;
    float scale, softcap;
    uint32_t* status;
};
int launch_window_attention(const WindowAttnParams& p, int elem, int num_sms, cudaStream_t s);

#ifdef __CUDACC__
// A kernel that gave up a wait still has copies under way into its shared memory: they get 2 ms (they take
// microseconds) before the block leaves.
__device__ __forceinline__ void drain_copies(volatile uint32_t* abort_flag) {
    if (*abort_flag)
        for (int i = 0; i < 500; ++i) __nanosleep(4000);
}
__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// a 16-byte chunk of T as f32 values and back
template <typename T> __device__ __forceinline__ void unpack16(const uint4& r, float* o);
template <> __device__ __forceinline__ void unpack16<float>(const uint4& r, float* o) {
    o[0] = __uint_as_float(r.x);
    o[1] = __uint_as_float(r.y);
    o[2] = __uint_as_float(r.z);
    o[3] = __uint_as_float(r.w);
}
template <> __device__ __forceinline__ void unpack16<__nv_bfloat16>(const uint4& r, float* o) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        o[2 * i] = __uint_as_float(w[i] << 16);
        o[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}
template <> __device__ __forceinline__ void unpack16<__half>(const uint4& r, float* o) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        o[2 * i] = f.x;
        o[2 * i + 1] = f.y;
    }
}
// two f32 -> two packed values of T, rounded to nearest even
template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) { return pack_bf16(lo, hi); }
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template <typename T> __device__ __forceinline__ uint4 pack16(const float* x) {
    if constexpr (sizeof(T) == 4) {
        return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
    } else {
        return make_uint4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7]));
    }
}
#endif

}  // namespace cmfc
