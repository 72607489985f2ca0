// Matrix products in 8-bit integers with a scale for each token and each output channel:
//   y[m, n] = (sum_k x[m, k] w[n, k]) * (x_scale[m] * w_scale[n])
// The sum is exact in 32-bit integers (|x|, |w| <= 128 and K <= 131071), whatever the order, so every form
// below and every split of K gives the same bits; one rounding to f32, the product of the two scales, their
// product, and one rounding to the output type follow.
#include <atomic>

#include "i8_gemm.cuh"

namespace cmfc {
namespace {

// ---- any shape, stride and alignment: 64 x 64 tiles on the dot-product unit ----
constexpr int GT = 64, GK = 64;
template <typename T>
__global__ void __launch_bounds__(256) i8_any_kernel(I8Params p) {
    __shared__ int xs[GT][GK / 4 + 1], ws[GT][GK / 4 + 1];  // four levels a word, rows on shifted banks
    const int64_t m0 = (int64_t)blockIdx.y * GT, n0 = (int64_t)blockIdx.x * GT;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    int acc[4][4] = {};
    for (int64_t k0 = 0; k0 < p.K; k0 += GK) {
        __syncthreads();
        for (int t = threadIdx.x; t < GT * GK; t += 256) {
            const int r = t / GK, c = t % GK;
            const bool in_k = k0 + c < p.K;
            reinterpret_cast<int8_t*>(&xs[r][0])[c] = in_k && m0 + r < p.M ? p.x[(m0 + r) * p.ldx + k0 + c] : (int8_t)0;
            reinterpret_cast<int8_t*>(&ws[r][0])[c] = in_k && n0 + r < p.N ? p.w[(n0 + r) * p.ldw + k0 + c] : (int8_t)0;
        }
        __syncthreads();
#pragma unroll 4
        for (int c = 0; c < GK / 4; ++c) {
            int a[4], b[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                a[i] = xs[ty + 16 * i][c];
                b[i] = ws[tx + 16 * i][c];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(a[i], b[j], acc[i][j]);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t m = m0 + ty + 16 * i, n = n0 + tx + 16 * j;
            if (m < p.M && n < p.N)
                static_cast<T*>(p.y)[m * p.ldy + n] = from_f32<T>(i8_scaled(acc[i][j], p.x_scale[m], p.w_scale[n]));
        }
}

template <typename T>
void launch_any(const I8Params& p, cudaStream_t s) {
    i8_any_kernel<T><<<dim3((unsigned)((p.N + GT - 1) / GT), (unsigned)((p.M + GT - 1) / GT)), 256, 0, s>>>(p);
}

}  // namespace

int launch_i8_matmat(const I8Params& p, int num_sms, cudaStream_t s) {
    (void)num_sms;
    if ((p.M + GT - 1) / GT > 65535) return fail(ERR_UNSUPPORTED, "i8_matmat: too many tokens for rows that are not 16-byte aligned");
    if (p.out_elem == ET_F32) launch_any<float>(p, s);
    else if (p.out_elem == ET_F16) launch_any<__half>(p, s);
    else launch_any<__nv_bfloat16>(p, s);
    CMFC_CUDA(cudaGetLastError());
    return OK;
}

}  // namespace cmfc
