// Matrix products in 8-bit integers with a scale for each token and each output channel:
//   y[m, n] = (sum_k x[m, k] w[n, k]) * (x_scale[m] * w_scale[n])
// The sum is exact in 32-bit integers (|x|, |w| <= 128 and K <= 131071), whatever the order, so every form
// below and every split of K gives the same bits; one rounding to f32, the product of the two scales, their
// product, and one rounding to the output type follow.
#include <atomic>
#include <type_traits>

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

// ---- up to 16 tokens: a stream of the weights through the warp-level 8-bit MMA ----
// Bound: memory, N K bytes of weights.  A block owns 16 weight rows; its 8 warps take 64-byte pieces of k in turn
// and add their integer sums in shared memory at the end.  Both operands go from global memory straight
// into MMA fragments: the contraction may run over k in any order as long as both operands use the same one,
// so a lane loads 16 consecutive levels of its row (and of its token) and they serve two m16n8k32 products.
// No staging and no barrier in the loop: up to UNROLL x 3 16-byte loads per lane are in flight.
constexpr int ROWS_WARPS = 8;
constexpr int ROWS_MAX_TOKENS = 16;
__device__ __forceinline__ void mma_m16n8k32_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <typename X>
__device__ __forceinline__ void round_tokens(const I8Params& p, const X* __restrict__ act, int64_t ld_act, int8_t* levels, float* scales, int* scratch) {
    constexpr int V = 16 / sizeof(X);
    const int chunks = (int)(p.K / V), warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    unsigned* tops = reinterpret_cast<unsigned*>(scratch);  // [tokens][warps]
    for (int m = 0; m < p.M; ++m) {
        unsigned top = 0;
        for (int c = threadIdx.x; c < chunks; c += 32 * ROWS_WARPS) {
            float v[V];
            unpack16<X>(__ldg(reinterpret_cast<const uint4*>(act + m * ld_act) + c), v);
#pragma unroll
            for (int e = 0; e < V; ++e) top = max(top, __float_as_uint(v[e]) & 0x7fffffffu);
        }
        top = __reduce_max_sync(0xffffffffu, top);
        if (lane == 0) tops[m * ROWS_WARPS + warp] = top;
    }
    __syncthreads();
    for (int m = 0; m < p.M; ++m) {
        unsigned top = 0;
#pragma unroll
        for (int w = 0; w < ROWS_WARPS; ++w) top = max(top, tops[m * ROWS_WARPS + w]);
        const RowScale rs(top);
        if (threadIdx.x == 0) scales[m] = rs.scale;
        for (int c = threadIdx.x; c < chunks; c += 32 * ROWS_WARPS) {
            rs.store<X>(levels + m * (p.K + 16) + c * V, __ldg(reinterpret_cast<const uint4*>(act + m * ld_act) + c));
        }
    }
    __syncthreads();
}

// X is int8_t (levels and scales are there), or the activations' type: then every block rounds the tokens itself first
// (quantize_rows's arithmetic, level for level), which saves a launch where the tokens are few and short.  The
// first weights are already on their way meanwhile.
template <typename T, typename X, int NT>  // NT groups of eight tokens
__global__ void __launch_bounds__(32 * ROWS_WARPS) i8_rows_kernel(I8Params p, const X* __restrict__ act, int64_t ld_act) {
    constexpr bool FUSED = !std::is_same<X, int8_t>::value;
    extern __shared__ __align__(16) int8_t levels[];  // FUSED: [tokens][K + 16], rows shifted by 16 bytes
    __shared__ int red[ROWS_WARPS][16][8 * NT + 1];
    __shared__ float scales[FUSED ? 8 : 1];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int64_t n0 = (int64_t)blockIdx.x * 16;
    const int8_t* w0 = p.w + min(n0 + g, p.N - 1) * p.ldw + t * 16;       // rows behind the last are read as the last
    const int8_t* w1 = p.w + min(n0 + g + 8, p.N - 1) * p.ldw + t * 16;   // and not written
    const int8_t* x[NT];
    bool live[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        live[i] = i * 8 + g < p.M;
        if constexpr (FUSED) x[i] = levels + (live[i] ? i * 8 + g : 0) * (p.K + 16) + t * 16;
        else x[i] = p.x + (live[i] ? i * 8 + g : 0) * p.ldx + t * 16;
    }
    int acc[NT][4] = {};
    constexpr int UNROLL = 4;
    const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
    constexpr int STEP = ROWS_WARPS * 64 * UNROLL;
    uint4 a[2][UNROLL][2], b[UNROLL][NT];
    auto load_w = [&](uint4 (&w)[UNROLL][2], int k0) {
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const int k = k0 + u * ROWS_WARPS * 64;
            const bool in = k + t * 16 < (int)p.K;  // K is a multiple of 16
            w[u][0] = in ? __ldg(reinterpret_cast<const uint4*>(w0 + k)) : zero;
            w[u][1] = in ? __ldg(reinterpret_cast<const uint4*>(w1 + k)) : zero;
        }
    };
    auto multiply = [&](const uint4 (&w)[UNROLL][2], int k0) {
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const int k = k0 + u * ROWS_WARPS * 64;
            const bool in = k + t * 16 < (int)p.K;
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                if constexpr (FUSED) b[u][i] = in && live[i] ? *reinterpret_cast<const uint4*>(x[i] + k) : zero;
                else b[u][i] = in && live[i] ? __ldg(reinterpret_cast<const uint4*>(x[i] + k)) : zero;
            }
        }
#pragma unroll
        for (int u = 0; u < UNROLL; ++u)
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                mma_m16n8k32_s8(acc[i], w[u][0].x, w[u][1].x, w[u][0].y, w[u][1].y, b[u][i].x, b[u][i].y);
                mma_m16n8k32_s8(acc[i], w[u][0].z, w[u][1].z, w[u][0].w, w[u][1].w, b[u][i].z, b[u][i].w);
            }
    };
    int k0 = warp * 64;
    load_w(a[0], k0);
    wait_for_quantizer();  // the weights do not depend on it
    if constexpr (FUSED) round_tokens<X>(p, act, ld_act, levels, scales, &red[0][0][0]);
    for (; k0 < (int)p.K; k0 += 2 * STEP) {  // the next piece of the weights is on its way while one is multiplied
        load_w(a[1], k0 + STEP);
        multiply(a[0], k0);
        load_w(a[0], k0 + 2 * STEP);
        multiply(a[1], k0 + STEP);
    }
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        red[warp][g][i * 8 + 2 * t] = acc[i][0];
        red[warp][g][i * 8 + 2 * t + 1] = acc[i][1];
        red[warp][g + 8][i * 8 + 2 * t] = acc[i][2];
        red[warp][g + 8][i * 8 + 2 * t + 1] = acc[i][3];
    }
    __syncthreads();
    const int r = threadIdx.x & 15, m = threadIdx.x >> 4;  // 16 tokens in one go
    if (m < 8 * NT && m < p.M && n0 + r < p.N) {
        int sum = 0;
#pragma unroll
        for (int v = 0; v < ROWS_WARPS; ++v) sum += red[v][r][m];
        static_cast<T*>(p.y)[m * p.ldy + n0 + r] = from_f32<T>(i8_scaled(sum, FUSED ? scales[FUSED ? m : 0] : p.x_scale[m], p.w_scale[n0 + r]));
    }
}

template <typename T>
cudaError_t launch_rows(const I8Params& p, cudaStream_t s) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3((unsigned)((p.N + 15) / 16));
    cfg.blockDim = dim3(32 * ROWS_WARPS);
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = p.behind_quantizer ? 1 : 0;
    const int8_t* none = nullptr;
    if (p.M <= 8) return cudaLaunchKernelEx(&cfg, i8_rows_kernel<T, int8_t, 1>, p, none, (int64_t)0);
    return cudaLaunchKernelEx(&cfg, i8_rows_kernel<T, int8_t, 2>, p, none, (int64_t)0);
}

template <typename T, typename X>
int launch_fused(const I8Params& p, const void* act, int64_t ld_act, cudaStream_t s) {
    i8_rows_kernel<T, X, 1><<<(unsigned)((p.N + 15) / 16), 32 * ROWS_WARPS, (size_t)(p.M * (p.K + 16)), s>>>(p, static_cast<const X*>(act), ld_act);
    CMFC_CUDA(cudaGetLastError());
    return OK;
}
template <typename T>
int launch_fused_x(const I8Params& p, const void* act, int elem, int64_t ld_act, cudaStream_t s) {
    if (elem == ET_F32) return launch_fused<T, float>(p, act, ld_act, s);
    if (elem == ET_F16) return launch_fused<T, __half>(p, act, ld_act, s);
    return launch_fused<T, __nv_bfloat16>(p, act, ld_act, s);
}

template <typename T>
void launch_any(const I8Params& p, cudaStream_t s) {
    i8_any_kernel<T><<<dim3((unsigned)((p.N + GT - 1) / GT), (unsigned)((p.M + GT - 1) / GT)), 256, 0, s>>>(p);
}

}  // namespace

// Rounding inside the product: every block of 16 weight rows does it again, from L2, for all tokens.
// One token of 2304 through 2304 rows: 4.4 us, two launches 5.8; through 9216 rows 10.3 and 8.9; eight tokens 16.3 and 6.4.
bool i8_fused_supported(const I8Params& p, const void* act, int elem, int64_t ld_act) {
    return p.M <= 8 && p.M * p.K <= 4608 && p.N <= 4608 && p.K % 16 == 0 && !((reinterpret_cast<uintptr_t>(act) | reinterpret_cast<uintptr_t>(p.w)) & 15) && p.ldw % 16 == 0 &&
           (ld_act * (int64_t)elem_bytes(elem)) % 16 == 0;
}
int launch_i8_fused(const I8Params& p, const void* act, int elem, int64_t ld_act, cudaStream_t s) {
    if (p.out_elem == ET_F32) return launch_fused_x<float>(p, act, elem, ld_act, s);
    if (p.out_elem == ET_F16) return launch_fused_x<__half>(p, act, elem, ld_act, s);
    return launch_fused_x<__nv_bfloat16>(p, act, elem, ld_act, s);
}

int launch_i8_matmat(const I8Params& p, int num_sms, cudaStream_t s) {
    const bool aligned = !((reinterpret_cast<uintptr_t>(p.x) | reinterpret_cast<uintptr_t>(p.w)) & 15) && p.ldx % 16 == 0 && p.ldw % 16 == 0;
    // us here / on CTA pairs (rows x columns of the weights): 1 token 2304 x 2304 2.9 / 7.2, 18432 x 2304 11.1 / 11.9; 8 tokens
    // 2304 x 9216 9.1 / 11.3, 18432 x 2304 11.9 / 11.9; 16 tokens 4096 x 4096 6.9 / 9.9, 2304 x 9216 11.7 / 11.3, 18432 x 2304 15.8 / 12.1
    if (aligned && p.M <= ROWS_MAX_TOKENS && p.K % 16 == 0 && (p.M <= 8 || p.N * p.K <= (int64_t)20 << 20)) {
        CMFC_CUDA(p.out_elem == ET_F32 ? launch_rows<float>(p, s) : p.out_elem == ET_F16 ? launch_rows<__half>(p, s) : launch_rows<__nv_bfloat16>(p, s));
        return OK;
    }
    if (aligned) return launch_i8_pair(p, num_sms, s);
    if ((p.M + GT - 1) / GT > 65535) return fail(ERR_UNSUPPORTED, "i8_matmat: too many tokens for rows that are not 16-byte aligned");
    if (p.out_elem == ET_F32) launch_any<float>(p, s);
    else if (p.out_elem == ET_F16) launch_any<__half>(p, s);
    else launch_any<__nv_bfloat16>(p, s);
    CMFC_CUDA(cudaGetLastError());
    return OK;
}

}  // namespace cmfc
