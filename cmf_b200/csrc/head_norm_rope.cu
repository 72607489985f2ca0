// Norms of query and key heads with the position rotation in the same pass, and the row quantizer of
// the 8-bit products: bandwidth-bound row kernels on the caller's device tensors.
//
// Per (token, head): y = x / sqrt(mean(x^2) + eps) * w, then every pair (a, b) of the first `rot`
// dims becomes (a c - b s, a s + b c) with c, s of the token's position; the other dims pass through.
// Pairs are neighbours (2i, 2i + 1) or halves (i, i + rot / 2).  Statistics and arithmetic are f32,
// the result is rounded once to the tensors' type.
//
// Bound: memory.  A head is read once and written once; the norm's gain and the position's cos / sin
// are read once per (token, up to HEADS_PER_ITEM heads) and stay in registers.  A lane owns two
// 16-byte chunks of a head that hold both members of its pairs (neighbouring chunks, or the same
// chunk of either half), so the rotation needs no exchange between lanes; a head takes a group of
// 4 to 32 lanes and a warp works on 32 / group items.  Measured, 8704 tokens x 32 heads of 96: f32 37 to 40 us (5.6 TB/s, 0.85 of
// a copy's rate); bf16 27 us (4.1 TB/s), where the conversions and the reduction of 16 values a lane and head hold up the loads; one
// token 2.2 us.  Items by a 2-D grid, a loop over tokens and a register cap were each slower.
#include "i8_gemm.cuh"

namespace cmfc {
namespace {

// heads in flight of a lane; 2 / 3 / 8 instead: 17.7 / 18.3 / 24.4 us against 16.5 (5531 tokens, 8 + 4 heads of 256, f16)
constexpr int HEADS_PER_ITEM = 4;

// N (a multiple of 4) values from a 16-byte aligned place
template <int N>
__device__ __forceinline__ void load_f32(const float* p, float* o) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
        const float4 v = __ldg(reinterpret_cast<const float4*>(p + i));
        o[i] = v.x;
        o[i + 1] = v.y;
        o[i + 2] = v.z;
        o[i + 3] = v.w;
    }
}

template <typename T, bool HALF, int LANES>
__global__ void __launch_bounds__(128) norm_rope_kernel(NormRopeParams p, int heads_per_item, int q_items, int items_per_token) {
    constexpr int V = 16 / sizeof(T);  // elements of a 16-byte chunk
    const int u = threadIdx.x % LANES;                 // this lane's unit: two chunks, V pairs
    const int units = p.hd / (2 * V), rot_units = p.rot / (2 * V);
    const uint32_t item = blockIdx.x * (128 / LANES) + threadIdx.x / LANES;  // fewer than 2^31
    const bool active = u < units && item < (uint32_t)p.n * items_per_token;
    const int64_t t = active ? item / (uint32_t)items_per_token : 0;
    const int part = active ? (int)(item % (uint32_t)items_per_token) : 0;
    const bool is_q = part < q_items;
    const int head0 = (is_q ? part : part - q_items) * heads_per_item;
    const int heads = active ? min(heads_per_item, (is_q ? p.nh : p.nkv) - head0) : 0;
    const HeadView in = is_q ? p.q : p.k, out = is_q ? p.q_out : p.k_out;
    const bool rotated = u < rot_units;
    const int d0 = HALF && rotated ? u * V : u * 2 * V;
    const int d1 = HALF && rotated ? p.rot / 2 + u * V : d0 + V;
    float w[2 * V], cs[V], sn[V];
    bool bad = false;
    if (active) {
        const float* g = is_q ? p.norm_q : p.norm_k;
        load_f32<V>(g + d0, w);
        load_f32<V>(g + d1, w + V);
        const int64_t pos = p.positions ? (p.pos64 ? static_cast<const int64_t*>(p.positions)[t]
                                                   : (int64_t)static_cast<const int32_t*>(p.positions)[t])
                                        : t;
        bad = pos < 0 || pos >= p.table_rows;
        if (rotated && !bad) {
            load_f32<V>(p.cos_t + pos * (p.rot / 2) + u * V, cs);
            load_f32<V>(p.sin_t + pos * (p.rot / 2) + u * V, sn);
        }
    }
    const T* src = static_cast<const T*>(in.p) + t * in.row + (int64_t)head0 * in.head;
    T* dst = static_cast<T*>(const_cast<void*>(out.p)) + t * out.row + (int64_t)head0 * out.head;
    uint4 raw[HEADS_PER_ITEM][2];
#pragma unroll
    for (int h = 0; h < HEADS_PER_ITEM; ++h)
        if (h < heads) {
            raw[h][0] = *reinterpret_cast<const uint4*>(src + h * in.head + d0);
            raw[h][1] = *reinterpret_cast<const uint4*>(src + h * in.head + d1);
        }
#pragma unroll
    for (int h = 0; h < HEADS_PER_ITEM; ++h) {
        // every lane of the warp takes part in the group's sum, with nothing to add where it has no head
        if (h >= heads_per_item) break;
        float x[2 * V], ss = 0.0f;
        if (h < heads) {
            unpack16<T>(raw[h][0], x);
            unpack16<T>(raw[h][1], x + V);
#pragma unroll
            for (int i = 0; i < 2 * V; ++i) ss = fmaf(x[i], x[i], ss);
        }
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        if (h >= heads) continue;
        const float inv = bad ? __int_as_float(0x7fc00000) : 1.0f / sqrtf(ss / (float)p.hd + p.eps);
#pragma unroll
        for (int i = 0; i < 2 * V; ++i) x[i] = (x[i] * inv) * w[i];
        if (rotated && !bad) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                float& a = HALF ? x[i] : x[2 * i];
                float& b = HALF ? x[V + i] : x[2 * i + 1];
                const float ra = fmaf(a, cs[i], -(b * sn[i])), rb = fmaf(a, sn[i], b * cs[i]);
                a = ra;
                b = rb;
            }
        }
        __stcs(reinterpret_cast<uint4*>(dst + h * out.head + d0), pack16<T>(x));
        __stcs(reinterpret_cast<uint4*>(dst + h * out.head + d1), pack16<T>(x + V));
    }
}

// Any head size, rotation, stride and alignment: one warp per (token, head), a pair per lane.
// Lane i reads and writes the same pairs, so an output that is the input itself is fine here too.
template <typename T, bool HALF>
__global__ void __launch_bounds__(128) norm_rope_any_kernel(NormRopeParams p) {
    const int lane = threadIdx.x & 31;
    const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int all = p.nh + p.nkv;
    if (item >= p.n * all) return;
    const int64_t t = item / all;
    const int hh = (int)(item % all);
    const bool is_q = hh < p.nh;
    const int h = is_q ? hh : hh - p.nh;
    const HeadView in = is_q ? p.q : p.k, out = is_q ? p.q_out : p.k_out;
    const float* g = is_q ? p.norm_q : p.norm_k;
    const T* src = static_cast<const T*>(in.p) + t * in.row + (int64_t)h * in.head;
    T* dst = static_cast<T*>(const_cast<void*>(out.p)) + t * out.row + (int64_t)h * out.head;
    float ss = 0.0f;
    for (int d = lane; d < p.hd; d += 32) {
        const float x = to_f32(src[d]);
        ss = fmaf(x, x, ss);
    }
    ss = warp_sum(ss);
    const int64_t pos = p.positions ? (p.pos64 ? static_cast<const int64_t*>(p.positions)[t]
                                               : (int64_t)static_cast<const int32_t*>(p.positions)[t])
                                    : t;
    const bool bad = pos < 0 || pos >= p.table_rows;
    const float inv = bad ? __int_as_float(0x7fc00000) : 1.0f / sqrtf(ss / (float)p.hd + p.eps);
    __syncwarp();  // the sums have read what the loops below overwrite when the output is the input
    const int half = p.rot / 2;
    for (int i = lane; i < half; i += 32) {
        const int da = HALF ? i : 2 * i, db = HALF ? i + half : 2 * i + 1;
        const float a = (to_f32(src[da]) * inv) * g[da], b = (to_f32(src[db]) * inv) * g[db];
        const float c = bad ? 1.0f : p.cos_t[pos * half + i], s = bad ? 0.0f : p.sin_t[pos * half + i];
        dst[da] = from_f32<T>(fmaf(a, c, -(b * s)));
        dst[db] = from_f32<T>(fmaf(a, s, b * c));
    }
    for (int d = p.rot + lane; d < p.hd; d += 32) dst[d] = from_f32<T>((to_f32(src[d]) * inv) * g[d]);
}

template <typename T, bool HALF, int LANES>
void norm_rope_lanes(const NormRopeParams& p, cudaStream_t s) {
    // few values: a head per lane group, so that the heads spread over the SMs; many: four heads share the gain and the
    // rotation that a group holds in registers.  us, one / four (heads of 96, 32 of them, bf16): 1 token 2.2 / 3.1, 300
    // tokens 3.3 / 3.9, 512 tokens 4.6 / 4.0, 8704 tokens 47 / 27; heads of 256, 12 of them: 300 tokens 3.2 / 3.6, 512
    // tokens 4.3 / 4.2, 1000 tokens 6.4 / 4.8
    const int per = p.n * (p.nh + p.nkv) * p.hd >= (int64_t)5 << 18 ? HEADS_PER_ITEM : 1;
    const int q_items = (p.nh + per - 1) / per, items = q_items + (p.nkv + per - 1) / per;
    const int64_t groups = p.n * items, per_block = 128 / LANES;
    norm_rope_kernel<T, HALF, LANES><<<(unsigned)((groups + per_block - 1) / per_block), 128, 0, s>>>(p, per, q_items, items);
}

template <typename T, bool HALF>
void norm_rope_typed(const NormRopeParams& p, cudaStream_t s) {
    constexpr int V = 16 / sizeof(T);
    auto fits = [](const HeadView& v) {
        return (reinterpret_cast<uintptr_t>(v.p) & 15) == 0 && v.row % V == 0 && v.head % V == 0;
    };
    auto aligned = [](const float* f) { return (reinterpret_cast<uintptr_t>(f) & 15) == 0; };
    const int units = p.hd / (2 * V);
    // the 16-byte form needs aligned rows, heads, gains and tables, and whole units of two chunks (rot / 2
    // is then a multiple of V, so every table row starts on 16 bytes too)
    if (p.hd % (2 * V) || p.rot % (2 * V) || units > 32 || !aligned(p.cos_t) || !aligned(p.sin_t) ||
        (p.nh && !aligned(p.norm_q)) || (p.nkv && !aligned(p.norm_k)) || (p.nh && !(fits(p.q) && fits(p.q_out))) ||
        (p.nkv && !(fits(p.k) && fits(p.k_out)))) {
        const int64_t items = p.n * (p.nh + p.nkv);
        norm_rope_any_kernel<T, HALF><<<(unsigned)((items + 3) / 4), 128, 0, s>>>(p);
    } else if (units <= 4) {
        norm_rope_lanes<T, HALF, 4>(p, s);
    } else if (units <= 8) {
        norm_rope_lanes<T, HALF, 8>(p, s);
    } else if (units <= 16) {
        norm_rope_lanes<T, HALF, 16>(p, s);
    } else {
        norm_rope_lanes<T, HALF, 32>(p, s);
    }
}

// ---------------- rows to 8 bits ----------------
// Bound: memory, the activations once and the levels once.  A row is read once into registers by a warp (short rows)
// or a block of 256 threads, CH 16-byte chunks a thread; what does not fit is read again, from L2.  Measured, bf16, 8704 rows:
// 2304 columns 13.9 us (4.3 TB/s), 9216 columns 48 us (5.0 TB/s); f32, 2304 columns 21 us (4.7 TB/s).
constexpr int QUANT_THREADS = 256;

// top of the bit patterns of |x| over a chunk, NaN above infinity above every number; 16-bit types two at a time
template <typename T>
__device__ __forceinline__ void chunk_top(const uint4& r, unsigned& top) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4) top = max(top, w[i] & 0x7fffffffu);
        else top = __vmaxu2(top, w[i] & 0x7fff7fffu);
    }
}
// ... and what chunk_top() left as the f32 bit pattern
template <typename T>
__device__ __forceinline__ unsigned top_f32(unsigned top) {
    if constexpr (sizeof(T) == 4) {
        return top;
    } else {
        top = max(top & 0xffffu, top >> 16);
        const unsigned short h = (unsigned short)top;
        return __float_as_uint(to_f32(*reinterpret_cast<const T*>(&h))) & 0x7fffffffu;
    }
}

// TPR threads per row (32 or 256), CH chunks kept by each
template <typename T, int TPR, int CH>
__global__ void __launch_bounds__(QUANT_THREADS) quantize_rows_kernel(const T* __restrict__ x, int64_t ldx, int rows, int chunks,
                                                                      int8_t* __restrict__ q, int64_t ldq, float* __restrict__ scale) {
    constexpr int V = 16 / (int)sizeof(T);
    let_product_start();
    const int64_t r = (int64_t)blockIdx.x * (QUANT_THREADS / TPR) + threadIdx.x / TPR;
    if (TPR == 32 && r >= rows) return;  // a whole warp
    const int t = threadIdx.x % TPR;
    const uint4* src = reinterpret_cast<const uint4*>(x + r * ldx);
    int8_t* dst = q + r * ldq;
    uint4 raw[CH];
    unsigned top = 0;
#pragma unroll
    for (int i = 0; i < CH; ++i) raw[i] = t + i * TPR < chunks ? __ldg(src + t + i * TPR) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
    for (int i = 0; i < CH; ++i) chunk_top<T>(raw[i], top);
    for (int c = t + CH * TPR; c < chunks; c += TPR) chunk_top<T>(__ldg(src + c), top);
    top = __reduce_max_sync(0xffffffffu, top_f32<T>(top));
    if constexpr (TPR > 32) {
        __shared__ unsigned red[TPR / 32];
        if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = top;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < TPR / 32; ++i) top = max(top, red[i]);
    }
    const RowScale rs(top);
    if (t == 0) scale[r] = rs.scale;
#pragma unroll
    for (int i = 0; i < CH; ++i)
        if (t + i * TPR < chunks) rs.store<T>(dst + (t + i * TPR) * V, raw[i]);
    for (int c = t + CH * TPR; c < chunks; c += TPR) rs.store<T>(dst + c * V, __ldg(src + c));
}

// rows of any length, pitch and alignment, value by value
template <typename T>
__global__ void __launch_bounds__(QUANT_THREADS) quantize_rows_any_kernel(const T* __restrict__ x, int64_t ldx, int cols, int8_t* __restrict__ q,
                                                                          int64_t ldq, float* __restrict__ scale) {
    let_product_start();
    const int64_t r = blockIdx.x;
    const T* src = x + r * ldx;
    int8_t* dst = q + r * ldq;
    __shared__ unsigned red[QUANT_THREADS / 32];
    unsigned top = 0;
    for (int c = threadIdx.x; c < cols; c += QUANT_THREADS) top = max(top, __float_as_uint(to_f32(src[c])) & 0x7fffffffu);
    top = __reduce_max_sync(0xffffffffu, top);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < QUANT_THREADS / 32; ++i) top = max(top, red[i]);
    const RowScale rs(top);
    if (threadIdx.x == 0) scale[r] = rs.scale;
    for (int c = threadIdx.x; c < cols; c += QUANT_THREADS) dst[c] = rs.level(to_f32(src[c]));
}

template <typename T>
void quantize_rows_typed(const void* x, int64_t rows, int64_t cols, int64_t ldx, int8_t* q, int64_t ldq, float* scale, cudaStream_t s) {
    constexpr int V = 16 / sizeof(T);
    const bool vec = !(reinterpret_cast<uintptr_t>(x) & 15) && !(reinterpret_cast<uintptr_t>(q) & 7) && cols % V == 0 && ldx % V == 0 && ldq % V == 0;
    const T* xt = static_cast<const T*>(x);
    const int chunks = (int)(cols / V);
    if (!vec) {
        quantize_rows_any_kernel<T><<<(unsigned)rows, QUANT_THREADS, 0, s>>>(xt, ldx, (int)cols, q, ldq, scale);
    } else if (chunks <= 32 * 16 && rows >= (chunks <= 32 * 4 ? 768 : 2560)) {
        // a warp per row keeps up to 16 chunks a lane in registers and needs no block barrier; with few rows a block per row
        // has more loads under way.  us, warp / block (bf16): 1024 columns 512 rows 2.4 / 2.2, 800 rows 2.4 / 2.5, 8704 rows 6.2
        // / 12.8; 2304 columns 800 rows 3.8 / 2.9, 1600 rows 4.8 / 4.2, 8704 rows 13.9 / 17.6
        const unsigned blocks = (unsigned)((rows + 7) / 8);
        if (chunks <= 32 * 4) quantize_rows_kernel<T, 32, 4><<<blocks, QUANT_THREADS, 0, s>>>(xt, ldx, (int)rows, chunks, q, ldq, scale);
        else if (chunks <= 32 * 8) quantize_rows_kernel<T, 32, 8><<<blocks, QUANT_THREADS, 0, s>>>(xt, ldx, (int)rows, chunks, q, ldq, scale);
        else if (chunks <= 32 * 12) quantize_rows_kernel<T, 32, 12><<<blocks, QUANT_THREADS, 0, s>>>(xt, ldx, (int)rows, chunks, q, ldq, scale);
        else quantize_rows_kernel<T, 32, 16><<<blocks, QUANT_THREADS, 0, s>>>(xt, ldx, (int)rows, chunks, q, ldq, scale);
    } else if (chunks <= 256 * 2) {
        quantize_rows_kernel<T, 256, 2><<<(unsigned)rows, QUANT_THREADS, 0, s>>>(xt, ldx, (int)rows, chunks, q, ldq, scale);
    } else if (chunks <= 256 * 4) {
        quantize_rows_kernel<T, 256, 4><<<(unsigned)rows, QUANT_THREADS, 0, s>>>(xt, ldx, (int)rows, chunks, q, ldq, scale);
    } else {
        quantize_rows_kernel<T, 256, 8><<<(unsigned)rows, QUANT_THREADS, 0, s>>>(xt, ldx, (int)rows, chunks, q, ldq, scale);
    }
}

}  // namespace

int launch_norm_rope(const NormRopeParams& p, int elem, bool half_split, cudaStream_t s) {
    if (elem == ET_F32) half_split ? norm_rope_typed<float, true>(p, s) : norm_rope_typed<float, false>(p, s);
    else if (elem == ET_F16) half_split ? norm_rope_typed<__half, true>(p, s) : norm_rope_typed<__half, false>(p, s);
    else half_split ? norm_rope_typed<__nv_bfloat16, true>(p, s) : norm_rope_typed<__nv_bfloat16, false>(p, s);
    CMFC_CUDA(cudaGetLastError());
    return OK;
}

int launch_quantize_rows(const void* x, int elem, int64_t rows, int64_t cols, int64_t ldx, int8_t* q, int64_t ldq, float* scale,
                         cudaStream_t s) {
    if (elem == ET_F32) quantize_rows_typed<float>(x, rows, cols, ldx, q, ldq, scale, s);
    else if (elem == ET_F16) quantize_rows_typed<__half>(x, rows, cols, ldx, q, ldq, scale, s);
    else quantize_rows_typed<__nv_bfloat16>(x, rows, cols, ldx, q, ldq, scale, s);
    CMFC_CUDA(cudaGetLastError());
    return OK;
}

}  // namespace cmfc
