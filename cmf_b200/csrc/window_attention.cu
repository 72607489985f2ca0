// Causal attention with a sliding window and first tokens that stay visible, over packed sequences or
// caches, any head size up to 256, any stride, f32 / f16 / bf16: the form for calls whose rows are not 16-byte
// aligned.  The others go to window_prefill.cu, window_tokens.cu and window_f32.cu.
//
//   query i of a sequence with Lq queries and Lk keys stands at position p = Lk - Lq + i and sees key j
//   when j <= p and (p - j < window or j < sinks);   s = scale q.k (soft cap: s = cap tanh(s / cap));
//   out = sum_j exp(s_j - max) v_j / sum_j exp(s_j - max), and 0 for a query that sees no key.
//
// One block owns 64 rows of one key head: a row is (query, head of the group), so the heads that share
// keys share every key tile.  One pass over the visible key tiles of 64 with the running maximum and sum of
// the softmax; scores and outputs are 4 x 4 and 4 x hd / 16 register tiles per thread, all in f32.
// Bound: the FMA pipe, fed from shared memory.
#include <atomic>

#include "window_attention.cuh"

namespace cmfc {
namespace {

constexpr int BM = 64, BN = 64, THREADS = 256;

template <int HDP>
constexpr int any_smem_floats() { return BM * (HDP + 4) + BN * (HDP + 4) + BN * HDP + BM * (BN + 4); }

template <typename T, int HDP>
__global__ void __launch_bounds__(THREADS) window_any_kernel(const __grid_constant__ WindowAttnParams p) {
    extern __shared__ float sm[];
    constexpr int LD = HDP + 4;  // 16-byte rows whose banks shift by four
    float* Qs = sm;                // [BM][LD]
    float* Ks = Qs + BM * LD;      // [BN][LD]
    float* Vs = Ks + BN * LD;      // [BN][HDP]
    float* Ps = Vs + BN * HDP;     // [BM][BN + 4]
    const int group = p.nh / p.nkv, kvh = blockIdx.y;
    SeqTile st;
    if (!find_tile(p, blockIdx.x, BM, group, st)) return;
    const int rows = st.q_len * group;       // of this sequence and key head
    const int r0 = st.tile * BM;
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const T* qp = static_cast<const T*>(p.q.p);
    const T* kp = static_cast<const T*>(p.k.p) + (int64_t)kvh * p.k.head;
    const T* vp = static_cast<const T*>(p.v.p) + (int64_t)kvh * p.v.head;
    for (int t = tid; t < BM * HDP; t += THREADS) {
        const int r = t / HDP, d = t % HDP, row = r0 + r;
        float x = 0.0f;
        if (row < rows && d < p.hd)
            x = to_f32(qp[(st.q0 + row / group) * p.q.row + (int64_t)(kvh * group + row % group) * p.q.head + d]);
        Qs[r * LD + d] = x;
    }
    const int first_i = r0 / group, last_i = min(rows - 1, r0 + BM - 1) / group;
    const KeyTiles kt = key_tiles(p, st, first_i, last_i, BN);
    float m[4], l[4], acc[4][HDP / 16];
    int pos[4];
#pragma unroll
    for (int a = 0; a < 4; ++a) {
        m[a] = -INFINITY;
        l[a] = 0.0f;
        const int row = r0 + ty * 4 + a;
        pos[a] = row < rows ? st.k_len - st.q_len + row / group : -1;
#pragma unroll
        for (int c = 0; c < HDP / 16; ++c) acc[a][c] = 0.0f;
    }
    for (int it = 0; it < kt.count; ++it) {
        const int j0 = kt.at(it) * BN;
        __syncthreads();
        for (int t = tid; t < BN * HDP; t += THREADS) {
            const int j = t / HDP, d = t % HDP;
            float kx = 0.0f, vx = 0.0f;
            if (j0 + j < st.k_len && d < p.hd) {
                kx = to_f32(kp[(st.k0 + j0 + j) * p.k.row + d]);
                vx = to_f32(vp[(st.k0 + j0 + j) * p.v.row + d]);
            }
            Ks[j * LD + d] = kx;
            Vs[j * HDP + d] = vx;
        }
        __syncthreads();
        float s[4][4];
#pragma unroll
        for (int a = 0; a < 4; ++a)
#pragma unroll
            for (int b = 0; b < 4; ++b) s[a][b] = 0.0f;
#pragma unroll 4
        for (int d = 0; d < HDP; d += 4) {
            float4 qv[4], kv[4];
#pragma unroll
            for (int a = 0; a < 4; ++a) qv[a] = *reinterpret_cast<const float4*>(Qs + (ty * 4 + a) * LD + d);
#pragma unroll
            for (int b = 0; b < 4; ++b) kv[b] = *reinterpret_cast<const float4*>(Ks + (tx + 16 * b) * LD + d);
#pragma unroll
            for (int a = 0; a < 4; ++a)
#pragma unroll
                for (int b = 0; b < 4; ++b)
                    s[a][b] = fmaf(qv[a].x, kv[b].x, fmaf(qv[a].y, kv[b].y, fmaf(qv[a].z, kv[b].z, fmaf(qv[a].w, kv[b].w, s[a][b]))));
        }
#pragma unroll
        for (int a = 0; a < 4; ++a) {
            float top = -INFINITY;
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const int j = j0 + tx + 16 * b;
                s[a][b] = sees(p, pos[a], j) ? score(s[a][b], p.scale, p.softcap) : -INFINITY;
                top = fmaxf(top, s[a][b]);
            }
#pragma unroll
            for (int o = 8; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            const float mn = fmaxf(m[a], top), ref = mn == -INFINITY ? 0.0f : mn;
            const float alpha = expf(m[a] - ref);
            m[a] = mn;
            float sum = 0.0f;
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const float e = expf(s[a][b] - ref);
                sum += e;
                Ps[(ty * 4 + a) * (BN + 4) + tx + 16 * b] = e;
            }
#pragma unroll
            for (int o = 8; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            l[a] = l[a] * alpha + sum;
#pragma unroll
            for (int c = 0; c < HDP / 16; ++c) acc[a][c] *= alpha;
        }
        __syncwarp();  // a row's weights are written and read by the same half warp
#pragma unroll 2
        for (int j = 0; j < BN; j += 4) {
            float4 pw[4];
#pragma unroll
            for (int a = 0; a < 4; ++a) pw[a] = *reinterpret_cast<const float4*>(Ps + (ty * 4 + a) * (BN + 4) + j);
#pragma unroll
            for (int jj = 0; jj < 4; ++jj)
#pragma unroll
                for (int c = 0; c < HDP / 64; ++c) {
                    const float4 v = *reinterpret_cast<const float4*>(Vs + (j + jj) * HDP + c * 64 + tx * 4);
#pragma unroll
                    for (int a = 0; a < 4; ++a) {
                        const float w = jj == 0 ? pw[a].x : jj == 1 ? pw[a].y : jj == 2 ? pw[a].z : pw[a].w;
                        acc[a][c * 4] = fmaf(w, v.x, acc[a][c * 4]);
                        acc[a][c * 4 + 1] = fmaf(w, v.y, acc[a][c * 4 + 1]);
                        acc[a][c * 4 + 2] = fmaf(w, v.z, acc[a][c * 4 + 2]);
                        acc[a][c * 4 + 3] = fmaf(w, v.w, acc[a][c * 4 + 3]);
                    }
                }
        }
    }
    unsigned redo = 0;
#pragma unroll
    for (int a = 0; a < 4; ++a) {
        const int row = r0 + ty * 4 + a;
        const bool any = pos[a] >= 0;  // from position 0 on a query sees at least its own key
        const float inv = any ? 1.0f / l[a] : 0.0f;
        bool fine = true;
        T* dst = static_cast<T*>(const_cast<void*>(p.out.p)) + (st.q0 + row / group) * p.out.row +
                 (int64_t)(kvh * group + row % group) * p.out.head;
#pragma unroll
        for (int c = 0; c < HDP / 16; ++c) {
            const int d = (c >> 2) * 64 + tx * 4 + (c & 3);
            const float o = any ? acc[a][c] * inv : 0.0f;
            fine = fine && isfinite(o);
            if (row < rows && d < p.hd) dst[d] = from_f32<T>(o);
        }
        const unsigned bad = __ballot_sync(0xffffffffu, row < rows && !fine);
        // rows ty * 4 + a of the two half warps
        if (bad & 0xffffu) redo |= 1u << a;
        if (bad >> 16) redo |= 16u << a;
    }
    // a non-finite value may come from a key that only other rows of the tile see (0 * inf): such rows
    // are computed again from the keys they see
    __syncwarp();
    for (; redo; redo &= redo - 1) {
        const int b = __ffs(redo) - 1;
        const int row = r0 + (ty & ~1) * 4 + b;  // b = half * 4 + a, the half warps are ty and ty + 1
        redo_row<T>(p, st, kvh, row);
    }
}

template <typename T, int HDP>
int launch_any_hd(const WindowAttnParams& p, cudaStream_t s) {
    static std::atomic<bool> configured[64];
    int dev = 0;
    CMFC_CUDA(cudaGetDevice(&dev));
    constexpr int SMEM = any_smem_floats<HDP>() * 4;
    if (!configured[dev & 63]) {
        CMFC_CUDA(cudaFuncSetAttribute(window_any_kernel<T, HDP>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM));
        configured[dev & 63] = true;
    }
    window_any_kernel<T, HDP><<<dim3((unsigned)max_tiles(p, BM), p.nkv), THREADS, SMEM, s>>>(p);
    CMFC_CUDA(cudaGetLastError());
    return OK;
}
template <typename T>
int launch_any(const WindowAttnParams& p, cudaStream_t s) {
    if (p.hd <= 64) return launch_any_hd<T, 64>(p, s);
    if (p.hd <= 128) return launch_any_hd<T, 128>(p, s);
    return launch_any_hd<T, 256>(p, s);
}

}  // namespace

int launch_window_any(const WindowAttnParams& p, int elem, cudaStream_t s) {
    if (elem == ET_F32) return launch_any<float>(p, s);
    if (elem == ET_F16) return launch_any<__half>(p, s);
    return launch_any<__nv_bfloat16>(p, s);
}

int launch_window_attention(const WindowAttnParams& p, int elem, int num_sms, cudaStream_t s) {
    if (window_few_rows(p, num_sms) && window_tokens_supported(p, elem)) return launch_window_tokens(p, elem, num_sms, s);
    if (window_prefill_supported(p, elem)) return launch_window_prefill(p, elem, s);
    if (window_f32_supported(p, elem)) return launch_window_f32(p, num_sms, s);
    return launch_window_any(p, elem, s);
}

}  // namespace cmfc
