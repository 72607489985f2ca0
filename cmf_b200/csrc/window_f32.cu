// Windowed causal attention on f32 tensors with 16-byte aligned rows: prompts and chunks.  The definition is in
// window_attention.cu; rows, tiles and the softmax are the ones there.
//
// Bound: the FMA pipe (4 hd FMA per visible pair).  A block owns 64 rows of one key head.  Scores are 4 x 4 register tiles,
// outputs 4 x hd / 16, both fed from shared memory: 8 16-byte loads for 64 FMA of a thread.  K and V tiles of 64 keys
// take turns in two buffers filled by cp.async: V(j) is on its way while S(j) is computed, K(j + 1) while P V(j) is.
#include <atomic>

#include "window_attention.cuh"

namespace cmfc {
namespace {

constexpr int BM = 64, BN = 64, THREADS = 256;

template <int HDP>
constexpr int smem_floats() { return BM * (HDP + 4) + 2 * BN * (HDP + 4) + BM * (BN + 4); }

// 16 bytes, or zeros
__device__ __forceinline__ void copy16(float* dst, const float* src, bool live) {
    const int n = live ? 16 : 0;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(n) : "memory");
}

template <int HDP>
__global__ void __launch_bounds__(THREADS) window_f32_kernel(const __grid_constant__ WindowAttnParams p) {
    extern __shared__ float sm[];
    constexpr int LD = HDP + 4;  // 16-byte rows whose banks shift by four
    float* Qs = sm;                 // [BM][LD]
    float* buf = Qs + BM * LD;      // two tiles [BN][LD]: K(j) in the first, V(j) in the second
    float* Ps = buf + 2 * BN * LD;  // [BM][BN + 4]
    const int group = p.nh / p.nkv, kvh = blockIdx.x % p.nkv;
    SeqTile st;
    if (!find_tile(p, (gridDim.x - 1 - blockIdx.x) / p.nkv, BM, group, st)) return;
    const int rows = st.q_len * group, r0 = st.tile * BM;
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const float* qp = static_cast<const float*>(p.q.p);
    const float* kp = static_cast<const float*>(p.k.p) + st.k0 * p.k.row + (int64_t)kvh * p.k.head;
    const float* vp = static_cast<const float*>(p.v.p) + st.k0 * p.v.row + (int64_t)kvh * p.v.head;
    const int first_i = r0 / group, last_i = min(rows - 1, r0 + BM - 1) / group;
    const KeyTiles kt = key_tiles(p, st, first_i, last_i, BN);
    // rows behind the last key that the block sees are zeros: they may hold anything
    const int end = min(st.k_len, st.k_len - st.q_len + last_i + 1);
    auto fetch = [&](float* dst, const float* src, int64_t pitch, int j0) {
        for (int t = tid; t < BN * (HDP / 4); t += THREADS) {
            const int j = t / (HDP / 4), d = t % (HDP / 4) * 4;
            const bool live = j0 + j < end && d < p.hd;
            copy16(dst + j * LD + d, live ? src + (int64_t)(j0 + j) * pitch + d : src, live);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    for (int t = tid; t < BM * (HDP / 4); t += THREADS) {
        const int r = t / (HDP / 4), d = t % (HDP / 4) * 4, row = r0 + r;
        const bool live = row < rows && d < p.hd;
        copy16(Qs + r * LD + d, live ? qp + (st.q0 + row / group) * p.q.row + (int64_t)(kvh * group + row % group) * p.q.head + d : qp, live);
    }
    if (kt.count) fetch(buf, kp, p.k.row, kt.at(0) * BN);
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
    float *Ks = buf, *Vs = buf + BN * LD;
    for (int it = 0; it < kt.count; ++it) {
        const int j0 = kt.at(it) * BN;
        fetch(Vs, vp, p.v.row, j0);
        asm volatile("cp.async.wait_group 1;" ::: "memory");  // K(it), and Q
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
                for (int b = 0; b < 4; ++b) {
                    s[a][b] = fmaf(qv[a].x, kv[b].x, s[a][b]);
                    s[a][b] = fmaf(qv[a].y, kv[b].y, s[a][b]);
                    s[a][b] = fmaf(qv[a].z, kv[b].z, s[a][b]);
                    s[a][b] = fmaf(qv[a].w, kv[b].w, s[a][b]);
                }
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
        __syncthreads();  // everybody is done with K(it)
        if (it + 1 < kt.count) {
            fetch(Ks, kp, p.k.row, kt.at(it + 1) * BN);
            asm volatile("cp.async.wait_group 1;" ::: "memory");
        } else {
            asm volatile("cp.async.wait_group 0;" ::: "memory");
        }
        __syncthreads();  // V(it) is there for everybody
#pragma unroll 2
        for (int j = 0; j < BN; j += 4) {
            float4 pw[4];
#pragma unroll
            for (int a = 0; a < 4; ++a) pw[a] = *reinterpret_cast<const float4*>(Ps + (ty * 4 + a) * (BN + 4) + j);
#pragma unroll
            for (int jj = 0; jj < 4; ++jj)
#pragma unroll
                for (int c = 0; c < HDP / 64; ++c) {
                    const float4 v = *reinterpret_cast<const float4*>(Vs + (j + jj) * LD + c * 64 + tx * 4);
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
        __syncthreads();  // everybody is done with V(it): its buffer takes V(it + 1)
    }
    unsigned redo = 0;
#pragma unroll
    for (int a = 0; a < 4; ++a) {
        const int row = r0 + ty * 4 + a;
        const bool any = pos[a] >= 0;  // from position 0 on a query sees at least its own key
        const float inv = any ? 1.0f / l[a] : 0.0f;
        bool fine = true;
        float* dst = static_cast<float*>(const_cast<void*>(p.out.p)) + (st.q0 + row / group) * p.out.row + (int64_t)(kvh * group + row % group) * p.out.head;
#pragma unroll
        for (int c = 0; c < HDP / 16; ++c) {
            const int d = (c >> 2) * 64 + tx * 4 + (c & 3);
            const float o = any ? acc[a][c] * inv : 0.0f;
            fine = fine && isfinite(o);
            if (row < rows && d < p.hd) dst[d] = o;
        }
        const unsigned bad = __ballot_sync(0xffffffffu, row < rows && !fine);
        if (bad & 0xffffu) redo |= 1u << a;   // rows ty * 4 + a of the two half warps
        if (bad >> 16) redo |= 16u << a;
    }
    // a non-finite value may come from a key that only other rows of the tile see (0 * inf): such rows are computed
    // again from the keys they see
    __syncwarp();
    for (; redo; redo &= redo - 1) redo_row<float>(p, st, kvh, r0 + (ty & ~1) * 4 + __ffs(redo) - 1);
}

template <int HDP>
int launch_hdp(const WindowAttnParams& p, cudaStream_t s) {
    static std::atomic<bool> configured[64];
    int dev = 0;
    CMFC_CUDA(cudaGetDevice(&dev));
    constexpr int SMEM = smem_floats<HDP>() * 4;
    static_assert(SMEM <= 232448, "tiles fit shared memory");
    if (!configured[dev & 63]) {
        CMFC_CUDA(cudaFuncSetAttribute(window_f32_kernel<HDP>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM));
        configured[dev & 63] = true;
    }
    window_f32_kernel<HDP><<<(unsigned)(max_tiles(p, BM) * p.nkv), THREADS, SMEM, s>>>(p);
    CMFC_CUDA(cudaGetLastError());
    return OK;
}

}  // namespace

bool window_f32_supported(const WindowAttnParams& p, int elem) {
    auto fits = [](const HeadView& v) { return !(reinterpret_cast<uintptr_t>(v.p) & 15) && v.row % 4 == 0 && v.head % 4 == 0; };
    return elem == ET_F32 && p.hd % 4 == 0 && max_tiles(p, BM) * p.nkv < ((int64_t)1 << 31) && fits(p.q) && fits(p.k) && fits(p.v);
}

int launch_window_f32(const WindowAttnParams& p, cudaStream_t s) {
    if (p.hd <= 64) return launch_hdp<64>(p, s);
    if (p.hd <= 128) return launch_hdp<128>(p, s);
    return launch_hdp<256>(p, s);
}

}  // namespace cmfc
