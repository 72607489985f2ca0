// Windowed causal attention on f32 tensors with 16-byte aligned rows.  The definition is in window_attention.cu;
// rows, tiles and the softmax are the ones there.
//
// Prompts and chunks: bound by the FMA pipe (4 hd FMA per visible pair).  A block owns 64 rows of one key head.  Scores are 4 x
// 4 register tiles, outputs 4 x hd / 16, both fed from shared memory: 8 16-byte loads for 64 FMA of a thread.  K and V
// tiles of 64 keys have a buffer each, filled by cp.async: V(j) is on its way while S(j) is computed, K(j + 1) while P V(j)
// is.  Only K's rows are padded, so that two blocks of heads up to 128 share an SM (3000 tokens, 16 / 8 heads of 128: 985 us;
// one block 1130).  Larger tiles of a thread, which read less for each FMA (8 x 8 scores with the dims over four lanes, or 16 x
// 2 with half of the dims a warp), left too few warps to hide the reads: 1190 and 1092 us.
// Single tokens: bound by memory, the keys and values once.  A block owns 4 rows of one key head and a share of the key
// axis (see window_f32_tokens_kernel).
// Measured: prompts 27 to 37 TFLOP/s (FMA pipe half to two thirds busy; the rest is waiting for shared memory); 64 sequences x 4096
// keys x 4 heads of 256 495 us (4.3 TB/s), one sequence x 256 keys x 8 heads of 128 7.6 us.
#include <cooperative_groups.h>

#include <algorithm>
#include <atomic>

#include "window_attention.cuh"

namespace cmfc {
namespace {

namespace cg = cooperative_groups;

constexpr int BM = 64, BN = 64, THREADS = 256, MAX_SPLITS = 8;

template <int HDP>
constexpr int smem_floats() { return BM * HDP + BN * (HDP + 4) + BN * HDP + BM * BN; }

// 16 bytes, or zeros
__device__ __forceinline__ void copy16(float* dst, const float* src, bool live) {
    const int n = live ? 16 : 0;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(n) : "memory");
}

template <int HDP>
__global__ void __launch_bounds__(THREADS, HDP <= 128 ? 2 : 1) window_f32_kernel(const __grid_constant__ WindowAttnParams p) {
    constexpr int A = BM / 16;  // rows of a thread
    extern __shared__ float sm[];
    constexpr int LD = HDP + 4;  // 16-byte rows whose banks shift by four
    float* Qs = sm;              // [BM][HDP]
    float* Ks = Qs + BM * HDP;   // [BN][LD]
    float* Vs = Ks + BN * LD;    // [BN][HDP]
    float* Ps = Vs + BN * HDP;   // [BM][BN]
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
    auto fetch = [&](float* dst, int ld, const float* src, int64_t pitch, int j0) {
        for (int t = tid; t < BN * (HDP / 4); t += THREADS) {
            const int j = t / (HDP / 4), d = t % (HDP / 4) * 4;
            const bool live = j0 + j < end && d < p.hd;
            copy16(dst + j * ld + d, live ? src + (int64_t)(j0 + j) * pitch + d : src, live);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    for (int t = tid; t < BM * (HDP / 4); t += THREADS) {
        const int r = t / (HDP / 4), d = t % (HDP / 4) * 4, row = r0 + r;
        const bool live = row < rows && d < p.hd;
        copy16(Qs + r * HDP + d, live ? qp + (st.q0 + row / group) * p.q.row + (int64_t)(kvh * group + row % group) * p.q.head + d : qp, live);
    }
    if (kt.count) fetch(Ks, LD, kp, p.k.row, kt.at(0) * BN);
    float m[A], l[A];
    uint64_t acc[A][HDP / 32];  // pairs of dims
    int pos[A];
#pragma unroll
    for (int a = 0; a < A; ++a) {
        m[a] = -INFINITY;
        l[a] = 0.0f;
        const int row = r0 + ty * A + a;
        pos[a] = row < rows ? st.k_len - st.q_len + row / group : -1;
#pragma unroll
        for (int c = 0; c < HDP / 32; ++c) acc[a][c] = 0ull;
    }
    for (int it = 0; it < kt.count; ++it) {
        const int j0 = kt.at(it) * BN;
        fetch(Vs, HDP, vp, p.v.row, j0);
        asm volatile("cp.async.wait_group 1;" ::: "memory");  // K(it), and Q
        __syncthreads();
        // even and odd dims in the two halves of a packed sum: one instruction for two FMA
        uint64_t s2[A][4];
#pragma unroll
        for (int a = 0; a < A; ++a)
#pragma unroll
            for (int b = 0; b < 4; ++b) s2[a][b] = 0ull;
#pragma unroll 4
        for (int d = 0; d < HDP; d += 4) {
            ulonglong2 qv[A], kv[4];
#pragma unroll
            for (int a = 0; a < A; ++a) qv[a] = *reinterpret_cast<const ulonglong2*>(Qs + (ty * A + a) * HDP + d);
#pragma unroll
            for (int b = 0; b < 4; ++b) kv[b] = *reinterpret_cast<const ulonglong2*>(Ks + (tx + 16 * b) * LD + d);
#pragma unroll
            for (int a = 0; a < A; ++a)
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    s2[a][b] = fma_f32x2(qv[a].x, kv[b].x, s2[a][b]);
                    s2[a][b] = fma_f32x2(qv[a].y, kv[b].y, s2[a][b]);
                }
        }
        float s[A][4];
#pragma unroll
        for (int a = 0; a < A; ++a)
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                float lo, hi;
                unpack_f32x2(s2[a][b], lo, hi);
                s[a][b] = lo + hi;
            }
#pragma unroll
        for (int a = 0; a < A; ++a) {
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
                Ps[(ty * A + a) * BN + tx + 16 * b] = e;
            }
#pragma unroll
            for (int o = 8; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            l[a] = l[a] * alpha + sum;
            const uint64_t alpha2 = pack_f32x2(alpha, alpha);
#pragma unroll
            for (int c = 0; c < HDP / 32; ++c) acc[a][c] = mul_f32x2(acc[a][c], alpha2);
        }
        __syncthreads();  // everybody is done with K(it)
        if (it + 1 < kt.count) {
            fetch(Ks, LD, kp, p.k.row, kt.at(it + 1) * BN);
            asm volatile("cp.async.wait_group 1;" ::: "memory");
        } else {
            asm volatile("cp.async.wait_group 0;" ::: "memory");
        }
        __syncthreads();  // V(it) is there for everybody
#pragma unroll 2
        for (int j = 0; j < BN; j += 4) {
            float4 pw[A];
#pragma unroll
            for (int a = 0; a < A; ++a) pw[a] = *reinterpret_cast<const float4*>(Ps + (ty * A + a) * BN + j);
#pragma unroll
            for (int jj = 0; jj < 4; ++jj)
#pragma unroll
                for (int c = 0; c < HDP / 64; ++c) {
                    const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(Vs + (j + jj) * HDP + c * 64 + tx * 4);
#pragma unroll
                    for (int a = 0; a < A; ++a) {
                        const float w = jj == 0 ? pw[a].x : jj == 1 ? pw[a].y : jj == 2 ? pw[a].z : pw[a].w;
                        const uint64_t w2 = pack_f32x2(w, w);
                        acc[a][c * 2] = fma_f32x2(w2, v.x, acc[a][c * 2]);
                        acc[a][c * 2 + 1] = fma_f32x2(w2, v.y, acc[a][c * 2 + 1]);
                    }
                }
        }
        __syncthreads();  // everybody is done with V(it): its buffer takes V(it + 1)
    }
    unsigned redo = 0;
#pragma unroll
    for (int a = 0; a < A; ++a) {
        const int row = r0 + ty * A + a;
        const bool any = pos[a] >= 0;  // from position 0 on a query sees at least its own key
        const float inv = any ? 1.0f / l[a] : 0.0f;
        bool fine = true;
        float* dst = static_cast<float*>(const_cast<void*>(p.out.p)) + (st.q0 + row / group) * p.out.row + (int64_t)(kvh * group + row % group) * p.out.head;
#pragma unroll
        for (int c = 0; c < HDP / 32; ++c) {
            const int d = (c >> 1) * 64 + tx * 4 + (c & 1) * 2;
            float o[2];
            unpack_f32x2(acc[a][c], o[0], o[1]);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                o[e] = any ? o[e] * inv : 0.0f;
                fine = fine && isfinite(o[e]);
                if (row < rows && d + e < p.hd) dst[d + e] = o[e];
            }
        }
        const unsigned bad = __ballot_sync(0xffffffffu, row < rows && !fine);
        if (bad & 0xffffu) redo |= 1u << a;   // rows ty * A + a of the two half warps
        if (bad >> 16) redo |= 1u << (A + a);
    }
    // a non-finite value may come from a key that only other rows of the tile see (0 * inf): such rows are computed
    // again from the keys they see
    __syncwarp();
    for (; redo; redo &= redo - 1) redo_row<float>(p, st, kvh, r0 + (ty & ~1) * A + __ffs(redo) - 1);
}

// ---- single tokens ----
// A block owns 4 rows (query, head of the group) of one key head; the blocks of a cluster (up to 8) share the key axis, and
// their partial maxima, sums and outputs meet over distributed shared memory in a fixed order.  Per tile of 64 keys:
//   S       a thread owns one key and a quarter of the dims for all 4 rows, so a key is read from shared memory once;
//           the quarters meet in shared memory
//   softmax a warp per row, two keys a lane
//   P V     a thread owns 4 dims of all 4 rows and every (1024 / hd)-th key
// K and V tiles take turns in their buffers as for prompts.
constexpr int TR = 4;
template <int HDP>
constexpr int tokens_floats() { return 2 * BN * (HDP + 4) + TR * (HDP + 4) + 4 * BN * TR + BN * TR + 4 * TR; }

template <int HDP>
__global__ void __launch_bounds__(THREADS) window_f32_tokens_kernel(const __grid_constant__ WindowAttnParams p, int splits) {
    extern __shared__ __align__(16) float sm[];
    constexpr int LD = HDP + 4, GROUPS = THREADS / (HDP / 4);  // key groups of P V
    float *Ks = sm, *Vs = Ks + BN * LD;  // one tile each
    float* Qs = Vs + BN * LD;            // [TR][LD], at the end the block's output
    float* Sp = Qs + TR * LD;            // [4 quarters][BN][TR]
    float* Ps = Sp + 4 * BN * TR;        // [BN][TR]
    float* al = Ps + BN * TR;            // [TR] factors, [TR] maxima, [TR] sums, a word of rows to compute again
    unsigned* bad_rows = reinterpret_cast<unsigned*>(al + 3 * TR);
    const int group = p.nh / p.nkv, split = blockIdx.x % splits, kvh = blockIdx.x / splits % p.nkv;
    SeqTile st;
    if (!find_tile(p, blockIdx.x / splits / p.nkv, TR, group, st)) return;  // the same answer for the whole cluster
    const int r0 = st.tile * TR, rows = min(st.q_len * group - r0, TR), shift = st.k_len - st.q_len;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const float* qp = static_cast<const float*>(p.q.p);
    const float* kp = static_cast<const float*>(p.k.p) + st.k0 * p.k.row + (int64_t)kvh * p.k.head;
    const float* vp = static_cast<const float*>(p.v.p) + st.k0 * p.v.row + (int64_t)kvh * p.v.head;
    const int last_i = (r0 + rows - 1) / group;
    const KeyTiles kt = key_tiles(p, st, r0 / group, last_i, BN);
    const int t0 = (int)((int64_t)split * kt.count / splits), t1 = (int)((int64_t)(split + 1) * kt.count / splits);
    const int end = min(st.k_len, shift + last_i + 1);  // rows behind the last key that the block sees are zeros
    auto fetch = [&](float* dst, const float* src, int64_t pitch, int j0) {
        for (int t = tid; t < BN * (HDP / 4); t += THREADS) {
            const int j = t / (HDP / 4), d = t % (HDP / 4) * 4;
            const bool live = j0 + j < end && d < p.hd;
            copy16(dst + j * LD + d, live ? src + (int64_t)(j0 + j) * pitch + d : src, live);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    for (int t = tid; t < TR * (HDP / 4); t += THREADS) {
        const int r = t / (HDP / 4), d = t % (HDP / 4) * 4, row = r0 + r;
        const bool live = r < rows && d < p.hd;
        copy16(Qs + r * LD + d, live ? qp + (st.q0 + row / group) * p.q.row + (int64_t)(kvh * group + row % group) * p.q.head + d : qp, live);
    }
    if (t0 < t1) fetch(Ks, kp, p.k.row, kt.at(t0) * BN);
    const int pos = warp < rows ? shift + (r0 + warp) / group : -1;  // warps 0 - 3: of their softmax row
    float m = -INFINITY, l = 0.0f;
    float acc[TR][4] = {};
    const int key = tid & 63, quarter = tid >> 6;
    const int d4 = tid % (HDP / 4) * 4, kg = tid / (HDP / 4);
    for (int it = t0; it < t1; ++it) {
        const int j0 = kt.at(it) * BN;
        fetch(Vs, vp, p.v.row, j0);
        asm volatile("cp.async.wait_group 1;" ::: "memory");  // K(it), and Q
        __syncthreads();
        float s[TR] = {};
#pragma unroll 8
        for (int d = quarter * (HDP / 4); d < (quarter + 1) * (HDP / 4); d += 4) {
            const float4 k = *reinterpret_cast<const float4*>(Ks + key * LD + d);
#pragma unroll
            for (int r = 0; r < TR; ++r) {
                const float4 q = *reinterpret_cast<const float4*>(Qs + r * LD + d);
                s[r] = fmaf(q.x, k.x, s[r]);
                s[r] = fmaf(q.y, k.y, s[r]);
                s[r] = fmaf(q.z, k.z, s[r]);
                s[r] = fmaf(q.w, k.w, s[r]);
            }
        }
        *reinterpret_cast<float4*>(Sp + (quarter * BN + key) * TR) = make_float4(s[0], s[1], s[2], s[3]);
        __syncthreads();  // everybody is done with K(it)
        const bool more = it + 1 < t1;
        if (more) fetch(Ks, kp, p.k.row, kt.at(it + 1) * BN);
        if (warp < TR) {
            float x[2], top = -INFINITY;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int k = lane + 32 * e;
                const float dot = (Sp[k * TR + warp] + Sp[(BN + k) * TR + warp]) + (Sp[(2 * BN + k) * TR + warp] + Sp[(3 * BN + k) * TR + warp]);
                x[e] = sees(p, pos, j0 + k) ? score(dot, p.scale, p.softcap) : -INFINITY;
                top = fmaxf(top, x[e]);
            }
#pragma unroll
            for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            const float mn = fmaxf(m, top), ref = mn == -INFINITY ? 0.0f : mn;
            const float alpha = mn == m ? 1.0f : expf(m - ref);
            m = mn;
            float sum = 0.0f;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float w = expf(x[e] - ref);
                sum += w;
                Ps[(lane + 32 * e) * TR + warp] = w;
            }
            l = l * alpha + warp_sum(sum);
            if (lane == 0) al[warp] = alpha;
        }
        if (more) asm volatile("cp.async.wait_group 1;" ::: "memory");
        else asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncthreads();  // V(it), the weights and the factors are there for everybody
        const float4 f = *reinterpret_cast<const float4*>(al);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            acc[0][e] *= f.x;
            acc[1][e] *= f.y;
            acc[2][e] *= f.z;
            acc[3][e] *= f.w;
        }
#pragma unroll 4
        for (int j = kg; j < BN; j += GROUPS) {
            const float4 w = *reinterpret_cast<const float4*>(Ps + j * TR), v = *reinterpret_cast<const float4*>(Vs + j * LD + d4);
            const float ww[TR] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int r = 0; r < TR; ++r) {
                acc[r][0] = fmaf(ww[r], v.x, acc[r][0]);
                acc[r][1] = fmaf(ww[r], v.y, acc[r][1]);
                acc[r][2] = fmaf(ww[r], v.z, acc[r][2]);
                acc[r][3] = fmaf(ww[r], v.w, acc[r][3]);
            }
        }
        __syncthreads();  // everybody is done with V(it): its buffer takes V(it + 1)
    }
    if (t0 >= t1) {
        asm volatile("cp.async.wait_all;" ::: "memory");
        __syncthreads();
    }
    // the key groups meet in K's space, the block's result goes to Q's
    float* part = Ks;  // [GROUPS][TR][HDP]
#pragma unroll
    for (int r = 0; r < TR; ++r) *reinterpret_cast<float4*>(part + (kg * TR + r) * HDP + d4) = make_float4(acc[r][0], acc[r][1], acc[r][2], acc[r][3]);
    if (warp < TR && lane == 0) {
        al[TR + warp] = m;
        al[2 * TR + warp] = l;
    }
    if (tid == 0) *bad_rows = 0;
    __syncthreads();
    for (int i = tid; i < TR * HDP; i += THREADS) {
        float sum = 0.0f;
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) sum += part[g * TR * HDP + i];
        Qs[i / HDP * LD + i % HDP] = sum;
    }
    cg::cluster_group cluster = cg::this_cluster();
    if (splits > 1) cluster.sync();
    else __syncthreads();
    // block c of the cluster finishes rows c, c + splits, ...
    const int own = rows > split ? (rows - split + splits - 1) / splits : 0;
    for (int i = tid; i < own * (HDP / 4); i += THREADS) {
        const int r = split + i / (HDP / 4) * splits, d = i % (HDP / 4) * 4, row = r0 + r;
        float ms[MAX_SPLITS], top = -INFINITY, sum = 0.0f, f[4] = {};
#pragma unroll
        for (int z = 0; z < MAX_SPLITS; ++z) {
            ms[z] = z < splits ? *cluster.map_shared_rank(al + TR + r, z) : -INFINITY;
            top = fmaxf(top, ms[z]);
        }
#pragma unroll
        for (int z = 0; z < MAX_SPLITS; ++z)
            if (z < splits) {
                const float w = ms[z] == top ? 1.0f : expf(ms[z] - top);
                const float4 v = *reinterpret_cast<const float4*>(cluster.map_shared_rank(Qs + r * LD + d, z));
                f[0] = fmaf(w, v.x, f[0]);
                f[1] = fmaf(w, v.y, f[1]);
                f[2] = fmaf(w, v.z, f[2]);
                f[3] = fmaf(w, v.w, f[3]);
                sum = fmaf(w, *cluster.map_shared_rank(al + 2 * TR + r, z), sum);
            }
        const bool any = shift + row / group >= 0;  // from position 0 on a query sees at least its own key
        const float inv = any ? 1.0f / sum : 0.0f;
        float* dst = static_cast<float*>(const_cast<void*>(p.out.p)) + (st.q0 + row / group) * p.out.row + (int64_t)(kvh * group + row % group) * p.out.head;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (d + e < p.hd) {
                const float o = any ? f[e] * inv : 0.0f;
                dst[d + e] = o;
                if (!isfinite(o)) atomicOr(bad_rows, 1u << r);
            }
    }
    __syncthreads();
    // 0 * inf from a key that only other rows of the block see: such rows are computed again from the keys they see
    unsigned bad = *bad_rows;
    for (int i = 0; bad; bad &= bad - 1, ++i)
        if (i % (THREADS / 32) == warp) redo_row<float>(p, st, kvh, r0 + __ffs(bad) - 1);
    if (splits > 1) cluster.sync();  // nobody's shared memory goes away while another block reads it
}

template <int HDP>
int launch_prompts(const WindowAttnParams& p, cudaStream_t s) {
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
template <int HDP>
int launch_tokens(const WindowAttnParams& p, cudaStream_t s) {
    static std::atomic<int> clusters_of[64][MAX_SPLITS + 1];  // clusters that run at once, a property of the device
    int dev = 0;
    CMFC_CUDA(cudaGetDevice(&dev));
    constexpr int SMEM = tokens_floats<HDP>() * 4;
    static_assert(SMEM <= 232448 && THREADS / (HDP / 4) * TR * HDP <= BN * (HDP + 4), "tiles fit shared memory, partial outputs a tile");
    auto kernel = window_f32_tokens_kernel<HDP>;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = SMEM;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (!clusters_of[dev & 63][1]) {
        CMFC_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM));
        for (int n = MAX_SPLITS; n >= 1; n /= 2) {
            attr[0].val.clusterDim.x = n;
            cfg.gridDim = dim3(n);
            int active = 0;
            CMFC_CUDA(cudaOccupancyMaxActiveClusters(&active, kernel, &cfg));
            clusters_of[dev & 63][n] = active > 0 ? active : 1;
        }
    }
    // As for the 16-bit types (window_tokens.cu): cut only while all shares run at once, and keep a key tile each (one
    // sequence x 8 heads of 128 x 256 / 512 keys: 7.6 / 7.8 us, with two tiles each 9.1 / 9.5, with eight 12.7 / 21.8).
    int splits = 1;
    while (splits < MAX_SPLITS && window_items(p, TR) <= clusters_of[dev & 63][2 * splits] && window_range(p) / (2 * splits) >= BN) splits *= 2;
    attr[0].val.clusterDim.x = splits;
    cfg.gridDim = dim3((unsigned)(max_tiles(p, TR) * p.nkv * splits));
    CMFC_CUDA(cudaLaunchKernelEx(&cfg, kernel, p, splits));
    return OK;
}
template <int HDP>
int launch_hdp(const WindowAttnParams& p, int num_sms, cudaStream_t s) {
    if (window_few_rows(p, num_sms)) return launch_tokens<HDP>(p, s);
    return launch_prompts<HDP>(p, s);
}

}  // namespace

bool window_f32_supported(const WindowAttnParams& p, int elem) {
    auto fits = [](const HeadView& v) { return !(reinterpret_cast<uintptr_t>(v.p) & 15) && v.row % 4 == 0 && v.head % 4 == 0; };
    return elem == ET_F32 && p.hd % 4 == 0 && max_tiles(p, TR) * p.nkv * MAX_SPLITS < ((int64_t)1 << 31) && fits(p.q) && fits(p.k) && fits(p.v);
}

int launch_window_f32(const WindowAttnParams& p, int num_sms, cudaStream_t s) {
    if (p.hd <= 64) return launch_hdp<64>(p, num_sms, s);
    if (p.hd <= 128) return launch_hdp<128>(p, num_sms, s);
    return launch_hdp<256>(p, num_sms, s);
}

}  // namespace cmfc
