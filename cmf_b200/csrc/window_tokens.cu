// Windowed causal attention for single tokens (and a few queries per sequence) over caches, f16 / bf16, head
// sizes up to 256.  The definition is in window_attention.cu.
//
// Bound: memory, the keys and values that are seen, once.  A block owns up to 16 rows of one key head (a row is (query,
// head of the group)), so all heads that share keys read them together, and a share of the key axis: the blocks
// of a cluster (up to 8) split it and join their partial maxima, sums and outputs over distributed shared memory,
// in a fixed order, so one launch does the whole thing without a workspace.
//   warp 0      TMA producer: tiles of 32 keys (16 of the largest heads), K and V, 128-byte swizzle, through a ring of 64 to
//               96 KB; two blocks share an SM, so up to 192 KB are on their way and one block's start and end hide
//               behind the other
//   other warps 16 keys at a time each, teams of one or two warps taking tiles in turn: S = Q K^T by m16n8k16 (rows of
//               queries beside each other, f32 sums), mask, soft cap, running maximum, exp2, O += P V
// Measured, bf16: 64 sequences x 4096 keys x 4 heads of 256 165 us, x 8 heads of 128 167 us (6.5 TB/s, a copy's rate); one
// sequence x 131072 keys x 8 heads of 128 115 us (4.7 TB/s); one sequence x 1000 keys 10 us, of which 5 are the launch of the
// cluster, its joining and the way of the first tile.
// Rows of V that no row of the block sees are zeroed in shared memory first (0 x NaN), and rows whose result is not
// finite are computed again key by key (redo_row).
#include <cooperative_groups.h>

#include <atomic>
#include <type_traits>

#include "window_attention.cuh"

namespace cmfc {
namespace {

namespace cg = cooperative_groups;

constexpr int ROWS = 16, MAX_WARPS = 8;
constexpr int MAX_SPLITS = 8;
constexpr float LOG2E = 1.4426950408889634f;

template <int HDP, int W>
struct Smem {
    static constexpr int KEYS = HDP <= 128 ? 32 : 16;  // of a tile; a warp takes 16
    static constexpr int WARPS = W, THREADS = 32 * (1 + W);
    static constexpr int WPT = KEYS / 16, TEAMS = WARPS / WPT;  // warps that share a tile, teams that take tiles in turn
    static constexpr int KTILE = KEYS * HDP * 2, STAGE = 2 * KTILE;
    static constexpr int STAGES = HDP == 128 && W == 4 ? 6 : 12;
    // A stage always belongs to the same team: a warp that met only some of a barrier's phases could not tell by
    // the parity whether the one before its own is complete.
    static_assert(STAGES % TEAMS == 0 && STAGES / TEAMS >= 2, "stages are dealt to the teams in turn; one holds the next tile");
    static constexpr int PER_SM = HDP <= 128 && W == 4 ? 2 : 1;
    static constexpr int PARTS = (WARPS + 1) * ROWS * HDP * 4;
    static constexpr int RING = STAGES * STAGE > PARTS ? STAGES * STAGE : PARTS;
    static constexpr int Q_LD = HDP + 8;  // rows shifted by 16 bytes: ldmatrix without conflicts
    static constexpr int Q = ROWS * Q_LD * 2;
    // after the loop the ring's space holds every warp's O [16][HDP] f32 and the block's joined one
    static constexpr int TOTAL = RING + Q + 1024 + 1536;
};
struct Tail {
    uint64_t full[12], empty[12];
    float m[MAX_WARPS + 1][ROWS], l[MAX_WARPS + 1][ROWS];  // the last ones: the whole block's
    unsigned bad;
    uint32_t abort_flag;
};
static_assert(sizeof(Tail) <= 1536, "barriers and statistics fit their place");

template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<T, __half>::value)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void load_3d(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst), "l"(map),
                 "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
                 : "memory");
}
// address of 16-byte unit `unit` (8 dims) of key row `row` in a K or V tile: chunks of 64 dims, KEYS rows of 128 swizzled bytes
template <int KEYS>
__device__ __forceinline__ uint32_t tile_at(uint32_t base, int row, int unit) {
    return base + (unit >> 3) * (KEYS * 128) + row * 128 + (((unit & 7) ^ (row & 7)) << 4);
}

template <typename T, int HDP, Cap CAP, int W>
__global__ void __launch_bounds__(32 * (1 + W), (Smem<HDP, W>::PER_SM))
window_tokens_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ WindowAttnParams p, int splits) {
    using L = Smem<HDP, W>;
    constexpr int NC = HDP / 64, KEYS = L::KEYS, WARPS = L::WARPS, THREADS = L::THREADS;
    // key heads next to each other: their keys lie next to each other too, and DRAM pages are read while open
    const int group = p.nh / p.nkv, split = blockIdx.x % splits, kvh = blockIdx.x / splits % p.nkv;
    SeqTile st;
    if (!find_tile(p, blockIdx.x / splits / p.nkv, ROWS, group, st)) return;  // the same answer for the whole cluster
    const int r0 = st.tile * ROWS, rows = min(st.q_len * group - r0, ROWS);
    const int shift = st.k_len - st.q_len;
    const int first_i = r0 / group, last_i = (r0 + rows - 1) / group;
    const KeyTiles kt = key_tiles(p, st, first_i, last_i, KEYS);
    const int t0 = (int)((int64_t)split * kt.count / splits), t1 = (int)((int64_t)(split + 1) * kt.count / splits);

    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    T* qs = reinterpret_cast<T*>(smem + L::RING);
    Tail* tail = reinterpret_cast<Tail*>(smem + L::RING + L::Q);
    volatile uint32_t* abort_flag = &tail->abort_flag;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < L::STAGES; ++s) {
            mbar_init(&tail->full[s], 1);
            mbar_init(&tail->empty[s], L::WPT);
        }
        tail->abort_flag = 0;
        tail->bad = 0;
        mbar_fence_init();
        tma_prefetch_desc(&tm_k);
        tma_prefetch_desc(&tm_v);
    }
    __syncthreads();

    float o[HDP / 8][4];
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
    const int g = lane >> 2, t4 = lane & 3;
    if (warp == 0) {
        if (elect_one()) {
            for (int t = t0; t < t1; ++t) {
                const int it = t - t0, s = it % L::STAGES;
                if (!mbar_wait<40>(&tail->empty[s], ((it / L::STAGES) & 1u) ^ 1u, abort_flag, 1)) break;
                mbar_expect_tx(&tail->full[s], L::STAGE);
                const uint32_t dst = smem_u32(smem) + s * L::STAGE;
                const int row = (int)st.k0 + kt.at(t) * KEYS;
                for (int c = 0; c < NC; ++c) load_3d(dst + c * KEYS * 128, &tm_k, &tail->full[s], c * 64, kvh, row);
                for (int c = 0; c < NC; ++c) load_3d(dst + L::KTILE + c * KEYS * 128, &tm_v, &tail->full[s], c * 64, kvh, row);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < HDP / 8; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[i][e] = 0.0f;
        // the queries, 16 bytes at a time; rows and dims that do not exist are zeros
        for (int i = threadIdx.x - 32; i < ROWS * (HDP / 8); i += 32 * WARPS) {
            const int r = i / (HDP / 8), d = i % (HDP / 8) * 8, row = r0 + r;
            uint4 x = make_uint4(0u, 0u, 0u, 0u);
            if (r < rows && d < p.hd)
                x = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.q.p) + (st.q0 + row / group) * p.q.row + (int64_t)(kvh * group + row % group) * p.q.head + d);
            *reinterpret_cast<uint4*>(qs + r * L::Q_LD + d) = x;
        }
        asm volatile("bar.sync 1, %0;" ::"n"(32 * WARPS) : "memory");
        const int w = warp - 1, team = w / L::WPT, half = w % L::WPT;
        const uint32_t qa = smem_u32(qs) + ((lane & 15) * L::Q_LD + (lane >> 4) * 8) * 2;  // ldmatrix: 16 rows x 16 dims
        uint32_t qf[HDP <= 128 ? HDP / 16 : 1][4];  // small heads keep the queries in registers
        if constexpr (HDP <= 128) {
#pragma unroll
            for (int k = 0; k < HDP / 16; ++k) ldsm4(qf[k], qa + k * 32);
        }
        const int pos0 = g < rows ? shift + (r0 + g) / group : -1, pos1 = g + 8 < rows ? shift + (r0 + g + 8) / group : -1;
        const float sc = p.scale * LOG2E, cap2 = p.softcap * LOG2E, to_y = CAP ? p.scale / p.softcap : 0.0f;
        const int pos_min = shift + first_i, seen_last = shift + last_i;
        const int seen_low = (int)max((int64_t)0, (int64_t)pos_min - p.window + 1);
        auto ready = [&](int t) {
            const int it = t - t0;
            // the lanes leave the polling loop one by one: ldmatrix and mma want the warp together
            return __all_sync(0xffffffffu, mbar_wait(&tail->full[it % L::STAGES], (it / L::STAGES) & 1u, abort_flag, 2)) != 0;
        };
        auto stage_at = [&](int t) { return smem_u32(smem) + (t - t0) % L::STAGES * L::STAGE; };
        // S of 16 keys: even and odd steps of 16 dims in sums of their own, so that four chains of products run side by side
        auto scores = [&](uint32_t ks, float (&s)[2][4]) {
            float odd[2][4];
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[n][e] = odd[n][e] = 0.0f;
#pragma unroll
            for (int k = 0; k < HDP / 16; ++k) {
                float(&sk)[2][4] = k & 1 ? odd : s;
                // keys 0-7 and 8-15 of the half, dims 0-7 and 8-15 of the step
                uint32_t b[4];
                ldsm4(b, tile_at<KEYS>(ks, half * 16 + (lane & 7) + ((lane >> 4) << 3), 2 * k + ((lane >> 3) & 1)));
                if constexpr (HDP <= 128) {
                    mma16816<T>(sk[0], qf[k][0], qf[k][1], qf[k][2], qf[k][3], b[0], b[1]);
                    mma16816<T>(sk[1], qf[k][0], qf[k][1], qf[k][2], qf[k][3], b[2], b[3]);
                } else {
                    uint32_t a[4];
                    ldsm4(a, qa + k * 32);
                    mma16816<T>(sk[0], a[0], a[1], a[2], a[3], b[0], b[1]);
                    mma16816<T>(sk[1], a[0], a[1], a[2], a[3], b[2], b[3]);
                }
            }
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[n][e] += odd[n][e];
        };
        float cur[2][4], nxt[2][4];
        int t = t0 + team;
        bool ok = t < t1 && ready(t);
        if (ok) scores(stage_at(t), cur);
        for (; ok && t < t1; t += L::TEAMS) {
            // S of the warp's next tile is on its way through the MMA unit while this one's softmax runs; behind
            // the last tile it is computed once more from the same keys and not used
            const bool more = t + L::TEAMS < t1;
            if (more && !ready(t + L::TEAMS)) break;
            scores(stage_at(more ? t + L::TEAMS : t), nxt);
            const int j0 = kt.at(t) * KEYS + half * 16;
            const uint32_t vs = stage_at(t) + L::KTILE;
            float x[2][4];  // log2 units
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    x[n][e] = CAP ? cap2 * (CAP == CAP_NEAR ? cap_tanh_far(cur[n][e] * to_y) : cap_tanh(cur[n][e] * to_y)) : cur[n][e] * sc;
            if (j0 + 15 > pos_min || ((int64_t)seen_last - j0 >= p.window && j0 + 16 > p.sinks)) {  // some row does not see all 16 keys
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[n][e] = sees(p, e < 2 ? pos0 : pos1, j0 + n * 8 + 2 * t4 + (e & 1)) ? x[n][e] : -INFINITY;
                // rows of V that nobody sees: zeros, 16 bytes at a time
                for (int i = lane; i < 16 * (HDP / 8); i += 32) {
                    const int j = j0 + i / (HDP / 8);
                    if (j > seen_last || (j < seen_low && j >= p.sinks))
                        asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(tile_at<KEYS>(vs, half * 16 + i / (HDP / 8), i % (HDP / 8))), "r"(0u) : "memory");
                }
                __syncwarp();
            }
            float alpha[2], ref[2];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                float mx = fmaxf(fmaxf(x[0][2 * r], x[0][2 * r + 1]), fmaxf(x[1][2 * r], x[1][2 * r + 1]));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                const float mn = fmaxf(m[r], mx);
                ref[r] = mn == -INFINITY ? 0.0f : mn;
                alpha[r] = mn == m[r] ? 1.0f : ex2_approx(m[r] - ref[r]);  // an unchanged infinite maximum too
                m[r] = mn;
            }
            if (__any_sync(0xffffffffu, alpha[0] != 1.0f || alpha[1] != 1.0f)) {
#pragma unroll
                for (int i = 0; i < HDP / 8; ++i) {
                    o[i][0] *= alpha[0];
                    o[i][1] *= alpha[0];
                    o[i][2] *= alpha[1];
                    o[i][3] *= alpha[1];
                }
                l[0] *= alpha[0];
                l[1] *= alpha[1];
            }
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    x[n][e] = ex2_approx(x[n][e] - ref[e >> 1]);
                    l[e >> 1] += x[n][e];  // the sum takes the weights before their rounding to T
                }
            const uint32_t a0 = pack2<T>(x[0][0], x[0][1]), a1 = pack2<T>(x[0][2], x[0][3]), a2 = pack2<T>(x[1][0], x[1][1]),
                           a3 = pack2<T>(x[1][2], x[1][3]);
#pragma unroll
            for (int d = 0; d < HDP / 16; ++d) {
                // keys 0-7 and 8-15, dims 0-7 and 8-15 of the step, transposed
                uint32_t b[4];
                ldsm4_t(b, tile_at<KEYS>(vs, half * 16 + (lane & 15), 2 * d + (lane >> 4)));
                mma16816<T>(o[2 * d], a0, a1, a2, a3, b[0], b[1]);
                mma16816<T>(o[2 * d + 1], a0, a1, a2, a3, b[2], b[3]);
            }
            // The slot's next tile is written by the async proxy: every lane's reads are ordered before that.  (Without
            // the fence, two blocks on an SM read a few rows of a next tile once in some ten thousand blocks.)
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&tail->empty[(t - t0) % L::STAGES]);
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) cur[n][e] = nxt[n][e];
        }
    }
    __syncthreads();  // every tile of the ring is consumed (or a wait gave up): its space is free
    drain_copies(abort_flag);
    float* part = reinterpret_cast<float*>(smem);  // [WARPS + 1][16][HDP], the last one for the block
    if (warp > 0) {
        const int w = warp - 1;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
            if (t4 == 0) {
                tail->m[w][g + 8 * r] = m[r];
                tail->l[w][g + 8 * r] = l[r];
            }
        }
#pragma unroll
        for (int i = 0; i < HDP / 8; ++i) {
            *reinterpret_cast<float2*>(part + (w * ROWS + g) * HDP + i * 8 + 2 * t4) = make_float2(o[i][0], o[i][1]);
            *reinterpret_cast<float2*>(part + (w * ROWS + g + 8) * HDP + i * 8 + 2 * t4) = make_float2(o[i][2], o[i][3]);
        }
    }
    __syncthreads();
    // join the warps: rows [0, rows)
    float* mine = part + WARPS * ROWS * HDP;
    for (int i = threadIdx.x; i < rows * (HDP / 4); i += THREADS) {
        const int r = i / (HDP / 4), d = i % (HDP / 4) * 4;
        float top = tail->m[0][r];
#pragma unroll
        for (int w = 1; w < WARPS; ++w) top = fmaxf(top, tail->m[w][r]);
        float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const float f = tail->m[w][r] == top ? 1.0f : ex2_approx(tail->m[w][r] - top);
            const float4 v = *reinterpret_cast<const float4*>(part + (w * ROWS + r) * HDP + d);
            acc.x = fmaf(f, v.x, acc.x);
            acc.y = fmaf(f, v.y, acc.y);
            acc.z = fmaf(f, v.z, acc.z);
            acc.w = fmaf(f, v.w, acc.w);
            sum = fmaf(f, tail->l[w][r], sum);
        }
        *reinterpret_cast<float4*>(mine + r * HDP + d) = acc;
        if (d == 0) {
            tail->m[MAX_WARPS][r] = top;
            tail->l[MAX_WARPS][r] = sum;
        }
    }
    cg::cluster_group cluster = cg::this_cluster();
    if (splits > 1) cluster.sync();
    else __syncthreads();
    // join the blocks: block c of the cluster finishes rows c, c + splits, ...
    const int own = rows > split ? (rows - split + splits - 1) / splits : 0;
    for (int i = threadIdx.x; i < own * (HDP / 4); i += THREADS) {
        const int r = split + i / (HDP / 4) * splits, d = i % (HDP / 4) * 4, row = r0 + r;
        float4 acc = *reinterpret_cast<const float4*>(mine + r * HDP + d);
        float sum = tail->l[MAX_WARPS][r];
        if (splits > 1) {
            float ms[MAX_SPLITS], top = -INFINITY;
#pragma unroll
            for (int s = 0; s < MAX_SPLITS; ++s) {
                ms[s] = s < splits ? *cluster.map_shared_rank(&tail->m[MAX_WARPS][r], s) : -INFINITY;
                top = fmaxf(top, ms[s]);
            }
            acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            sum = 0.0f;
#pragma unroll
            for (int s = 0; s < MAX_SPLITS; ++s)
                if (s < splits) {
                    const float f = ms[s] == top ? 1.0f : ex2_approx(ms[s] - top);
                    const float4 v = *reinterpret_cast<const float4*>(cluster.map_shared_rank(mine + r * HDP + d, s));
                    acc.x = fmaf(f, v.x, acc.x);
                    acc.y = fmaf(f, v.y, acc.y);
                    acc.z = fmaf(f, v.z, acc.z);
                    acc.w = fmaf(f, v.w, acc.w);
                    sum = fmaf(f, *cluster.map_shared_rank(&tail->l[MAX_WARPS][r], s), sum);
                }
        }
        const bool any = shift + row / group >= 0;  // from position 0 on a query sees at least its own key
        const float inv = any ? 1.0f / sum : 0.0f;
        const float f[4] = {any ? acc.x * inv : 0.0f, any ? acc.y * inv : 0.0f, any ? acc.z * inv : 0.0f, any ? acc.w * inv : 0.0f};
        T* dst = static_cast<T*>(const_cast<void*>(p.out.p)) + (st.q0 + row / group) * p.out.row + (int64_t)(kvh * group + row % group) * p.out.head;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (d + e < p.hd) {
                dst[d + e] = from_f32<T>(f[e]);
                if (!isfinite(f[e])) atomicOr(&tail->bad, 1u << r);
            }
    }
    __syncthreads();
    unsigned bad = tail->bad;
    for (int i = 0; bad; bad &= bad - 1, ++i)
        if (i % (THREADS / 32) == warp) redo_row<T>(p, st, kvh, r0 + __ffs(bad) - 1);
    if (threadIdx.x == 0 && tail->abort_flag) atomicCAS(p.status, 0u, 0xA00u | tail->abort_flag);
    if (splits > 1) cluster.sync();  // nobody's shared memory goes away while another block reads it
}

template <typename T, int HDP, Cap CAP, int W>
int launch_form(const CUtensorMap& tm_k, const CUtensorMap& tm_v, const WindowAttnParams& p, cudaStream_t s) {
    static std::atomic<int> clusters_of[64][MAX_SPLITS + 1];  // clusters that run at once, a property of the device
    int dev = 0;
    CMFC_CUDA(cudaGetDevice(&dev));
    auto kernel = window_tokens_kernel<T, HDP, CAP, W>;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.blockDim = dim3(Smem<HDP, W>::THREADS);
    cfg.dynamicSmemBytes = Smem<HDP, W>::TOTAL;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (!clusters_of[dev & 63][1]) {
        CMFC_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Smem<HDP, W>::TOTAL));
        for (int n = MAX_SPLITS; n >= 1; n /= 2) {
            attr[0].val.clusterDim.x = n;
            cfg.gridDim = dim3(n);
            int active = 0;
            CMFC_CUDA(cudaOccupancyMaxActiveClusters(&active, kernel, &cfg));
            clusters_of[dev & 63][n] = active > 0 ? active : 1;
        }
    }
    // Cut the key axis only as far as all shares still run at once and keep 128 keys: a cluster waits until all of its
    // blocks find room (64 sequences x 4 key heads of 256 x 4096 keys: uncut 164 us, in two 192, in four 226; one
    // sequence x 8 heads of 128 x 4096 keys: uncut 40 us, in two 24, in four 16, in eight 12).
    const int64_t items = window_items(p, ROWS), range = window_range(p);
    int splits = 1;
    while (splits < MAX_SPLITS && items <= clusters_of[dev & 63][2 * splits] && range / (2 * splits) >= 128) splits *= 2;
    attr[0].val.clusterDim.x = splits;
    cfg.gridDim = dim3((unsigned)(max_tiles(p, ROWS) * p.nkv * splits));
    CMFC_CUDA(cudaLaunchKernelEx(&cfg, kernel, tm_k, tm_v, p, splits));
    return OK;
}
template <typename T, int HDP, int W>
int launch_warps(const CUtensorMap& tm_k, const CUtensorMap& tm_v, const WindowAttnParams& p, cudaStream_t s) {
    switch (cap_form(p)) {
        case NO_CAP: return launch_form<T, HDP, NO_CAP, W>(tm_k, tm_v, p, s);
        case CAP_NEAR: return launch_form<T, HDP, CAP_NEAR, W>(tm_k, tm_v, p, s);
        default: return launch_form<T, HDP, CAP_ANY, W>(tm_k, tm_v, p, s);
    }
}
template <typename T, int HDP>
int launch_hdp(const CUtensorMap& tm_k, const CUtensorMap& tm_v, const WindowAttnParams& p, int num_sms, cudaStream_t s) {
    // A warp's step over 16 keys is a chain of about 1200 clocks whatever else runs.  Few items: eight warps a block, one
    // block per SM (one sequence x 8 heads of 128 x 131072 keys: 115 us, with four warps 174); many: four warps, two
    // blocks per SM, one of which starts or ends while the other reads (64 sequences x 8 heads of 128 x 4096 keys: 167 us,
    // with eight warps 188).  Heads of 256 leave room for the tiles of four warps.
    if constexpr (HDP <= 128) {
        if (window_items(p, ROWS) <= num_sms / 2)
            return launch_warps<T, HDP, 8>(tm_k, tm_v, p, s);
    }
    return launch_warps<T, HDP, 4>(tm_k, tm_v, p, s);
}
template <typename T>
int launch_typed(const CUtensorMap& tm_k, const CUtensorMap& tm_v, const WindowAttnParams& p, int num_sms, cudaStream_t s) {
    if (p.hd <= 64) return launch_hdp<T, 64>(tm_k, tm_v, p, num_sms, s);
    if (p.hd <= 128) return launch_hdp<T, 128>(tm_k, tm_v, p, num_sms, s);
    return launch_hdp<T, 256>(tm_k, tm_v, p, num_sms, s);
}

}  // namespace

bool window_tokens_supported(const WindowAttnParams& p, int elem) {
    constexpr int64_t MOST = (int64_t)1 << 38;  // strides of a tensor map stay below 2^40 bytes
    auto fits = [&](const HeadView& v, int heads) {
        return !(reinterpret_cast<uintptr_t>(v.p) & 15) && v.row > 0 && v.row < MOST && v.row % 8 == 0 &&
               (heads == 1 || (v.head > 0 && v.head < MOST && v.head % 8 == 0));
    };
    // queries come by 16-byte loads (any stride that keeps them aligned), keys and values by TMA
    return elem != ET_F32 && max_tiles(p, ROWS) * p.nkv * MAX_SPLITS < ((int64_t)1 << 31) && p.hd % 8 == 0 && p.k_rows > 0 && !(reinterpret_cast<uintptr_t>(p.q.p) & 15) && p.q.row % 8 == 0 &&
           p.q.head % 8 == 0 && fits(p.k, p.nkv) && fits(p.v, p.nkv);
}

int launch_window_tokens(const WindowAttnParams& p, int elem, int num_sms, cudaStream_t s) {
    CUtensorMap tm_k, tm_v;
    auto map = [&](CUtensorMap* m, const HeadView& v) {
        return make_tensor_map_heads16(m, v.p, (uint64_t)p.hd, (uint64_t)p.nkv, (uint64_t)p.k_rows, (uint64_t)(p.nkv == 1 ? v.row : v.head) * 2,
                                       (uint64_t)v.row * 2, 64, 1, p.hd <= 128 ? Smem<128, 4>::KEYS : Smem<256, 4>::KEYS);
    };
    if (map(&tm_k, p.k) != OK || map(&tm_v, p.v) != OK) return launch_window_any(p, elem, s);  // a layout that no tensor map describes
    if (elem == ET_F16) return launch_typed<__half>(tm_k, tm_v, p, num_sms, s);
    return launch_typed<__nv_bfloat16>(tm_k, tm_v, p, num_sms, s);
}

}  // namespace cmfc
