// Windowed causal attention for prompts and chunks of prompts on the tensor cores (f16 / bf16, head sizes
// up to 256), flash style: scores never leave the SM.  The definition is in window_attention.cu.
//
// A tile is 128 rows of one key head: a row is (query, head of the group), so one K / V tile serves all heads
// that share it, and the masked corner of a tile is 128 / group queries wide instead of 128.  Per key tile of 128:
//   S = Q K^T     tcgen05.mma, both operands from shared memory (TMA, 128-byte swizzle, chunks of 64 dims)
//   softmax       one row per thread: tcgen05.ld of the row, scale (or soft cap), mask on the tiles that need one,
//                 running maximum moved lazily (only when it grows by more than 8 in log2 units), exp2, row sum
//                 in f32, P rounded to the operand type (its products are summed in f32) and written over S
//   O += P V      tcgen05.mma with P as the tensor-memory A operand; V is used as it lies in memory (keys x dims),
//                 the MN-major form of the B operand, so nothing is transposed
// Two streams keep the tensor pipe and the softmax warps busy at the same time.  Head sizes up to 128: two query
// tiles that share every K / V tile (S and O of both fill the 512 columns of tensor memory).  Above, or when a
// sequence has only one tile left: one query tile with two S buffers, S(j + 1) computed during softmax(j).
// Either way step u of the sequence "P V (u), then S (u + 2)" is issued by one thread in the same order.
//
// K and V travel through one ring of 16 KB slots: a K chunk is 64 dims x 128 keys, a V chunk 8192 / dims keys x
// all dims, so that the P V products keep their full N and a large head still has several loads in flight.
//
// Bound: up to dims of 128 the chain softmax -> P V -> S of a stream (about 3900 clocks for a pair of tiles of which the
// products take 2050); above, the products' reads of shared memory (3700 clocks a step); with a soft cap the FMA pipe.
// Measured, 8192 tokens: 32 / 8 heads of 128 533 us = 1031 TFLOP/s; 8 / 4 heads of 256, window 4096 226 us = 911 TFLOP/s,
// with a soft cap 303 us = 681.
//
// Rows of V behind the last key that a tile sees are zeroed in shared memory before they are used: they are another
// sequence's, or memory that nobody wrote, and 0 x NaN would spread.  Rows whose result is not finite, or that met a
// NaN score, are computed again key by key (redo_row), so that what a row does not see never reaches it.
#include <atomic>
#include <type_traits>

#include "window_attention.cuh"

namespace cmfc {
namespace {

constexpr int QT = 128, KT = 128;
constexpr int SLOT = 16384;
constexpr float LOG2E = 1.4426950408889634f;

template <int HDP> __host__ __device__ constexpr int q_tiles() { return HDP <= 128 ? 2 : 1; }
template <int HDP> __host__ __device__ constexpr int slots() { return HDP == 64 ? 12 : 10; }
constexpr int THREADS = 32 * (2 + 8);
template <int HDP> __host__ __device__ constexpr int q_bytes() { return QT * HDP * 2; }
constexpr int BARS_BYTES = 3 * 1024;
template <int HDP> __host__ __device__ constexpr int smem_bytes() { return q_tiles<HDP>() * q_bytes<HDP>() + slots<HDP>() * SLOT + BARS_BYTES; }

struct Bars {
    uint64_t q_full;
    uint64_t full[12], empty[12];
    // one of each per stream (query tile, or S buffer); the phase before the one that anybody waits for is
    // always known to be complete, so its parity is enough
    uint64_t s_full[2], p_full[2], o_done[2];
    // one query tile: reference of the rows' exponentials, handed from warp to warp between the groups; their parts of
    // the row sums with the reference each is relative to; rows to compute again
    uint64_t ref_full[2][4];
    float ref[QT];
    float2 part[2][QT];
    uint8_t bad[QT];
    uint32_t tmem_base, abort_flag;
};
static_assert(sizeof(Bars) <= BARS_BYTES && smem_bytes<64>() <= 232448 && smem_bytes<128>() <= 232448 && smem_bytes<256>() <= 232448, "barriers and row statistics fit their place");

// kind::f16, f32 accumulator, A and B of one 16-bit type (f16: 0, bf16: 1); b_mn: B is MN-major
template <typename T>
__device__ __forceinline__ uint32_t idesc16(uint32_t n, bool b_mn) {
    const uint32_t f = sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    return (1u << 4) | (f << 7) | (f << 10) | ((b_mn ? 1u : 0u) << 16) | ((n >> 3) << 17) | ((QT >> 4) << 24);
}
// MN-major operand in 128-byte swizzled rows of 64 values: groups of 64 values `group_bytes` apart, groups of
// eight k rows 1024 bytes apart
__device__ __forceinline__ uint64_t smem_desc_mn(uint32_t addr, uint32_t group_bytes) {
    uint64_t d = 0;
    d |= (uint64_t)((addr & 0x3FFFFu) >> 4);
    d |= (uint64_t)(group_bytes >> 4) << 16;
    d |= (uint64_t)(1024u >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}
__device__ __forceinline__ void load_3d(void* dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(dst)),
                 "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
                 : "memory");
}
// maxima that keep a NaN
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// bit i: the row at position pos sees key j0 + i
__device__ __forceinline__ uint32_t seen_bits(const WindowAttnParams& p, int pos, int j0) {
    auto below = [](int64_t n) -> uint32_t { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; };  // bits [0, n)
    const uint32_t causal = below((int64_t)pos - j0 + 1);
    const uint32_t passed = below((int64_t)pos - p.window + 1 - j0) & ~below((int64_t)p.sinks - j0);
    return causal & ~passed;
}

template <typename T, int HDP, int POLY_OF_8, Cap CAP>
__global__ void __launch_bounds__(THREADS, 1)
window_prefill_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                      const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ WindowAttnParams p, int tile_tokens, int out_vec) {
    constexpr int NC = HDP / 64;             // chunks of a K or V tile
    constexpr int VK = SLOT / (HDP * 2);     // keys of a V chunk
    constexpr int SLOTS = slots<HDP>();
    constexpr int TILES = q_tiles<HDP>();
    const int group = p.nh / p.nkv, kvh = blockIdx.x % p.nkv;
    SeqTile st;
    // the last tiles of a sequence see the most keys: they start first, all heads of a tile together
    if (!find_tile(p, (gridDim.x - 1 - blockIdx.x) / p.nkv, TILES * tile_tokens * group, group, st)) return;
    const int i0 = st.tile * TILES * tile_tokens;             // first query of the block
    const int shift = st.k_len - st.q_len;
    const int last_i = min(st.q_len, i0 + TILES * tile_tokens) - 1;
    const bool two = TILES == 2 && i0 + tile_tokens < st.q_len;  // two query tiles, or one with two S buffers
    const KeyTiles kt = key_tiles(p, st, i0, last_i, KT);
    const int n = kt.count;

    extern __shared__ __align__(1024) uint8_t smem[];  // whole swizzle patterns of 1024 bytes
    uint8_t* ring = smem + TILES * q_bytes<HDP>();
    Bars* bars = reinterpret_cast<Bars*>(ring + SLOTS * SLOT);
    volatile uint32_t* abort_flag = &bars->abort_flag;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        mbar_init(&bars->q_full, 1);
        for (int s = 0; s < SLOTS; ++s) {
            mbar_init(&bars->full[s], 1);
            mbar_init(&bars->empty[s], 1);
        }
        for (int x = 0; x < 2; ++x) {
            mbar_init(&bars->s_full[x], 1);
            mbar_init(&bars->p_full[x], 4);
            mbar_init(&bars->o_done[x], 1);
            for (int w = 0; w < 4; ++w) mbar_init(&bars->ref_full[x][w], 1);
        }
        bars->abort_flag = 0;
        mbar_fence_init();
        tma_prefetch_desc(&tm_q);
        tma_prefetch_desc(&tm_k);
        tma_prefetch_desc(&tm_v);
    }
    if (warp == 1) {
        tmem_alloc(&bars->tmem_base, 512);
        tmem_relinquish();
    }
    // rows of a tile that the group does not fill (128 = 42 x 3 + 2) hold zeros: their scores need no mask
    const int used = tile_tokens * group;
    for (int i = threadIdx.x; i < (QT - used) * 8 * NC * TILES; i += THREADS)
        *reinterpret_cast<uint4*>(smem + (i / ((QT - used) * 8)) * (QT * 128) + used * 128 + (i % ((QT - used) * 8)) * 16) = make_uint4(0u, 0u, 0u, 0u);
    for (int i = threadIdx.x; i < QT; i += THREADS) bars->bad[i] = 0;
    fence_proxy_async_smem();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = bars->tmem_base;
    const uint32_t o_col = 256;

    if (warp == 0) {
        // ---------------- TMA producer ----------------
        if (n > 0 && elect_one()) {
            const int tiles = two ? 2 : 1;
            mbar_expect_tx(&bars->q_full, (uint32_t)(tiles * NC * tile_tokens * group * 128));
            for (int t = 0; t < tiles; ++t)
                for (int c = 0; c < NC; ++c)
                    load_3d(smem + t * q_bytes<HDP>() + c * QT * 128, &tm_q, &bars->q_full, c * 64, kvh * group,
                            (int)st.q0 + i0 + t * tile_tokens);
            uint32_t it = 0;
            auto slot = [&](uint32_t& s) {
                s = it % SLOTS;
                const bool ok = mbar_wait<100>(&bars->empty[s], ((it / SLOTS) & 1u) ^ 1u, abort_flag, 1);
                if (ok) mbar_expect_tx(&bars->full[s], SLOT);
                ++it;
                return ok;
            };
            auto load_k = [&](int j) {
                for (int c = 0; c < NC; ++c) {
                    uint32_t s;
                    if (!slot(s)) return false;
                    load_3d(ring + s * SLOT, &tm_k, &bars->full[s], c * 64, kvh, (int)st.k0 + kt.at(j) * KT);
                }
                return true;
            };
            auto load_v = [&](int j) {
                for (int c = 0; c < NC; ++c) {
                    uint32_t s;
                    if (!slot(s)) return false;
                    for (int d = 0; d < NC; ++d)
                        load_3d(ring + s * SLOT + d * VK * 128, &tm_v, &bars->full[s], d * 64, kvh, (int)st.k0 + kt.at(j) * KT + c * VK);
                }
                return true;
            };
            // in the order in which the MMA warp uses them
            if (two) {
                for (int j = 0; j < n; ++j)
                    if (!load_k(j) || !load_v(j)) break;
            } else if (load_k(0)) {
                for (int j = 0; j < n; ++j)
                    if ((j + 1 < n && !load_k(j + 1)) || !load_v(j)) break;
            }
        }
    } else if (warp == 1) {
        // ---------------- MMA issuer ----------------
        if (n > 0) {
            const bool leader = elect_one();
            const uint32_t idesc_s = idesc16<T>(KT, false), idesc_o = idesc16<T>((uint32_t)(p.hd + 15) / 16 * 16, true);
            const int ksteps = (p.hd + 15) / 16;
            const int steps = two ? 2 * n : n;
            auto k_index = [&](int j) { return (uint32_t)((two ? 2 * j : j == 0 ? 0 : 2 * j - 1) * NC); };
            auto v_index = [&](int j) { return (uint32_t)((two ? 2 * j + 1 : j < n - 1 ? 2 * j + 2 : 2 * n - 1) * NC); };
            // The thread that issues runs alone, an instruction every few clocks, and a product of 128 x 128 x 16 takes 64:
            // descriptors are made once and stepped by adding to their address field (16-byte units, 14 bits).
            const uint64_t q_desc = smem_desc_kmajor(smem_u32(smem), 128), k_desc = smem_desc_kmajor(smem_u32(ring), 128),
                           v_desc = smem_desc_mn(smem_u32(ring), VK * 128);
            const bool whole = ksteps == HDP / 16;
            // The warp stays together, waits included (descriptors live in uniform registers, which lanes that run
            // apart would share); only the products and commits are the leader's.
            auto arrived = [&](uint64_t* bar, uint32_t parity, uint32_t site) {
                return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, site)) != 0;
            };
            auto landed = [&](uint32_t index) {
#pragma unroll
                for (uint32_t i = 0; i < NC; ++i)
                    if (!arrived(&bars->full[(index + i) % SLOTS], ((index + i) / SLOTS) & 1u, 2)) return false;
                return true;
            };
            auto issue_s = [&](int u) {
                const int j = two ? u >> 1 : u, x = u & 1;
                const bool last_use = !two || x == 1;  // the second query tile comes behind the first
                const uint64_t qd = q_desc + (two ? x : 0) * (q_bytes<HDP>() >> 4);
                const uint32_t d = tmem + x * 128, index = k_index(j);
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    const uint32_t s = (index + c) % SLOTS;
                    const uint64_t kd = k_desc + s * (SLOT >> 4);
                    if (leader) {
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            if (whole || 4 * c + k < ksteps) mma_ss(d, qd + c * (QT * 128 >> 4) + k * 2, kd + k * 2, idesc_s, (c | k) != 0);
                        if (last_use) tc_commit(&bars->empty[s]);
                    }
                }
                if (leader) tc_commit(&bars->s_full[x]);
                __syncwarp();
            };
            auto issue_o = [&](int u) {
                const int j = two ? u >> 1 : u, x = u & 1;
                const bool last_use = !two || x == 1;
                const uint32_t d = tmem + o_col + (two ? x * 128 : 0), a = tmem + x * 128, index = v_index(j);
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    const uint32_t s = (index + c) % SLOTS;
                    const uint64_t vd = v_desc + s * (SLOT >> 4);
                    if (leader) {
#pragma unroll
                        for (int k = 0; k < VK / 16; ++k) {
                            if (c == 0 && k == 0) mma_ts(d, a, vd, idesc_o, j != 0);
                            else mma_ts(d, a + (c * VK + k * 16) / 2, vd + k * (2048 >> 4), idesc_o, 1u);
                        }
                        if (last_use) tc_commit(&bars->empty[s]);
                    }
                }
                if (leader) tc_commit(&bars->o_done[x]);
                __syncwarp();
            };
            bool ok = arrived(&bars->q_full, 0, 4) && landed(k_index(0));
            tc_fence_after();
            if (ok) issue_s(0);
            if (ok && steps > 1) {
                ok = two || landed(k_index(1));
                if (ok) issue_s(1);
            }
            for (int u = 0; ok && u < steps; ++u) {
                const int j = two ? u >> 1 : u;
                // what this step needs from memory, while the softmax is still at work on its P
                if (!two || (u & 1) == 0) {
                    ok = landed(v_index(j)) && (u + 2 >= steps || landed(k_index(two ? j + 1 : j + 2)));
                    if (!ok) break;
                    const int seen = shift + last_i + 1 - kt.at(j) * KT;  // keys of this tile that some row of the block sees
                    if (seen < KT) {
                        for (int c = 0; c < NC; ++c) {
                            uint8_t* slot = ring + (v_index(j) + c) % SLOTS * SLOT;
                            const int r0 = max(0, min(VK, seen - c * VK)), units = (VK - r0) * 8;  // 16-byte pieces of a group of 64 dims
                            for (int g = 0; g < NC; ++g)
                                for (int i = lane; i < units; i += 32) *reinterpret_cast<uint4*>(slot + g * VK * 128 + r0 * 128 + i * 16) = make_uint4(0u, 0u, 0u, 0u);
                        }
                        fence_proxy_async_smem();
                        __syncwarp();
                    }
                }
                ok = arrived(&bars->p_full[u & 1], (u >> 1) & 1u, 5);
                if (!ok) break;
                tc_fence_after();
                issue_o(u);
                if (u + 2 < steps) issue_s(u + 2);
            }
        }
    } else {
        // ---------------- softmax warps: group x of four warps owns stream x ----------------
        // Two query tiles: every key tile of query tile x.  One query tile: every other key tile; the reference of
        // the exponentials, which both groups' P must share, goes from one to the other through shared memory as soon as a
        // group knows the maximum of its tile, so that one group's exponentials run beside the other's maximum.
        const int x = (warp - 2) >> 2;
        const int quarter = warp & 3, r = quarter * 32 + lane;
        const uint32_t lane_addr = (uint32_t)(quarter * 32) << 16;
        const int qi = i0 + (two ? x * tile_tokens : 0) + r / group;  // query of this row
        const bool live = r < used && qi < st.q_len;
        const int pos = live ? shift + qi : -1;
        const uint32_t s_at = tmem + lane_addr + x * 128, o_at = tmem + lane_addr + o_col + (two ? x * 128 : 0);
        const float c = p.scale * LOG2E, cap2 = p.softcap * LOG2E, to_y = CAP ? p.scale / p.softcap : 0.0f;
        // Soft cap: where all scores of a warp's rows lie in cap_tanh's polynomial range, its coefficients for a score s instead
        // of y = s to_y, times cap log2(e), leave seven packed instructions for the exponents of two scores
        float cap_c[6] = {1.0f, -0.3333296776f, 0.1332551539f, -0.0533498190f, 0.0195937864f, -0.0047239522f};
        auto tanh_of = [](float y) { return CAP == CAP_NEAR ? cap_tanh_far(y) : cap_tanh(y); };
        if (CAP) {
            float f = cap2 * to_y;
#pragma unroll
            for (int k = 0; k < 6; ++k, f *= to_y * to_y) cap_c[k] *= f;
        }
        const int step = two ? 1 : 2;
        float m_ref = -INFINITY;                  // reference of O: exponents are s - m_ref
        float l = 0.0f, l_ref = -INFINITY;        // this thread's part of the row sum and its reference
        bool bad = false, ok = true;
        for (int j = two ? 0 : x; j < n; j += step) {
            const uint32_t ph = (uint32_t)(two ? j : j >> 1) & 1u;
            // the lanes leave a polling loop one by one: tcgen05.ld wants the warp together
            if (!__all_sync(0xffffffffu, mbar_wait<20>(&bars->s_full[x], ph, abort_flag, 6))) { ok = false; break; }
            tc_fence_after();
            uint32_t v[4][32];
#pragma unroll
            for (int ch = 0; ch < 4; ++ch) tmem_ld_x32(s_at + ch * 32, v[ch]);
            tc_wait_ld();
            const int j0 = kt.at(j) * KT;
            const bool whole = r >= used || (j0 + KT - 1 <= pos && ((int64_t)pos - j0 < p.window || j0 + KT <= p.sinks));
            const bool masked = __any_sync(0xffffffffu, !whole);
            if (masked) {
#pragma unroll
                for (int ch = 0; ch < 4; ++ch) {
                    const uint32_t bits = r >= used ? 0xffffffffu : seen_bits(p, pos, j0 + ch * 32);
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        if (!(bits >> i & 1u)) v[ch][i] = 0xff800000u;
                }
            }
            float mxs[8];
#pragma unroll
            for (int a = 0; a < 8; ++a) mxs[a] = -INFINITY;
#pragma unroll
            for (int ch = 0; ch < 4; ++ch)
#pragma unroll
                for (int i = 0; i < 32; i += 2)
                    mxs[(i >> 1) & 7] = max3_nan(mxs[(i >> 1) & 7], __uint_as_float(v[ch][i]), __uint_as_float(v[ch][i + 1]));
            const float mx = max_nan(max3_nan(max3_nan(mxs[0], mxs[1], mxs[2]), mxs[3], mxs[4]), max3_nan(mxs[5], mxs[6], mxs[7]));
            bool small = false;  // every score of the warp's rows lies where the polynomial holds (a masked tile's do not)
            if (CAP) {
                float mns[4] = {INFINITY, INFINITY, INFINITY, INFINITY};
#pragma unroll
                for (int ch = 0; ch < 4; ++ch)
#pragma unroll
                    for (int i = 0; i < 32; i += 2)
                        mns[(i >> 1) & 3] = fminf(mns[(i >> 1) & 3], fminf(__uint_as_float(v[ch][i]), __uint_as_float(v[ch][i + 1])));
                small = __all_sync(0xffffffffu, (CAP == CAP_NEAR || to_y <= 1e3f) && fmaxf(mx, -fminf(fminf(mns[0], mns[1]), fminf(mns[2], mns[3]))) * to_y <= TANH_POLY_MAX);
            }
            // the cap keeps the order: the largest capped score is the capped largest score
            const float m_cand = !CAP ? mx * c : mx == -INFINITY ? mx : cap2 * tanh_of(mx * to_y);
            bad = bad || m_cand != m_cand;
            if (!two && j > 0) {
                if (!__all_sync(0xffffffffu, mbar_wait(&bars->ref_full[x ^ 1][quarter], (uint32_t)((j - 1) >> 1) & 1u, abort_flag, 9))) { ok = false; break; }
                m_ref = bars->ref[r];
            }
            const bool moved = m_cand > m_ref + 8.0f || (m_ref == -INFINITY && m_cand > -INFINITY);
            const float alpha = moved ? ex2_approx(m_ref - m_cand) : 1.0f;
            if (moved) m_ref = m_cand;
            if (!two) {
                bars->ref[r] = m_ref;
                __syncwarp();
                if (lane == 0) mbar_arrive(&bars->ref_full[x][quarter]);
            }
            if (j > 0 && __any_sync(0xffffffffu, moved)) {
                // P V of the query tile's previous key tile has to be in O (with two query tiles S(j) was issued
                // behind it, with two S buffers before it); the next one waits for this warp's P
                if (!__all_sync(0xffffffffu, mbar_wait(&bars->o_done[two ? x : x ^ 1], (uint32_t)(two ? j - 1 : (j - 1) >> 1) & 1u, abort_flag, 7))) {
                    ok = false;
                    break;
                }
                tc_fence_after();
#pragma unroll 1
                for (int ch = 0; ch < (p.hd + 7) / 8; ++ch) {
                    uint32_t o[8];
                    tmem_ld_x8(o_at + ch * 8, o);
                    tc_wait_ld();
#pragma unroll
                    for (int i = 0; i < 8; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                    tmem_st_x8(o_at + ch * 8, o);
                }
            }
            if (l_ref != m_ref) {
                l *= ex2_approx(l_ref - m_ref);
                l_ref = m_ref;
            }
            const float ref = m_ref == -INFINITY ? 0.0f : m_ref;
            const uint64_t c2 = pack_f32x2(c, c), nm2 = pack_f32x2(-ref, -ref);
            uint64_t sums[4] = {0ull, 0ull, 0ull, 0ull};
            // exponents of two scores -> weights, their sum and P; one straight run of code for either form of the cap
            auto weights = [&](auto exponent) {
#pragma unroll
                for (int ch = 0; ch < 4; ++ch) {
                    uint32_t pk[16];
#pragma unroll
                    for (int i = 0; i < 32; i += 2) {
                        float t0, t1, e0, e1;
                        unpack_f32x2(exponent(pack_f32x2(__uint_as_float(v[ch][i]), __uint_as_float(v[ch][i + 1]))), t0, t1);
                        if ((((i >> 1) & 7) * POLY_OF_8) % 8 < POLY_OF_8) {
                            ex2_poly_x2<true>(t0, t1, e0, e1);
                        } else {
                            e0 = ex2_approx(t0);
                            e1 = ex2_approx(t1);
                        }
                        sums[(i >> 1) & 3] = add_f32x2(sums[(i >> 1) & 3], pack_f32x2(e0, e1));
                        pk[i >> 1] = pack2<T>(e0, e1);
                    }
                    tmem_st_x16(s_at + ch * 16, pk);
                }
            };
            if (!CAP) {
                weights([&](uint64_t sv) { return fma_f32x2(sv, c2, nm2); });
            } else if (small) {
                weights([&](uint64_t sv) {  // seven instructions for two scores: s P'(s^2) - ref
                    const uint64_t z = mul_f32x2(sv, sv);
                    uint64_t q = pack_f32x2(cap_c[5], cap_c[5]);
#pragma unroll
                    for (int k = 4; k >= 0; --k) q = fma_f32x2(q, z, pack_f32x2(cap_c[k], cap_c[k]));
                    return fma_f32x2(sv, q, nm2);
                });
            } else {
#pragma unroll
                for (int ch = 0; ch < 4; ++ch) {
                    const uint32_t bits = r >= used || !masked ? 0xffffffffu : seen_bits(p, pos, j0 + ch * 32);
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        v[ch][i] = bits >> i & 1u ? __float_as_uint(tanh_of(__uint_as_float(v[ch][i]) * to_y) * cap2) : 0xff800000u;
                }
                weights([&](uint64_t sv) { return add_f32x2(sv, nm2); });
            }
            tc_wait_st();
            {
                float s0, s1;
                unpack_f32x2(add_f32x2(add_f32x2(sums[0], sums[1]), add_f32x2(sums[2], sums[3])), s0, s1);
                l += s0 + s1;
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars->p_full[x]);
        }
        if (!two) {
            // The groups' parts of the row sum meet; all eight warps get here whether or not a wait gave up.
            bars->part[x][r] = make_float2(l, l_ref);
            if (bad) bars->bad[r] = 1;
            asm volatile("bar.sync 1, 256;" ::: "memory");
            const float2 other = bars->part[x ^ 1][r];
            const float m = fmaxf(l_ref, other.y);  // the later of the two: a reference only grows
            l = (l_ref == m ? l : l * ex2_approx(l_ref - m)) + (other.y == m ? other.x : other.x * ex2_approx(other.y - m));
            bad = bars->bad[r] != 0;
        }
        if (n > 0 && ok) {
            const int last = two ? x : (n - 1) & 1;
            ok = __all_sync(0xffffffffu, mbar_wait(&bars->o_done[last], (uint32_t)(two ? n - 1 : (n - 1) >> 1) & 1u, abort_flag, 8)) != 0;
        }
        if (ok) {
            tc_fence_after();
            const float inv = pos >= 0 ? 1.0f / l : 0.0f;
            T* dst = static_cast<T*>(const_cast<void*>(p.out.p)) + (st.q0 + qi) * p.out.row + (int64_t)(kvh * group + r % group) * p.out.head;
            // one query tile: each group writes half of the row
            const int chunks = (p.hd + 15) / 16, half = (chunks + 1) / 2;
            const int ch0 = two || x == 0 ? 0 : half, ch1 = two || x == 1 ? chunks : half;
            for (int ch = ch0; ch < ch1; ++ch) {
                uint32_t o[16];
                __syncwarp();  // the stores below leave lanes apart, tcgen05.ld wants the warp together
                if (n > 0) {
                    tmem_ld_x16(o_at + ch * 16, o);
                    tc_wait_ld();
                }
                float f[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    f[i] = pos >= 0 && n > 0 ? __uint_as_float(o[i]) * inv : 0.0f;  // a query that sees no key: zeros
                    bad = bad || !isfinite(f[i]);
                }
                if (live) {
                    if (out_vec) {
                        *reinterpret_cast<uint4*>(dst + ch * 16) = pack16<T>(f);
                        if (ch * 16 + 8 < p.hd) *reinterpret_cast<uint4*>(dst + ch * 16 + 8) = pack16<T>(f + 8);
                    } else {
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            if (ch * 16 + i < p.hd) dst[ch * 16 + i] = from_f32<T>(f[i]);
                    }
                }
            }
            if (!two) {
                // either group may have found the row bad; both have written their halves when one computes it again
                if (bad) bars->bad[r] = 1;
                asm volatile("bar.sync 1, 256;" ::: "memory");
                bad = x == 0 && bars->bad[r] != 0;
            }
            unsigned redo = __ballot_sync(0xffffffffu, bad && pos >= 0);
            __syncwarp();
            for (; redo; redo &= redo - 1) redo_row<T>(p, st, kvh, (i0 + (two ? x * tile_tokens : 0)) * group + quarter * 32 + __ffs(redo) - 1);
        } else if (!two) {
            asm volatile("bar.sync 1, 256;" ::: "memory");  // the other group may wait here
        }
    }

    tc_fence_before();
    __syncthreads();
    drain_copies(abort_flag);
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
    if (threadIdx.x == 0 && bars->abort_flag) atomicCAS(p.status, 0u, 0x900u | bars->abort_flag);
}

template <typename T, int HDP, int POLY, Cap CAP>
int launch_form(const CUtensorMap& tm_q, const CUtensorMap& tm_k, const CUtensorMap& tm_v, const WindowAttnParams& p, int tile_tokens, cudaStream_t s) {
    static std::atomic<bool> configured[64];
    int dev = 0;
    CMFC_CUDA(cudaGetDevice(&dev));
    auto kernel = window_prefill_kernel<T, HDP, POLY, CAP>;
    if (!configured[dev & 63]) {
        CMFC_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes<HDP>()));
        configured[dev & 63] = true;
    }
    const int out_vec = !(reinterpret_cast<uintptr_t>(p.out.p) & 15) && p.out.row % 8 == 0 && p.out.head % 8 == 0 && p.hd % 8 == 0;
    const int64_t blocks = p.q_rows / (q_tiles<HDP>() * tile_tokens) + p.seqs;
    kernel<<<(unsigned)(blocks * p.nkv), THREADS, smem_bytes<HDP>(), s>>>(tm_q, tm_k, tm_v, p, tile_tokens, out_vec);
    CMFC_CUDA(cudaGetLastError());
    return OK;
}
template <typename T, int HDP>
int launch_hdp(const CUtensorMap& tm_q, const CUtensorMap& tm_k, const CUtensorMap& tm_v, const WindowAttnParams& p, int tile_tokens, cudaStream_t s) {
    constexpr int POLY = HDP <= 128 ? 2 : 0;
    switch (cap_form(p)) {
        case NO_CAP: return launch_form<T, HDP, POLY, NO_CAP>(tm_q, tm_k, tm_v, p, tile_tokens, s);
        case CAP_NEAR: return launch_form<T, HDP, POLY, CAP_NEAR>(tm_q, tm_k, tm_v, p, tile_tokens, s);
        default: return launch_form<T, HDP, POLY, CAP_ANY>(tm_q, tm_k, tm_v, p, tile_tokens, s);
    }
}
template <typename T>
int launch_typed(const CUtensorMap& tm_q, const CUtensorMap& tm_k, const CUtensorMap& tm_v, const WindowAttnParams& p, int tile_tokens, cudaStream_t s) {
    if (p.hd <= 64) return launch_hdp<T, 64>(tm_q, tm_k, tm_v, p, tile_tokens, s);
    if (p.hd <= 128) return launch_hdp<T, 128>(tm_q, tm_k, tm_v, p, tile_tokens, s);
    return launch_hdp<T, 256>(tm_q, tm_k, tm_v, p, tile_tokens, s);
}

}  // namespace

bool window_prefill_supported(const WindowAttnParams& p, int elem) {
    constexpr int64_t MOST = (int64_t)1 << 38;  // strides of a tensor map stay below 2^40 bytes
    // TMA: 16-byte aligned bases and strides (and no broadcast ones); the softmax takes its row maximum before
    // it scales, so the scale must be positive
    auto fits = [&](const HeadView& v, int heads) {
        return !(reinterpret_cast<uintptr_t>(v.p) & 15) && v.row > 0 && v.row < MOST && v.row % 8 == 0 &&
               (heads == 1 || (v.head > 0 && v.head < MOST && v.head % 8 == 0));
    };
    const int64_t group = p.nh / p.nkv;
    return elem != ET_F32 && p.scale > 0.0f && p.k_rows > 0 && group <= QT && (p.q_rows / (QT / group) + p.seqs) * p.nkv < ((int64_t)1 << 31) &&
           fits(p.q, p.nh) && fits(p.k, p.nkv) && fits(p.v, p.nkv);
}

int launch_window_prefill(const WindowAttnParams& p, int elem, cudaStream_t s) {
    const int group = p.nh / p.nkv, tile_tokens = QT / group;
    const int hdp = p.hd <= 64 ? 64 : p.hd <= 128 ? 128 : 256;
    CUtensorMap tm_q, tm_k, tm_v;
    // [rows, heads, hd] views; a single head's stride is never used
    auto map = [&](CUtensorMap* m, const HeadView& v, int64_t rows, int heads, int box_heads, int box_rows) {
        return make_tensor_map_heads16(m, v.p, (uint64_t)p.hd, (uint64_t)heads, (uint64_t)rows, (uint64_t)(heads == 1 ? v.row : v.head) * 2,
                                       (uint64_t)v.row * 2, 64, (uint32_t)box_heads, (uint32_t)box_rows);
    };
    if (map(&tm_q, p.q, p.q_rows, p.nh, group, tile_tokens) != OK || map(&tm_k, p.k, p.k_rows, p.nkv, 1, KT) != OK ||
        map(&tm_v, p.v, p.k_rows, p.nkv, 1, SLOT / (hdp * 2)) != OK)
        return launch_window_any(p, elem, s);  // a layout that no tensor map describes
    if (elem == ET_F16) return launch_typed<__half>(tm_q, tm_k, tm_v, p, tile_tokens, s);
    return launch_typed<__nv_bfloat16>(tm_q, tm_k, tm_v, p, tile_tokens, s);
}

}  // namespace cmfc
