// 8-bit products on the tensor cores: y = (x w^T) scaled, on CTA pairs (tcgen05 kind::i8, cta_group::2).
//
// A tile of a pair is 256 weight rows x up to 256 tokens.  The weights are the A operand (M = 256, 128 rows in
// each CTA's shared memory), the tokens the B operand (N = 32 .. 256 in steps of 32, half of them staged by each CTA),
// so any number of tokens finds a tile of its own size: 333 tokens are two tiles of 192, not two of 256.  Both
// operands come by TMA (128 levels of k a stage, 128-byte swizzle) and the integer sums stay in tensor memory
// (128 lanes = weight rows, one column per token), two accumulators of 256 columns, so that a tile is
// drained while the next one is multiplied.
//   warp 0         TMA producer (both CTAs; the pair's bytes are counted on the even CTA's barrier)
//   warp 1         MMA issuer (even CTA)
//   warps 2 - 9    epilogue: tcgen05.ld, integer -> f32, both scales, rounded to the output type, 32 x 32 chunks staged
//                  in shared memory and written by TMA stores (plain stores where the output is not 16-byte aligned)
// Few tiles (a batch of some hundred tokens, a narrow matrix): the K axis is cut into 2 to 4 slices, one per
// pair of a cluster of 4 to 8 CTAs; the slices' integer sums meet over distributed shared memory in the
// stages' own space.  Integer sums are exact, so neither the cut nor the batch changes a bit of the result.
//
// Bound: the tensor pipe, and close behind it L2 -> SM (a 256 x 256 tile takes 64 KB per 128 levels of k, which at
// the full 8-bit rate is near the 64 bytes a clock that an SM can take).  Measured, bf16 out: 8704 x 18432 x 2304 244 us =
// 3030 TOP/s, 0.92 of twice the bf16 rate of a library product.
#include <cooperative_groups.h>

#include <algorithm>
#include <atomic>

#include "i8_gemm.cuh"

namespace cmfc {
namespace {

namespace cg = cooperative_groups;

constexpr int TW = 128;            // weight rows per CTA (256 per pair)
constexpr int TT = 256;            // most tokens of a tile
constexpr int BK = 128;            // levels of k per stage: one 128-byte swizzled row
constexpr int STAGES = 6;
constexpr int W_STAGE = TW * BK;       // 16 KiB
constexpr int X_STAGE = TT / 2 * BK;   // 16 KiB
constexpr int STAGE = W_STAGE + X_STAGE;
constexpr int EPI_WARPS = 8;
constexpr int THREADS = 32 * (2 + EPI_WARPS);
constexpr int CHUNK = 32 * 32 * 4;     // an epilogue warp's staged chunk: 32 tokens x 32 weight rows
constexpr int SMEM_BYTES = STAGES * STAGE + EPI_WARPS * CHUNK + 1024 + 256;
constexpr int TMEM_COLS = 512;
constexpr int MAX_SPLITS = 4;
constexpr uint32_t PEER_MASK = 0xFEFFFFFFu;  // clears the lowest CTA-rank bit of a shared::cluster address
static_assert(TT * TW * 4 <= STAGES * STAGE, "a slice's sums fit the space of the stages");

struct Bars {
    uint64_t full[STAGES];     // even CTA: both CTAs' halves of both operands have landed
    uint64_t empty[STAGES];    // the pair's MMAs of the stage are done (multicast commit)
    uint64_t acc_full[2];      // accumulator complete (multicast commit)
    uint64_t acc_empty[2];     // even CTA: both CTAs drained it
    uint32_t tmem_base;
    uint32_t abort_flag;
};

struct Plan {
    int tt;        // tokens per tile, a multiple of 32
    int tiles_m, tiles_n, kblocks, splits;
    int tma_out;
};

// kind::i8: S32 accumulator (2) at [4, 6), signed 8-bit A and B (1) at [7, 10) and [10, 13), N >> 3 at [17, 23), M >> 4 at [24, 29)
__device__ __forceinline__ uint32_t idesc_i8(uint32_t m, uint32_t n) {
    return (2u << 4) | (1u << 7) | (1u << 10) | ((n >> 3) << 17) | ((m >> 4) << 24);
}
__device__ __forceinline__ void mma_i8_pair(uint32_t d_tmem, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n"
        "}\n" ::"r"(d_tmem),
        "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void commit_pair(uint64_t* bar, uint16_t ctas) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)), "h"(ctas)
        : "memory");
}
__device__ __forceinline__ void arrive_even(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(smem_u32(bar) & PEER_MASK) : "memory");
}
__device__ __forceinline__ void load_pair(void* dst, const CUtensorMap* map, uint64_t* bar, int x, int y) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(smem_u32(dst)),
        "l"(map), "r"(smem_u32(bar) & PEER_MASK), "r"(x), "r"(y)
        : "memory");
}

// tiles of a launch, groups of eight token tiles under every weight tile: what runs at the same time
// shares its operands in L2
__device__ __forceinline__ void tile_at(const Plan& pl, int tile, int& tm, int& tn) {
    constexpr int G = 8;
    const int per = G * pl.tiles_n, g = tile / per, first = g * G;
    const int rows = min(G, pl.tiles_m - first), r = tile - g * per;
    tm = first + r % rows;
    tn = r / rows;
}

template <typename T>
__device__ __forceinline__ void store_one(const I8Params& p, int64_t m, int64_t n, int acc, float xs, float ws) {
    static_cast<T*>(p.y)[m * p.ldy + n] = from_f32<T>(i8_scaled(acc, xs, ws));
}

template <typename T>
__global__ void __launch_bounds__(THREADS, 1)
i8_pair_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w,
               const __grid_constant__ CUtensorMap tm_y, I8Params p, Plan pl) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* chunks = smem + STAGES * STAGE;
    Bars* bars = reinterpret_cast<Bars*>(chunks + EPI_WARPS * CHUNK);
    volatile uint32_t* abort_flag = &bars->abort_flag;
    cg::cluster_group cluster = cg::this_cluster();
    const int crank = (int)cluster.block_rank(), rank = crank & 1, slice = crank >> 1;
    const uint16_t both = (uint16_t)(3u << (crank & ~1));
    const int unit = blockIdx.x / (2 * pl.splits), units = gridDim.x / (2 * pl.splits);
    const int tiles = pl.tiles_m * pl.tiles_n;
    const int kb0 = (int)((int64_t)slice * pl.kblocks / pl.splits), kb1 = (int)((int64_t)(slice + 1) * pl.kblocks / pl.splits);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t xbytes = (uint32_t)(pl.tt / 2 * BK);

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&bars->full[s], 1);
            mbar_init(&bars->empty[s], 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(&bars->acc_full[a], 1);
            mbar_init(&bars->acc_empty[a], 2 * EPI_WARPS);
        }
        bars->abort_flag = 0;
        mbar_fence_init();
        tma_prefetch_desc(&tm_x);
        tma_prefetch_desc(&tm_w);
        if (pl.tma_out) tma_prefetch_desc(&tm_y);
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bars->tmem_base)), "r"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    cluster.sync();  // every barrier is initialised before anyone signals across the pair
    tc_fence_after();
    const uint32_t tmem = bars->tmem_base;
    wait_for_quantizer();

    if (warp == 0) {
        if (elect_one()) {
            uint32_t it = 0;
            for (int tile = unit; tile < tiles && !*abort_flag; tile += units) {
                int tm, tn;
                tile_at(pl, tile, tm, tn);
                const int n0 = tn * 2 * TW + rank * TW, m0 = tm * pl.tt + rank * (pl.tt / 2);
                for (int kb = kb0; kb < kb1; ++kb, ++it) {
                    const int s = it % STAGES;
                    if (!mbar_wait<100>(&bars->empty[s], ((it / STAGES) & 1u) ^ 1u, abort_flag, 1)) break;
                    if (rank == 0) mbar_expect_tx(&bars->full[s], 2 * (W_STAGE + xbytes));
                    load_pair(smem + s * STAGE, &tm_w, &bars->full[s], kb * BK, n0);
                    load_pair(smem + s * STAGE + W_STAGE, &tm_x, &bars->full[s], kb * BK, m0);
                }
            }
        }
    } else if (warp == 1) {
        if (rank == 0 && elect_one()) {
            const uint32_t idesc = idesc_i8(2 * TW, (uint32_t)pl.tt);
            uint32_t it = 0, ti = 0;
            for (int tile = unit; tile < tiles && !*abort_flag; tile += units, ++ti) {
                const uint32_t a = ti & 1u;
                if (!mbar_wait(&bars->acc_empty[a], ((ti >> 1) & 1u) ^ 1u, abort_flag, 2)) break;
                tc_fence_after();
                bool ok = true;
                for (int kb = kb0; kb < kb1; ++kb, ++it) {
                    const int s = it % STAGES;
                    if (!mbar_wait(&bars->full[s], (it / STAGES) & 1u, abort_flag, 3)) { ok = false; break; }
                    tc_fence_after();
                    const uint32_t ws = smem_u32(smem + s * STAGE), xs = ws + W_STAGE;
#pragma unroll
                    for (int j = 0; j < BK / 32; ++j)
                        mma_i8_pair(tmem + a * TT, smem_desc_kmajor(ws + j * 32, 128), smem_desc_kmajor(xs + j * 32, 128), idesc, kb != kb0 || j != 0);
                    commit_pair(&bars->empty[s], both);
                }
                if (!ok) break;
                commit_pair(&bars->acc_full[a], both);
            }
        }
    } else {
        const int quarter = warp & 3, ehalf = (warp - 2) >> 2;
        const uint32_t lane_addr = (uint32_t)(quarter * 32) << 16;
        T* stage = reinterpret_cast<T*>(chunks + (warp - 2) * CHUNK);
        int* sums = reinterpret_cast<int*>(smem);  // a slice's sums, [token][weight row], when K is cut
        bool pending = false;
        uint32_t ti = 0;
        for (int tile = unit; tile < tiles && !*abort_flag; tile += units, ++ti) {
            int tm, tn;
            tile_at(pl, tile, tm, tn);
            const uint32_t a = ti & 1u;
            if (!__all_sync(0xffffffffu, mbar_wait<40>(&bars->acc_full[a], (ti >> 1) & 1u, abort_flag, 4))) break;
            tc_fence_after();
            const int row = quarter * 32 + lane;
            const int64_t n = (int64_t)tn * 2 * TW + rank * TW + row;
            const float ws = n < p.N ? p.w_scale[n] : 0.0f;
            const int nchunks = pl.tt / 32;
            for (int c = ehalf; c < nchunks; c += 2) {
                uint32_t v[32];
                __syncwarp();  // the plain stores below leave lanes apart, tcgen05.ld wants the warp together
                tmem_ld_x32(tmem + lane_addr + a * TT + c * 32, v);
                tc_wait_ld();
                if (c + 2 >= nchunks) {  // this warp's last load of the accumulator
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) arrive_even(&bars->acc_empty[a]);
                }
                if (pl.splits > 1) {
#pragma unroll
                    for (int j = 0; j < 32; ++j) sums[(c * 32 + j) * TW + row] = (int)v[j];
                    continue;
                }
                const int64_t mb = (int64_t)tm * pl.tt + c * 32;
                if (mb >= p.M) continue;
                const float xs_lane = mb + lane < p.M ? p.x_scale[mb + lane] : 0.0f;
                if (pl.tma_out) {
                    if (pending) bulk_wait_group_read0();
                    __syncwarp();
#pragma unroll
                    for (int j = 0; j < 32; ++j)
                        stage[j * 32 + lane] = from_f32<T>(i8_scaled((int)v[j], __shfl_sync(0xffffffffu, xs_lane, j), ws));
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        tma_store_2d(&tm_y, stage, (int)(n - lane), (int)mb);
                        bulk_commit_group();
                        pending = true;
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 32; ++j) {
                        const float xs = __shfl_sync(0xffffffffu, xs_lane, j);
                        if (mb + j < p.M && n < p.N) store_one<T>(p, mb + j, n, (int)v[j], xs, ws);
                    }
                }
            }
            // with fewer chunks than warps a lane quarter's second warp loads nothing and still hands over
            if (ehalf >= nchunks) {
                __syncwarp();
                if (lane == 0) arrive_even(&bars->acc_empty[a]);
            }
        }
        if (pending) bulk_wait_group0();
    }

    tc_fence_before();
    __syncthreads();
    drain_copies(abort_flag);
    cluster.sync();  // the pair's MMAs and signals are done, and with a cut K every slice's sums are written
    if (pl.splits > 1) {
        // one tile per cluster: this CTA finishes the tokens of its slice's share for its 128 weight rows
        int tm, tn;
        tile_at(pl, unit, tm, tn);
        // (four rows a thread, four tokens in flight: the remote loads are what takes time here)
        const int row = lane * 4;
        const int64_t n = (int64_t)tn * 2 * TW + rank * TW + row;
        const int t0 = slice * pl.tt / pl.splits, t1 = (slice + 1) * pl.tt / pl.splits;
        const int4* part[MAX_SPLITS];
#pragma unroll
        for (int s = 0; s < MAX_SPLITS; ++s)
            part[s] = static_cast<const int4*>(cluster.map_shared_rank(static_cast<void*>(smem), (unsigned)(2 * (s < pl.splits ? s : 0) + rank))) + lane;
        float ws[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) ws[e] = n + e < p.N ? p.w_scale[n + e] : 0.0f;
        constexpr int FLY = 4;
        for (int tb = t0 + warp; tb < t1; tb += FLY * (THREADS / 32)) {
            int4 acc[FLY];
#pragma unroll
            for (int f = 0; f < FLY; ++f) {
                const int t = tb + f * (THREADS / 32);
                acc[f] = make_int4(0, 0, 0, 0);
#pragma unroll
                for (int s = 0; s < MAX_SPLITS; ++s)
                    if (s < pl.splits && t < t1) {
                        const int4 v = part[s][t * (TW / 4)];
                        acc[f].x += v.x;
                        acc[f].y += v.y;
                        acc[f].z += v.z;
                        acc[f].w += v.w;
                    }
            }
#pragma unroll
            for (int f = 0; f < FLY; ++f) {
                const int t = tb + f * (THREADS / 32);
                const int64_t m = (int64_t)tm * pl.tt + t;
                if (t >= t1 || m >= p.M) continue;
                const float xs = p.x_scale[m];
                const int a[4] = {acc[f].x, acc[f].y, acc[f].z, acc[f].w};
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (n + e < p.N) store_one<T>(p, m, n + e, a[e], xs, ws[e]);
            }
        }
        cluster.sync();  // nobody's shared memory goes away while another CTA reads it
    }
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
    }
    if (threadIdx.x == 0 && bars->abort_flag) atomicCAS(p.status, 0u, 0x800u | bars->abort_flag);
}

template <typename T>
int launch_typed(const I8Params& p, int num_sms, cudaStream_t stream) {
    static std::atomic<int> clusters_of[64][MAX_SPLITS + 1];  // co-resident clusters per split, a property of the device
    int dev = 0;
    CMFC_CUDA(cudaGetDevice(&dev));
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = SMEM_BYTES;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (!clusters_of[dev & 63][1]) {
        CMFC_CUDA(cudaFuncSetAttribute(i8_pair_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES));
        for (int s = MAX_SPLITS; s >= 1; --s) {
            attr[0].val.clusterDim.x = 2 * s;
            cfg.gridDim = dim3(2 * s);
            int n = 0;
            CMFC_CUDA(cudaOccupancyMaxActiveClusters(&n, i8_pair_kernel<T>, &cfg));
            clusters_of[dev & 63][s] = n > 0 ? n : 1;
        }
    }
    Plan pl;
    const int64_t tiles_m = (p.M + TT - 1) / TT, tiles_n = (p.N + 2 * TW - 1) / (2 * TW);
    pl.tiles_m = (int)tiles_m;
    pl.tiles_n = (int)tiles_n;
    pl.tt = (int)((((p.M + tiles_m - 1) / tiles_m) + 31) / 32 * 32);
    pl.kblocks = (int)((p.K + BK - 1) / BK);
    // K is cut as far as all tiles still run at once.  Joining the slices costs 2 us with few tokens a tile and 5 with many, a
    // stage of work 0.2 us.  us, cut / whole (tokens x weight rows x columns): 32 x 2304 x 1024 7.0 / 6.2, x 2304 7.4 / 7.6, x 9216
    // 11.4 / 19.2; 333 x 2304 x 2304 12.0 / 11.1, x 3456 12.9 / 13.3, x 9216 17.0 / 23.4; 512 x 2304 x 2304 13.8 / 12.9, x 9216 20.2 / 28.6
    const int64_t tiles = tiles_m * tiles_n;
    pl.splits = 1;
    for (int s = 2; s <= MAX_SPLITS; ++s)
        if (tiles <= clusters_of[dev & 63][s] && pl.kblocks >= 10 + pl.tt / 16) pl.splits = s;
    const int es = (int)elem_bytes(p.out_elem);
    pl.tma_out = pl.splits == 1 && !(reinterpret_cast<uintptr_t>(p.y) & 15) && (p.ldy * es) % 16 == 0;
    CUtensorMap tm_x, tm_w, tm_y;
    CMFC_TRY(make_tensor_map_2d(&tm_w, p.w, 1, (uint64_t)p.N, (uint64_t)p.K, (uint64_t)p.ldw, TW, BK, 3));
    CMFC_TRY(make_tensor_map_2d(&tm_x, p.x, 1, (uint64_t)p.M, (uint64_t)p.K, (uint64_t)p.ldx, pl.tt / 2, BK, 3));
    tm_y = tm_x;
    if (pl.tma_out) CMFC_TRY(make_tensor_map_2d(&tm_y, p.y, es, (uint64_t)p.M, (uint64_t)p.N, (uint64_t)p.ldy * es, 32, 32, 0));
    const int64_t most = pl.splits > 1 ? tiles : std::min<int64_t>(tiles, num_sms / 2);
    attr[0].val.clusterDim.x = 2 * pl.splits;
    cfg.gridDim = dim3((unsigned)(most * 2 * pl.splits));
    cfg.numAttrs = p.behind_quantizer ? 2 : 1;
    CMFC_CUDA(cudaLaunchKernelEx(&cfg, i8_pair_kernel<T>, tm_x, tm_w, tm_y, p, pl));
    return OK;
}

}  // namespace

int launch_i8_pair(const I8Params& p, int num_sms, cudaStream_t s) {
    if (p.out_elem == ET_F32) return launch_typed<float>(p, num_sms, s);
    if (p.out_elem == ET_F16) return launch_typed<__half>(p, num_sms, s);
    return launch_typed<__nv_bfloat16>(p, num_sms, s);
}

}  // namespace cmfc
