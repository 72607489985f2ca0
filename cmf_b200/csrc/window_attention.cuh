// Shared by the windowed-attention kernels: which rows and keys a block works on, the mask and the score.
#pragma once
#include <algorithm>

#include "text_ops.cuh"

namespace cmfc {

int launch_window_any(const WindowAttnParams& p, int elem, cudaStream_t s);
bool window_prefill_supported(const WindowAttnParams& p, int elem);
int launch_window_prefill(const WindowAttnParams& p, int elem, cudaStream_t s);
bool window_f32_supported(const WindowAttnParams& p, int elem);
int launch_window_f32(const WindowAttnParams& p, int num_sms, cudaStream_t s);
bool window_tokens_supported(const WindowAttnParams& p, int elem);
int launch_window_tokens(const WindowAttnParams& p, int elem, int num_sms, cudaStream_t s);

// Upper bound of the row tiles of all sequences: every sequence adds at most one partial tile.
inline int64_t max_tiles(const WindowAttnParams& p, int rows_per_tile) {
    return p.q_rows * (p.nh / p.nkv) / rows_per_tile + p.seqs;
}

// The lengths are on the device: where a launch is cut by how much there is to do, the host goes by the tensors' sizes
// and the window, and a wrong guess costs time only.
inline int64_t window_items(const WindowAttnParams& p, int rows_per_tile) {  // row tiles x key heads
    return std::max<int64_t>(1, (p.q_rows * (p.nh / p.nkv) / p.seqs + rows_per_tile - 1) / rows_per_tile) * p.seqs * p.nkv;
}
inline int64_t window_range(const WindowAttnParams& p) {  // keys of a row
    return std::min<int64_t>((int64_t)p.window + p.sinks, std::max<int64_t>(1, p.k_rows / p.seqs));
}

// Few rows: the single-token kernels (tiles of 4 or 16 rows, the key axis cut); many: the prompt kernels (tiles of 64 or 128
// rows over all keys).  A prompt tile costs the same for one row as for all, so the former win up to 16 rows a sequence, and
// longer where 16-row tiles are no more than the SMs: there prompt tiles leave most of them idle.  us, single-token kernel / prompt kernel:
//                                            bf16                          f32
//   sequences x key heads x dims x keys      16 rows   24 rows   128 rows  16 rows     24 rows     128 rows
//   64 x 8 x 128 x 2048                      94 / 122  136 / 123 442 / 130 626 / 1151  928 / 1152  4737 / 2000
//   64 x 4 x 256 x 1024                      63 / 60   96 / 60   338 / 68  440 / 534   688 / 535   3481 / 1074
//   8 x 8 x 64 x 4096                        18 / 47   25 / 47   79 / 40   130 / 368   228 / 368   882 / 608
//   1 x 8 x 128 x 8192                       16 / 93   22 / 93   35 / 91   58 / 1139   76 / 1139   397 / 1141
inline bool window_few_rows(const WindowAttnParams& p, int num_sms) {
    return p.q_rows * (p.nh / p.nkv) <= 16 * (int64_t)p.seqs || window_items(p, 16) <= num_sms;
}

// Soft caps of the 16-bit forms.  Ordinary ones take tanh from one quotient, off by up to 2 x 2^-24 of the cap: 3e-5 at 256, far
// below a rounding of the weights (prompts: outside the range of a polynomial whose coefficients hold powers of scale /
// cap, which must stay f32 numbers).  Others go by the size of each score.  us, ordinary / any: 8192 tokens, 8 / 4 heads of
// 256 303 / 343; 64 tokens over 4096 keys x 4 heads of 256 160 / 169.
enum Cap { NO_CAP, CAP_NEAR, CAP_ANY };
inline Cap cap_form(const WindowAttnParams& p) {
    return !(p.softcap > 0.0f) ? NO_CAP : p.softcap <= 256.0f && p.scale <= 1e3f * p.softcap ? CAP_NEAR : CAP_ANY;
}

#ifdef __CUDACC__

struct SeqTile {
    int64_t q0, k0;     // first query row, first key row
    int q_len, k_len;
    int tile;           // row tile inside the sequence
};

// The caller's offsets are device data that the host never sees: they are clamped to the tensors, so a
// wrong value can give wrong results but no access out of range.
__device__ __forceinline__ void load_seq(const WindowAttnParams& p, int s, SeqTile& st) {
    if (!p.q_start) {
        st.q0 = st.k0 = 0;
        st.q_len = (int)p.q_rows;
        st.k_len = (int)p.k_rows;
        return;
    }
    const int64_t a = min(max((int64_t)p.q_start[s], (int64_t)0), p.q_rows);
    const int64_t b = min(max((int64_t)p.q_start[s + 1], a), p.q_rows);
    st.q0 = a;
    st.q_len = (int)(b - a);
    st.k0 = min(max((int64_t)p.k_start[s], (int64_t)0), p.k_rows);
    st.k_len = (int)min(max((int64_t)p.k_len[s], (int64_t)0), p.k_rows - st.k0);
}

// Sequence and row tile of number `index` in the row tiles of all sequences: every warp counts the tiles
// of 32 sequences at a time.  False: there is no such tile (the grid is an upper bound).
__device__ __forceinline__ bool find_tile(const WindowAttnParams& p, int64_t index, int rows_per_tile, int group, SeqTile& st) {
    const int lane = threadIdx.x & 31;
    int64_t before = 0;
    for (int s0 = 0; s0 < p.seqs; s0 += 32) {
        SeqTile mine;
        mine.q_len = 0;
        if (s0 + lane < p.seqs) load_seq(p, s0 + lane, mine);
        const int64_t tiles = ((int64_t)mine.q_len * group + rows_per_tile - 1) / rows_per_tile;
        int64_t upto = tiles;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, index < before + upto);
        if (hit) {
            const int src = __ffs(hit) - 1;
            st.tile = (int)(index - (before + __shfl_sync(0xffffffffu, upto - tiles, src)));
            load_seq(p, s0 + src, st);
            return true;
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
    return false;
}

// Key tiles that some query of [first_i, last_i] sees: those of the sinks, then those of the window.
struct KeyTiles {
    int sink_tiles, low_tile, count;
    __device__ __forceinline__ int at(int it) const { return it < sink_tiles ? it : low_tile + (it - sink_tiles); }
};
__device__ __forceinline__ KeyTiles key_tiles(const WindowAttnParams& p, const SeqTile& st, int first_i, int last_i, int n) {
    KeyTiles kt;
    const int shift = st.k_len - st.q_len;
    const int first = shift + first_i, last = shift + last_i;  // positions; below 0: sees nothing
    if (last < 0) {
        kt.sink_tiles = kt.low_tile = kt.count = 0;
        return kt;
    }
    const int low = (int)max((int64_t)0, (int64_t)first - p.window + 1);  // first key of the earliest window
    kt.low_tile = low / n;
    const int sink_keys = min(p.sinks, low);
    kt.sink_tiles = min((sink_keys + n - 1) / n, kt.low_tile);
    kt.count = kt.sink_tiles + (last / n - kt.low_tile + 1);
    return kt;
}

__device__ __forceinline__ bool sees(const WindowAttnParams& p, int pos, int j) {
    return j <= pos && (pos - j < p.window || j < p.sinks);
}
__device__ __forceinline__ float score(float dot, float scale, float softcap) {
    const float s = dot * scale;
    return softcap > 0.0f ? softcap * tanhf(s / softcap) : s;
}

// tanh(y) for the 16-bit forms, relative error about 2^-22: up to |y| = 0.75 y P(y^2), P of degree 5 fitted to
// tanh(sqrt z) / sqrt z on [0, 0.5625] at Chebyshev points (3e-8, 1.1e-7 with f32 roundings; the quotient below would lose
// what a large cap makes of a small y); above 1 - 2 / (2^(2 y log2 e) + 1) on the special-function unit.
constexpr float TANH_POLY_MAX = 0.75f;
__device__ __forceinline__ float cap_tanh_far(float y) { return 1.0f - __fdividef(2.0f, ex2_approx(y * (2.0f * 1.4426950408889634f)) + 1.0f); }
__device__ __forceinline__ float cap_tanh(float y) {
    const float z = y * y;
    float q = -0.0047239522f;
    q = fmaf(q, z, 0.0195937864f);
    q = fmaf(q, z, -0.0533498190f);
    q = fmaf(q, z, 0.1332551539f);
    q = fmaf(q, z, -0.3333296776f);
    q = fmaf(q, z, 1.0f);
    return fabsf(y) <= TANH_POLY_MAX ? y * q : cap_tanh_far(y);
}

// One warp, one (query, head) row, key by key over exactly the keys that the row sees: rows whose tile
// result is not finite come here, so that an infinity or a NaN among keys or values that the row does not
// see cannot reach it, and one that it does see gives what the formula gives.
template <typename T>
__device__ __noinline__ void redo_row(const WindowAttnParams& p, SeqTile st, int kvh, int row) {
    const int lane = threadIdx.x & 31;
    const int group = p.nh / p.nkv;
    const int64_t qi = st.q0 + row / group;
    const int head = kvh * group + row % group;
    const int pos = st.k_len - st.q_len + row / group;
    const T* q = static_cast<const T*>(p.q.p) + qi * p.q.row + (int64_t)head * p.q.head;
    const T* k = static_cast<const T*>(p.k.p) + st.k0 * p.k.row + (int64_t)kvh * p.k.head;
    const T* v = static_cast<const T*>(p.v.p) + st.k0 * p.v.row + (int64_t)kvh * p.v.head;
    T* out = static_cast<T*>(const_cast<void*>(p.out.p)) + qi * p.out.row + (int64_t)head * p.out.head;
    float qv[8], acc[8], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int c = 0; c < 8; ++c) {
        qv[c] = lane + 32 * c < p.hd ? to_f32(q[lane + 32 * c]) : 0.0f;
        acc[c] = 0.0f;
    }
    const int low = (int)max((int64_t)0, (int64_t)pos - p.window + 1);
    for (int j = p.sinks > 0 ? 0 : low; j <= pos; ++j) {
        if (j >= p.sinks && j < low) j = low;
        float dot = 0.0f;
#pragma unroll
        for (int c = 0; c < 8; ++c)
            if (lane + 32 * c < p.hd) dot = fmaf(qv[c], to_f32(k[j * p.k.row + lane + 32 * c]), dot);
        const float s = score(warp_sum(dot), p.scale, p.softcap);
        const float mn = s != s ? s : fmaxf(m, s);  // a NaN score makes the row NaN
        const float alpha = mn == m ? 1.0f : expf(m - mn), e = s == -INFINITY ? 0.0f : expf(s - mn);
        m = mn;
        l = l * alpha + e;
#pragma unroll
        for (int c = 0; c < 8; ++c)
            if (lane + 32 * c < p.hd) acc[c] = acc[c] * alpha + e * to_f32(v[j * p.v.row + lane + 32 * c]);
    }
    const float inv = 1.0f / l;  // every score -inf: 0 / 0, NaN as the formula
#pragma unroll
    for (int c = 0; c < 8; ++c)
        if (lane + 32 * c < p.hd) out[lane + 32 * c] = from_f32<T>(acc[c] * inv);
}

#endif  // __CUDACC__

}  // namespace cmfc
