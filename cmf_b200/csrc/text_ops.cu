// C ABI of the text-layer operators (include/cmf_cuda.h): argument checks, then one or two launches on the
// caller's stream.  Nothing here allocates, synchronizes or keeps anything between calls, so the calls
// can be captured into a graph (after the device's context exists) and issued from several streams.
#include <limits.h>
#include <math.h>

#include "../../include/cmf_cuda.h"
#include "i8_gemm.cuh"
#include "runtime.h"
#include "text_ops.cuh"

using namespace cmfc;

namespace {

#define NEED(cond, msg) \
    if (!(cond)) return fail(ERR_BAD_ARG, msg)

static_assert(CMFC_ET_F32 == ET_F32 && CMFC_ET_F16 == ET_F16 && CMFC_ET_BF16 == ET_BF16, "element types of the header");

// counts stay a tile below 2^31, so that the end of the last tile is a number too
constexpr size_t MOST = (size_t)INT_MAX - 1023;

bool elem_ok(int e) { return e == ET_F32 || e == ET_F16 || e == ET_BF16; }

// Makes `device` current for the launches of one entry and puts the caller's device back; the device's
// context (SM count, status word) is created on its first use.
struct OnDevice {
    int before = -1;
    Context* c = nullptr;
    int enter(int device, cudaStream_t s) {
        CMFC_CUDA(cudaGetDevice(&before));
        if (before != device) {
            const cudaError_t e = cudaSetDevice(device);
            if (e != cudaSuccess) {
                before = -1;
                return fail(ERR_BAD_ARG, "no such CUDA device " + std::to_string(device));
            }
        }
        c = ctx_of_device(device, s);
        return c ? OK : ERR_CUDA;
    }
    ~OnDevice() {
        int now = -1;
        if (before >= 0 && cudaGetDevice(&now) == cudaSuccess && now != before) cudaSetDevice(before);
    }
};

void count_launches(Context* c, uint64_t n) { __atomic_fetch_add(&c->launches, n, __ATOMIC_RELAXED); }

// [rows, heads, hd] with these strides: do no two elements share an address?
bool distinct(int64_t rows, int64_t heads, int64_t hd, int64_t row, int64_t head) {
    if (rows == 0 || heads == 0) return true;
    if (rows > 1 && heads > 1) {
        const bool heads_inside = head <= row;
        const int64_t lo = heads_inside ? head : row, lo_n = heads_inside ? heads : rows, hi = heads_inside ? row : head;
        return lo >= hd && (hi - hd) / lo >= lo_n - 1;
    }
    if (rows > 1) return row >= hd;
    return heads <= 1 || head >= hd;
}
constexpr int64_t MAX_STRIDE = (int64_t)1 << 40;  // in a tensor that exists, rows x stride stays far below 2^63
bool stride_ok(int64_t s) { return s >= 0 && s < MAX_STRIDE; }

bool on_elements(const void* p, int elem) { return reinterpret_cast<uintptr_t>(p) % (size_t)elem_bytes(elem) == 0; }

template <class F>
int guarded(F f) {
    try {
        return f();
    } catch (...) {  // building a message can run out of memory; nothing may leave a C entry
        return ERR_OOM;
    }
}

int quantize_rows_impl(int device, const void* x, int elem, size_t rows, size_t cols, int64_t ldx, int8_t* q, int64_t ldq,
                       float* scale, cudaStream_t s) {
    NEED(elem_ok(elem), "quantize_rows: unknown element type");
    NEED(rows <= MOST && cols >= 1 && cols <= MOST, "quantize_rows: rows must be at most 2^31 - 1024, cols in [1, 2^31 - 1024]");
    if (rows == 0) return OK;
    NEED(x && q && scale, "quantize_rows: null pointer");
    NEED(on_elements(x, elem) && on_elements(scale, ET_F32), "quantize_rows: a pointer is off its element's boundary");
    NEED(stride_ok(ldx) && stride_ok(ldq) && (rows == 1 || (ldx >= (int64_t)cols && ldq >= (int64_t)cols)),
         "quantize_rows: a row pitch is shorter than a row");
    OnDevice on;
    CMFC_TRY(on.enter(device, s));
    CMFC_TRY(launch_quantize_rows(x, elem, (int64_t)rows, (int64_t)cols, ldx, q, ldq, scale, s));
    count_launches(on.c, 1);
    return OK;
}

int64_t up16(size_t v) { return (int64_t)((v + 15) / 16 * 16); }
// the pitch of a single row is never used: any that suits the aligned forms will do
int64_t pitch(size_t rows, size_t cols, int64_t ld) { return rows == 1 ? up16(cols) : ld; }

I8Params i8_params(const int8_t* wq, int64_t ldw, const float* ws, size_t b, size_t rows, size_t cols, void* y, int elem, int64_t ldy) {
    I8Params p = {};
    p.w = wq;
    p.w_scale = ws;
    p.y = y;
    p.ldw = pitch(rows, cols, ldw);
    p.ldy = pitch(b, rows, ldy);
    p.M = (int64_t)b;
    p.N = (int64_t)rows;
    p.K = (int64_t)cols;
    p.out_elem = elem;
    return p;
}

int i8_matmat_impl(int device, const int8_t* xq, int64_t ldx, const float* xs, const int8_t* wq, int64_t ldw, const float* ws,
                   size_t b, size_t rows, size_t cols, void* y, int elem, int64_t ldy, cudaStream_t s) {
    NEED(elem_ok(elem), "i8_matmat: unknown output type");
    NEED(b <= MOST && rows >= 1 && rows <= MOST, "i8_matmat: b must be at most 2^31 - 1024, rows in [1, 2^31 - 1024]");
    NEED(cols >= 1, "i8_matmat: cols must not be 0");
    if (cols > (size_t)I8_MAX_K) return fail(ERR_UNSUPPORTED, "i8_matmat: cols above 131071 could overflow the 32-bit sum");
    if (b == 0) return OK;
    NEED(xq && xs && wq && ws && y, "i8_matmat: null pointer");
    NEED(on_elements(xs, ET_F32) && on_elements(ws, ET_F32) && on_elements(y, elem), "i8_matmat: a pointer is off its element's boundary");
    NEED(stride_ok(ldx) && stride_ok(ldw) && stride_ok(ldy), "i8_matmat: bad row pitch");
    NEED((b == 1 || ldx >= (int64_t)cols) && (rows == 1 || ldw >= (int64_t)cols) && (b == 1 || ldy >= (int64_t)rows),
         "i8_matmat: a row pitch is shorter than a row");
    OnDevice on;
    CMFC_TRY(on.enter(device, s));
    I8Params p = i8_params(wq, ldw, ws, b, rows, cols, y, elem, ldy);
    p.x = xq;
    p.x_scale = xs;
    p.ldx = pitch(b, cols, ldx);
    p.status = on.c->status;
    CMFC_TRY(launch_i8_matmat(p, on.c->num_sms, s));
    count_launches(on.c, 1);
    return OK;
}

size_t i8_linear_workspace(const void* x, int elem, int64_t ldx, const int8_t* wq, int64_t ldw, size_t b, size_t rows, size_t cols) {
    if (b > MOST || cols > (size_t)I8_MAX_K || rows > MOST || !elem_ok(elem)) return 0;  // refused by the call itself
    const I8Params p = i8_params(wq, ldw, nullptr, b, rows, cols, nullptr, ET_F32, (int64_t)rows);
    return i8_fused_supported(p, x, elem, pitch(b, cols, ldx)) ? 0 : b * (size_t)up16(cols) + 4 * b;
}

int i8_linear_impl(int device, const void* x, int elem, int64_t ldx, const int8_t* wq, int64_t ldw, const float* ws, size_t b,
                   size_t rows, size_t cols, void* y, int y_elem, int64_t ldy, void* work, size_t work_bytes, cudaStream_t s) {
    NEED(elem_ok(elem) && elem_ok(y_elem), "i8_linear: unknown element type");
    NEED(b <= MOST && rows >= 1 && rows <= MOST, "i8_linear: b must be at most 2^31 - 1024, rows in [1, 2^31 - 1024]");
    NEED(cols >= 1, "i8_linear: cols must not be 0");
    if (cols > (size_t)I8_MAX_K) return fail(ERR_UNSUPPORTED, "i8_linear: cols above 131071 could overflow the 32-bit sum");
    if (b == 0) return OK;
    NEED(x && wq && ws && y, "i8_linear: null pointer");
    NEED(on_elements(x, elem) && on_elements(ws, ET_F32) && on_elements(y, y_elem), "i8_linear: a pointer is off its element's boundary");
    NEED(stride_ok(ldx) && stride_ok(ldw) && stride_ok(ldy), "i8_linear: bad row pitch");
    NEED((b == 1 || ldx >= (int64_t)cols) && (rows == 1 || ldw >= (int64_t)cols) && (b == 1 || ldy >= (int64_t)rows),
         "i8_linear: a row pitch is shorter than a row");
    OnDevice on;
    CMFC_TRY(on.enter(device, s));
    I8Params p = i8_params(wq, ldw, ws, b, rows, cols, y, y_elem, ldy);
    p.status = on.c->status;
    if (i8_fused_supported(p, x, elem, pitch(b, cols, ldx))) {
        CMFC_TRY(launch_i8_fused(p, x, elem, pitch(b, cols, ldx), s));
        count_launches(on.c, 1);
        return OK;
    }
    const size_t levels = b * (size_t)up16(cols);
    NEED(work && !(reinterpret_cast<uintptr_t>(work) & 15) && work_bytes >= levels + 4 * b,
         "i8_linear: this call needs a 16-byte aligned workspace of cmfc_i8_linear_workspace() bytes");
    int8_t* q = static_cast<int8_t*>(work);
    float* scale = reinterpret_cast<float*>(q + levels);
    CMFC_TRY(launch_quantize_rows(x, elem, p.M, p.K, ldx, q, up16(cols), scale, s));
    p.x = q;
    p.x_scale = scale;
    p.ldx = up16(cols);
    p.behind_quantizer = 1;
    CMFC_TRY(launch_i8_matmat(p, on.c->num_sms, s));
    count_launches(on.c, 2);
    return OK;
}

int qk_norm_rope_impl(int device, const cmfc_qk_norm_rope_args* a, cudaStream_t s) {
    NEED(a, "qk_norm_rope: null arguments");
    NEED(elem_ok(a->elem), "qk_norm_rope: unknown element type");
    NEED(a->nh + (uint64_t)a->nkv >= 1 && a->nh <= 65536 && a->nkv <= 65536, "qk_norm_rope: bad head counts");
    NEED(a->hd >= 1 && a->hd <= 65536, "qk_norm_rope: bad head size");
    NEED(a->rot <= a->hd && a->rot % 2 == 0, "qk_norm_rope: rot must be even and at most hd");
    NEED(a->eps >= 0.0f && isfinite(a->eps), "qk_norm_rope: eps must not be negative");
    if (a->n == 0) return OK;
    NEED(a->table_rows >= 1 && a->table_rows <= INT_MAX, "qk_norm_rope: empty or oversized cos / sin table");
    if (a->n > INT_MAX || a->n * (a->nh + (uint64_t)a->nkv) > INT_MAX)
        return fail(ERR_UNSUPPORTED, "qk_norm_rope: more than 2^31 heads in one call");
    NEED((!a->nh || (a->q && a->q_out && a->norm_q)) && (!a->nkv || (a->k && a->k_out && a->norm_k)) &&
             (!a->rot || (a->cos_t && a->sin_t)),
         "qk_norm_rope: null pointer");
    NEED(on_elements(a->q, a->elem) && on_elements(a->k, a->elem) && on_elements(a->q_out, a->elem) && on_elements(a->k_out, a->elem) &&
             on_elements(a->norm_q, ET_F32) && on_elements(a->norm_k, ET_F32) && on_elements(a->cos_t, ET_F32) && on_elements(a->sin_t, ET_F32) &&
             reinterpret_cast<uintptr_t>(a->positions) % (a->positions_64 ? 8 : 4) == 0,
         "qk_norm_rope: a pointer is off its element's boundary");
    const int64_t st[8] = {a->q_row, a->q_head, a->k_row, a->k_head, a->q_out_row, a->q_out_head, a->k_out_row, a->k_out_head};
    for (int64_t v : st) NEED(stride_ok(v), "qk_norm_rope: bad stride");
    NEED(distinct((int64_t)a->n, a->nh, a->hd, a->q_out_row, a->q_out_head) && distinct((int64_t)a->n, a->nkv, a->hd, a->k_out_row, a->k_out_head),
         "qk_norm_rope: heads of an output overlap");
    OnDevice on;
    CMFC_TRY(on.enter(device, s));
    NormRopeParams p;
    p.q = {a->q, a->q_row, a->q_head};
    p.k = {a->k, a->k_row, a->k_head};
    p.q_out = {a->q_out, a->q_out_row, a->q_out_head};
    p.k_out = {a->k_out, a->k_out_row, a->k_out_head};
    p.norm_q = a->norm_q;
    p.norm_k = a->norm_k;
    p.cos_t = a->cos_t;
    p.sin_t = a->sin_t;
    p.positions = a->positions;
    p.n = (int64_t)a->n;
    p.table_rows = (int64_t)a->table_rows;
    p.nh = (int)a->nh;
    p.nkv = (int)a->nkv;
    p.hd = (int)a->hd;
    p.rot = (int)a->rot;
    p.pos64 = a->positions_64;
    p.eps = a->eps;
    CMFC_TRY(launch_norm_rope(p, a->elem, a->half_split != 0, s));
    count_launches(on.c, 1);
    return OK;
}

int window_attention_impl(int device, const cmfc_window_attention_args* a, cudaStream_t s) {
    NEED(a, "window_attention: null arguments");
    NEED(elem_ok(a->elem), "window_attention: unknown element type");
    NEED(a->nh >= 1 && a->nkv >= 1 && a->nh % a->nkv == 0 && a->nh <= 65535, "window_attention: nh must be a positive multiple of nkv");
    NEED(a->hd >= 1, "window_attention: empty heads");
    if (a->hd > 256) return fail(ERR_UNSUPPORTED, "window_attention: head sizes above 256 are not implemented");
    NEED(isfinite(a->scale) && isfinite(a->softcap) && a->softcap >= 0.0f, "window_attention: scale and softcap must be finite, softcap not negative");
    NEED(a->q_rows <= MOST && a->k_rows <= MOST && a->q_rows * (a->nh / a->nkv) <= MOST, "window_attention: more than 2^31 - 1024 rows");
    const bool packed = a->q_start || a->k_start || a->k_len;
    NEED(!packed || (a->q_start && a->k_start && a->k_len), "window_attention: q_start, k_start and k_len come together");
    NEED(packed ? a->seqs <= 1u << 30 : a->seqs == 1, "window_attention: without q_start there is one sequence");
    if (a->q_rows == 0 || a->seqs == 0) return OK;
    NEED(a->q && a->out && (a->k_rows == 0 || (a->k && a->v)), "window_attention: null pointer");
    NEED(on_elements(a->q, a->elem) && on_elements(a->k, a->elem) && on_elements(a->v, a->elem) && on_elements(a->out, a->elem) &&
             on_elements(a->q_start, ET_F32) && on_elements(a->k_start, ET_F32) && on_elements(a->k_len, ET_F32),
         "window_attention: a pointer is off its element's boundary");
    const int64_t st[8] = {a->q_row, a->q_head, a->k_row, a->k_head, a->v_row, a->v_head, a->out_row, a->out_head};
    for (int64_t v : st) NEED(stride_ok(v), "window_attention: bad stride");
    NEED(distinct((int64_t)a->q_rows, a->nh, a->hd, a->out_row, a->out_head), "window_attention: heads of the output overlap");
    OnDevice on;
    CMFC_TRY(on.enter(device, s));
    WindowAttnParams p;
    p.q = {a->q, a->q_row, a->q_head};
    p.k = {a->k, a->k_row, a->k_head};
    p.v = {a->v, a->v_row, a->v_head};
    p.out = {a->out, a->out_row, a->out_head};
    p.q_start = a->q_start;
    p.k_start = a->k_start;
    p.k_len = a->k_len;
    p.q_rows = (int64_t)a->q_rows;
    p.k_rows = (int64_t)a->k_rows;
    p.seqs = (int)a->seqs;
    p.nh = (int)a->nh;
    p.nkv = (int)a->nkv;
    p.hd = (int)a->hd;
    p.window = a->window == 0 || a->window > INT_MAX ? INT_MAX : (int)a->window;
    p.sinks = a->sinks > INT_MAX ? INT_MAX : (int)a->sinks;
    p.scale = a->scale;
    p.softcap = a->softcap;
    p.status = on.c->status;
    CMFC_TRY(launch_window_attention(p, a->elem, on.c->num_sms, s));
    count_launches(on.c, 1);
    return OK;
}

}  // namespace

extern "C" int cmfc_quantize_rows(int device, const void* x, int elem, size_t rows, size_t cols, int64_t ldx, int8_t* q,
                                  int64_t ldq, float* scale, void* stream) {
    return guarded([&] { return quantize_rows_impl(device, x, elem, rows, cols, ldx, q, ldq, scale, (cudaStream_t)stream); });
}

extern "C" int cmfc_i8_matmat(int device, const int8_t* xq, int64_t ldx, const float* x_scale, const int8_t* wq, int64_t ldw,
                              const float* w_scale, size_t b, size_t rows, size_t cols, void* y, int elem, int64_t ldy,
                              void* stream) {
    return guarded([&] {
        return i8_matmat_impl(device, xq, ldx, x_scale, wq, ldw, w_scale, b, rows, cols, y, elem, ldy, (cudaStream_t)stream);
    });
}

extern "C" size_t cmfc_i8_linear_workspace(const void* x, int elem, int64_t ldx, const int8_t* wq, int64_t ldw, size_t b,
                                           size_t rows, size_t cols) {
    return i8_linear_workspace(x, elem, ldx, wq, ldw, b, rows, cols);
}

extern "C" int cmfc_i8_linear(int device, const void* x, int elem, int64_t ldx, const int8_t* wq, int64_t ldw, const float* w_scale,
                              size_t b, size_t rows, size_t cols, void* y, int y_elem, int64_t ldy, void* work, size_t work_bytes,
                              void* stream) {
    return guarded([&] {
        return i8_linear_impl(device, x, elem, ldx, wq, ldw, w_scale, b, rows, cols, y, y_elem, ldy, work, work_bytes, (cudaStream_t)stream);
    });
}

extern "C" int cmfc_qk_norm_rope(int device, const cmfc_qk_norm_rope_args* a, void* stream) {
    return guarded([&] { return qk_norm_rope_impl(device, a, (cudaStream_t)stream); });
}

extern "C" int cmfc_window_attention(int device, const cmfc_window_attention_args* a, void* stream) {
    return guarded([&] { return window_attention_impl(device, a, (cudaStream_t)stream); });
}

// The engine's q8_matmat with the activations rounded to 8 bits as well: host f32 in and out, the
// container's q8_row levels and row scales as they are.
extern "C" int cmfc_q8_matmat_i8(cmfc_model* m, int64_t idx, const float* xs, size_t b, size_t rows, size_t cols, float* out) {
    return guarded([&]() -> int {
        NEED(m && xs && out && b > 0, "q8_matmat_i8: null argument or empty batch");
        Context* c = ctx();
        if (!c) return last_error().empty() ? fail(ERR_CUDA, "no CUDA device") : ERR_CUDA;
        DevWeight* w = nullptr;
        CMFC_TRY(get_weight(c, m->m, idx, &w));
        if (w->dtype != DT_Q8) return fail(ERR_UNSUPPORTED, "q8_matmat_i8: tensor " + m->m->recs[idx].name + " is not q8_row");
        if ((size_t)w->rows != rows || (size_t)w->cols != cols)
            return fail(ERR_SHAPE, "q8_matmat_i8: rows/cols disagree with the tensor's directory record");
        DevBuf &xf = c->buf("mm_xf"), &xq = c->buf("mm_xb"), &y = c->buf("mm_y"), &sc = c->buf("mm_xs");
        CMFC_TRY(xf.ensure(b * cols * 4));
        CMFC_TRY(xq.ensure(b * cols));
        CMFC_TRY(sc.ensure(b * 4));
        CMFC_TRY(y.ensure(b * rows * 4));
        CMFC_CUDA(cudaMemcpyAsync(xf.p, xs, b * cols * 4, cudaMemcpyHostToDevice, c->stream));
        CMFC_TRY(quantize_rows_impl(c->device, xf.p, ET_F32, b, cols, (int64_t)cols, xq.as<int8_t>(), (int64_t)cols, sc.as<float>(), c->stream));
        CMFC_TRY(i8_matmat_impl(c->device, xq.as<int8_t>(), (int64_t)cols, sc.as<float>(), reinterpret_cast<const int8_t*>(w->plane),
                                (int64_t)cols, w->scales, b, rows, cols, y.p, ET_F32, (int64_t)rows, c->stream));
        CMFC_CUDA(cudaMemcpyAsync(out, y.p, b * rows * 4, cudaMemcpyDeviceToHost, c->stream));
        return check_status(c, "q8_matmat_i8");
    });
}
