"""Operators of text-model attention layers on torch CUDA tensors: head norms with the position rotation,
causal attention with a sliding window, and matrix products in 8-bit integers.

Unlike the facade in :mod:`cmf_b200.gpu`, whose functions take host arrays and return when the result is
there, these take the caller's device tensors and enqueue their work on torch's current stream of the
tensors' device: they return at once, can be captured into a CUDA graph (after one call outside of it) and
may run on several streams.  They compute forward results only: a tensor that requires a gradient is
refused while gradients are enabled.  A wrong argument raises :class:`CmfCudaError` before anything is launched.

They have no counterpart in the reference's facade; torch is imported on the first call.
"""
import struct

from ._lib import CmfCudaError, check, lib

_BAD_ARG, _UNSUPPORTED, _SHAPE = -1, -2, -3
_ALL = 2 ** 31 - 1  # no sequence is longer
# the argument structs of include/cmf_cuda.h in the platform's own layout
_ROPE = struct.Struct("@9P8q2Q4I3if")    # cmfc_qk_norm_rope_args
_ATTN = struct.Struct("@7P8q4Q4I2fi4x")  # cmfc_window_attention_args
_torch = None
_elem_of = None   # element type id of a dtype, or None
_stream = None    # raw handle of torch's current stream on a device
_grad_on = None


def _load():
    global _torch, _elem_of, _stream, _grad_on
    import torch
    _elem_of = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}.get
    _stream = torch._C._cuda_getCurrentRawStream
    _grad_on = torch.is_grad_enabled
    _torch = torch


def _fail(code, msg):
    raise CmfCudaError(code, msg)


# A call of a few microseconds is mostly its checks: they are written as plain comparisons, and what is wrong is
# found out in words only when one of them fails.

def _elem(name, t):
    e = _elem_of(t.dtype)
    return e if e is not None else _fail(_UNSUPPORTED, f"{name}: {t.dtype} is not float32, float16 or bfloat16")


def _device(what, tensors):
    """Index of the one CUDA device that holds all tensors."""
    dev = tensors[0].get_device()
    for t in tensors:
        if t.get_device() != dev:
            _fail(_BAD_ARG, f"{what}: tensors on {tensors[0].device} and {t.device}")
    if dev < 0:
        _fail(_BAD_ARG, f"{what}: tensors must be on a CUDA device, not {tensors[0].device}")
    return dev


def _no_grad(what, tensors):
    if _grad_on():
        for t in tensors:
            if t.requires_grad:
                _fail(_UNSUPPORTED, f"{what}: no backward pass; call it under torch.no_grad()")


def _heads(name, t, shape, dtype):
    """Strides (token, head) of a [tokens, heads, hd] tensor whose heads are contiguous."""
    if t.shape != shape or t.dtype != dtype:
        _fail(_SHAPE, f"{name} must be {tuple(shape)} {dtype}, not {tuple(t.shape)} {t.dtype}")
    row, head, one = t.stride()
    if one != 1 and shape[2] > 1:
        _fail(_SHAPE, f"{name}: the values of a head must be contiguous")
    return row, head


def _three(name, t):
    if t.dim() != 3:
        _fail(_SHAPE, f"{name} must be [tokens, heads, hd], not {tuple(t.shape)}")
    return t.shape


def _plain(name, t, shape, dtype):
    if t.shape != shape or t.dtype != dtype or not t.is_contiguous():
        _fail(_SHAPE, f"{name} must be contiguous {tuple(shape)} {dtype}, not {tuple(t.shape)} {t.dtype}")


def _rows(name, t):
    """Row pitch of a [rows, columns] tensor with contiguous rows."""
    if t.dim() != 2 or (t.shape[1] > 1 and t.stride(1) != 1):
        _fail(_SHAPE, f"{name} must be [rows, columns] with contiguous rows")
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def quantize_rows(x):
    """Rows to 8 bits: ``scale = max |x| / 127`` (times the f32 number next to 1 / 127, as torch divides a CUDA
    tensor by a number) and ``q = rint(x / scale)`` for each row of ``x`` [b, cols].  Returns ``(q, scale)``, int8
    [b, cols] and float32 [b].  A row of zeros gives scale 0; a row that holds an infinity or a NaN gives scale
    NaN and levels 0."""
    if _torch is None:
        _load()
    ldx, elem = _rows("x", x), _elem("x", x)
    b, cols = x.shape
    if cols == 0:
        _fail(_SHAPE, "quantize_rows: x has no columns")
    _no_grad("quantize_rows", (x,))
    dev = _device("quantize_rows", (x,))
    # rows of the levels start on 16 bytes, as the product's tensor-core form wants them
    q = x.new_empty((b, (cols + 15) // 16 * 16), dtype=_torch.int8)
    if cols % 16:
        q = q[:, :cols]
    scale = x.new_empty(b, dtype=_torch.float32)
    check(lib().cmfc_quantize_rows(dev, x.data_ptr(), elem, b, cols, ldx, q.data_ptr(), (cols + 15) // 16 * 16, scale.data_ptr(), _stream(dev)))
    return q, scale


def _weights(what, w_q, w_scale, cols):
    ldw = _rows("w_q", w_q)
    rows = w_q.shape[0]
    if w_q.dtype != _torch.int8:
        _fail(_UNSUPPORTED, f"{what}: w_q must be int8")
    if w_q.shape[1] != cols or cols == 0 or rows == 0:
        _fail(_SHAPE, f"{what}: {cols} columns of activations and w_q {tuple(w_q.shape)} do not multiply")
    _plain("w_scale", w_scale, (rows,), _torch.float32)
    return ldw, rows


def _result(what, x, b, rows, out_dtype, out):
    """(out, its element type, its pitch), new unless given."""
    if out is None:
        elem = _elem_of(out_dtype)
        if elem is None:
            _fail(_UNSUPPORTED, f"{what}: {out_dtype} is not float32, float16 or bfloat16")
        return None, elem, rows
    if out.shape != (b, rows) or (out_dtype is not None and out.dtype != out_dtype):
        _fail(_SHAPE, f"out must be {(b, rows)} {out_dtype}, not {tuple(out.shape)} {out.dtype}")
    return out, _elem("out", out), _rows("out", out)


def i8_matmat(x_q, x_scale, w_q, w_scale, out_dtype=None, out=None):
    """``y[m, n] = (sum_k x_q[m, k] w_q[n, k]) * (x_scale[m] * w_scale[n])``: int8 levels ``x_q`` [b, cols] and ``w_q``
    [rows, cols] with float32 scales [b] and [rows]; the sum is exact.  ``y`` is [b, rows] of ``out_dtype``
    (float32 by default, float16, bfloat16), or written to ``out``."""
    if _torch is None:
        _load()
    ldx = _rows("x_q", x_q)
    b, cols = x_q.shape
    if x_q.dtype != _torch.int8:
        _fail(_UNSUPPORTED, "i8_matmat: x_q must be int8")
    ldw, rows = _weights("i8_matmat", w_q, w_scale, cols)
    _plain("x_scale", x_scale, (b,), _torch.float32)
    y, elem, ldy = _result("i8_matmat", x_q, b, rows, out_dtype or (out.dtype if out is not None else _torch.float32), out)
    tensors = (x_q, x_scale, w_q, w_scale) if y is None else (x_q, x_scale, w_q, w_scale, y)
    _no_grad("i8_matmat", tensors)
    dev = _device("i8_matmat", tensors)
    if y is None:
        y = x_q.new_empty((b, rows), dtype=out_dtype or _torch.float32)
    check(lib().cmfc_i8_matmat(dev, x_q.data_ptr(), ldx, x_scale.data_ptr(), w_q.data_ptr(), ldw, w_scale.data_ptr(), b, rows, cols,
                               y.data_ptr(), elem, ldy, _stream(dev)))
    return y


def i8_linear(x, w_q, w_scale, out_dtype=None, out=None):
    """``x`` [b, cols] (float32, float16, bfloat16) through 8-bit weights: :func:`quantize_rows`, then
    :func:`i8_matmat`, in one call and with the same bits.  ``w_q`` int8 [rows, cols] and ``w_scale`` float32 [rows] are a
    q8_row tensor's levels and row scales.  The result has x's type unless ``out_dtype`` or ``out`` says otherwise."""
    if _torch is None:
        _load()
    ldx, x_elem = _rows("x", x), _elem("x", x)
    b, cols = x.shape
    ldw, rows = _weights("i8_linear", w_q, w_scale, cols)
    y, elem, ldy = _result("i8_linear", x, b, rows, out_dtype or (out.dtype if out is not None else x.dtype), out)
    tensors = (x, w_q, w_scale) if y is None else (x, w_q, w_scale, y)
    _no_grad("i8_linear", tensors)
    dev = _device("i8_linear", tensors)
    if y is None:
        y = x.new_empty((b, rows), dtype=out_dtype or x.dtype)
    L, xp, wp = lib(), x.data_ptr(), w_q.data_ptr()
    nbytes = L.cmfc_i8_linear_workspace(xp, x_elem, ldx, wp, ldw, b, rows, cols)
    work = x.new_empty(nbytes, dtype=_torch.uint8) if nbytes else None   # goes back to torch's pool of this stream
    check(L.cmfc_i8_linear(dev, xp, x_elem, ldx, wp, ldw, w_scale.data_ptr(), b, rows, cols, y.data_ptr(), elem, ldy,
                           work.data_ptr() if nbytes else None, nbytes, _stream(dev)))
    return y


def qk_norm_rope(q, k, norm_q, norm_k, cos, sin, positions=None, eps=1e-5, half_split=False, q_out=None, k_out=None):
    """Norms of query and key heads and the position rotation in one pass.

    ``q`` [n, nh, hd] and ``k`` [n, nkv, hd] (any strides between tokens and heads, such as views of a fused
    projection; ``k`` may be None): ``y = x / sqrt(mean(x^2) + eps) * norm`` for every head, then the pairs (a, b) of the
    first ``2 * cos.shape[1]`` dims, neighbours or with ``half_split`` the halves ``(i, i + rot / 2)``, become ``(a c - b s, a s
    + b c)``.  ``cos`` / ``sin`` are float32 [positions, rot / 2]; ``positions`` int32 or int64 [n] (default 0 .. n - 1); a
    position outside the table makes the token's heads NaN.  Returns ``(q, k)`` in new tensors or in ``q_out`` /
    ``k_out``, which may be ``q`` and ``k`` themselves."""
    if _torch is None:
        _load()
    f32 = _torch.float32
    dtype, elem = q.dtype, _elem("q", q)
    n, nh, hd = shape = _three("q", q)
    q_row, q_head = _heads("q", q, shape, dtype)
    _plain("norm_q", norm_q, (hd,), f32)
    tensors = [q, norm_q, cos, sin]
    nkv = k_row = k_head = 0
    if k is not None:
        nkv = _three("k", k)[1]
        k_row, k_head = _heads("k", k, (n, nkv, hd), dtype)
        _plain("norm_k", norm_k, (hd,), f32)
        tensors += (k, norm_k)
    elif k_out is not None:
        _fail(_BAD_ARG, "k_out without k")
    if cos.dim() != 2:
        _fail(_SHAPE, "cos must be [positions, rot / 2]")
    table, half = cos.shape
    _plain("cos", cos, (table, half), f32)
    _plain("sin", sin, (table, half), f32)
    if 2 * half > hd:
        _fail(_SHAPE, f"cos has {half} pairs, a head of {hd} has {hd // 2}")
    pos_ptr = pos64 = 0
    if positions is not None:
        if positions.dtype == _torch.int64:
            pos64 = 1
        elif positions.dtype != _torch.int32:
            _fail(_UNSUPPORTED, "positions must be int32 or int64")
        _plain("positions", positions, (n,), positions.dtype)
        tensors.append(positions)
        pos_ptr = positions.data_ptr()
    qo_row, qo_head, ko_row, ko_head = nh * hd, hd, nkv * hd, hd
    if q_out is not None:
        qo_row, qo_head = _heads("q_out", q_out, (n, nh, hd), dtype)
        tensors.append(q_out)
    if k_out is not None:
        ko_row, ko_head = _heads("k_out", k_out, (n, nkv, hd), dtype)
        tensors.append(k_out)
    _no_grad("qk_norm_rope", tensors)
    dev = _device("qk_norm_rope", tensors)
    if q_out is None:
        q_out = q.new_empty((n, nh, hd))
    if k_out is None and k is not None:
        k_out = k.new_empty((n, nkv, hd))
    if n == 0 or nh + nkv == 0 or hd == 0:
        return q_out, k_out
    args = _ROPE.pack(q.data_ptr(), k.data_ptr() if nkv else 0, q_out.data_ptr(), k_out.data_ptr() if nkv else 0,
                      norm_q.data_ptr(), norm_k.data_ptr() if nkv else 0, cos.data_ptr(), sin.data_ptr(), pos_ptr,
                      q_row, q_head, k_row, k_head, qo_row, qo_head, ko_row, ko_head, n, table, nh, nkv, hd, 2 * half,
                      elem, pos64, bool(half_split), eps)
    check(lib().cmfc_qk_norm_rope(dev, args, _stream(dev)))
    return q_out, k_out


def window_attention(q, k, v, window=None, sinks=0, scale=None, softcap=0.0, q_start=None, k_start=None, k_len=None, out=None):
    """Causal attention with a sliding window and first tokens that stay visible.

    ``q`` [rows, nh, hd], ``k`` and ``v`` [key rows, nkv, hd] (any strides between rows and heads; nh a multiple of nkv; hd
    up to 256).  Sequence ``z`` has the query rows ``q_start[z] : q_start[z + 1]`` and the ``k_len[z]`` key rows from
    ``k_start[z]`` on (int32 tensors on the same device): packed prompts, or slots of a cache seen as rows.  Its
    queries are its last positions, so a prompt, a chunk behind a cache and a single token are the same call;
    without the three there is one sequence of all rows.  A query at position p sees key j when ``j <= p`` and
    (``p - j < window`` or ``j < sinks``); ``window`` None sees everything before it.  ``scale`` is ``hd ** -0.5`` by default;
    ``softcap > 0`` caps the scaled scores, ``cap * tanh(s / cap)``.  A query that sees no key gets zeros; query rows
    outside every sequence are not written.  Returns ``out`` like q, new unless given (it must not overlap the inputs)."""
    if _torch is None:
        _load()
    dtype, elem = q.dtype, _elem("q", q)
    rows, nh, hd = shape = _three("q", q)
    q_row, q_head = _heads("q", q, shape, dtype)
    krows, nkv, _ = _three("k", k)
    kshape = (krows, nkv, hd)
    k_row, k_head = _heads("k", k, kshape, dtype)
    v_row, v_head = _heads("v", v, kshape, dtype)
    if nkv == 0 or nh % nkv or nh == 0 or hd == 0:
        _fail(_SHAPE, f"window_attention: {nh} query heads over {nkv} key heads of {hd}")
    if window is None:
        window = 0
    elif window < 1 or int(window) != window:
        _fail(_BAD_ARG, "window must be a whole number of at least 1 (a query's own key), or None")
    if sinks < 0 or int(sinks) != sinks:
        _fail(_BAD_ARG, "sinks must be a whole number and not negative")
    tensors = [q, k, v]
    seqs, qs, ks, kl = 1, 0, 0, 0
    if q_start is not None or k_start is not None or k_len is not None:
        if q_start is None or k_start is None or k_len is None:
            _fail(_BAD_ARG, "q_start, k_start and k_len come together")
        if k_len.dim() != 1:
            _fail(_SHAPE, "k_len must be [sequences]")
        i32 = _torch.int32
        seqs = k_len.shape[0]
        _plain("q_start", q_start, (seqs + 1,), i32)
        _plain("k_start", k_start, (seqs,), i32)
        _plain("k_len", k_len, (seqs,), i32)
        tensors += (q_start, k_start, k_len)
        qs, ks, kl = q_start.data_ptr(), k_start.data_ptr(), k_len.data_ptr()
    o_row, o_head = nh * hd, hd
    if out is not None:
        o_row, o_head = _heads("out", out, shape, dtype)
        tensors.append(out)
    _no_grad("window_attention", tensors)
    dev = _device("window_attention", tensors)
    if out is None:
        out = q.new_empty(shape)
    if rows == 0 or seqs == 0:
        return out
    args = _ATTN.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), qs, ks, kl, q_row, q_head, k_row, k_head, v_row, v_head,
                      o_row, o_head, rows, krows, min(int(window), _ALL), min(int(sinks), _ALL), seqs, nh, nkv, hd, hd ** -0.5 if scale is None else scale, softcap, elem)
    check(lib().cmfc_window_attention(dev, args, _stream(dev)))
    return out
