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
# the argument structs of include/cmf_cuda.h in the platform's own layout
_ROPE = struct.Struct("@9P8q2Q4I3if")    # cmfc_qk_norm_rope_args
_ATTN = struct.Struct("@7P8q4Q4I2fi4x")  # cmfc_window_attention_args
_torch = None
_ELEM = {}


def _load():
    global _torch
    if _torch is None:
        import torch
        _ELEM.update({torch.float32: 0, torch.float16: 1, torch.bfloat16: 2})
        _torch = torch
    return _torch


def _fail(code, msg):
    raise CmfCudaError(code, msg)


def _elem(name, t):
    try:
        return _ELEM[t.dtype]
    except KeyError:
        _fail(_UNSUPPORTED, f"{name}: {t.dtype} is not float32, float16 or bfloat16")


def _on_device(what, *tensors):
    """Index of the one CUDA device that holds all tensors."""
    dev = tensors[0].device
    for t in tensors:
        if t.device != dev:
            _fail(_BAD_ARG, f"{what}: tensors on {dev} and {t.device}")
        if t.requires_grad and _torch.is_grad_enabled():
            _fail(_UNSUPPORTED, f"{what}: no backward pass; call it under torch.no_grad()")
    if dev.type != "cuda":
        _fail(_BAD_ARG, f"{what}: tensors must be on a CUDA device, not {dev}")
    return dev.index


def _stream(device):
    return _torch._C._cuda_getCurrentRawStream(device)


def _heads(name, t):
    """Strides (token, head) of a [tokens, heads, hd] tensor whose heads are contiguous."""
    if t.dim() != 3:
        _fail(_SHAPE, f"{name} must be [tokens, heads, hd], not {tuple(t.shape)}")
    row, head, one = t.stride()
    if one != 1 and t.shape[2] > 1:
        _fail(_SHAPE, f"{name}: the values of a head must be contiguous")
    return row, head


def _same(name, t, shape, dtype):
    if t.shape != shape or t.dtype != dtype:
        _fail(_SHAPE, f"{name} must be {tuple(shape)} {dtype}, not {tuple(t.shape)} {t.dtype}")


def _plain(name, t, shape, dtype):
    _same(name, t, shape, dtype)
    if not t.is_contiguous():
        _fail(_SHAPE, f"{name} must be contiguous")


def _rows(name, t):
    if t.dim() != 2 or (t.shape[1] > 1 and t.stride(1) != 1):
        _fail(_SHAPE, f"{name} must be [rows, columns] with contiguous rows")
    return max(t.stride(0), t.shape[1]) if t.shape[0] <= 1 else t.stride(0)


def quantize_rows(x):
    """Rows to 8 bits: ``scale = max |x| / 127`` and ``q = rint(x / scale)`` for each row of ``x`` [b, cols].
    Returns ``(q, scale)``, int8 [b, cols] and float32 [b].  A row of zeros gives scale 0; a row that holds an
    infinity or a NaN gives scale NaN and levels 0."""
    torch = _load()
    ldx, elem = _rows("x", x), _elem("x", x)
    b, cols = x.shape
    if cols == 0:
        _fail(_SHAPE, "quantize_rows: x has no columns")
    dev = _on_device("quantize_rows", x)
    # rows of the levels start on 16 bytes, as the product's tensor-core form wants them
    q = torch.empty((b, (cols + 15) // 16 * 16), dtype=torch.int8, device=x.device)[:, :cols]
    scale = torch.empty(b, dtype=torch.float32, device=x.device)
    check(lib().cmfc_quantize_rows(dev, x.data_ptr(), elem, b, cols, ldx, q.data_ptr(), q.stride(0), scale.data_ptr(), _stream(dev)))
    return q, scale


def i8_matmat(x_q, x_scale, w_q, w_scale, out_dtype=None, out=None):
    """``y[m, n] = (sum_k x_q[m, k] w_q[n, k]) * (x_scale[m] * w_scale[n])``: int8 levels ``x_q`` [b, cols] and ``w_q``
    [rows, cols] with float32 scales [b] and [rows]; the sum is exact.  ``y`` is [b, rows] of ``out_dtype``
    (float32 by default, float16, bfloat16), or written to ``out``."""
    torch = _load()
    ldx, ldw = _rows("x_q", x_q), _rows("w_q", w_q)
    b, cols = x_q.shape
    rows = w_q.shape[0]
    if x_q.dtype != torch.int8 or w_q.dtype != torch.int8:
        _fail(_UNSUPPORTED, "i8_matmat: x_q and w_q must be int8")
    if w_q.shape[1] != cols or cols == 0 or rows == 0:
        _fail(_SHAPE, f"i8_matmat: x_q {tuple(x_q.shape)} and w_q {tuple(w_q.shape)} do not multiply")
    _plain("x_scale", x_scale, (b,), torch.float32)
    _plain("w_scale", w_scale, (rows,), torch.float32)
    if out is None:
        out_dtype = out_dtype or torch.float32
        if out_dtype not in _ELEM:
            _fail(_UNSUPPORTED, f"i8_matmat: {out_dtype} is not float32, float16 or bfloat16")
        dev = _on_device("i8_matmat", x_q, x_scale, w_q, w_scale)
        out = torch.empty((b, rows), dtype=out_dtype, device=x_q.device)
    else:
        _same("out", out, (b, rows), out_dtype or out.dtype)
        dev = _on_device("i8_matmat", x_q, x_scale, w_q, w_scale, out)
    ldy, elem = _rows("out", out), _elem("out", out)
    check(lib().cmfc_i8_matmat(dev, x_q.data_ptr(), ldx, x_scale.data_ptr(), w_q.data_ptr(), ldw, w_scale.data_ptr(), b, rows, cols,
                               out.data_ptr(), elem, ldy, _stream(dev)))
    return out


def i8_linear(x, w_q, w_scale, out_dtype=None, out=None):
    """``x`` [b, cols] (float32, float16, bfloat16) through 8-bit weights: :func:`quantize_rows`, then
    :func:`i8_matmat`.  ``w_q`` int8 [rows, cols] and ``w_scale`` float32 [rows] are a q8_row tensor's levels and row
    scales.  The result has x's type unless ``out_dtype`` or ``out`` says otherwise."""
    q, scale = quantize_rows(x)
    return i8_matmat(q, scale, w_q, w_scale, out_dtype or (out.dtype if out is not None else x.dtype), out)


def qk_norm_rope(q, k, norm_q, norm_k, cos, sin, positions=None, eps=1e-5, half_split=False, q_out=None, k_out=None):
    """Norms of query and key heads and the position rotation in one pass.

    ``q`` [n, nh, hd] and ``k`` [n, nkv, hd] (any strides between tokens and heads, such as views of a fused
    projection; ``k`` may be None): ``y = x / sqrt(mean(x^2) + eps) * norm`` for every head, then the pairs (a, b) of the
    first ``2 * cos.shape[1]`` dims, neighbours or with ``half_split`` the halves ``(i, i + rot / 2)``, become ``(a c - b s, a s
    + b c)``.  ``cos`` / ``sin`` are float32 [positions, rot / 2]; ``positions`` int32 or int64 [n] (default 0 .. n - 1); a
    position outside the table makes the token's heads NaN.  Returns ``(q, k)`` in new tensors or in ``q_out`` /
    ``k_out``, which may be ``q`` and ``k`` themselves."""
    torch = _load()
    elem = _elem("q", q)
    q_row, q_head = _heads("q", q)
    n, nh, hd = q.shape
    nkv = 0
    tensors = [q, norm_q, cos, sin]
    _plain("norm_q", norm_q, (hd,), torch.float32)
    if k is not None:
        nkv = k.shape[1] if k.dim() == 3 else 0
        k_row, k_head = _heads("k", k)
        _same("k", k, (n, nkv, hd), q.dtype)
        _plain("norm_k", norm_k, (hd,), torch.float32)
        tensors += [k, norm_k]
    else:
        k_row = k_head = 0
    if cos.dim() != 2:
        _fail(_SHAPE, "cos must be [positions, rot / 2]")
    table, half = cos.shape
    _plain("cos", cos, (table, half), torch.float32)
    _plain("sin", sin, (table, half), torch.float32)
    if 2 * half > hd:
        _fail(_SHAPE, f"cos has {half} pairs, a head of {hd} has {hd // 2}")
    pos_ptr = pos64 = 0
    if positions is not None:
        if positions.dtype not in (torch.int32, torch.int64):
            _fail(_UNSUPPORTED, "positions must be int32 or int64")
        _plain("positions", positions, (n,), positions.dtype)
        pos64 = int(positions.dtype == torch.int64)
        tensors.append(positions)
    if q_out is not None:
        _same("q_out", q_out, (n, nh, hd), q.dtype)
        tensors.append(q_out)
    if k_out is not None:
        if k is None:
            _fail(_BAD_ARG, "k_out without k")
        _same("k_out", k_out, (n, nkv, hd), q.dtype)
        tensors.append(k_out)
    dev = _on_device("qk_norm_rope", *tensors)
    if positions is not None:
        pos_ptr = positions.data_ptr()
    if q_out is None:
        q_out = torch.empty((n, nh, hd), dtype=q.dtype, device=q.device)
    if k is not None and k_out is None:
        k_out = torch.empty((n, nkv, hd), dtype=q.dtype, device=q.device)
    qo_row, qo_head = _heads("q_out", q_out)
    ko_row, ko_head = _heads("k_out", k_out) if k is not None else (0, 0)
    if n == 0 or nh + nkv == 0 or hd == 0:
        return q_out, k_out
    args = _ROPE.pack(q.data_ptr(), k.data_ptr() if nkv else 0, q_out.data_ptr(), k_out.data_ptr() if nkv else 0,
                      norm_q.data_ptr(), norm_k.data_ptr() if nkv else 0, cos.data_ptr(), sin.data_ptr(), pos_ptr,
                      q_row, q_head, k_row, k_head, qo_row, qo_head, ko_row, ko_head, n, table, nh, nkv, hd, 2 * half,
                      elem, pos64, int(half_split), eps)
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
    torch = _load()
    elem = _elem("q", q)
    q_row, q_head = _heads("q", q)
    k_row, k_head = _heads("k", k)
    v_row, v_head = _heads("v", v)
    rows, nh, hd = q.shape
    krows, nkv = k.shape[0], k.shape[1]
    _same("k", k, (krows, nkv, hd), q.dtype)
    _same("v", v, (krows, nkv, hd), q.dtype)
    if nkv == 0 or nh % nkv or nh == 0 or hd == 0:
        _fail(_SHAPE, f"window_attention: {nh} query heads over {nkv} key heads of {hd}")
    if window is not None and window < 1:
        _fail(_BAD_ARG, "window must be at least 1 (a query's own key), or None")
    if sinks < 0:
        _fail(_BAD_ARG, "sinks must not be negative")
    tensors = [q, k, v]
    seqs, qs, ks, kl = 1, 0, 0, 0
    if q_start is not None or k_start is not None or k_len is not None:
        if q_start is None or k_start is None or k_len is None:
            _fail(_BAD_ARG, "q_start, k_start and k_len come together")
        if k_len.dim() != 1:
            _fail(_SHAPE, "k_len must be [sequences]")
        seqs = k_len.shape[0]
        _plain("q_start", q_start, (seqs + 1,), torch.int32)
        _plain("k_start", k_start, (seqs,), torch.int32)
        _plain("k_len", k_len, (seqs,), torch.int32)
        tensors += [q_start, k_start, k_len]
    if out is not None:
        _same("out", out, (rows, nh, hd), q.dtype)
        tensors.append(out)
    dev = _on_device("window_attention", *tensors)
    if out is None:
        out = torch.empty((rows, nh, hd), dtype=q.dtype, device=q.device)
    o_row, o_head = _heads("out", out)
    if rows == 0 or seqs == 0:
        return out
    if q_start is not None:
        qs, ks, kl = q_start.data_ptr(), k_start.data_ptr(), k_len.data_ptr()
    args = _ATTN.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), qs, ks, kl, q_row, q_head, k_row, k_head, v_row, v_head,
                      o_row, o_head, rows, krows, window or 0, sinks, seqs, nh, nkv, hd, hd ** -0.5 if scale is None else scale,
                      softcap, elem)
    check(lib().cmfc_window_attention(dev, args, _stream(dev)))
    return out
