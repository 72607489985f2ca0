"""Refusals of the text-layer operators: no GPU is touched before the arguments are right."""
import ctypes as C

import pytest
import torch

from cmf_b200 import CmfCudaError, lib, ops


def refused(code, f, *a, **kw):
    with pytest.raises(CmfCudaError) as e:
        f(*a, **kw)
    assert e.value.code == code, str(e.value)


def heads(n=4, h=2, hd=16, dtype=torch.float32):
    return torch.zeros(n, h, hd, dtype=dtype)


def rope(q=None, k=None, **kw):
    q = heads() if q is None else q
    k = heads() if k is None else k
    a = dict(norm_q=torch.ones(16), norm_k=torch.ones(16), cos=torch.ones(8, 8), sin=torch.ones(8, 8))
    a.update(kw)
    return ops.qk_norm_rope(q, k, **a)


def test_norm_rope_refuses():
    refused(-1, rope)                                                   # right in all but the device
    refused(-2, rope, q=heads(dtype=torch.float64))
    refused(-3, rope, q=torch.zeros(4, 32))
    refused(-3, rope, q=heads().transpose(1, 2))                        # heads not contiguous
    refused(-3, rope, k=heads(n=3))
    refused(-3, rope, k=heads(dtype=torch.float16))
    refused(-3, rope, norm_q=torch.ones(15))
    refused(-3, rope, norm_k=torch.ones(16, dtype=torch.float16))
    refused(-3, rope, cos=torch.ones(8, 9), sin=torch.ones(8, 9))       # more pairs than the head has
    refused(-3, rope, sin=torch.ones(8, 7))
    refused(-3, rope, cos=torch.ones(8, 16)[:, ::2], sin=torch.ones(8, 8))
    refused(-2, rope, positions=torch.zeros(4))
    refused(-3, rope, positions=torch.zeros(5, dtype=torch.int32))
    refused(-3, rope, q_out=heads(n=5))
    refused(-3, rope, k_out=heads(dtype=torch.bfloat16))
    refused(-2, rope, q=heads().requires_grad_())


def attn(q=None, k=None, v=None, **kw):
    return ops.window_attention(heads(h=4) if q is None else q, heads() if k is None else k, heads() if v is None else v, **kw)


def test_window_attention_refuses():
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    refused(-1, attn)
    refused(-2, attn, q=heads(h=4, dtype=torch.float64))
    refused(-3, attn, q=heads(h=3))                                     # 3 query heads over 2 key heads
    refused(-3, attn, k=heads(hd=8))
    refused(-3, attn, v=heads(n=5))
    refused(-3, attn, v=heads(dtype=torch.float16))
    refused(-3, attn, q=torch.zeros(4, 64))
    refused(-1, attn, window=0)
    refused(-1, attn, window=-5)
    refused(-1, attn, sinks=-1)
    refused(-1, attn, window=2.5)
    refused(-1, attn, sinks=0.5)
    refused(-1, attn, q_start=i32(0, 4))
    refused(-3, attn, q_start=i32(0, 4), k_start=i32(0, 0), k_len=i32(4))
    refused(-3, attn, q_start=i32(0, 2, 4), k_start=i32(0), k_len=i32(4))
    refused(-3, attn, q_start=torch.tensor([0, 4]), k_start=i32(0), k_len=i32(4))
    refused(-3, attn, out=heads(h=3))
    refused(-2, attn, k=heads().requires_grad_())


def test_products_refuse():
    x, w, s = torch.zeros(4, 32), torch.zeros(8, 32, dtype=torch.int8), torch.ones(8)
    xq, xs = torch.zeros(4, 32, dtype=torch.int8), torch.ones(4)
    refused(-1, ops.quantize_rows, x)
    refused(-2, ops.quantize_rows, x.double())
    refused(-3, ops.quantize_rows, x[0])
    refused(-3, ops.quantize_rows, x[:, :0])
    refused(-3, ops.quantize_rows, x.t())
    refused(-2, ops.quantize_rows, x.clone().requires_grad_())
    refused(-1, ops.i8_matmat, xq, xs, w, s)
    refused(-2, ops.i8_matmat, x, xs, w, s)
    refused(-3, ops.i8_matmat, xq, xs, w[:, :16], s)
    refused(-3, ops.i8_matmat, xq, xs, w, s[:7])
    refused(-3, ops.i8_matmat, xq, xs.half(), w, s)
    refused(-3, ops.i8_matmat, xq, xs, w, s, out=torch.zeros(4, 9))
    refused(-2, ops.i8_matmat, xq, xs, w, s, out_dtype=torch.float64)
    refused(-1, ops.i8_linear, x, w, s)
    refused(-3, ops.i8_linear, x, w[:, :16], s)
    refused(-2, ops.i8_linear, x, x, s)
    refused(-2, ops.i8_linear, x.int(), w, s)
    refused(-3, ops.i8_linear, x, w, s, out=torch.zeros(8, 4))
    refused(-3, ops.i8_linear, x, w, s, out_dtype=torch.float32, out=torch.zeros(4, 8, dtype=torch.float16))


def test_library_refuses_before_any_device_call():
    """The C entries check sizes, strides and pointers themselves."""
    L, p = lib(), C.c_void_p(256)

    def rope_args(**kw):
        a = dict(ptrs=[256] * 9, strides=[32, 16] * 4, n=4, table=8, nh=2, nkv=2, hd=16, rot=16, elem=0, pos64=0, half=0, eps=1e-5)
        a.update(kw)
        return ops._ROPE.pack(*a["ptrs"], *a["strides"], a["n"], a["table"], a["nh"], a["nkv"], a["hd"], a["rot"], a["elem"], a["pos64"],
                              a["half"], a["eps"])

    for kw, code in [(dict(elem=3), -1), (dict(nh=0, nkv=0), -1), (dict(hd=0, rot=0), -1), (dict(rot=15), -1), (dict(rot=18), -1),
                     (dict(eps=-1.0), -1), (dict(eps=float("nan")), -1), (dict(ptrs=[0] * 9), -1), (dict(table=0), -1),
                     (dict(strides=[32, 16, 32, 16, 32, 8, 32, 16]), -1), (dict(strides=[-32, 16] + [32, 16] * 3), -1),
                     (dict(ptrs=[258] + [256] * 8), -1), (dict(ptrs=[256] * 8 + [260], pos64=1), -1), (dict(ptrs=[256] * 7 + [254, 256], elem=2), -1),
                     (dict(strides=[32, 16] * 2 + [2 ** 39, 16, 2 ** 39, 2 ** 39 + 8], n=2 ** 28), -1), (dict(n=2 ** 30), -2)]:
        assert L.cmfc_qk_norm_rope(0, rope_args(**kw), None) == code, (kw, L.cmfc_last_error())
    assert L.cmfc_qk_norm_rope(0, None, None) == -1
    assert L.cmfc_qk_norm_rope(0, rope_args(n=0), None) == 0

    def attn_args(**kw):
        a = dict(ptrs=[256] * 4 + [0] * 3, strides=[64, 16, 32, 16, 32, 16, 64, 16], q_rows=4, k_rows=4, window=0, sinks=0, seqs=1, nh=4, nkv=2,
                 hd=16, scale=0.25, softcap=0.0, elem=0)
        a.update(kw)
        return ops._ATTN.pack(*a["ptrs"], *a["strides"], a["q_rows"], a["k_rows"], a["window"], a["sinks"], a["seqs"], a["nh"], a["nkv"],
                              a["hd"], a["scale"], a["softcap"], a["elem"])

    for kw, code in [(dict(elem=-1), -1), (dict(nh=3), -1), (dict(nkv=0), -1), (dict(hd=0), -1), (dict(hd=257), -2), (dict(scale=float("inf")), -1),
                     (dict(softcap=-1.0), -1), (dict(seqs=2), -1), (dict(ptrs=[256] * 4 + [256, 0, 0]), -1), (dict(ptrs=[0] * 7), -1),
                     (dict(q_rows=2 ** 31), -1), (dict(k_rows=2 ** 31 - 100), -1), (dict(q_rows=2 ** 30), -1), (dict(strides=[64, 16, 32, 16, 32, 16, 64, 8]), -1),
                     (dict(strides=[64, 16, 32, -16, 32, 16, 64, 16]), -1), (dict(ptrs=[256, 258, 256, 256, 0, 0, 0]), -1),
                     (dict(ptrs=[256, 257, 256, 256, 0, 0, 0], elem=1), -1), (dict(ptrs=[256] * 4 + [256, 258, 256]), -1)]:
        assert L.cmfc_window_attention(0, attn_args(**kw), None) == code, (kw, L.cmfc_last_error())
    assert L.cmfc_window_attention(0, None, None) == -1
    assert L.cmfc_window_attention(0, attn_args(q_rows=0), None) == 0

    q = lambda **kw: L.cmfc_quantize_rows(*{**dict(dev=0, x=p, elem=0, rows=4, cols=8, ldx=8, q=p, ldq=8, s=p, st=None), **kw}.values())  # noqa: E731
    assert q(elem=9) == -1 and q(cols=0) == -1 and q(x=None) == -1 and q(ldx=7) == -1 and q(ldq=7) == -1 and q(ldx=-8) == -1
    assert q(x=C.c_void_p(258)) == -1 and q(s=C.c_void_p(257)) == -1
    assert q(rows=0) == 0 and q(rows=2 ** 31 - 1) == -1 and q(cols=2 ** 31, ldx=2 ** 31, ldq=2 ** 31) == -1
    m = lambda **kw: L.cmfc_i8_matmat(*{**dict(dev=0, x=p, ldx=8, xs=p, w=p, ldw=8, ws=p, b=4, rows=4, cols=8, y=p, elem=0, ldy=4, st=None),  # noqa: E731
                                        **kw}.values())
    assert m(elem=9) == -1 and m(rows=0) == -1 and m(cols=0) == -1 and m(w=None) == -1 and m(ldx=7) == -1 and m(ldy=3) == -1
    assert m(cols=131072, ldx=131072, ldw=131072) == -2
    assert m(ws=C.c_void_p(258)) == -1 and m(y=C.c_void_p(258)) == -1 and m(y=C.c_void_p(257), elem=2) == -1
    assert m(b=0) == 0
    # the workspace of i8_linear: none for a few short aligned tokens, levels and scales otherwise
    assert L.cmfc_i8_linear_workspace(p, 2, 64, p, 64, 1, 8, 64) == 0
    assert L.cmfc_i8_linear_workspace(p, 2, 64, p, 64, 9, 8, 64) == 9 * 64 + 36
    assert L.cmfc_i8_linear_workspace(C.c_void_p(258), 2, 64, p, 64, 2, 8, 64) == 2 * 64 + 8
    assert L.cmfc_i8_linear_workspace(p, 2, 33, p, 33, 2, 8, 33) == 2 * 48 + 8
    li = lambda **kw: L.cmfc_i8_linear(*{**dict(dev=0, x=p, elem=0, ldx=8, w=p, ldw=8, ws=p, b=4, rows=4, cols=8, y=p, ye=0, ldy=4, work=p, nb=100,  # noqa: E731
                                                st=None), **kw}.values())
    assert li(elem=9) == -1 and li(ye=9) == -1 and li(rows=0) == -1 and li(cols=0) == -1 and li(x=None) == -1 and li(ldx=7) == -1 and li(ldy=3) == -1
    assert li(cols=131072, ldx=131072, ldw=131072) == -2
    assert li(b=0) == 0
    assert L.cmfc_q8_matmat_i8(None, 0, p, 1, 1, 1, p) == -1
