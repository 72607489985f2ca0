"""Definitions of the text-layer operators in 64 bits, and how far a result may be from them.

Tolerances are per element and follow from the arithmetic: a rounding to type T is off by at most
u(T) = finfo(T).eps / 2 relative to the value, every f32 operation by 2^-24, and sums of n terms by n 2^-24 times
the sum of the terms' magnitudes."""
import torch

F32 = 2.0 ** -24


def unit(dtype):
    return torch.finfo(dtype).eps / 2


def subnormal(dtype):
    """Below the smallest normal number the numbers of a type are smallest_normal * eps apart (f16: 2^-24), and a
    rounding is off by up to half of that whatever the value: u relative to the value is not enough there.  (Twice
    that half, for the f32 result that is rounded may itself be on the other side of a tie.)"""
    f = torch.finfo(dtype)
    return f.smallest_normal * f.eps


def norm_rope(x, weight, cos, sin, half_split, eps=1e-5):
    """x [n, heads, hd]; cos / sin [n, rot / 2] -> (result f64, tolerance f64)."""
    u, x_type = unit(x.dtype), x.dtype
    x = x.double()
    hd, rot = x.shape[-1], 2 * cos.shape[1]
    y = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * weight.double()
    c, s = cos.double()[:, None], sin.double()[:, None]
    if half_split:
        ia, ib = torch.arange(rot // 2), torch.arange(rot // 2) + rot // 2
    else:
        ia, ib = torch.arange(rot // 2) * 2, torch.arange(rot // 2) * 2 + 1
    out, size = y.clone(), y.abs()
    a, b = y[..., ia], y[..., ib]
    out[..., ia], out[..., ib] = a * c - b * s, a * s + b * c
    size[..., ia] = size[..., ib] = a.abs() + b.abs()
    # the sum of squares is a chain of at most hd / 32 + 5 or 16 + 5 terms, halved by the root; division, root,
    # two products and the rotation's three operations follow
    ops = max(16, hd // 32) / 2 + 12
    return out, u * out.abs() + ops * F32 * size + subnormal(x_type)


def quantize_rows(x):
    """The levels and scales bit for bit: the scale is the f32 product with the f32 number next to 1 / 127, the levels
    come from a correctly rounded f32 division."""
    x = x.float().cpu()
    top = x.abs().amax(1)
    scale = top * (torch.tensor(1.0) / torch.tensor(127.0))
    finite = torch.isfinite(x).all(1)
    safe = torch.where(finite & (scale > 0), scale, torch.ones_like(scale))
    q = torch.where((finite & (scale > 0))[:, None], x / safe[:, None], torch.zeros_like(x)).round().clamp(-127, 127).to(torch.int8)
    return q, torch.where(finite, scale, torch.full_like(scale, float("nan")))


def i8_matmat(x_q, x_scale, w_q, w_scale, out_dtype):
    """Exact integer sums; conversion, the scales' product and the last product are each one f32 rounding."""
    acc = (x_q.double() @ w_q.double().t())
    y = acc * x_scale.double()[:, None] * w_scale.double()
    return y, (3.01 * F32 + unit(out_dtype)) * y.abs() + subnormal(out_dtype)


def window_attention(q, k, v, lens, key_start, key_len, window, sinks, scale, softcap):
    """q [rows, nh, hd]; sequences one after the other -> (result f64, tolerance f64), rows outside: NaN."""
    dtype, u = q.dtype, unit(q.dtype)
    rows, nh, hd = q.shape
    group = nh // k.shape[1]
    out = torch.full((rows, nh, hd), float("nan"), dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    r0 = 0
    for length, k0, lk in zip(lens, key_start, key_len):
        if length == 0:
            continue
        pos = torch.arange(length, device=q.device)[:, None] + (lk - length)
        j = torch.arange(lk, device=q.device)[None]
        seen = (j <= pos) & ((pos - j < window) | (j < sinks))
        for h in range(nh):
            qq = q[r0:r0 + length, h].double()
            kk, vv = k[k0:k0 + lk, h // group].double(), v[k0:k0 + lk, h // group].double()
            # what a row does not see has no part in it, whatever it holds: keys and values that no query sees are
            # taken out, and the others' products are formed only where they are seen
            used = seen.any(0)
            kk, vv = torch.where(used[:, None], kk, 0.0), torch.where(used[:, None], vv, 0.0)
            s = (qq @ kk.t()) * scale
            size = (qq.abs() @ kk.abs().t()) * abs(scale)
            if softcap:
                s = softcap * torch.tanh(s / softcap)
            s = torch.where(seen, s, torch.full_like(s, -torch.inf))
            size = torch.where(seen, size, torch.zeros_like(size))
            top = s.amax(1, keepdim=True) if lk else s.new_zeros((length, 1))
            e = torch.where(seen, torch.exp(s - top), torch.zeros_like(s))
            p = e / e.sum(1, keepdim=True)
            p = torch.where(seen.any(1, keepdim=True), p, torch.zeros_like(p))
            if torch.isfinite(vv).all():
                o, ov = p @ vv, p @ vv.abs()
            else:  # 0 x inf only where the row sees it
                o = torch.stack([(p[i][seen[i]][:, None] * vv[seen[i]]).sum(0) for i in range(length)])
                ov = torch.zeros_like(o)
            out[r0:r0 + length, h] = o
            # scores: hd products and sums, scaling, and for the cap two roundings of the quotient, the quotient
            # of 2^x + 1 (3 operations, 2^x itself 4 F32) and the product, all relative to at most softcap
            ds = ((hd + 3) * F32 * size).amax(1, keepdim=True) if lk else torch.zeros((length, 1), dtype=torch.float64, device=q.device)
            if softcap:
                ds = ds + 12 * F32 * softcap
            # weights: the exponential's error (2^-21, or 1e-4 of the cubic that 16-bit forms use beside it),
            # their rounding to the type, the rounding of the exponent's argument (8 bits of it before the
            # point: 2^-24 x 256), and the f32 sums over the keys
            n = seen.sum(1, keepdim=True)
            a = 2 * ds + (2.0 ** -21 if dtype == torch.float32 else 1e-4 + u) + 256 * F32 + 2 * (n + 8) * F32
            tol[r0:r0 + length, h] = (u + 4 * F32) * o.abs() + a * (ov + o.abs()) + subnormal(dtype)
        r0 += length
    return out, tol


def check(got, want, tol):
    """got within tol of want; NaN and infinities in the same places."""
    got = got.double()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), "NaN in other places"
    assert torch.equal(got[~fine].nan_to_num(nan=0.0), want[~fine].nan_to_num(nan=0.0))
    over = ((got - want).abs() - tol)[fine]
    if over.numel():
        i = int(over.argmax())
        assert float(over[i]) <= 0, (f"off by {float((got - want).abs()[fine][i]):.3g}, allowed {float(tol[fine][i]):.3g}, "
                                     f"value {float(want[fine][i]):.3g}")
