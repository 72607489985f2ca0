"""Head norms with rotation, windowed attention and 8-bit products against their definitions in 64 bits."""
import numpy as np
import pytest
import torch

from tests import text_ops_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_wait_ran_out():
    """After every test: no kernel gave up a bounded wait."""
    yield
    from cmf_b200 import gpu
    torch.cuda.synchronize()
    gpu.synchronize()


TYPES = [torch.float32, torch.float16, torch.bfloat16]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


# ---------------- head norms with the position rotation ----------------

def rope_inputs(n, nh, nkv, hd, rot, dtype, seed=0, table=50):
    g = gen(seed)
    qkv = randn(g, n, nh + 2 * nkv, hd, dtype=dtype) * 1.5
    angle = torch.arange(table, dtype=torch.float64, device="cuda")[:, None] * 100.0 ** (-torch.arange(rot // 2, device="cuda").double() / max(1, rot // 2))
    return (qkv, 1 + 0.3 * randn(g, hd), 1 + 0.3 * randn(g, hd), angle.cos().float(), angle.sin().float(),
            torch.randint(0, table, (n,), generator=g, device="cuda"))


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,nh,nkv,hd,rot", [(1, 24, 8, 96, 96), (37, 8, 4, 256, 192), (5, 3, 1, 64, 64), (130, 5, 2, 128, 32), (700, 24, 8, 32, 32),
                                              (3, 2, 1, 20, 10), (4, 2, 2, 7, 6), (2, 1, 1, 512, 512), (3, 4, 2, 48, 0), (2, 3, 1, 1, 0)])
def test_norm_rope(n, nh, nkv, hd, rot, dtype, half):
    from cmf_b200 import ops
    qkv, wq, wk, cos, sin, pos = rope_inputs(n, nh, nkv, hd, rot, dtype)
    q, k = qkv[:, :nh], qkv[:, nh:nh + nkv]
    for positions in (pos, pos.int()):
        qo, ko = ops.qk_norm_rope(q, k, wq, wk, cos, sin, positions=positions, half_split=half)
        ref.check(qo, *ref.norm_rope(q, wq, cos[pos], sin[pos], half))
        ref.check(ko, *ref.norm_rope(k, wk, cos[pos], sin[pos], half))


@pytest.mark.parametrize("dtype,hd", [(torch.bfloat16, 96), (torch.float32, 30)])
def test_norm_rope_in_place_default_positions_and_layouts(dtype, hd):
    from cmf_b200 import ops
    qkv, wq, wk, cos, sin, _ = rope_inputs(33, 6, 2, hd, hd, dtype, table=33)
    before = qkv.clone()
    q, k = qkv[:, :6], qkv[:, 6:8]
    qo, ko = ops.qk_norm_rope(q, k, wq, wk, cos, sin, eps=1e-3, q_out=q, k_out=k)
    assert qo is q and ko is k
    ref.check(q, *ref.norm_rope(before[:, :6], wq, cos, sin, False, 1e-3))
    ref.check(k, *ref.norm_rope(before[:, 6:8], wk, cos, sin, False, 1e-3))
    assert torch.equal(qkv[:, 8:], before[:, 8:])                       # the values beside them
    # head-major output, and an input whose rows start off the 16-byte boundary
    major = torch.full((6, 33, hd), 7.0, dtype=dtype, device="cuda")
    odd = torch.empty(33 * 6 * (hd + 1) + 1, dtype=dtype, device="cuda")[1:].view(33, 6, hd + 1)[..., :hd]
    odd.copy_(before[:, :6])
    only, none = ops.qk_norm_rope(odd, None, wq, None, cos, sin, half_split=True, q_out=major.transpose(0, 1))
    assert none is None
    ref.check(only, *ref.norm_rope(before[:, :6], wq, cos, sin, True))


def test_norm_rope_positions_outside_the_table_and_empty_calls():
    from cmf_b200 import ops
    for hd in (64, 10):
        qkv, wq, wk, cos, sin, pos = rope_inputs(6, 2, 1, hd, hd, torch.float32)
        pos[1], pos[4] = -1, 50
        for positions in (pos, pos.int()):
            qo, ko = ops.qk_norm_rope(qkv[:, :2], qkv[:, 2:3], wq, wk, cos, sin, positions=positions)
            bad = torch.tensor([False, True, False, False, True, False], device="cuda")
            assert torch.isnan(qo[bad]).all() and torch.isnan(ko[bad]).all()
            want, tol = ref.norm_rope(qkv[:, :2], wq, cos[pos.clamp(0, 49)], sin[pos.clamp(0, 49)], False)
            ref.check(qo[~bad], want[~bad], tol[~bad])
    e = qkv[:0]
    qo, ko = ops.qk_norm_rope(e[:, :2], e[:, 2:3], wq, wk, cos, sin)
    assert qo.shape == (0, 2, 10) and ko.shape == (0, 1, 10)


def test_norm_rope_rows_of_zeros_and_non_finite_rows_stay_apart():
    from cmf_b200 import ops
    qkv, wq, wk, cos, sin, _ = rope_inputs(4, 2, 1, 64, 64, torch.bfloat16)
    qkv[0, 0] = 0
    qkv[1, 0, 5] = float("nan")
    qo, _ = ops.qk_norm_rope(qkv[:, :2], None, wq, None, cos, sin)
    assert (qo[0, 0] == 0).all() and torch.isnan(qo[1, 0]).all()
    assert torch.isfinite(qo[1, 1]).all() and torch.isfinite(qo[2:]).all()


# ---------------- 8-bit products ----------------

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("b,cols", [(1, 1), (3, 17), (5, 64), (2, 2304), (7, 9216), (2, 9000), (4, 40000)])
def test_quantize_rows(b, cols, dtype):
    from cmf_b200 import ops
    g = gen(b * cols)
    wide = randn(g, b, cols + 5, dtype=dtype)
    wide[:, 0] *= 11
    for x in (wide[:, :cols], wide[:, 3:3 + cols], wide[:, :cols].contiguous()):
        q, s = ops.quantize_rows(x)
        wq, ws = ref.quantize_rows(x)
        assert torch.equal(q.cpu(), wq) and torch.equal(s.cpu(), ws)


@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_rows_near_ties(dtype):
    """Values on and beside every half of every maximum's grid: levels k + 1/2 in all roundings, where the quotient's own
    rounding decides."""
    from cmf_b200 import ops
    g = gen(9)
    tops = (torch.rand(700, 1, generator=g, device="cuda") * 4 + 0.01).to(dtype).float()
    tops[:8, 0] = torch.tensor([127.0, 254.0, 3.96875, 1.0, 1e-4, 300.0, 0.49609375, 2.0])
    halves = (torch.arange(127, device="cuda").float() + 0.5)[None] * (tops / 127)
    x = torch.cat([tops, halves, -halves, halves * (1 + 2e-7), halves * (1 - 2e-7), halves * (1 + 1.3e-7), halves * (1 - 1.3e-7)], 1)
    x = torch.cat([x, x[:, :1].expand(-1, (-x.shape[1]) % 16)], 1)
    x = torch.minimum(torch.maximum(x.to(dtype), -tops.to(dtype)), tops.to(dtype))
    for scale in (1.0, 2.0 ** -20, 2.0 ** 11) if dtype != torch.float16 else (1.0,):
        y = (x * scale).contiguous()
        q, s = ops.quantize_rows(y)
        wq, ws = ref.quantize_rows(y)
        assert torch.equal(q.cpu(), wq) and torch.equal(s.cpu(), ws)
        q, s = ops.quantize_rows(y[:20])                    # a block per row instead of a warp
        assert torch.equal(q.cpu(), wq[:20]) and torch.equal(s.cpu(), ws[:20])


def test_quantize_rows_zeros_ties_tiny_and_non_finite():
    from cmf_b200 import ops
    x = torch.zeros(7, 32, device="cuda")
    x[1, :4] = torch.tensor([127.0, 0.5, 1.5, -2.5])     # scale 1: ties to even
    x[2, 3], x[3, 5] = float("inf"), float("nan")
    x[4, 0] = 1e-45                                       # the scale underflows to 0
    x[5, :3] = torch.tensor([2e-43, -1e-43, 1e-43])       # a subnormal scale
    x[6, 0] = 3.4e38
    q, s = ops.quantize_rows(x)
    wq, ws = ref.quantize_rows(x)
    assert torch.equal(q.cpu(), wq)
    assert torch.equal(s.cpu().nan_to_num(nan=-1.0), ws.nan_to_num(nan=-1.0))
    assert q[1, :4].tolist() == [127, 0, 2, -2] and torch.isnan(s[2:4]).all() and s[0] == 0 and s[4] == 0
    q, s = ops.quantize_rows(x[:0])
    assert q.shape == (0, 32) and s.shape == (0,)
    y = ops.i8_matmat(*ops.quantize_rows(x), torch.ones(4, 32, dtype=torch.int8, device="cuda"), torch.ones(4, device="cuda"))
    assert torch.isnan(y[2:4]).all() and (y[0] == 0).all() and torch.isfinite(y[1]).all()


SHAPES = [(1, 1, 1), (1, 2304, 2304), (2, 100, 48), (3, 16, 33), (8, 300, 512), (9, 130, 2304), (16, 256, 9216), (17, 64, 4096), (33, 1000, 144),
          (64, 2304, 2304), (65, 129, 130), (127, 256, 128), (128, 128, 16), (200, 2300, 1040), (256, 256, 2304), (257, 520, 80), (333, 2304, 1184),
          (700, 768, 4608), (1031, 2304, 256), (2500, 1280, 176)]


@pytest.mark.parametrize("out", TYPES)
@pytest.mark.parametrize("b,rows,cols", SHAPES)
def test_i8_matmat(b, rows, cols, out):
    from cmf_b200 import ops
    g = gen(b + rows * 7 + cols)
    xq = torch.randint(-128, 128, (b, cols), generator=g, device="cuda", dtype=torch.int8)
    wq = torch.randint(-128, 128, (rows, cols), generator=g, device="cuda", dtype=torch.int8)
    xs, ws = torch.rand(b, generator=g, device="cuda") * 1e-3, torch.rand(rows, generator=g, device="cuda") * 1e-3
    y = ops.i8_matmat(xq, xs, wq, ws, out_dtype=out)
    assert y.dtype == out
    ref.check(y, *ref.i8_matmat(xq, xs, wq, ws, out))


def test_i8_matmat_largest_sums():
    """-128 x -128 in every place: the sums are what 32 bits hold."""
    from cmf_b200 import ops
    for b, cols in ((1, 131071), (40, 131056), (300, 16384)):
        xq = torch.full((b, cols), -128, dtype=torch.int8, device="cuda")
        wq = torch.full((256, cols), -128, dtype=torch.int8, device="cuda")
        one = torch.ones(300, device="cuda")
        y = ops.i8_matmat(xq, one[:b], wq, one[:256])
        assert (y == float(np.float32(16384 * cols))).all()


@pytest.mark.parametrize("b", [1, 12, 40, 300])
def test_i8_matmat_pitches_alignment_and_neighbours(b):
    from cmf_b200 import ops
    g = gen(b)
    rows, cols = 300, 272
    xw = torch.randint(-128, 128, (b, cols + 37), generator=g, device="cuda", dtype=torch.int8)
    ww = torch.randint(-128, 128, (rows, cols + 48), generator=g, device="cuda", dtype=torch.int8)
    xs, ws = torch.rand(b, generator=g, device="cuda"), torch.rand(rows, generator=g, device="cuda")
    for xo, wo, yo in ((0, 0, 0), (3, 0, 1), (0, 16, 4), (16, 5, 3)):
        x, w = xw[:, xo:xo + cols], ww[:, wo:wo + cols]
        for out in TYPES:
            canvas = torch.full((b + 2, rows + 9), 5.0, dtype=out, device="cuda")
            y = canvas[1:1 + b, yo:yo + rows]
            assert ops.i8_matmat(x, xs * 1e-2, w, ws * 1e-2, out=y) is y
            ref.check(y, *ref.i8_matmat(x, xs * 1e-2, w, ws * 1e-2, out))
            canvas[1:1 + b, yo:yo + rows] = 5.0
            assert (canvas == 5.0).all()                   # nothing beside the result was written
    assert ops.i8_matmat(xw[:0, :cols], xs[:0], ww[:, :cols], ws).shape == (0, rows)


def test_q8_matmat_i8_beside_q8_matmat(tmp_path):
    """The facade's entry on a q8_row tensor: the same bits as the two operators on its planes, and as near to
    q8_matmat as the activations' rounding allows."""
    from cmf_b200 import CmfCudaError, Model, gpu, ops
    from oracle import codecs as oc
    from tests.modelfile import single_weight_file
    rows, cols = 384, 2304
    rng = np.random.default_rng(3)
    w = (rng.standard_normal((rows, cols)) * 0.02).astype(np.float32)
    path = str(tmp_path / "w.cmf")
    single_weight_file(path, [("w", oc.Q8_ROW, w), ("w4", oc.Q4TP, w)])
    gpu.set_current_device(0)
    with Model(path) as m:
        idx = m.index("w")
        payload = m.tensor_bytes(idx)
        wq = torch.from_numpy(payload[:rows * cols].view(np.int8).reshape(rows, cols).copy()).cuda()
        ws = torch.from_numpy(payload[rows * cols:].view(np.float16).astype(np.float32)).cuda()
        for b in (1, 5, 300):
            x = rng.standard_normal((b, cols)).astype(np.float32)
            y, near = np.empty((b, rows), np.float32), np.empty((b, rows), np.float32)
            assert gpu.q8_matmat_i8(m, idx, x, b, rows, cols, y)
            assert np.array_equal(y, ops.i8_linear(torch.from_numpy(x).cuda(), wq, ws).cpu().numpy())
            gpu.q8_matmat(m, idx, None, x, b, rows, cols, near)
            # half a level of scale / 1 on each activation, half a bf16 step (2^-8) on q8_matmat's side
            wd = wq.double().abs().cpu().numpy() * ws.double().cpu().numpy()[:, None]
            tol = (np.abs(x).max(1, keepdims=True) / 127 / 2 * (1 + 1e-5)) * wd.sum(1) + (2.0 ** -8 + 1e-5) * (np.abs(x) @ wd.T)
            assert (np.abs(y - near) <= tol).all()
        with pytest.raises(CmfCudaError) as e:
            gpu.q8_matmat_i8(m, m.index("w4"), x, 300, rows, cols, y)
        assert e.value.code == -2
        with pytest.raises(CmfCudaError) as e:
            gpu.q8_matmat_i8(m, idx, x.reshape(-1), 600, rows, cols // 2, np.empty(600 * rows, np.float32))
        assert e.value.code == -3


# ---------------- windowed attention ----------------

def attn_inputs(lens, prior, nh, nkv, hd, dtype, seed=0, slots=None, junk=0.0):
    """Packed sequences, or slots of a cache (`slots` rows each) whose rows behind a sequence hold `junk`."""
    g = gen(seed)
    total = [a + b for a, b in zip(lens, prior)]
    starts = [i * slots for i in range(len(lens))] if slots else [sum(total[:i]) for i in range(len(lens))]
    rows = slots * len(lens) if slots else sum(total)
    q = randn(g, sum(lens), nh, hd, dtype=dtype) * 1.5
    k, v = randn(g, rows, nkv, hd, dtype=dtype), randn(g, rows, nkv, hd, dtype=dtype)
    if slots:
        for s, t in zip(starts, total):
            k[s + t:s + slots] = junk
            v[s + t:s + slots] = junk
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    return q, k, v, starts, total, dict(q_start=i32([sum(lens[:i]) for i in range(len(lens) + 1)]), k_start=i32(starts), k_len=i32(total))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("nh,nkv,hd", [(6, 2, 96), (4, 2, 64), (8, 4, 256), (2, 1, 128), (5, 1, 32), (3, 3, 80), (7, 1, 40), (2, 2, 20), (1, 1, 1), (16, 1, 128), (40, 1, 64)])
@pytest.mark.parametrize("window,sinks,cap", [(None, 0, 0.0), (100, 4, 0.0), (33, 0, 20.0), (1, 0, 0.0), (130, 140, 0.0)])
def test_prompts(nh, nkv, hd, window, sinks, cap, dtype):
    from cmf_b200 import ops
    lens = [1, 130, 0, 65, 300]
    q, k, v, starts, total, where = attn_inputs(lens, [0] * 5, nh, nkv, hd, dtype)
    out = ops.window_attention(q, k, v, window=window, sinks=sinks, softcap=cap, **where)
    ref.check(out, *ref.window_attention(q, k, v, lens, starts, total, window or 1 << 30, sinks, hd ** -0.5, cap))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("nh,nkv,hd", [(6, 2, 96), (8, 4, 256), (9, 1, 128), (4, 4, 64), (3, 1, 72), (33, 1, 128), (2, 1, 30)])
@pytest.mark.parametrize("window,sinks,cap", [(None, 0, 0.0), (200, 4, 50.0), (1, 0, 0.0), (64, 70, 0.0), (16, 1, 0.0)])
def test_single_tokens_over_a_cache(nh, nkv, hd, window, sinks, cap, dtype):
    """Slots of a cache whose unused rows hold NaN; lengths of one, around tiles, and a sequence with no query."""
    from cmf_b200 import ops
    lens = [1, 1, 1, 0, 1, 1, 1]
    prior = [0, 15, 16, 40, 127, 300, 699]
    q, k, v, starts, total, where = attn_inputs(lens, prior, nh, nkv, hd, dtype, slots=704, junk=float("nan"))
    out = ops.window_attention(q, k, v, window=window, sinks=sinks, softcap=cap, **where)
    ref.check(out, *ref.window_attention(q, k, v, lens, starts, total, window or 1 << 30, sinks, hd ** -0.5, cap))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nh,nkv,hd", [(8, 4, 256), (6, 2, 96), (4, 4, 64)])
def test_many_single_tokens_over_long_caches(nh, nkv, hd, dtype):
    """Enough blocks and tiles that every ring wraps many times under load; each call gives the first one's bits."""
    from cmf_b200 import ops
    prior = [4095 - 61 * i for i in range(48)]
    q, k, v, starts, total, where = attn_inputs([1] * 48, prior, nh, nkv, hd, dtype, slots=4096)
    first = ops.window_attention(q, k, v, sinks=2, **where)
    ref.check(first, *ref.window_attention(q, k, v, [1] * 48, starts, total, 1 << 30, 2, hd ** -0.5, 0.0))
    outs = [ops.window_attention(q, k, v, sinks=2, **where) for _ in range(200)]
    assert all(torch.equal(o, first) for o in outs)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("nh,nkv,hd", [(6, 2, 96), (8, 4, 256), (4, 1, 128)])
@pytest.mark.parametrize("window,sinks,cap", [(None, 0, 0.0), (150, 4, 0.0), (20, 0, 30.0)])
@pytest.mark.parametrize("lens,prior", [([3, 1, 5, 2], [50, 700, 0, 127]), ([100, 7, 260], [300, 129, 1]), ([64], [999])])
def test_chunks_behind_a_cache(lens, prior, nh, nkv, hd, window, sinks, cap, dtype):
    from cmf_b200 import ops
    q, k, v, starts, total, where = attn_inputs(lens, prior, nh, nkv, hd, dtype, slots=1100, junk=float("inf"))
    out = ops.window_attention(q, k, v, window=window, sinks=sinks, softcap=cap, **where)
    ref.check(out, *ref.window_attention(q, k, v, lens, starts, total, window or 1 << 30, sinks, hd ** -0.5, cap))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_one_long_sequence_without_offsets(hd, dtype):
    from cmf_b200 import ops
    q, k, v, starts, total, _ = attn_inputs([1500], [0], 4, 2, hd, dtype)
    out = ops.window_attention(q, k, v, window=700, sinks=3, scale=0.2)
    ref.check(out, *ref.window_attention(q, k, v, [1500], [0], [1500], 700, 3, 0.2, 0.0))
    one = ops.window_attention(q[-1:], k, v, window=700, sinks=3, scale=0.2)
    ref.check(one, *ref.window_attention(q[-1:], k, v, [1], [0], [1500], 700, 3, 0.2, 0.0))


@pytest.mark.parametrize("dtype", TYPES)
def test_queries_without_keys_and_rows_outside_every_sequence(dtype):
    """More queries than keys: the first ones stand before the first key and get zeros; rows before the first and
    behind the last sequence are left as they were."""
    from cmf_b200 import ops
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    for nh, nkv, hd in ((4, 2, 64), (2, 1, 256), (2, 2, 20)):
        g = gen(1)
        q, k, v = randn(g, 60, nh, hd, dtype=dtype), randn(g, 50, nkv, hd, dtype=dtype), randn(g, 50, nkv, hd, dtype=dtype)
        out = torch.full_like(q, 3.0)
        ops.window_attention(q, k, v, window=9, sinks=1, q_start=i32(5, 15, 35, 36, 40), k_start=i32(0, 4, 30, 50), k_len=i32(4, 0, 20, 0), out=out)
        assert (out[:5] == 3.0).all() and (out[40:] == 3.0).all()
        want, tol = ref.window_attention(q[5:40], k, v, [10, 20, 1, 4], [0, 4, 30, 50], [4, 0, 20, 0], 9, 1, hd ** -0.5, 0.0)
        assert (out[5:11] == 0).all() and (out[15:35] == 0).all() and (out[36:40] == 0).all()
        ref.check(out[5:40], want, tol)
        # no keys at all, no queries at all
        assert (ops.window_attention(q, k[:0], v[:0]) == 0).all()
        assert ops.window_attention(q[:0], k, v).shape == (0, nh, hd)


@pytest.mark.parametrize("dtype", TYPES)
def test_offsets_outside_the_tensors_are_clamped(dtype):
    from cmf_b200 import ops
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    for hd in (64, 24):
        g = gen(2)
        q, k, v = randn(g, 40, 2, hd, dtype=dtype), randn(g, 50, 1, hd, dtype=dtype), randn(g, 50, 1, hd, dtype=dtype)
        for qs, ks, kl in (((-7, 10, 10 ** 9), (-3, 45), (20, 10 ** 9)), ((30, 10, 5), (10 ** 9, 0), (-5, 2 ** 31 - 1))):
            out = ops.window_attention(q, k, v, q_start=i32(*qs), k_start=i32(*ks), k_len=i32(*kl))
            torch.cuda.synchronize()
            assert out.shape == q.shape
        # the first set is a right one after clamping
        out = ops.window_attention(q, k, v, q_start=i32(-7, 10, 10 ** 9), k_start=i32(-3, 45), k_len=i32(20, 10 ** 9))
        ref.check(out, *ref.window_attention(q, k, v, [10, 30], [0, 45], [20, 5], 1 << 30, 0, hd ** -0.5, 0.0))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("where", ["k", "v"])
def test_non_finite_keys_reach_only_the_rows_that_see_them(dtype, bad, where):
    """One bad key in the middle: rows before it and rows whose window has passed it are as if it were not there."""
    from cmf_b200 import ops
    for nh, nkv, hd, lens, prior in ((4, 2, 64, [300], [0]), (2, 1, 256, [200], [60]), (3, 1, 128, [9], [150]), (2, 1, 36, [100], [100])):
        q, k, v, starts, total, w = attn_inputs(lens, prior, nh, nkv, hd, dtype)
        at = prior[0] + lens[0] // 2
        (k if where == "k" else v)[at, 0, 3] = bad
        out = ops.window_attention(q, k, v, window=lens[0] // 4, sinks=2, **w)
        pos = torch.arange(lens[0], device="cuda") + prior[0]
        sees = (pos >= at) & (pos - at < lens[0] // 4)
        k2, v2 = k.clone(), v.clone()
        k2[at, 0], v2[at, 0] = 1.0, 1.0
        want, tol = ref.window_attention(q, k2, v2, lens, starts, total, lens[0] // 4, 2, hd ** -0.5, 0.0)
        free = ~sees
        ref.check(out[free], want[free], tol[free])
        heads = slice(0, nh // nkv)
        if where == "v":
            hit = out[sees][:, heads, 3].double()
            assert torch.isnan(hit).all() if bad != bad else (hit == bad).all()
        elif bad != bad:
            assert torch.isnan(out[sees][:, heads]).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_large_scores_and_rising_maxima(dtype):
    """Scores that rise by hundreds from key to key, and rows whose scores are all far below zero."""
    from cmf_b200 import ops
    for nh, nkv, hd, n in ((4, 2, 64, 400), (2, 1, 256, 300), (4, 2, 128, 1)):
        q, k, v, _, _, _ = attn_inputs([n], [400 - n], nh, nkv, hd, dtype)
        q[:, 0::2, 0], q[:, 1::2, 0] = 4.0, -4.0
        k[:, :, 0] = torch.linspace(0, 200, k.shape[0], device="cuda")[:, None].to(dtype)
        out = ops.window_attention(q, k, v, window=250, sinks=5, scale=1.0)
        ref.check(out, *ref.window_attention(q, k, v, [n], [0], [400], 250, 5, 1.0, 0.0))


@pytest.mark.parametrize("nh,nkv,hd", [(8, 4, 256), (6, 2, 96), (4, 4, 64), (4, 1, 128)])
def test_many_prompt_tiles_give_the_same_bits(nh, nkv, hd):
    """Prompts and chunks over enough blocks and key tiles that every ring wraps many times, again and again."""
    from cmf_b200 import ops
    lens, prior = [700, 33, 1500, 129, 64], [900, 0, 300, 2000, 5]
    q, k, v, starts, total, where = attn_inputs(lens, prior, nh, nkv, hd, torch.bfloat16)
    first = ops.window_attention(q, k, v, window=1100, sinks=3, softcap=20.0, **where)
    ref.check(first, *ref.window_attention(q, k, v, lens, starts, total, 1100, 3, hd ** -0.5, 20.0))
    outs = [ops.window_attention(q, k, v, window=1100, sinks=3, softcap=20.0, **where) for _ in range(100)]
    assert all(torch.equal(o, first) for o in outs)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cap", [1e-3, 0.5, 3.0, 256.0, 257.0, 1e4, 1e9])
def test_caps_far_below_and_above_the_scores(dtype, cap):
    """Scores of several units under a cap that they all reach, that some reach, and that none comes near."""
    from cmf_b200 import ops
    for nh, nkv, hd, n in ((4, 2, 64, 200), (2, 1, 256, 150), (4, 2, 128, 1), (4, 2, 256, 1)):
        q, k, v, _, _, _ = attn_inputs([n], [260 - n], nh, nkv, hd, dtype)
        out = ops.window_attention(q * 3, k, v, window=200, softcap=cap)
        want, tol = ref.window_attention(q * 3, k, v, [n], [0], [260], 200, 0, hd ** -0.5, cap)
        if cap > 1e3:  # the cap changes nothing: the tolerance that grows with it has to hold without it too
            want, tol = ref.window_attention(q * 3, k, v, [n], [0], [260], 200, 0, hd ** -0.5, 0.0)
            # y P(y^2) or tanhf: 6 roundings of a score of at most 3 x 1.5 x 6 x 6 = 162
            tol = tol + 2 * 6 * 162 * ref.F32 * v.double().abs().max()
        ref.check(out, want, tol)


@pytest.mark.parametrize("dtype", TYPES)
def test_scales_of_zero_and_below(dtype):
    from cmf_b200 import ops
    for nh, nkv, hd, n in ((4, 2, 64, 200), (2, 1, 256, 1), (24, 24, 32, 200)):
        q, k, v, _, _, _ = attn_inputs([n], [230 - n], nh, nkv, hd, dtype)
        for scale, cap in ((0.0, 0.0), (-0.3, 0.0), (-0.2, 2.0), (1e-6, 0.0)):
            out = ops.window_attention(q, k, v, window=180, sinks=1, scale=scale, softcap=cap)
            ref.check(out, *ref.window_attention(q, k, v, [n], [0], [230], 180, 1, scale, cap))


def with_rows_behind(monkeypatch):
    """window_attention with so many rows behind the last sequence that a call goes to the kernels for prompts, whose
    choice goes by the tensors' sizes; strides and alignment stay as they were."""
    from cmf_b200 import ops
    plain = ops.window_attention

    def longer(t, rows):
        nh, hd = t.shape[1:]
        row, head = t.stride(0), t.stride(1)
        head = rows * row if head >= row else head  # heads before tokens
        skip = t.data_ptr() % 16 // t.element_size()
        at = torch.full((skip + rows * row + nh * head + hd,), 7.0, dtype=t.dtype, device=t.device)
        u = at.as_strided((rows, nh, hd), (row, head, 1), skip)
        u[:t.shape[0]] = t
        return u

    def call(q, k, v, q_start=None, k_start=None, k_len=None, out=None, **kw):
        i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
        n = q.shape[0]
        if n == 0:
            return plain(q, k, v, **kw)
        if q_start is None:
            q_start, k_start, k_len = i32(0, n), i32(0), i32(k.shape[0])
        rows = n + 2400 * len(k_start) * k.shape[1] // q.shape[1]
        o = longer(torch.empty_like(q) if out is None else out, rows)
        plain(longer(q, rows), k, v, q_start=q_start, k_start=k_start, k_len=k_len, out=o, **kw)
        assert (o[n:] == 7.0).all()
        return o[:n] if out is None else out.copy_(o[:n])
    monkeypatch.setattr(ops, "window_attention", call)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("nh,nkv,hd", [(6, 2, 96), (4, 2, 64), (8, 4, 256), (2, 1, 128), (3, 3, 80), (7, 1, 40), (2, 2, 20), (40, 1, 64)])
def test_prompt_kernels_on_calls_of_any_size(monkeypatch, nh, nkv, hd, dtype):
    with_rows_behind(monkeypatch)
    for window, sinks, cap in ((None, 0, 0.0), (100, 4, 0.0), (33, 0, 20.0), (1, 0, 0.0), (130, 140, 0.0)):
        test_prompts(nh, nkv, hd, window, sinks, cap, dtype)
    for lens, prior in (([3, 1, 5, 2], [50, 700, 0, 127]), ([100, 7, 260], [300, 129, 1]), ([64], [999])):
        test_chunks_behind_a_cache(lens, prior, nh, nkv, hd, 150, 4, 30.0, dtype)
    test_single_tokens_over_a_cache(nh, nkv, hd, 64, 70, 0.0, dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_prompt_kernels_on_the_calls_that_can_go_wrong(monkeypatch, dtype):
    with_rows_behind(monkeypatch)
    test_queries_without_keys_and_rows_outside_every_sequence(dtype)
    test_large_scores_and_rising_maxima(dtype)
    test_scales_of_zero_and_below(dtype)
    for bad in (float("nan"), float("inf"), -float("inf")):
        for where in ("k", "v"):
            test_non_finite_keys_reach_only_the_rows_that_see_them(dtype, bad, where)
    for cap in (1e-3, 0.5, 3.0, 256.0, 257.0, 1e4, 1e9):
        test_caps_far_below_and_above_the_scores(dtype, cap)
    for n in (1, 200):
        test_strides_and_layouts(dtype, n)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n", [1, 200])
def test_strides_and_layouts(dtype, n):
    """Views of a fused projection, head-major tensors, rows off the 16-byte boundary, heads broadcast with stride 0."""
    from cmf_b200 import ops
    g = gen(4)
    nh, nkv, hd, lk = 6, 2, 64, 260
    fused = randn(g, lk, nh + 2 * nkv, hd, dtype=dtype)
    odd = randn(g, lk, nh + 2 * nkv, hd + 3, dtype=dtype)[..., 1:1 + hd]
    major = randn(g, nh + 2 * nkv, lk, hd, dtype=dtype).transpose(0, 1)
    for x in (fused, odd, major):
        q, k, v = x[lk - n:, :nh], x[:, nh:nh + nkv], x[:, nh + nkv:]
        out = torch.full((nh, n, hd + 5), 3.0, dtype=dtype, device="cuda")
        ops.window_attention(q, k, v, window=77, out=out[..., 2:2 + hd].transpose(0, 1))
        ref.check(out[..., 2:2 + hd].transpose(0, 1), *ref.window_attention(q, k, v, [n], [0], [lk], 77, 0, hd ** -0.5, 0.0))
        assert (out[..., :2] == 3.0).all() and (out[..., 2 + hd:] == 3.0).all()
    k, v = fused[:, :1].expand(lk, nkv, hd), fused[:, 1:2].expand(lk, nkv, hd)
    ref.check(ops.window_attention(fused[:n, :nh], k, v), *ref.window_attention(fused[:n, :nh], k, v, [n], [0], [lk], 1 << 30, 0, hd ** -0.5, 0.0))


def test_rows_beyond_two_to_the_31_elements():
    """A cache whose later slots lie past 2^31 (and 2^32) elements."""
    from cmf_b200 import ops
    slots, slot, hd = 9, 2 ** 19, 1024          # rows of 1024 elements, heads at their beginning
    cache = torch.empty(slots * slot, hd, dtype=torch.bfloat16, device="cuda")
    assert cache.numel() > 2 ** 32
    g = gen(5)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    k, v = cache.view(-1, 8, 128)[:, :2], cache.view(-1, 8, 128)[:, 2:4]
    starts, lens = [0, 4 * slot + 17, 8 * slot + 1000], [40, 300, 333]
    for s, n in zip(starts, lens):
        cache[s:s + n] = randn(g, n, hd, dtype=torch.bfloat16)
    for ql in ([1, 1, 1], [30, 200, 333]):
        q = randn(g, sum(ql), 4, 128, dtype=torch.bfloat16)
        out = ops.window_attention(q, k, v, window=100, sinks=2, q_start=i32(0, ql[0], ql[0] + ql[1], sum(ql)), k_start=i32(*starts), k_len=i32(*lens))
        ref.check(out, *ref.window_attention(q, k, v, ql, starts, lens, 100, 2, 128 ** -0.5, 0.0))
    del cache, k, v
    torch.cuda.empty_cache()


# ---------------- together, on streams, in graphs ----------------

def layer(ops, x, w, cache_k, cache_v, where, first_row, positions, out_dtype=torch.bfloat16):
    """One attention layer of a text model: projections in 8 bits, norms + rotation, cache, windowed attention."""
    nh, nkv, hd = 8, 2, 64
    qkv = ops.i8_linear(x, *w["qkv"], out_dtype=out_dtype).view(x.shape[0], nh + 2 * nkv, hd)
    q, k = ops.qk_norm_rope(qkv[:, :nh], qkv[:, nh:nh + nkv], w["nq"], w["nk"], w["cos"], w["sin"], positions=positions, half_split=True)
    cache_k[first_row] = k
    cache_v[first_row] = qkv[:, nh + nkv:]
    a = ops.window_attention(q, cache_k, cache_v, window=90, sinks=4, softcap=30.0, **where)
    return ops.i8_linear(a.view(x.shape[0], nh * hd), *w["o"], out_dtype=out_dtype)


def layer_weights(g):
    def lin(rows, cols):
        w = randn(g, rows, cols) * cols ** -0.5
        s = w.abs().amax(1) / 127
        return (w / s[:, None]).round().to(torch.int8), s
    angle = torch.arange(400, device="cuda").double()[:, None] * 10000.0 ** (-torch.arange(32, device="cuda").double() / 32)
    return dict(qkv=lin(12 * 64, 512), o=lin(512, 512), nq=1 + 0.1 * randn(g, 64), nk=1 + 0.1 * randn(g, 64), cos=angle.cos().float(), sin=angle.sin().float())


def test_a_layer_over_a_prompt_equals_the_layer_token_by_token():
    """A prompt in one call, in chunks, and token by token over the cache, the single tokens replayed from a graph."""
    from cmf_b200 import ops
    g = gen(6)
    w = layer_weights(g)
    n, slot = 300, 384
    x = randn(g, n, 512, dtype=torch.bfloat16)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731

    def caches():
        return [torch.full((2 * slot, 2, 64), float("nan"), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    rows = torch.arange(n, device="cuda")
    kc, vc = caches()
    whole = layer(ops, x, w, kc, vc, dict(q_start=i32(0, n), k_start=i32(0), k_len=i32(n)), rows, rows)
    kd, vd = caches()
    parts, at = [], 0
    for m in (200, 3, 60):
        r = torch.arange(at, at + m, device="cuda")
        parts.append(layer(ops, x[at:at + m], w, kd, vd, dict(q_start=i32(0, m), k_start=i32(slot), k_len=i32(at + m)), slot + r, r))
        at += m
    # token by token: the graph reads its inputs, its position and its cache length from the same tensors each time
    xin, row, pos, klen = x[at:at + 1].clone(), torch.tensor([slot + at], device="cuda"), torch.tensor([at], device="cuda"), i32(at + 1)
    where = dict(q_start=i32(0, 1), k_start=i32(slot), k_len=klen)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer(ops, xin, w, kd, vd, where, row, pos)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layer(ops, xin, w, kd, vd, where, row, pos)
    for t in range(at, n):
        xin.copy_(x[t:t + 1])
        row.fill_(slot + t)
        pos.fill_(t)
        klen.fill_(t + 1)
        graph.replay()
        parts.append(y.clone())
    got = torch.cat(parts)
    assert torch.isfinite(whole).all()
    assert torch.equal(kc[:n], kd[slot:slot + n]) and torch.equal(vc[:n], vd[slot:slot + n])   # 8-bit products: the same bits for any batch
    # attention sums in another order, its result rounded to bf16 (2^-9 each), then to 8 bits (half a level of
    # max / 127): relative to the largest value of a row at most 2^-8 + 1 / 127 for each, carried by |w|
    wd = w["o"][0].double().abs() * w["o"][1].double()[:, None]
    a_top = 6.0 * torch.ones(n, 1, device="cuda", dtype=torch.float64)   # |values| of a projection of unit inputs stay below 6
    tol = a_top * (2.0 ** -8 + 1 / 127) * wd.sum(1) + 2.0 ** -8 * whole.double().abs()
    assert ((got.double() - whole.double()).abs() <= tol).all()
    rel = ((got.double() - whole.double()).norm() / whole.double().norm()).item()
    assert rel < 2.0 ** -8 + 1 / 127, rel


def test_calls_on_other_streams_in_two_graphs_and_at_once():
    """Every operator on two streams at the same time and from two captured graphs replayed side by side gives the
    bits of a lone call: nothing is shared between calls."""
    from cmf_b200 import ops
    g = gen(7)
    q, k, v, _, _, where = attn_inputs([1] * 9, [500 + 60 * i for i in range(9)], 8, 2, 128, torch.bfloat16, slots=1100)
    pq, pk, pv, _, _, pwhere = attn_inputs([700, 900], [0, 0], 4, 2, 64, torch.float16)
    x = randn(g, 70, 1024, dtype=torch.bfloat16)
    w = torch.randint(-127, 128, (768, 1024), generator=g, device="cuda", dtype=torch.int8)
    s = torch.rand(768, generator=g, device="cuda")
    qkv, nq, nk, cos, sin, pos = rope_inputs(65, 6, 2, 64, 64, torch.bfloat16)

    def every():
        return [ops.window_attention(q, k, v, window=400, **where), ops.window_attention(pq, pk, pv, window=300, **pwhere),
                ops.i8_linear(x, w, s), ops.i8_linear(x[:2], w, s), *ops.qk_norm_rope(qkv[:, :6], qkv[:, 6:8], nq, nk, cos, sin, positions=pos)]
    want = every()
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(3):
        for st in (a, b):
            with torch.cuda.stream(st):
                got.append(every())
    graphs = []
    for st in (a, b):
        gr = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(gr, stream=st):
            graphs.append((gr, every()))
    for _ in range(3):
        for st, (gr, _) in zip((a, b), graphs):
            with torch.cuda.stream(st):
                gr.replay()
    torch.cuda.synchronize()
    for outs in got + [o for _, o in graphs]:
        for x1, x2 in zip(outs, want):
            assert torch.equal(x1, x2)


def test_threads_call_at_once_each_on_its_stream():
    import threading
    from cmf_b200 import ops
    g = gen(11)
    q, k, v, _, _, where = attn_inputs([1, 3, 90], [300, 20, 500], 6, 2, 96, torch.bfloat16)
    x = randn(g, 40, 512, dtype=torch.float16)
    w, s = torch.randint(-127, 128, (256, 512), generator=g, device="cuda", dtype=torch.int8), torch.rand(256, generator=g, device="cuda")
    qkv, nq, nk, cos, sin, pos = rope_inputs(65, 6, 2, 64, 64, torch.float32)

    def every():
        return [ops.window_attention(q, k, v, window=100, **where), ops.i8_linear(x, w, s), *ops.quantize_rows(x),
                *ops.qk_norm_rope(qkv[:, :6], qkv[:, 6:8], nq, nk, cos, sin, positions=pos)]
    want = every()
    torch.cuda.synchronize()
    got, errors = [], []

    def work():
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got.append(every())
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # reported by the test's own thread
            errors.append(e)
    threads = [threading.Thread(target=work) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors and len(got) == 80
    assert all(torch.equal(a, b) for outs in got for a, b in zip(outs, want))


@pytest.mark.parametrize("dtype", TYPES)
def test_sequences_that_share_key_rows(dtype):
    """A common beginning of several sequences, read by all of them in place."""
    from cmf_b200 import ops
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    g = gen(12)
    for lens in ([1, 1, 1, 1], [5, 40, 1, 70]):
        q = randn(g, sum(lens), 4, 64, dtype=dtype)
        k, v = randn(g, 300, 2, 64, dtype=dtype), randn(g, 300, 2, 64, dtype=dtype)
        starts, total = [0, 0, 10, 0], [300, 250, 100, 300]
        qs = [sum(lens[:i]) for i in range(5)]
        out = ops.window_attention(q, k, v, window=200, sinks=7, q_start=i32(*qs), k_start=i32(*starts), k_len=i32(*total))
        ref.check(out, *ref.window_attention(q, k, v, lens, starts, total, 200, 7, 0.125, 0.0))


CAPTURE = """
import torch
from cmf_b200 import ops
x = torch.randn(40, 4, 64, device="cuda")
ops.quantize_rows(x[:, 0])                     # the device's context exists; no other kernel has run yet
torch.cuda.synchronize()
w, s = torch.randint(-9, 9, (64, 256), device="cuda", dtype=torch.int8), torch.ones(64, device="cuda")
def calls():
    out = []
    for t in (torch.float32, torch.float16, torch.bfloat16):
        for y in (x.to(t), x.to(t)[..., :20]):
            out.append(ops.window_attention(y, y[:, :2], y[:, 2:], window=9, softcap=5.0))
            out.append(ops.window_attention(y[:1], y[:, :2], y[:, 2:]))
        out += [ops.i8_linear(x.to(t).view(40, 256)[:b], w, s) for b in (1, 12, 40)]
        out += ops.qk_norm_rope(x.to(t), None, s, None, x[:, 0, :32].contiguous(), x[:, 1, :32].contiguous())[:1]
    return out
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = calls()
graph.replay()
torch.cuda.synchronize()
for a, b in zip(got, calls()):
    assert torch.equal(a, b)
print("captured")
"""


def test_first_launches_may_be_captured():
    """A process whose first call of most kernels is inside a capture."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", CAPTURE], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


def test_the_first_call_on_a_device_is_refused_inside_a_capture():
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    code = """
import torch
from cmf_b200 import CmfCudaError, ops
x = torch.ones(4, 64, device="cuda")
torch.cuda.synchronize()
try:
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        try:
            ops.quantize_rows(x)
            code = 0
        except CmfCudaError as e:
            code = e.code
        x.add_(1)
finally:
    print("code", code)
q, s = ops.quantize_rows(x)
torch.cuda.synchronize()
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "code -" in r.stdout, r.stdout + r.stderr[-2000:]


def test_the_status_word_is_clear_and_launches_are_counted():
    from cmf_b200 import gpu, ops
    gpu.set_current_device(0)
    before = gpu.launch_count()
    w, s = torch.ones(16, 64, dtype=torch.int8, device="cuda"), torch.ones(16, device="cuda")
    ops.i8_matmat(*ops.quantize_rows(torch.ones(2, 64, device="cuda")), w, s)
    torch.cuda.synchronize()
    gpu.synchronize()                       # no kernel gave up a wait
    assert gpu.launch_count() == before + 2


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("b,rows,cols", [(1, 2304, 2304), (1, 40, 16), (3, 130, 4096), (8, 300, 4096), (8, 64, 4112), (9, 64, 512), (4, 33, 100), (1, 7, 33), (300, 520, 272)])
def test_i8_linear_is_the_two_operators_in_one(b, rows, cols, dtype):
    """Bit for bit, whether the product rounds the tokens itself or not; rows off the 16-byte boundary too."""
    from cmf_b200 import ops
    g = gen(b + rows)
    wide = randn(g, b, cols + 9, dtype=dtype)
    wide[0, cols // 2] = 40.0
    w = torch.randint(-128, 128, (rows, cols + 16), generator=g, device="cuda", dtype=torch.int8)
    s = torch.rand(rows, generator=g, device="cuda") * 1e-2
    for x, wq in ((wide[:, :cols].contiguous(), w[:, :cols].contiguous()), (wide[:, 1:1 + cols], w[:, :cols]), (wide[:, :cols].contiguous(), w[:, 3:3 + cols])):
        for out in TYPES:
            want = ops.i8_matmat(*ops.quantize_rows(x), wq, s, out_dtype=out)
            assert torch.equal(ops.i8_linear(x, wq, s, out_dtype=out), want)
            canvas = torch.full((b, rows + 5), 3.0, dtype=out, device="cuda")
            ops.i8_linear(x, wq, s, out=canvas[:, 2:2 + rows])
            assert torch.equal(canvas[:, 2:2 + rows], want) and (canvas[:, :2] == 3.0).all() and (canvas[:, 2 + rows:] == 3.0).all()
    assert ops.i8_linear(x, wq, s).dtype == dtype
    bad = wide[:, :cols].contiguous()
    bad[b - 1, 0] = float("inf")
    y = ops.i8_linear(bad, w[:, :cols].contiguous(), s)
    assert torch.isnan(y[b - 1]).all() and torch.isfinite(y[:b - 1].float()).all()
    assert (ops.i8_linear(torch.zeros_like(bad), w[:, :cols].contiguous(), s) == 0).all()
