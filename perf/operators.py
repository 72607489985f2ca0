"""What is measured of the operators for text-model attention layers: head norms with the position rotation, causal
attention with a sliding window and first tokens that stay visible, and matrix products in 8-bit integers.

``own`` chooses between the plain form (elementary torch operations in 32 bits) and the framework's kernels."""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # head norms + rotation.  One generated token of the 24 / 8 x 96 head layout: launch latency.
        dict(name="rope_one_token", op="rope", n=1, nh=24, nkv=8, hd=96, rot=96, half=False, type="bf16", table=8192),
        # a pair of 1024 x 1024 sequences with their captions (2 x 4352 tokens), f32 projections as the GEMMs write them
        dict(name="rope_two_images", op="rope", n=8704, nh=24, nkv=8, hd=96, rot=96, half=False, type="f32", table=8704),
        # an odd batch of prompts in the 8 / 4 x 256 layout, half-split pairs, three quarters of a head rotated
        dict(name="rope_prompts", op="rope", n=5531, nh=8, nkv=4, hd=256, rot=192, half=True, type="f16", table=16384),
        # windowed attention.  One prompt twice as long as the 4096 window, logits capped at 50, wide heads
        dict(name="attn_long_prompt", op="attn", lens="8192", prior="0", nh=8, nkv=4, hd=256, window=4096, sinks=0, cap=50.0, type="bf16"),
        # a ragged batch, one token to a few thousand, in the 24 / 8 x 96 layout, four first tokens always visible
        dict(name="attn_ragged_batch", op="attn", lens="1,77,513,2999,130,1024,1531", prior="0,0,0,0,0,0,0", nh=24, nkv=8, hd=96,
             window=1000, sinks=4, cap=0.0, type="bf16"),
        # chunks of prompts appended behind what their caches already hold
        dict(name="attn_chunks", op="attn", lens="512,300,512,999", prior="4096,1000,7000,0", nh=16, nkv=4, hd=128, window=2048, sinks=16,
             cap=0.0, type="f16"),
        # one generated token of one short sequence: launch latency
        dict(name="attn_one_token", op="attn", lens="1", prior="130", nh=24, nkv=8, hd=96, window=4096, sinks=4, cap=0.0, type="bf16"),
        # one generated token for each of 64 sequences with caches around and beyond the window
        dict(name="attn_tokens_64", op="attn", lens=",".join(["1"] * 64), prior=",".join(str(700 + 117 * i) for i in range(64)), nh=8, nkv=4,
             hd=256, window=4096, sinks=4, cap=50.0, type="bf16"),
        # 32-bit queries, keys and values (the prompt encoder's own type)
        dict(name="attn_f32", op="attn", lens="1200,331", prior="0,0", nh=8, nkv=4, hd=256, window=512, sinks=0, cap=50.0, type="f32"),
        # 8-bit products.  One token through a square projection: launch latency and the weights' bytes
        dict(name="i8_one_token", op="i8", m=1, n=2304, k=2304, type="bf16", out="f32"),
        # an odd number of tokens through a down projection
        dict(name="i8_down_333", op="i8", m=333, n=2304, k=9216, type="f16", out="f32"),
        # a pair of 1024 x 1024 sequences through the gate / up projection
        dict(name="i8_gate_up", op="i8", m=8704, n=18432, k=2304, type="bf16", out="bf16"),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "attn", "attn", "attn", "i8"])
    if op == "rope":
        hd = rng.choice([64, 96, 128, 256])
        nkv = rng.choice([1, 2, 4, 8])
        rot = hd if rng.random() < 0.7 else hd // 2
        n = _spread(rng, 1, 8704)
        return dict(op="rope", n=n, nh=nkv * rng.choice([1, 2, 3, 4]), nkv=nkv, hd=hd, rot=rot, half=rng.random() < 0.5,
                    type=rng.choice(["f32", "f16", "bf16"]), table=max(n, _spread(rng, 1000, 16384)))
    if op == "attn":
        nkv = rng.choice([1, 2, 4, 8])
        type_ = rng.choice(["bf16", "bf16", "f16", "f32"])
        form = rng.choice(["prompts", "chunks", "tokens"])
        if form == "tokens":
            count = _spread(rng, 1, 64)
            lens, prior = [1] * count, [_spread(rng, 1, 8000) for _ in range(count)]
        else:
            count = rng.randint(1, 6)
            most = 3000 if type_ != "f32" else 1200
            lens = [_spread(rng, 1, most) for _ in range(count)]
            prior = [_spread(rng, 1, 3000) if form == "chunks" else 0 for _ in range(count)]
        return dict(op="attn", lens=",".join(map(str, lens)), prior=",".join(map(str, prior)), nh=nkv * rng.choice([1, 2, 3, 4]), nkv=nkv,
                    hd=rng.choice([64, 96, 128, 256]), window=_spread(rng, 16, 8192), sinks=rng.choice([0, 0, 4, 16, 130]),
                    cap=rng.choice([0.0, 0.0, 50.0]), type=type_)
    return dict(op="i8", m=_spread(rng, 1, 4352), n=16 * _spread(rng, 16, 576), k=16 * _spread(rng, 16, 576),
                type=rng.choice(["f32", "f16", "bf16"]), out=rng.choice(["f32", "bf16", "f16"]))


def _ints(text):
    return [int(x) for x in text.split(",")]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def prepare(case, seed):
    g, dev = _gen(seed), "cuda"
    st = dict(case)
    if case["op"] == "rope":
        # a fused projection's output: queries, keys and values of a token side by side
        n, nh, nkv, hd = case["n"], case["nh"], case["nkv"], case["hd"]
        qkv = torch.randn(n, nh + 2 * nkv, hd, generator=g, device=dev) * 1.7
        qkv = qkv.to(TYPES[case["type"]])
        st["q"], st["k"] = qkv[:, :nh], qkv[:, nh:nh + nkv]
        st["norm_q"] = 1.0 + 0.2 * torch.randn(hd, generator=g, device=dev)
        st["norm_k"] = 1.0 + 0.2 * torch.randn(hd, generator=g, device=dev)
        angle = torch.arange(case["table"], dtype=torch.float64, device=dev)[:, None] * 10000.0 ** (
            -torch.arange(case["rot"] // 2, dtype=torch.float64, device=dev) * 2 / case["rot"])
        st["cos"], st["sin"] = angle.cos().float(), angle.sin().float()
        st["positions"] = torch.randint(0, case["table"], (n,), generator=g, device=dev, dtype=torch.int32)
        return st
    if case["op"] == "attn":
        lens, prior = _ints(case["lens"]), _ints(case["prior"])
        nh, nkv, hd, t = case["nh"], case["nkv"], case["hd"], TYPES[case["type"]]
        total = [a + b for a, b in zip(lens, prior)]
        if any(prior):
            cap = (max(total) + 127) // 128 * 128       # a cache of equal slots
            starts, rows = [i * cap for i in range(len(lens))], cap * len(lens)
        else:
            starts = [sum(total[:i]) for i in range(len(total))]
            rows = sum(total)
        st["q"] = torch.randn(sum(lens), nh, hd, generator=g, device=dev, dtype=t) * 1.5
        st["k"] = torch.randn(rows, nkv, hd, generator=g, device=dev, dtype=t)
        st["v"] = torch.randn(rows, nkv, hd, generator=g, device=dev, dtype=t)
        st["q_start"] = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=dev)
        st["k_start"] = torch.tensor(starts, dtype=torch.int32, device=dev)
        st["k_len"] = torch.tensor(total, dtype=torch.int32, device=dev)
        st["max_q"], st["max_k"] = max(lens), max(total)
        st["scale"] = hd ** -0.5
        return st
    m, n, k = case["m"], case["n"], case["k"]
    x = torch.randn(m, k, generator=g, device=dev)
    x[:, torch.randint(0, k, (max(1, k // 300),), generator=g, device=dev)] *= 12.0     # channels with large activations
    st["x"] = x.to(TYPES[case["type"]])
    w = torch.randn(n, k, generator=g, device=dev) * 0.02
    st["w_scale"] = w.abs().amax(1) / 127
    st["w_q"] = (w / st["w_scale"][:, None]).round().to(torch.int8)
    return st


def _plain_rope(x, weight, cos, sin, rot, half, eps=1e-5):
    y = x.float()
    y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + eps) * weight
    r, rest = y[..., :rot], y[..., rot:]
    c, s = cos[:, None], sin[:, None]
    if half:
        a, b = r[..., :rot // 2], r[..., rot // 2:]
        r = torch.cat([a * c - b * s, a * s + b * c], -1)
    else:
        a, b = r[..., 0::2], r[..., 1::2]
        r = torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2)
    return torch.cat([r, rest], -1).to(x.dtype)


def _plain_attention(st):
    q, k, v, q_start, k_start, k_len = st["q"], st["k"], st["v"], st["q_start"], st["k_start"], st["k_len"]
    count, nkv, hd, group = k_len.numel(), st["nkv"], st["hd"], st["nh"] // st["nkv"]
    i, j = torch.arange(st["max_q"], device=q.device), torch.arange(st["max_k"], device=q.device)
    q_len = q_start[1:] - q_start[:-1]
    qp = q[(q_start[:-1, None] + i).clamp(max=q.shape[0] - 1)].float()           # [count, max_q, nh, hd]
    at = (k_start[:, None] + j).clamp(max=k.shape[0] - 1)
    kp, vp = k[at].float(), v[at].float()                                        # [count, max_k, nkv, hd]
    qp = qp.reshape(count, -1, nkv, group, hd).permute(0, 2, 3, 1, 4)
    s = torch.matmul(qp.reshape(count, nkv, -1, hd), kp.permute(0, 2, 3, 1)).reshape(count, nkv, group, len(i), len(j))
    s = s * st["scale"]
    if st["cap"]:
        s = st["cap"] * torch.tanh(s / st["cap"])
    p = (k_len - q_len)[:, None, None] + i[None, :, None]
    seen = (j <= p) & ((p - j < st["window"]) | (j < st["sinks"]))
    s = s.masked_fill(~seen[:, None, None], -math.inf)
    e = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e30))
    o = torch.matmul((e / e.sum(-1, keepdim=True).clamp(min=1e-30)).reshape(count, nkv, -1, len(j)), vp.permute(0, 2, 1, 3))
    o = o.reshape(count, nkv * group, len(i), hd)
    t = torch.arange(q.shape[0], device=q.device)
    b = torch.searchsorted(q_start[1:].contiguous(), t.int(), right=True)
    return o[b, :, t - q_start[b]].to(q.dtype)


def _plain_i8(st):
    x = st["x"].float()
    scale = x.abs().amax(1, keepdim=True) / 127
    xq = (x / scale).round()
    return (torch.matmul(xq, st["w_q"].float().t()) * scale * st["w_scale"]).to(TYPES[st["out"]])


def run(st):
    if own:
        from cmf_b200 import ops
    if st["op"] == "rope":
        if own:
            return ops.qk_norm_rope(st["q"], st["k"], st["norm_q"], st["norm_k"], st["cos"], st["sin"], positions=st["positions"],
                                    half_split=st["half"])
        cos, sin = st["cos"][st["positions"]], st["sin"][st["positions"]]
        return (_plain_rope(st["q"], st["norm_q"], cos, sin, st["rot"], st["half"]),
                _plain_rope(st["k"], st["norm_k"], cos, sin, st["rot"], st["half"]))
    if st["op"] == "attn":
        if own:
            return ops.window_attention(st["q"], st["k"], st["v"], window=st["window"], sinks=st["sinks"], scale=st["scale"],
                                        softcap=st["cap"], q_start=st["q_start"], k_start=st["k_start"], k_len=st["k_len"])
        return _plain_attention(st)
    if own:
        return ops.i8_linear(st["x"], st["w_q"], st["w_scale"], out_dtype=TYPES[st["out"]])
    return _plain_i8(st)


def _pairs(length, prior, window, sinks):
    """(key rows that some query sees, query-key pairs) of one sequence."""
    pairs = 0
    for p in range(prior, prior + length):
        low = max(0, p - window + 1)
        pairs += p + 1 - low + min(sinks, low)
    low = max(0, prior - window + 1)
    return prior + length - low + min(sinks, low), pairs


def work(case):
    if case["op"] == "rope":
        values = case["n"] * (case["nh"] + case["nkv"]) * case["hd"]
        return {"bytes": 2 * values * BYTES[case["type"]] + case["n"] * (case["rot"] * 4 + 4), "flops": 8 * values}
    if case["op"] == "attn":
        lens = _ints(case["lens"])
        each = [_pairs(a, b, case["window"], case["sinks"]) for a, b in zip(lens, _ints(case["prior"]))]
        size = case["hd"] * BYTES[case["type"]]
        return {"bytes": 2 * sum(lens) * case["nh"] * size + 2 * sum(r for r, _ in each) * case["nkv"] * size,
                "flops": 4 * case["hd"] * case["nh"] * sum(p for _, p in each)}
    m, n, k = case["m"], case["n"], case["k"]
    return {"bytes": m * k * BYTES[case["type"]] + n * k + 4 * n + m * n * BYTES[case["out"]], "flops": 2 * m * n * k}


def _exact_head(x, weight, cos, sin, rot, half):
    x = x.double()
    x = x / (x.square().mean(-1, keepdim=True) + 1e-5).sqrt() * weight.double()
    z = torch.view_as_complex(torch.stack([x[..., :rot // 2], x[..., rot // 2:rot]] if half else [x[..., 0:rot:2], x[..., 1:rot:2]], -1).contiguous())
    z = torch.view_as_real(z * torch.complex(cos.double(), sin.double())[:, None])
    out = x.clone()
    if half:
        out[..., :rot // 2], out[..., rot // 2:rot] = z[..., 0], z[..., 1]
    else:
        out[..., 0:rot:2], out[..., 1:rot:2] = z[..., 0], z[..., 1]
    return out


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "rope":
        at = st["positions"].long()
        return tuple(_exact_head(st[x], st["norm_" + x], st["cos"][at], st["sin"][at], case["rot"], case["half"]) for x in ("q", "k"))
    if case["op"] == "attn":
        # sequence by sequence and key head by key head, in blocks of queries with the keys that the block can see
        out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
        group, first = case["nh"] // case["nkv"], 0
        for length, prior, start in zip(_ints(case["lens"]), _ints(case["prior"]), st["k_start"].tolist()):
            for i0 in range(0, length, 512):
                i1 = min(length, i0 + 512)
                low, high = max(0, prior + i0 - case["window"] + 1), prior + i1
                keys = torch.cat([torch.arange(min(case["sinks"], low)), torch.arange(low, high)]).cuda()
                pos = torch.arange(prior + i0, prior + i1, device="cuda")
                hidden = (keys[None] > pos[:, None]) | ((keys[None] <= pos[:, None] - case["window"]) & (keys[None] >= case["sinks"]))
                for h in range(case["nh"]):
                    kk, vv = st["k"][start + keys, h // group].double(), st["v"][start + keys, h // group].double()
                    s = st["q"][first + i0:first + i1, h].double() @ kk.t() * st["scale"]
                    if case["cap"]:
                        s = case["cap"] * torch.tanh(s / case["cap"])
                    out[first + i0:first + i1, h] = torch.softmax(s.masked_fill(hidden, -math.inf), -1) @ vv
            first += length
        return out
    # the 8-bit levels are part of the definition: scale and quotient are numbers of 32 bits, rounded from the exact ones
    x = st["x"].double()
    scale = (x.abs().amax(1, keepdim=True) / 127).float().double()
    levels = (x / scale).float().double().round()
    return (levels @ st["w_q"].double().t()) * scale * st["w_scale"].double()
