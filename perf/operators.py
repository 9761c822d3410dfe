"""Performance cases of the 4-bit serving operators.

Four kinds of work, each through the public entry points:

  w4      servoflow_amd.kernels.gemm_w4: a projection whose weights are 4-bit codes with a scale (and an optional
          zero point) for every group of 32, 64 or 128 inputs, on one token's row up to a few batches of rows.
  rope    servoflow_amd.kernels.heads_rope: a projection's rows split into query, key and value heads, the
          per-head RMSNorm and the position rotation of queries and keys in the same pass.
  cache   the same with keys and values going into a 4-bit cache (servoflow_amd.attention.Kv4Cache), and the
          written tokens read back.
  attn    servoflow_amd.attention.attention_kv4: attention over such a cache, from one token's query heads over a
          long context to the action tokens' cross-attention over the image keys.

Sizes are this repository's own (hidden 2048 = 32 heads x 64, 67 tokens, 4374 image keys, FFN 8192, SigLIP's
1152, batch 1 to 16) or generic ones of token-by-token decoding: head dims 64 and 128, 1 to 8 query heads for each
key head, contexts of up to 16384.

The cache's format: for every token, head and 64 channels mid = bf16((max + min) / 2), a = max |x - mid|,
s = (a rounded up to bf16) / 8, code = clamp(floor((x - mid) / s) + 8, 0, 15), 8 where s is 0; a code stands for
s * (code - 7.5) + mid.
"""
import math

import torch

own = False

DEV = "cuda:0"
EPS = 1e-6
_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # One token through a hidden x hidden projection: the smallest call, latency.
        {"name": "w4_token", "kind": "w4", "M": 1, "N": 2048, "K": 2048, "group": 128, "dtype": "bf16", "out": "bf16",
         "zeros": False, "act": "none", "bias": True},
        # One robot's 67 token rows through the QKV projection, with zero points.
        {"name": "w4_qkv_b1", "kind": "w4", "M": 67, "N": 6144, "K": 2048, "group": 64, "dtype": "fp16", "out": "fp16",
         "zeros": True, "act": "none", "bias": True},
        # Sixteen sequences decoding together through a wide matrix: the weight stream.
        {"name": "w4_tokens_b16", "kind": "w4", "M": 16, "N": 8192, "K": 8192, "group": 128, "dtype": "bf16",
         "out": "bf16", "zeros": False, "act": "none", "bias": False},
        # A ragged head over the image encoder's width: odd columns, small groups, GELU, fp32 out.
        {"name": "w4_odd", "kind": "w4", "M": 5, "N": 2051, "K": 1152, "group": 32, "dtype": "fp16", "out": "fp32",
         "zeros": True, "act": "gelu", "bias": True},
        # Eight sequences' next tokens at far positions, keys shared by four query heads each.
        {"name": "rope_token_b8", "kind": "rope", "B": 8, "S": 1, "Hq": 32, "Hkv": 8, "D": 128, "rot": 128,
         "pairs": "halves", "norm": True, "dtype": "bf16", "out": "bf16", "far": 1000000},
        # A long prompt with half of each head rotated in interleaved pairs.
        {"name": "rope_prompt", "kind": "rope", "B": 1, "S": 4374, "Hq": 32, "Hkv": 32, "D": 64, "rot": 32,
         "pairs": "interleaved", "norm": True, "dtype": "fp16", "out": "fp16", "far": 0},
        # Sixteen sequences' next tokens into the cache at ragged places.
        {"name": "cache_token_b16", "kind": "cache", "B": 16, "S": 1, "Hq": 32, "Hkv": 8, "D": 128, "rot": 128,
         "pairs": "halves", "norm": True, "dtype": "bf16", "out": "bf16", "cap": 4096},
        # One frame's image tokens written as a block's cached keys and values (normed keys, no rotation).
        {"name": "cache_frame", "kind": "cache", "B": 1, "S": 4374, "Hq": 0, "Hkv": 32, "D": 64, "rot": 0,
         "pairs": "halves", "norm": True, "dtype": "bf16", "out": "bf16", "cap": 4374},
        # One sequence's next token over a middling context: latency.
        {"name": "attn_token_b1", "kind": "attn", "B": 1, "Hq": 32, "Hkv": 8, "Sq": 1, "Sk": 2500, "D": 128,
         "dtype": "bf16", "out": "bf16", "mask": "none"},
        # Sixteen sequences of different length decoding together: the cache stream.
        {"name": "attn_tokens_b16", "kind": "attn", "B": 16, "Hq": 32, "Hkv": 8, "Sq": 1, "Sk": 16384, "D": 128,
         "dtype": "bf16", "out": "bf16", "mask": "ragged"},
        # Eight robots' action tokens over their six camera views.
        {"name": "attn_image_b8", "kind": "attn", "B": 8, "Hq": 32, "Hkv": 32, "Sq": 67, "Sk": 4374, "D": 64,
         "dtype": "bf16", "out": "bf16", "mask": "none"},
        # A chunk of a prompt behind what is cached, rows that see nothing among them.
        {"name": "attn_chunk", "kind": "attn", "B": 3, "Hq": 16, "Hkv": 4, "Sq": 130, "Sk": 1537, "D": 64,
         "dtype": "fp16", "out": "fp16", "mask": "causal"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["w4", "w4", "rope", "cache", "attn", "attn", "attn"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if kind == "w4":
        group = rng.choice([32, 64, 128, 128])
        M, N = rng.choice([1, _log_int(rng, 1, 16), _log_int(rng, 1, 268)]), _log_int(rng, 256, 8192)
        K = group * max(1, _log_int(rng, 256, 8192) // group)
        return {"kind": kind, "M": M, "N": N, "K": K, "group": group, "dtype": dtype,
                "out": rng.choice([dtype, dtype, "fp32"]), "zeros": rng.choice([False, True]),
                "act": rng.choice(["none", "none", "gelu", "silu"]), "bias": rng.choice([False, True])}
    D = rng.choice([64, 128])
    if kind in ("rope", "cache"):
        Hkv = rng.choice([1, 2, 4, 8, 8, 16, 32])
        Hq = Hkv * rng.choice([1, 2, 4, 8])
        B, S = _log_int(rng, 1, 16), rng.choice([1, _log_int(rng, 1, 4374)])
        while B * S * (Hq + 2 * Hkv) * D > 4374 * 96 * 64 and S > 1:
            S = max(1, S // 2)
        c = {"kind": kind, "B": B, "S": S, "Hq": Hq, "Hkv": Hkv, "D": D,
             "rot": rng.choice([D, D, D // 2, 16 * rng.randint(1, D // 16)]),
             "pairs": rng.choice(["halves", "interleaved"]), "norm": rng.choice([True, True, False]), "dtype": dtype,
             "out": dtype}
        if kind == "rope":
            return {**c, "out": rng.choice([dtype, dtype, "fp32"]), "far": rng.choice([0, 100000, 1000000])}
        return {**c, "cap": S + _log_int(rng, 1, 4096)}
    Hkv = rng.choice([1, 2, 4, 8, 8, 16, 32])
    Hq = Hkv * rng.choice([1, 2, 4, 8])
    B, Sk = _log_int(rng, 1, 16), _log_int(rng, 1, 16384)
    Sq = rng.choice([1, 1, 1, rng.randint(2, 8), 67, rng.randint(17, 256)])
    while (B * Hkv * Sk * D > 16 * 8 * 16384 * 128 or B * Hq * Sq * Sk > 8 * 32 * 67 * 4374) and Sk > 1:
        Sk = max(1, Sk // 2 + rng.randint(0, 1))
    return {"kind": kind, "B": B, "Hq": Hq, "Hkv": Hkv, "Sq": Sq, "Sk": Sk, "D": D, "dtype": dtype,
            "out": rng.choice([dtype, dtype, "fp32"]), "mask": rng.choice(["none", "ragged", "causal", "bytes"])}


# --- inputs ---------------------------------------------------------------


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) % (1 << 30) * 7919 + 29)
    return g


def _randn(g, *shape, dtype=torch.float32, std=1.0):
    return (torch.randn(*shape, device=DEV, generator=g) * std).to(dtype)


def _w4_inputs(case, seed):
    """Activations, and weights ~ N(0, 0.02) as a 4-bit checkpoint holds them: two codes a byte (the even input in
    the low half), a 16-bit scale and a zero point for each group."""
    g, dt = _gen(seed), _DT[case["dtype"]]
    M, N, K, G = (case[k] for k in ("M", "N", "K", "group"))
    w = _randn(g, N, K // G, G, std=0.02)
    if case["zeros"]:
        scale = ((w.amax(-1) - w.amin(-1)) / 15).to(dt)
        zero = torch.round(-w.amin(-1) / scale.float()).clamp(0, 15)
    else:
        scale = (w.abs().amax(-1) / 7).to(dt)
        zero = torch.full((N, K // G), 8.0, device=DEV)
    c = (torch.round(w / scale.float()[..., None]) + zero[..., None]).clamp(0, 15).to(torch.uint8).reshape(N, K)
    return {"a": _randn(g, M, K, dtype=dt), "codes": c[:, 0::2] | (c[:, 1::2] << 4), "scale": scale,
            "zero": zero.to(torch.uint8) if case["zeros"] else None,
            "bias": _randn(g, N, std=0.02) if case["bias"] else None}


def _rope_inputs(case, seed):
    """A projection's rows [B * S][(Hq + 2 Hkv) D], the norms' weights, the tokens' positions and the frequencies."""
    g, dt = _gen(seed), _DT[case["dtype"]]
    B, S, Hq, Hkv, D = (case[k] for k in ("B", "S", "Hq", "Hkv", "D"))
    t = {"p": _randn(g, B * S, (Hq + 2 * Hkv) * D, dtype=dt)}
    t["gq"], t["gk"] = ((1 + _randn(g, D, std=0.1)) if case["norm"] else None for _ in range(2))
    far = case["far"] if case["kind"] == "rope" else case["cap"] - S
    first = torch.randint(0, far + 1, (B, 1), device=DEV, generator=g, dtype=torch.int32)
    t["pos"] = (first + torch.arange(S, device=DEV, dtype=torch.int32)).contiguous()
    half = case["rot"] // 2
    t["freq"] = 10000.0 ** (-torch.arange(half, device=DEV, dtype=torch.float64) / max(half, 1))
    return t


def _attn_inputs(case, seed):
    """Queries, keys and values (keys with a channel-wise offset, as projections' biases leave), and the masks."""
    g, dt = _gen(seed), _DT[case["dtype"]]
    B, Hq, Hkv, Sq, Sk, D = (case[k] for k in ("B", "Hq", "Hkv", "Sq", "Sk", "D"))
    t = {"q": _randn(g, B, Hq, Sq, D, dtype=dt), "valid": None, "bytes": None}
    t["k"] = _randn(g, B, Hkv, Sk, D, dtype=dt) + _randn(g, 1, Hkv, 1, D, dtype=dt, std=0.5)
    t["v"] = _randn(g, B, Hkv, Sk, D, dtype=dt)
    if case["mask"] in ("ragged", "causal"):   # a causal row of fewer cached tokens than queries sees nothing
        t["valid"] = torch.randint(min(Sk, max(1, Sk // 4)), Sk + 1, (B,), device=DEV, generator=g, dtype=torch.int32)
        if case["mask"] == "causal" and Sq > 1:
            t["valid"][0] = min(Sk, Sq - Sq // 3)
    if case["mask"] == "bytes":
        t["bytes"] = torch.rand(B, Sk, device=DEV, generator=g) < 0.8
        t["bytes"][0] = False
    return t


def _quantise(x):
    """Codes, steps and middles of the cache's format for x [..., D] (64 channels a group)."""
    x = x.float().unflatten(-1, (-1, 64))
    mx, mn = x.amax(-1), x.amin(-1)
    mid = (0.5 * mx + 0.5 * mn).to(torch.bfloat16).float()
    a = torch.maximum(mx - mid, mid - mn)
    s = ((a.view(torch.int32) + 0xffff) & -65536).view(torch.float32) * 0.125
    c = torch.floor((x - mid[..., None]) / torch.where(s > 0, s, 1.0)[..., None]).clamp(-8, 7) + 8
    return torch.where(s[..., None] > 0, c, 8.0), s, mid


def _value(c, s, mid):
    return ((c - 7.5) * s[..., None] + mid[..., None]).flatten(-2)


def prepare(case, seed):
    if case["kind"] == "w4":
        t = _w4_inputs(case, seed)
        if own:   # the weights as the kernels read them, laid out once at load
            from servoflow_amd import kernels
            t["w"] = kernels.w4_pack(t.pop("codes"), t.pop("scale"), t.pop("zero"), group=case["group"])
        return {"case": case, **t}
    if case["kind"] in ("rope", "cache"):
        t = _rope_inputs(case, seed)
        if own and case["kind"] == "cache":
            from servoflow_amd.attention import Kv4Cache
            t["cache"] = Kv4Cache(case["B"], case["Hkv"], case["cap"], case["D"], DEV)
        return {"case": case, **t}
    t = _attn_inputs(case, seed)
    k, v = t.pop("k"), t.pop("v")
    if own:
        from servoflow_amd.attention import Kv4Cache
        t["cache"] = Kv4Cache(case["B"], case["Hkv"], case["Sk"], case["D"], DEV)
        t["cache"].write(k, v)
    else:
        for name, x in (("k", k), ("v", v)):
            c, s, mid = _quantise(x)
            c = c.flatten(-2).to(torch.uint8)
            t[name] = (c[..., 0::2] | (c[..., 1::2] << 4), s.to(torch.bfloat16), mid.to(torch.bfloat16))
    return {"case": case, **t}


# --- the operators' plain forms --------------------------------------------


def _unpack(c):
    return torch.stack((c & 15, c >> 4), -1).flatten(-2).float()


def _act(name, x):
    if name == "gelu":
        return 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)))
    return x / (1 + torch.exp(-x)) if name == "silu" else x


def _plain_w4(s, c):
    zero = s["zero"].float()[..., None] if c["zeros"] else 8.0
    w = (_unpack(s["codes"]).unflatten(-1, (-1, c["group"])) - zero) * s["scale"].float()[..., None]
    y = torch.matmul(s["a"].float(), w.flatten(-2).t())
    return _act(c["act"], y + s["bias"] if c["bias"] else y).to(_DT[c["out"]])


def _rotate(x, cos, sin, pairs):
    """x [B, S, H, rot], cos and sin [B, S, 1, rot / 2]."""
    if pairs == "halves":
        a, b = x.chunk(2, -1)
        return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)


def _heads(s, c):
    """Query, key and value heads [B, H, S, D] in 32 bits."""
    B, S, Hq, Hkv, D, rot = (c[k] for k in ("B", "S", "Hq", "Hkv", "D", "rot"))
    x = s["p"].float().reshape(B, S, Hq + 2 * Hkv, D)
    q, k, v = x.split((Hq, Hkv, Hkv), 2)
    if c["norm"]:
        q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + EPS) * s["gq"]
        k = k * torch.rsqrt(k.square().mean(-1, keepdim=True) + EPS) * s["gk"]
    if rot:
        ang = s["pos"].double()[..., None, None] * s["freq"]   # far positions: 64 bits
        cos, sin = torch.cos(ang).float(), torch.sin(ang).float()
        q, k = (torch.cat((_rotate(t[..., :rot], cos, sin, c["pairs"]), t[..., rot:]), -1) for t in (q, k))
    return tuple(t.transpose(1, 2) for t in (q, k, v))


def _plain_rope(s, c):
    return tuple(t.to(_DT[c["out"]]).contiguous() for t in _heads(s, c))


def _plain_cache(s, c):
    q, k, v = _heads(s, c)
    out = {n: _value(*_quantise(t.contiguous())).to(_DT[c["out"]]) for n, t in (("k", k), ("v", v))}
    if c["Hq"]:
        out["q"] = q.to(_DT[c["out"]]).contiguous()
    return out


def _visible(s, c):
    """Which keys each query sees, [B, 1, 1 or Sq, Sk], or None."""
    at = torch.arange(c["Sk"], device=DEV)
    if c["mask"] == "bytes":
        return s["bytes"][:, None, None, :]
    if c["mask"] == "ragged":
        return at < s["valid"][:, None, None, None]
    if c["mask"] == "causal":
        last = s["valid"][:, None, None, None] - c["Sq"] + torch.arange(c["Sq"], device=DEV)[:, None]
        return at <= last
    return None


def _plain_attn(s, c):
    B, Hq, Hkv, Sq, D = (c[k] for k in ("B", "Hq", "Hkv", "Sq", "D"))
    k, v = (_value(_unpack(t[0]).unflatten(-1, (-1, 64)), t[1].float(), t[2].float()) for t in (s["k"], s["v"]))
    q = s["q"].float().reshape(B, Hkv, Hq // Hkv * Sq, D) / math.sqrt(D)
    x = torch.matmul(q, k.transpose(2, 3).contiguous()).reshape(B, Hq, Sq, -1)
    see = _visible(s, c)
    if see is not None:
        x = x.masked_fill(~see, -math.inf)
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(m > -math.inf, m, 0.0))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.reshape(B, Hkv, -1, c["Sk"]), v).reshape(B, Hq, Sq, D)
    return (o / torch.where(total > 0, total, 1.0)).to(_DT[c["out"]])


# --- the framework's ---------------------------------------------------------


def _own_w4(s, c):
    from servoflow_amd import abi, kernels
    act = {"none": abi.SF_ACT_NONE, "gelu": abi.SF_ACT_GELU_TANH, "silu": abi.SF_ACT_SILU}[c["act"]]
    return kernels.gemm_w4(s["a"], s["w"], s["bias"], act=act, out_dtype=_DT[c["out"]])


def _own_rope(s, c):
    from servoflow_amd import kernels
    return kernels.heads_rope(s["p"], c["S"], (c["Hq"], c["Hkv"], c["Hkv"]), c["D"], gammas=(s["gq"], s["gk"]),
                              positions=s["pos"], inv_freq=s["freq"] if c["rot"] else None,
                              interleaved=c["pairs"] == "interleaved", eps=EPS, out_dtype=_DT[c["out"]])


def _own_cache(s, c):
    from servoflow_amd import kernels
    q = kernels.heads_rope(s["p"], c["S"], (c["Hq"], c["Hkv"], c["Hkv"]), c["D"], gammas=(s["gq"], s["gk"]),
                           positions=s["pos"], inv_freq=s["freq"] if c["rot"] else None,
                           interleaved=c["pairs"] == "interleaved", eps=EPS, out_dtype=_DT[c["out"]],
                           cache=s["cache"])[0]
    k, v = s["cache"].read(s["pos"], _DT[c["out"]])
    return {"k": k, "v": v, "q": q} if c["Hq"] else {"k": k, "v": v}


def _own_attn(s, c):
    from servoflow_amd.attention import attention_kv4
    return attention_kv4(s["q"], s["cache"], is_causal=c["mask"] == "causal", valid_len=s["valid"], kv_mask=s["bytes"],
                         out_dtype=_DT[c["out"]])


_PLAIN = {"w4": _plain_w4, "rope": _plain_rope, "cache": _plain_cache, "attn": _plain_attn}
_OWN = {"w4": _own_w4, "rope": _own_rope, "cache": _own_cache, "attn": _own_attn}


def run(s):
    return (_OWN if own else _PLAIN)[s["case"]["kind"]](s, s["case"])


# --- what a pass cannot do without ----------------------------------------


def work(case):
    e, o = _BYTES[case["dtype"]], _BYTES[case["out"]]
    if case["kind"] == "w4":
        M, N, K = case["M"], case["N"], case["K"]
        by = N * K / 2 + N * K // case["group"] * (3 if case["zeros"] else 2) + M * K * e + M * N * o
        return {"bytes": by + (4 * N if case["bias"] else 0), "flops": 2 * M * N * K}
    if case["kind"] in ("rope", "cache"):
        D, kv = case["D"], 2 * case["Hkv"]
        n = case["B"] * case["S"]
        values = n * (case["Hq"] + kv) * D
        by, fl = values * e + n * 4, values * 8
        if case["kind"] == "rope":
            return {"bytes": by + values * o, "flops": fl}
        codes = n * kv * (D // 2 + D // 64 * 4)   # written, and read back to their values
        return {"bytes": by + n * case["Hq"] * D * o + 2 * codes + n * kv * D * o, "flops": fl + 10 * n * kv * D}
    B, Hq, Hkv, Sq, Sk, D = (case[k] for k in ("B", "Hq", "Hkv", "Sq", "Sk", "D"))
    keys = {"none": 1.0, "bytes": 1.0}.get(case["mask"], 0.625) * Sk   # lengths are uniform in [Sk / 4, Sk]
    return {"bytes": B * Hkv * keys * (D + D // 64 * 8) + B * Hq * Sq * D * (e + o), "flops": 4 * B * Hq * Sq * keys * D}


# --- the same in 64 bits ---------------------------------------------------


def _levels64(x):
    """What the cache's format makes of x [..., D], from its definition."""
    y = x.double().reshape(*x.shape[:-1], x.shape[-1] // 64, 64)
    hi, lo = y.max(-1, keepdim=True).values, y.min(-1, keepdim=True).values
    mid = ((hi + lo) / 2).to(torch.bfloat16).double()
    a = (y - mid).abs().max(-1, keepdim=True).values
    e = torch.floor(torch.log2(a.clamp_min(1e-300)))
    ulp = torch.pow(torch.full_like(e, 2.0), e - 7)   # bf16 holds 8 significant bits
    step = torch.ceil(a / ulp) * ulp / 8
    n = torch.floor((y - mid) / torch.where(step > 0, step, torch.ones_like(step))).clamp(-8, 7)
    n = torch.where(step > 0, n, torch.zeros_like(n))
    return ((n + 0.5) * step + mid).reshape(x.shape)


def _exact_heads(case, seed):
    t = _rope_inputs(case, seed)
    B, S, Hq, Hkv, D, rot = (case[k] for k in ("B", "S", "Hq", "Hkv", "D", "rot"))
    x = t["p"].double().reshape(B, S, Hq + 2 * Hkv, D).permute(0, 2, 1, 3)
    out = []
    for part, gamma in ((x[:, :Hq], t["gq"]), (x[:, Hq:Hq + Hkv], t["gk"])):
        if case["norm"]:
            part = part / torch.sqrt((part * part).sum(-1, keepdim=True) / D + EPS) * gamma.double()
        if rot:
            i = torch.arange(rot // 2, device=DEV)
            i, j = (i, i + rot // 2) if case["pairs"] == "halves" else (2 * i, 2 * i + 1)
            turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEV), t["pos"].double()[:, None, :, None] * t["freq"])
            z = torch.complex(part[..., i], part[..., j]) * turn
            part = part.clone()
            part[..., i], part[..., j] = z.real, z.imag
        out.append(part)
    return out[0], out[1], x[:, Hq + Hkv:]


def _exact_attn(case, seed):
    t = _attn_inputs(case, seed)
    B, Hq, Hkv, Sq, Sk, D = (case[k] for k in ("B", "Hq", "Hkv", "Sq", "Sk", "D"))
    out = torch.zeros(B, Hq, Sq, D, dtype=torch.float64, device=DEV)
    for b in range(B):
        n = Sk if t["valid"] is None else int(t["valid"][b])
        k, v = _levels64(t["k"][b, :, :n]), _levels64(t["v"][b, :, :n])
        q = t["q"][b].double().reshape(Hkv, Hq // Hkv, Sq, D)
        for j in range(Hq // Hkv):
            x = torch.matmul(q[:, j], k.transpose(1, 2).contiguous()) / math.sqrt(D)
            if t["bytes"] is not None:
                x[..., ~t["bytes"][b, :n]] = -math.inf
            if case["mask"] == "causal":
                row = torch.arange(Sq, device=DEV)[:, None] + (n - Sq)
                x[:, torch.arange(n, device=DEV)[None, :] > row] = -math.inf
            p = torch.softmax(x, -1)
            p[torch.isnan(p)] = 0   # rows that see nothing
            out[b, j::Hq // Hkv] = torch.matmul(p, v)
    return out


def exact(case, seed):
    if case["kind"] == "w4":
        t, N, K, G = _w4_inputs(case, seed), case["N"], case["K"], case["group"]
        w = torch.empty(N, K, dtype=torch.float64, device=DEV)
        w[:, 0::2], w[:, 1::2] = (t["codes"] & 15).double(), (t["codes"] >> 4).double()
        w = w.reshape(N, K // G, G)
        w -= 8.0 if t["zero"] is None else t["zero"].double()[:, :, None]
        w *= t["scale"].double()[:, :, None]
        y = torch.matmul(t["a"].double(), w.reshape(N, K).t())
        return _act(case["act"], y if t["bias"] is None else y + t["bias"].double())
    if case["kind"] == "rope":
        return _exact_heads(case, seed)
    if case["kind"] == "cache":
        q, k, v = _exact_heads(case, seed)
        out = {"k": _levels64(k), "v": _levels64(v)}
        return {**out, "q": q} if case["Hq"] else out
    return _exact_attn(case, seed)
