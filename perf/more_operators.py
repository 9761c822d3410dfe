"""Performance cases of the operators of a decoding step that verifies a tree of drafted tokens.

Four kinds of work, each through the public entry points:

  i8      servoflow_amd.kernels.gemm_i8: a projection in 8-bit integers -- activations quantised by token, weights by
          output channel -- for the hundreds of rows that a tree has, where 4-bit weights stop paying.
  tree    servoflow_amd.attention.attention_kv4 with a draft_tree: every drafted token attends to what is cached and
          to its own ancestors among the drafted ones.
  sample  servoflow_amd.kernels.sample: one token from each row of logits, with temperature, top-k, top-p and min-p,
          from a given uniform number.
  commit  servoflow_amd.attention.draft_tree, accept_tree and Kv4Cache.keep: the tree's tables, the path of drafted
          tokens that the sampled ones confirm, and the cache with that path alone, around the write of the drafted
          tokens' keys and values and a read of what is kept.

Sizes are this repository's own (hidden 2048 = 32 heads x 64, 67 tokens, 4374 keys, FFN 8192, a width of 1152) or
generic ones of decoding: head dims 64 and 128, 1 to 8 query heads for each key head, contexts of up to 16384, trees
of up to 128 tokens, vocabularies of up to 131072.

Definitions that outputs depend on:
  8-bit rows: scale = max |x| / 127 in fp32, code = x / scale to the nearest integer, ties to even (0 for a row of
  zeros).
  4-bit cache: for every token, head and 64 channels mid = bf16((max + min) / 2), a = max |x - mid|, s = (a rounded
  up to bf16) / 8, code = clamp(floor((x - mid) / s) + 8, 0, 15), 8 where s is 0; a code stands for
  s * (code - 7.5) + mid.
  A tree: node j's parent comes before it (-1: none; node 0 is the root, the last token already decided).  The T nodes
  are the last T of a sequence's cached tokens, and the Sq queries the last Sq of them.
  Sampling: weights exp((l - max l) / temperature); tokens in falling order of l, ties by index; the first top_k of
  them; of these the fewest whose weights reach top_p of their sum; of these the ones of at least min_p times the
  largest; the first whose running sum exceeds u times the sum of what is left.  Temperature 0: the first.
"""
import math

import torch

own = False

DEV = "cuda:0"
_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # One robot's 67 token rows through the QKV projection.
        {"name": "i8_qkv_b1", "kind": "i8", "M": 67, "N": 6144, "K": 2048, "dtype": "bf16", "out": "bf16", "act": "none",
         "bias": True},
        # A long prompt through a wide matrix: the matrix units.
        {"name": "i8_prompt", "kind": "i8", "M": 4374, "N": 8192, "K": 8192, "dtype": "bf16", "out": "bf16",
         "act": "none", "bias": False},
        # A ragged head over a width of 1152: odd columns, few rows, GELU, fp32 out.
        {"name": "i8_odd", "kind": "i8", "M": 5, "N": 2051, "K": 1152, "dtype": "fp16", "out": "fp32", "act": "gelu",
         "bias": True},
        # One sequence's small tree over a middling context: latency.
        {"name": "tree_small", "kind": "tree", "B": 1, "Hq": 32, "Hkv": 8, "T": 8, "Sq": 8, "Sk": 2500, "D": 128,
         "dtype": "bf16", "out": "bf16", "short": False, "each": False},
        # Sixteen sequences of different length, each with its own tree.
        {"name": "tree_b16", "kind": "tree", "B": 16, "Hq": 32, "Hkv": 8, "T": 16, "Sq": 16, "Sk": 8192, "D": 128,
         "dtype": "bf16", "out": "bf16", "short": False, "each": True},
        # A wide tree over many key heads.
        {"name": "tree_wide", "kind": "tree", "B": 4, "Hq": 32, "Hkv": 32, "T": 64, "Sq": 64, "Sk": 4374, "D": 64,
         "dtype": "fp16", "out": "fp16", "short": False, "each": False},
        # The newest level of a tree alone, one sequence shorter than its tree, fp32 out.
        {"name": "tree_odd", "kind": "tree", "B": 3, "Hq": 16, "Hkv": 4, "T": 37, "Sq": 21, "Sk": 1537, "D": 64,
         "dtype": "fp16", "out": "fp32", "short": True, "each": True},
        # One sequence's next token: latency.
        {"name": "sample_token", "kind": "sample", "B": 1, "V": 32000, "dtype": "bf16", "rule": "top", "masked": False},
        # Every node of sixteen trees of sixteen, each row with its own parameters, greedy ones among them.
        {"name": "sample_tree", "kind": "sample", "B": 256, "V": 131072, "dtype": "bf16", "rule": "mixed",
         "masked": False},
        # An odd vocabulary with a grammar's forbidden tokens, temperature alone: most of the row stays in play.
        {"name": "sample_odd", "kind": "sample", "B": 37, "V": 50001, "dtype": "fp32", "rule": "temperature",
         "masked": True},
        # One sequence's tree, verified and kept in one layer's cache.
        {"name": "commit_b1", "kind": "commit", "B": 1, "T": 16, "H": 8, "D": 128, "dtype": "bf16", "cap": 2500},
        # Thirty-two sequences' wide trees.
        {"name": "commit_b32", "kind": "commit", "B": 32, "T": 64, "H": 32, "D": 64, "dtype": "bf16", "cap": 4374},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["i8", "i8", "tree", "tree", "tree", "sample", "sample", "sample", "commit"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if kind == "i8":
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        M, N = _log_int(rng, 1, 4374), _log_int(rng, 256, 8192)
        K = 16 * _log_int(rng, 16, 512)
        return {"kind": kind, "M": M, "N": N, "K": K, "dtype": dtype, "out": rng.choice([dtype, dtype, "fp32"]),
                "act": rng.choice(["none", "none", "gelu", "silu"]), "bias": rng.choice([False, True])}
    if kind == "sample":
        V = _log_int(rng, 1000, 131072)
        B = rng.choice([1, _log_int(rng, 1, 256)])
        return {"kind": kind, "B": B, "V": V, "dtype": rng.choice(["bf16", "fp16", "fp32"]),
                "rule": rng.choice(["top", "temperature", "mixed"]), "masked": rng.choice([False, False, True])}
    D, Hkv = rng.choice([64, 128]), rng.choice([1, 2, 4, 8, 8, 16, 32])
    if kind == "commit":
        B, T = _log_int(rng, 1, 32), _log_int(rng, 2, 128)
        while B * T * Hkv * D > 32 * 64 * 32 * 64:
            B = max(1, B // 2)
            T = max(2, T // 2)
        return {"kind": kind, "B": B, "T": T, "H": Hkv, "D": D, "dtype": dtype, "cap": T + _log_int(rng, 1, 4096)}
    Hq = Hkv * rng.choice([1, 2, 4, 8])
    B, T = _log_int(rng, 1, 16), _log_int(rng, 2, 128)
    Sq = rng.choice([T, T, rng.randint(1, T)])
    Sk = T + _log_int(rng, 1, 16384)
    while (B * Hkv * Sk * D > 16 * 8 * 8192 * 128 or B * Hq * Sq * Sk > 16 * 32 * 16 * 8192) and (B > 1 or Sk > 2 * T):
        B, Sk = max(1, B // 2), max(T + 1, Sk // 2 + rng.randint(0, 1))
    return {"kind": kind, "B": B, "Hq": Hq, "Hkv": Hkv, "T": T, "Sq": Sq, "Sk": Sk, "D": D, "dtype": dtype,
            "out": rng.choice([dtype, dtype, "fp32"]), "short": rng.choice([False, False, True]),
            "each": rng.choice([False, True])}


# --- inputs ---------------------------------------------------------------


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) % (1 << 30) * 6007 + 41)
    return g


def _randn(g, *shape, dtype=torch.float32, std=1.0):
    return (torch.randn(*shape, device=DEV, generator=g) * std).to(dtype)


def _randint(g, lo, hi, *shape):
    return torch.randint(lo, hi, shape, device=DEV, generator=g, dtype=torch.int32)


def _i8_inputs(case, seed):
    """Activations with a few channels far above the others, and weights ~ N(0, 0.02) as an 8-bit checkpoint holds them."""
    g, dt = _gen(seed), _DT[case["dtype"]]
    M, N, K = case["M"], case["N"], case["K"]
    gain = 1 + 7 * (torch.rand(K, device=DEV, generator=g) < 0.01)
    w = _randn(g, N, K, std=0.02)
    scale = w.abs().amax(1) / 127
    return {"a": (_randn(g, M, K) * gain).to(dt), "w": torch.round(w / scale[:, None]).to(torch.int8), "scale": scale,
            "bias": _randn(g, N, std=0.02) if case["bias"] else None}


def _parents(g, B, T):
    """Each node's parent among the eight before it, some of them the one before (chains)."""
    at = torch.arange(T, device=DEV, dtype=torch.int32)
    back = (torch.rand(B, T, device=DEV, generator=g).square() * 8).to(torch.int32) + 1
    return torch.where(at > 0, (at - back).clamp_min(0), -1)


def _tree_inputs(case, seed):
    g, dt = _gen(seed), _DT[case["dtype"]]
    B, Hq, Hkv, T, Sq, Sk, D = (case[k] for k in ("B", "Hq", "Hkv", "T", "Sq", "Sk", "D"))
    t = {"q": _randn(g, B, Hq, Sq, D, dtype=dt), "parents": _parents(g, B if case["each"] else 1, T)}
    t["k"] = _randn(g, B, Hkv, Sk, D, dtype=dt) + _randn(g, 1, Hkv, 1, D, dtype=dt, std=0.5)
    t["v"] = _randn(g, B, Hkv, Sk, D, dtype=dt)
    t["valid"] = _randint(g, max(T, Sk // 4), Sk + 1, B)
    if case["short"]:   # a sequence whose first nodes lie before its first token: rows that see nothing
        t["valid"][0] = T - T // 3
    return t


def _sample_inputs(case, seed):
    """Logits as a head leaves them: a broad bulk and a few tokens above it."""
    g, dt = _gen(seed), _DT[case["dtype"]]
    B, V = case["B"], case["V"]
    x = _randn(g, B, V, std=2.0)
    top = torch.randint(0, V, (B, 24), device=DEV, generator=g)
    lift = -3 * torch.log(torch.rand(B, 24, device=DEV, generator=g).clamp_min(1e-6)) + 5
    x = x.scatter_add(1, top, lift)
    if case["masked"]:
        x = torch.where(torch.rand(B, V, device=DEV, generator=g) < 0.3, -math.inf, x)
        x[:, 0] = 1.0
    t = {"logits": x.to(dt), "u": torch.rand(B, device=DEV, generator=g)}
    t["temperature"] = 0.5 + torch.rand(B, device=DEV, generator=g)
    t["top_k"] = t["top_p"] = t["min_p"] = None
    if case["rule"] != "temperature":
        t["top_k"] = torch.full((B,), 50, device=DEV, dtype=torch.int32)
        t["top_p"] = torch.full((B,), 0.9, device=DEV)
    if case["rule"] == "mixed":
        pick = torch.rand(4, B, device=DEV, generator=g)
        t["temperature"] = torch.where(pick[0] < 0.2, 0.0, t["temperature"])
        t["top_k"] = torch.where(pick[1] < 0.5, 0, _randint(g, 1, 200, B))
        t["top_p"] = torch.where(pick[2] < 0.4, 1.0, 0.5 + 0.5 * torch.rand(B, device=DEV, generator=g))
        t["min_p"] = torch.where(pick[3] < 0.5, 0.0, 0.1 * torch.rand(B, device=DEV, generator=g))
    return t


def _commit_inputs(case, seed):
    """Drafted tokens, and sampled ones of which most are a child's."""
    g, dt = _gen(seed), _DT[case["dtype"]]
    B, T, H, D = (case[k] for k in ("B", "T", "H", "D"))
    t = {"parents": _parents(g, B, T), "drafted": _randint(g, 0, 1000, B, T), "sampled": _randint(g, 0, 1000, B, T)}
    p, d = t["parents"].long(), t["drafted"]
    for j in range(1, T):   # the token of one of the children, seven nodes of eight
        take = torch.rand(B, device=DEV, generator=g) < 0.875
        row = torch.arange(B, device=DEV)[take]
        t["sampled"][row, p[take, j]] = d[take, j]
    t["k"], t["v"] = _randn(g, B, H, T, D, dtype=dt), _randn(g, B, H, T, D, dtype=dt)
    t["first"] = _randint(g, 0, case["cap"] - T + 1, B)
    t["slots"] = t["first"][:, None] + torch.arange(T, device=DEV, dtype=torch.int32)
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
    if case["kind"] == "i8":
        return {"case": case, **_i8_inputs(case, seed)}
    if case["kind"] == "sample":
        return {"case": case, **_sample_inputs(case, seed)}
    if case["kind"] == "commit":
        t = _commit_inputs(case, seed)
        if own:
            from servoflow_amd.attention import Kv4Cache
            t["cache"] = Kv4Cache(case["B"], case["H"], case["cap"], case["D"], DEV)
        return {"case": case, **t}
    t = _tree_inputs(case, seed)
    k, v = t.pop("k"), t.pop("v")
    if own:   # the tree's tables serve every layer of the step
        from servoflow_amd.attention import Kv4Cache, draft_tree
        t["cache"] = Kv4Cache(case["B"], case["Hkv"], case["Sk"], case["D"], DEV)
        t["cache"].write(k, v)
        t["tree"] = draft_tree(t["parents"])
    else:
        for name, x in (("k", k), ("v", v)):
            c, s, mid = _quantise(x)
            c = c.flatten(-2).to(torch.uint8)
            t[name] = (c[..., 0::2] | (c[..., 1::2] << 4), s.to(torch.bfloat16), mid.to(torch.bfloat16))
        t["see"] = _ancestors(t["parents"])
    return {"case": case, **t}


# --- the operators' plain forms --------------------------------------------


def _act(name, x):
    if name == "gelu":
        return 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)))
    return x / (1 + torch.exp(-x)) if name == "silu" else x


def _plain_i8(s, c):
    a = s["a"].float()
    scale = a.abs().amax(1, keepdim=True) / torch.full((), 127.0, device=a.device)   # (by a number: times its reciprocal)
    code = torch.round(a.double() / torch.where(scale > 0, scale, 1.0).double())   # next to a border: 64 bits
    y = torch.matmul(code, s["w"].double().t()).float()                            # whole numbers beyond 2^24
    y = y * scale * s["scale"]
    return _act(c["act"], y + s["bias"] if c["bias"] else y).to(_DT[c["out"]])


def _ancestors(parents):
    """see[b, j, i]: node i is node j or one of its ancestors."""
    B, T = parents.shape
    see = torch.zeros(B, T, T, dtype=torch.bool, device=DEV)
    row, p = torch.arange(B, device=DEV), parents.long()
    for j in range(T):
        see[:, j] = see[row, p[:, j].clamp_min(0)] & (p[:, j] >= 0)[:, None]
        see[:, j, j] = True
    return see


def _unpack(c):
    return torch.stack((c & 15, c >> 4), -1).flatten(-2).float()


def _plain_tree(s, c):
    B, Hq, Hkv, T, Sq, Sk, D = (c[k] for k in ("B", "Hq", "Hkv", "T", "Sq", "Sk", "D"))
    k, v = (_value(_unpack(t[0]).unflatten(-1, (-1, 64)), t[1].float(), t[2].float()) for t in (s["k"], s["v"]))
    q = s["q"].float().reshape(B, Hkv, Hq // Hkv * Sq, D) / math.sqrt(D)
    x = torch.matmul(q, k.transpose(2, 3).contiguous()).reshape(B, Hq, Sq, Sk)
    node = torch.arange(Sk, device=DEV) - (s["valid"].long()[:, None] - T)   # [B, Sk]: a slot's node, or before them
    mine = s["see"][:, T - Sq:].expand(B, Sq, T).gather(2, node.clamp(0, T - 1)[:, None].expand(B, Sq, Sk))
    see = (node < 0)[:, None] | ((node < T)[:, None] & mine)
    own_slot = s["valid"].long()[:, None] - Sq + torch.arange(Sq, device=DEV)   # a node before the first token: nothing
    x = x.masked_fill(~(see & (own_slot >= 0)[..., None])[:, None], -math.inf)
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(m > -math.inf, m, 0.0))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.reshape(B, Hkv, -1, Sk), v).reshape(B, Hq, Sq, D)
    return (o / torch.where(total > 0, total, 1.0)).to(_DT[c["out"]])


def _plain_sample(s, c):
    """In 64 bits: a sum over the vocabulary next to a border decides."""
    V = c["V"]
    t = s["temperature"].double()[:, None]
    greedy = t == 0
    x, order = torch.sort(s["logits"].float(), dim=1, descending=True, stable=True)
    w = torch.exp((x.double() - x[:, :1].double()) / torch.where(greedy, 1.0, t))
    at = torch.arange(V, device=DEV)
    keep = (at == 0) | ~greedy
    if s["top_k"] is not None:
        k = s["top_k"].long()[:, None]
        keep = keep & ((at < k) | (k <= 0))
    run = torch.cumsum(w * keep, 1)
    if s["top_p"] is not None:
        p = s["top_p"].double()[:, None]
        before = torch.cat((torch.zeros_like(run[:, :1]), run[:, :-1]), 1)
        keep = keep & ((before < p * run[:, -1:]) | (p >= 1) | (at == 0))
    if s["min_p"] is not None:
        keep = keep & (w >= s["min_p"].double()[:, None])
    run = torch.cumsum(w * keep, 1)
    total = run[:, -1:]
    j = (run <= s["u"].double()[:, None] * total).sum(1, keepdim=True).clamp_max(V - 1)
    j = torch.minimum(j, (w * keep > 0).sum(1, keepdim=True) - 1)
    return order.gather(1, j)[:, 0].to(torch.int32), torch.log(w.gather(1, j) / total)[:, 0].float()


def _plain_commit(s, c):
    B, T = c["B"], c["T"]
    p, drafted, sampled = s["parents"], s["drafted"], s["sampled"]
    depth = _ancestors(p).sum(2).to(torch.int32) - 1
    row, at = torch.arange(B, device=DEV), torch.arange(T, device=DEV)
    cur, live = torch.zeros(B, dtype=torch.long, device=DEV), torch.ones(B, dtype=torch.bool, device=DEV)
    nodes, tokens = (torch.full((B, T), -1, dtype=torch.int32, device=DEV) for _ in range(2))
    for i in range(T):
        nodes[:, i] = torch.where(live, cur.to(torch.int32), -1)
        tok = sampled[row, cur]
        tokens[:, i] = torch.where(live, tok, -1)
        child = (p == cur[:, None].to(torch.int32)) & (drafted == tok[:, None])
        nxt = torch.where(child, at, T).amin(1)
        live = live & (nxt < T)
        cur = torch.where(live, nxt, cur)
    count = (nodes >= 0).sum(1).to(torch.int32)
    pick = torch.where(nodes >= 0, nodes.long(), at)[:, None, :, None].expand(B, c["H"], T, c["D"])
    k, v = (_value(*_quantise(s[n])).gather(2, pick).to(_DT[c["dtype"]]) for n in ("k", "v"))
    return {"depth": depth, "nodes": nodes, "count": count, "tokens": tokens, "k": k, "v": v}


# --- the framework's ---------------------------------------------------------


def _own_i8(s, c):
    from servoflow_amd import abi, kernels
    act = {"none": abi.SF_ACT_NONE, "gelu": abi.SF_ACT_GELU_TANH, "silu": abi.SF_ACT_SILU}[c["act"]]
    return kernels.gemm_i8(s["a"], s["w"], s["scale"], bias=s["bias"], act=act, out_dtype=_DT[c["out"]])


def _own_tree(s, c):
    from servoflow_amd.attention import attention_kv4
    return attention_kv4(s["q"], s["cache"], valid_len=s["valid"], tree=s["tree"], out_dtype=_DT[c["out"]])


def _own_sample(s, c):
    from servoflow_amd import kernels
    return kernels.sample(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                          min_p=s["min_p"])


def _own_commit(s, c):
    from servoflow_amd.attention import accept_tree, draft_tree
    tree = draft_tree(s["parents"])
    s["cache"].write(s["k"], s["v"], s["slots"])
    nodes, count, tokens = accept_tree(tree, s["drafted"], s["sampled"])
    s["cache"].keep(nodes, s["first"])
    k, v = s["cache"].read(s["slots"], _DT[c["dtype"]])
    return {"depth": tree.depth, "nodes": nodes, "count": count, "tokens": tokens, "k": k, "v": v}


_PLAIN = {"i8": _plain_i8, "tree": _plain_tree, "sample": _plain_sample, "commit": _plain_commit}
_OWN = {"i8": _own_i8, "tree": _own_tree, "sample": _own_sample, "commit": _own_commit}


def run(s):
    return (_OWN if own else _PLAIN)[s["case"]["kind"]](s, s["case"])


# --- what a pass cannot do without ----------------------------------------


def work(case):
    e = _BYTES[case["dtype"]]
    if case["kind"] == "i8":
        M, N, K = case["M"], case["N"], case["K"]
        by = M * K * e + N * K + 4 * N * (2 if case["bias"] else 1) + M * N * _BYTES[case["out"]]
        return {"bytes": by, "flops": 2 * M * N * K}
    if case["kind"] == "sample":   # a difference, an exponential, a sum and a comparison for each logit
        return {"bytes": case["B"] * (case["V"] * e + 28), "flops": 4 * case["B"] * case["V"]}
    if case["kind"] == "commit":
        B, T, H, D = (case[k] for k in ("B", "T", "H", "D"))
        token = 2 * H * (D // 64) * 36   # written, half of them moved, read back
        return {"bytes": B * T * (2 * 2 * H * D * e + 3 * token + 7 * 4), "flops": 12 * B * T * 2 * H * D}
    B, Hq, Hkv, T, Sq, Sk, D = (case[k] for k in ("B", "Hq", "Hkv", "T", "Sq", "Sk", "D"))
    keys = (max(T, Sk // 4) + Sk) / 2   # lengths are uniform
    return {"bytes": B * Hkv * keys * (D + D // 64 * 8) + B * Hq * Sq * D * (e + _BYTES[case["out"]]),
            "flops": 4 * B * Hq * Sq * keys * D}


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


def _exact_i8(case, seed):
    t = _i8_inputs(case, seed)
    a = t["a"].double()
    step = torch.div(a.abs().max(1).values.float(), torch.full((a.shape[0],), 127.0, device=DEV)).double()
    q = a / step.clamp_min(1e-300)[:, None]
    lo = torch.floor(q)
    up = (q - lo > 0.5) | ((q - lo == 0.5) & (lo % 2 != 0))
    y = torch.matmul(lo + up, t["w"].double().t()) * step[:, None] * t["scale"].double()
    return _act(case["act"], y if t["bias"] is None else y + t["bias"].double())


def _exact_tree(case, seed):
    t = _tree_inputs(case, seed)
    B, Hq, Hkv, T, Sq, D = (case[k] for k in ("B", "Hq", "Hkv", "T", "Sq", "D"))
    G, par = Hq // Hkv, t["parents"].cpu().tolist()
    out = torch.zeros(B, Hq, Sq, D, dtype=torch.float64, device=DEV)
    for b in range(B):
        n = int(t["valid"][b])
        k, v = _levels64(t["k"][b, :, :n]), _levels64(t["v"][b, :, :n])
        hide = torch.zeros(Sq, n, dtype=torch.bool)
        mine = par[b if case["each"] else 0]
        for s in range(Sq):
            j = T - Sq + s
            hide[s, max(0, n - T):] = True
            if n - T + j < 0:
                hide[s] = True
                continue
            while j >= 0:
                if n - T + j >= 0:
                    hide[s, n - T + j] = False
                j = mine[j]
        hide = hide.to(DEV)
        q = t["q"][b].double().reshape(Hkv, G, Sq, D)
        for j in range(G):
            x = torch.matmul(q[:, j], k.transpose(1, 2).contiguous()) / math.sqrt(D)
            p = torch.softmax(x.masked_fill(hide, -math.inf), -1)
            out[b, j::G] = torch.matmul(torch.nan_to_num(p, nan=0.0), v)
    return out


def _exact_sample(case, seed):
    t = _sample_inputs(case, seed)
    tokens, logs = [], []
    at = lambda name, b, none: none if t[name] is None else t[name][b].item()   # noqa: E731
    for b in range(case["B"]):
        l = t["logits"][b].double()
        order = torch.argsort(-l, stable=True)
        temp, k, p = t["temperature"][b].item(), at("top_k", b, 0), at("top_p", b, 1.0)
        l = l[order]
        n = 1 if temp == 0 else int((l > -math.inf).sum()) if k <= 0 else min(k, int((l > -math.inf).sum()))
        lw = (l[:n] - l[0]) / (temp if temp else 1.0)
        w = torch.exp(lw)
        if p < 1:
            n = min(n, 1 + int((torch.cumsum(w, 0) < p * w.sum()).sum()))
        n = min(n, int((w >= at("min_p", b, 0.0)).sum()))
        run = torch.cumsum(w[:n], 0)
        j = min(n - 1, int(torch.searchsorted(run, t["u"][b].double() * run[-1], right=True)))
        tokens.append(order[j])
        logs.append(lw[j] - torch.log(run[-1]))
    return torch.stack(tokens).to(torch.int32), torch.stack(logs)


def _exact_commit(case, seed):
    t = _commit_inputs(case, seed)
    B, T = case["B"], case["T"]
    par, drafted, sampled = (t[n].cpu().tolist() for n in ("parents", "drafted", "sampled"))
    depth, nodes, tokens = [], [], []
    for b in range(B):
        d = []
        for j in range(T):
            d.append(0 if par[b][j] < 0 else d[par[b][j]] + 1)
        path = [0]
        while True:
            kids = [j for j in range(T) if par[b][j] == path[-1] and drafted[b][j] == sampled[b][path[-1]]]
            if not kids:
                break
            path.append(kids[0])
        depth.append(d)
        nodes.append(path)
        tokens.append([sampled[b][j] for j in path])
    full = lambda rows: torch.tensor([r + [-1] * (T - len(r)) for r in rows], dtype=torch.int32, device=DEV)   # noqa: E731
    k, v = _levels64(t["k"]), _levels64(t["v"])
    for x in (k, v):
        for b in range(B):
            x[b, :, :len(nodes[b])] = x[b][:, nodes[b]]
    return {"depth": full(depth), "nodes": full(nodes),
            "count": torch.tensor([len(r) for r in nodes], dtype=torch.int32, device=DEV), "tokens": full(tokens), "k": k, "v": v}


def exact(case, seed):
    return {"i8": _exact_i8, "tree": _exact_tree, "sample": _exact_sample, "commit": _exact_commit}[case["kind"]](case, seed)
