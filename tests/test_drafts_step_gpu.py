"""The operators of a step that verifies drafted tokens together, as a program uses them: a small decoder whose tree of
drafts goes through 8-bit projections, head norm + rotation into the 4-bit cache, attention of the tree, a head, the
sampler, the confirmed path and the cache with that path alone.

What such a step accepts has to be what the same decoder gives token by token, with the operators that were there
(causal attention, one query at a time): greedy tokens are equal, and cached tokens are equal bit for bit in the first
layer, whose inputs are.  Then the step captured and replayed, on two streams, and beyond 32 bits."""
import pytest
import torch

from servoflow_amd import kernels
from servoflow_amd.attention import Kv4Cache, accept_tree, attention_kv4, draft_tree

from _drafts import ancestors, random_parents
from _drafts import sample as plain_sample

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32


def _randn(seed, *shape, dtype=F32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def _int(t):
    return torch.as_tensor(t, dtype=torch.int32).to(DEV)


class Decoder:
    """Two layers of attention, a residual stream in fp32, a head; weights in 8 bits."""

    def __init__(self, B, cap, hidden=256, Hq=8, H=2, D=64, V=1000, layers=2, seed=3):
        self.B, self.Hq, self.H, self.D, self.V, self.hidden = B, Hq, H, D, V, hidden
        self.embed = _randn(seed, V, hidden).to(DEV)
        self.layers = []
        for n in range(layers):
            qkv = self.weights(seed + 10 * n + 1, (Hq + 2 * H) * D, hidden)
            out = self.weights(seed + 10 * n + 2, hidden, Hq * D)
            self.layers.append((qkv, out, Kv4Cache(B, H, cap, D, DEV)))
            self.layers[-1][2].data.fill_(0xff)
        self.head = self.weights(seed + 99, V, hidden)
        self.ones = torch.ones(hidden, device=DEV)
        self.freq = (10000.0 ** (-torch.arange(D // 2, dtype=torch.float64) / (D // 2))).to(DEV)

    @staticmethod
    def weights(seed, N, K):
        w = _randn(seed, N, K) * 0.06
        s = w.abs().amax(1) / 127
        return torch.round(w / s[:, None]).to(torch.int8).to(DEV), s.to(DEV)

    def logits(self, tokens, positions, valid, tree=None, causal=False, slots=None):
        """tokens [B, S] at positions, into slots; attention over valid tokens."""
        B, S = tokens.shape
        x = self.embed[tokens.reshape(-1).long()].clone()
        for qkv, out, cache in self.layers:
            p = kernels.gemm_i8(kernels.rmsnorm(x, self.ones), *qkv)
            q, _, _ = kernels.heads_rope(p, S, (self.Hq, self.H, self.H), self.D, positions=positions, inv_freq=self.freq,
                                         cache=cache, slots=slots)
            a = torch.empty(B, S, self.Hq, self.D, dtype=BF, device=DEV)
            attention_kv4(q, cache, out=a.transpose(1, 2), valid_len=valid, tree=tree, is_causal=causal)
            kernels.gemm_i8(a.reshape(B * S, -1), *out, out=x, accumulate=True)
        return kernels.gemm_i8(kernels.rmsnorm(x, self.ones), *self.head, out_dtype=F32).reshape(B, S, -1)

    def prompt(self, tokens):
        B, S = tokens.shape
        pos = torch.arange(S, dtype=torch.int32, device=DEV).expand(B, S).contiguous()
        return self.logits(tokens, pos, torch.full((B,), S, dtype=torch.int32, device=DEV), causal=True)

    def next(self, tokens, lengths):
        """One token each, behind `lengths` cached ones."""
        return self.logits(tokens[:, None], lengths[:, None].contiguous(), lengths + 1)[:, 0]

    def verify(self, tree, drafted, lengths, u, **rule):
        """A tree whose root is the last token decided, behind `lengths` cached ones: nodes, count, tokens, logits."""
        B, T = drafted.shape
        at = torch.arange(T, dtype=torch.int32, device=DEV)
        logits = self.logits(drafted, lengths[:, None] + tree.depth, lengths + T, tree=tree, slots=lengths[:, None] + at)
        sampled, _ = kernels.sample(logits.reshape(B * T, -1), u, **rule)
        nodes, count, tokens = accept_tree(tree, drafted, sampled.reshape(B, T))
        for _, _, cache in self.layers:
            cache.keep(nodes, lengths)
        return nodes, count, tokens, logits


def _drafts(tree, follow, wrong, seed):
    """Drafted tokens of a tree: node j carries the token that its depth has in `follow` on some path, others `wrong`."""
    g = torch.Generator().manual_seed(seed)
    parents, depth = tree.parents.cpu(), tree.depth.cpu()
    B, T = follow.shape[0], parents.shape[1]
    out = torch.empty(B, T, dtype=torch.int32)
    for b in range(B):
        p, d = parents[min(b, len(parents) - 1)], depth[min(b, len(depth) - 1)]
        for j in range(T):
            good = j == 0 or torch.rand((), generator=g) < 0.7
            out[b, j] = follow[b, int(d[j])] if good and int(d[j]) < follow.shape[1] else (wrong + j) % 1000
    return out


@pytest.mark.parametrize("T,each", [(6, False), (21, True), (40, True)])
def test_a_verified_tree_gives_what_token_by_token_gives(T, each):
    B, S0, steps = 3, 17, 12
    cap = S0 + 8 * T + steps
    prompt = torch.randint(0, 1000, (B, S0), generator=torch.Generator().manual_seed(5), dtype=torch.int32).to(DEV)
    # token by token, greedily
    ref = Decoder(B, cap)
    tok = ref.prompt(prompt)[:, -1].argmax(-1).to(torch.int32)
    seq, lengths = [tok], torch.full((B,), S0, dtype=torch.int32, device=DEV)
    for _ in range(steps):
        tok = ref.next(seq[-1], lengths).argmax(-1).to(torch.int32)
        seq.append(tok)
        lengths = lengths + 1
    seq = torch.stack(seq, 1).cpu()
    # by trees of drafts, right ones and wrong ones among them
    dec = Decoder(B, cap)
    root = dec.prompt(prompt)[:, -1].argmax(-1).to(torch.int32)
    assert torch.equal(root.cpu(), seq[:, 0])
    lengths = torch.full((B,), S0, dtype=torch.int32, device=DEV)
    done = [0] * B
    for step in range(4):
        parents = torch.stack([random_parents(T, 50 * step + b, back=3) for b in range(B if each else 1)])
        tree = draft_tree(_int(parents))
        follow = torch.stack([torch.nn.functional.pad(seq[b, done[b]:], (0, T))[:T] for b in range(B)])
        drafted = _drafts(tree, follow, 7 * step, step).to(DEV)
        u = torch.rand(B * T, generator=torch.Generator().manual_seed(step)).to(DEV)
        nodes, count, tokens, _ = dec.verify(tree, drafted, lengths, u, temperature=0.0)
        for b in range(B):
            n = int(count[b])
            path = nodes[b, :n].tolist()
            assert path[0] == 0 and all(int(parents[b if each else 0][j]) == i for i, j in zip(path, path[1:]))
            have = min(n, seq.shape[1] - 1 - done[b])
            assert tokens[b, :have].tolist() == seq[b, done[b] + 1:done[b] + 1 + have].tolist(), (step, b)
            done[b] = min(done[b] + n, seq.shape[1] - 1)
        lengths = lengths + count
        if max(done) >= steps - 2:
            break
    assert max(done) >= 4
    for b in range(B):   # the first layer's keys and values: the same rows went in
        n = min(int(lengths[b]), S0 + steps)
        for got, want in zip(dec.layers[0][2].read(dtype=F32), ref.layers[0][2].read(dtype=F32)):
            assert torch.equal(got[b, :, :n], want[b, :, :n])


def test_step_against_plain_forms():
    """One step's logits against 64 bits on the cached values, and its tokens against the plain sampler."""
    B, S0, T = 2, 40, 24
    dec = Decoder(B, 128, layers=1)
    dec.prompt(torch.randint(0, 1000, (B, S0), generator=torch.Generator().manual_seed(9), dtype=torch.int32).to(DEV))
    lengths = _int([S0, S0 - 13])
    parents = torch.stack([random_parents(T, 3 + b) for b in range(B)])
    tree = draft_tree(_int(parents))
    drafted = torch.randint(0, 1000, (B, T), generator=torch.Generator().manual_seed(1), dtype=torch.int32).to(DEV)
    u = torch.rand(B * T, generator=torch.Generator().manual_seed(2))
    rule = {"temperature": 0.8, "top_k": 60, "top_p": 0.9, "min_p": 0.01}
    nodes, count, tokens, logits = dec.verify(tree, drafted, lengths, u.to(DEV), **rule)
    sampled = torch.tensor([plain_sample(logits.reshape(B * T, -1)[i].cpu(), float(u[i]), float(torch.tensor(0.8)), 60,
                                         float(torch.tensor(0.9)), float(torch.tensor(0.01)))[0] for i in range(B * T)]).reshape(B, T)
    for b in range(B):
        path = [0]
        while True:
            kids = [j for j in range(path[-1] + 1, T) if int(parents[b, j]) == path[-1] and int(drafted[b, j]) == int(sampled[b, path[-1]])]
            if not kids:
                break
            path.append(kids[0])
        assert nodes[b, :len(path)].tolist() == path and int(count[b]) == len(path)
        assert tokens[b, :len(path)].tolist() == [int(sampled[b, j]) for j in path]
    see = ancestors(parents[0])
    assert see.sum() > T   # (branches)


def _inputs(B, T, n):
    out = []
    for i in range(n):
        parents = torch.stack([random_parents(T, 100 + 7 * i + b, back=3) for b in range(B)])
        drafted = torch.randint(0, 6, (B, T), generator=torch.Generator().manual_seed(i), dtype=torch.int32)
        out.append((parents, drafted, torch.rand(B * T, generator=torch.Generator().manual_seed(50 + i))))
    return out


def test_graph_replays_match_eager():
    """A captured step: trees, drafts, uniform numbers and lengths move on the device; eager work and waits between replays."""
    B, T, S0 = 2, 19, 25
    prompt = torch.randint(0, 1000, (B, S0), generator=torch.Generator().manual_seed(5), dtype=torch.int32).to(DEV)
    steps = _inputs(B, T, 5)
    rule = {"temperature": 0.5, "top_k": 4, "top_p": 0.95}
    eager = Decoder(B, 256)
    eager.prompt(prompt)
    lengths = torch.full((B,), S0, dtype=torch.int32, device=DEV)
    ref = []
    for parents, drafted, u in steps:
        tree = draft_tree(parents.to(DEV))
        nodes, count, tokens, logits = eager.verify(tree, drafted.to(DEV), lengths, u.to(DEV), **rule)
        ref.append(tuple(t.clone() for t in (nodes, count, tokens, logits)))
        lengths = lengths + count
    dec = Decoder(B, 256)
    dec.prompt(prompt)
    p, d, u, n = (torch.empty_like(t, device=DEV) for t in (steps[0][0], steps[0][1], steps[0][2], lengths))

    def step():
        return dec.verify(draft_tree(p), d, n, u, **rule)

    p.copy_(steps[0][0]), d.copy_(steps[0][1]), u.copy_(steps[0][2]), n.fill_(100)
    step()   # the kernels are loaded before the capture
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
        n += out[1]
    for _, _, c in dec.layers:
        c.data.fill_(0xff)
    dec.prompt(prompt)
    n.fill_(S0)
    for i, (parents, drafted, uu) in enumerate(steps):
        p.copy_(parents), d.copy_(drafted), u.copy_(uu)
        g.replay()
        for got, want in zip(out, ref[i]):
            assert torch.equal(got, want), i
        (torch.randn(512, 512, device=DEV) @ torch.randn(512, 512, device=DEV)).sum().item()
    assert torch.equal(n, lengths)


def test_graph_replays_of_the_sampler_and_the_products():
    """Captured alone, with workspaces that the capture keeps: rows in parts, 16-bit rows with the second launch, both products."""
    x32 = _randn(1, 3, 70001).to(DEV) * 2
    x16 = (_randn(2, 5, 70001) * 2).to(BF).to(DEV)
    u = torch.rand(5, generator=torch.Generator().manual_seed(1)).to(DEV)
    w, t = Decoder.weights(4, 300, 512)
    a = _randn(3, 200, 512, dtype=BF).to(DEV)

    def all_of_it():
        return (*kernels.sample(x32, u[:3], top_p=0.97), *kernels.sample(x16, u), kernels.gemm_i8(a, w, t), kernels.gemm_i8(a[:2], w, t))

    all_of_it()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = all_of_it()
    for i in range(4):
        x32.copy_(_randn(20 + i, 3, 70001) * 2)
        x16.copy_(_randn(30 + i, 5, 70001) * 2)
        a.copy_(_randn(40 + i, 200, 512))
        if i == 2:
            x16[1] = 0.25   # more than 65535 of one value
        g.replay()
        got = [o.clone() for o in out]
        for x, y in zip(got, all_of_it()):
            assert torch.equal(x, y), i


def test_streams():
    """Two programs at once, each with what it needs of its own."""
    B, T, Sk, D = 1, 16, 3000, 128
    tree = draft_tree(_int(random_parents(T, 4)))
    caches, qs, xs, refs = [], [], [], []
    w, t = Decoder.weights(4, 700, 512)
    u = torch.tensor([0.4, 0.9], device=DEV)
    for i in range(2):
        c = Kv4Cache(B, 2, Sk, D, DEV)
        c.write(_randn(70 + i, B, 2, Sk, D, dtype=BF).to(DEV), _randn(75 + i, B, 2, Sk, D, dtype=BF).to(DEV))
        caches.append(c), qs.append(_randn(80 + i, B, 8, T, D, dtype=BF).to(DEV)), xs.append(_randn(85 + i, 2, 90001).to(DEV) * 2)

    def work(i):
        a = attention_kv4(qs[i], caches[i], tree=tree, num_splits=6)
        return a, kernels.gemm_i8(a.reshape(-1, 512), w, t), *kernels.sample(xs[i], u, top_p=0.9)

    refs = [work(i) for i in range(2)]
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(15):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(work(i))
    torch.cuda.synchronize()
    for i in range(2):
        for o in outs[i]:
            assert all(torch.equal(x, y) for x, y in zip(o, refs[i]))


def test_beyond_32_bits():
    """Logits and activations of more than 2^32 bytes, their last rows; a cache of 4.5 GiB, its last tokens."""
    rows, V = 70000, 32768
    x = torch.zeros(rows, V, dtype=BF, device=DEV)
    assert x.numel() * 2 > 1 << 32
    tail = (_randn(5, 3, V) * 2).to(BF)
    x[-3:] = tail.to(DEV)
    u = torch.full((rows,), 0.37, device=DEV)
    tok, lp = kernels.sample(x, u, top_p=0.9)
    want, lw = kernels.sample(x[-3:].clone(), u[-3:], top_p=0.9)
    assert torch.equal(tok[-3:], want) and torch.equal(lp[-3:], lw)
    assert (tok[:-3] == tok[0]).all()
    del x
    M, K, N = 270000, 16384, 40
    a = torch.zeros(M, K, dtype=torch.int8, device=DEV)
    assert a.numel() > 1 << 32
    a[-70:] = torch.randint(-128, 128, (70, K), dtype=torch.int8, device=DEV)
    w, t = Decoder.weights(6, N, K)
    s = torch.ones(M, device=DEV)
    y = kernels.gemm_i8(a, w, t, s)
    assert torch.equal(y[-70:], kernels.gemm_i8(a[-70:].clone(), w, t, s[-70:])) and (y[:-70] == 0).all()
    del a
    B, H, D, cap, n = 4, 4, 64, 1 << 22, 40
    c = Kv4Cache(B, H, cap, D, DEV)
    assert c.data.numel() > 1 << 32
    at = _int(torch.arange(cap - n, cap).expand(B, n).contiguous())
    k, v = _randn(80, B, H, n, D, dtype=BF).to(DEV), _randn(81, B, H, n, D, dtype=BF).to(DEV)
    c.write(k, v, at)
    was = c.read(at, F32)
    nodes = torch.full((B, n), -1, dtype=torch.int32, device=DEV)
    nodes[:, :20] = torch.arange(0, 40, 2, dtype=torch.int32, device=DEV)
    c.keep(nodes, at[:, 0].contiguous())
    for got, old in zip(c.read(at, F32), was):
        assert torch.equal(got[:, :, :20], old[:, :, ::2]) and torch.equal(got[:, :, 20:], old[:, :, 20:])
    valid = torch.full((B,), cap, dtype=torch.int32, device=DEV)
    tree = draft_tree(_int(random_parents(n, 3)))
    mask = torch.zeros(B, cap, dtype=torch.bool, device=DEV)
    mask[:, -n:] = True
    q = _randn(82, B, 8, n, D, dtype=BF).to(DEV)
    kk, vv = c.read(at, F32)
    small = Kv4Cache(B, H, n, D, DEV)
    small.write(kk.to(BF), vv.to(BF))
    got = attention_kv4(q, c, valid_len=valid, kv_mask=mask, tree=tree, out_dtype=F32)
    from _drafts import attend_see, tree_sees
    ref = attend_see(q.cpu(), kk.cpu(), vv.cpu(), tree_sees([tree.parents[0].cpu()], n, n, [n] * B))
    assert float((got.cpu().double() - ref).abs().max()) <= 1e-4 * float(vv.abs().max())


def test_step_logits_in_64_bits():
    """Each stage of a verified step, both layers to the logits, from what went into it: norms, 8-bit products, rotated queries, what
    is cached, attention by the ancestors' mask over the cached values, the residual sum.  The kernels give the same in the step
    itself, bit for bit.  A norm takes sums of 256 squares, 16 roundings at most; products, rotation and attention: the
    tolerances of their own tests."""
    from _drafts import attend_see, quant, tree_sees
    from _quant4 import half_step, rotate
    B, S0, T = 2, 40, 24
    dec = Decoder(B, 128)
    dec.prompt(torch.randint(0, 1000, (B, S0), generator=torch.Generator().manual_seed(9), dtype=torch.int32).to(DEV))
    lengths = _int([S0, S0 - 13])
    parents = torch.stack([random_parents(T, 3 + b) for b in range(B)])
    assert all(len(set(p.tolist())) < T - 1 for p in parents)   # branches
    tree = draft_tree(_int(parents))
    drafted = torch.randint(0, 1000, (B, T), generator=torch.Generator().manual_seed(1), dtype=torch.int32).to(DEV)
    slots = lengths[:, None] + torch.arange(T, dtype=torch.int32, device=DEV)
    positions, valid = lengths[:, None] + tree.depth, lengths + T
    pos, freq = positions.cpu(), dec.freq.cpu()
    see = tree_sees(list(parents), T, 128, valid.tolist())
    Hq, H, D = dec.Hq, dec.H, dec.D

    def near(got, ref, tol, what):
        err = (got.cpu().double() - ref).abs()
        assert (err <= tol).all(), f"{what}: {float((err / tol.clamp_min(1e-300)).max())} of the tolerance"

    def normed(x, what):
        h = kernels.rmsnorm(x, dec.ones)
        y = x.cpu().double()
        ref = y / torch.sqrt(y.square().mean(1, keepdim=True) + 1e-6)
        near(h, ref, (2.0 ** -20 + half_step(BF)) * ref.abs(), what)
        return h

    def product(rows, w, t):
        codes, s = quant(rows.cpu())
        ref = (codes @ w.cpu().double().t()) * s.double()[:, None] * t.cpu().double()
        return ref, 6 * 2.0 ** -24 * ref.abs()

    x = dec.embed[drafted.reshape(-1).long()].clone()
    for n, (qkv, out, cache) in enumerate(dec.layers):
        h = normed(x, f"layer {n}: norm")
        p = kernels.gemm_i8(h, *qkv)
        ref, tol = product(h, *qkv)
        near(p, ref, tol + half_step(BF) * (ref.abs() + tol), f"layer {n}: qkv")
        q, _, _ = kernels.heads_rope(p, T, (Hq, H, H), D, positions=positions, inv_freq=dec.freq, cache=cache, slots=slots)
        heads = p.cpu().double().reshape(B, T, Hq + 2 * H, D).transpose(1, 2)
        ref = rotate(heads[:, :Hq], pos, freq, False)
        turn = 40 * 2.0 ** -24 * 2 * heads.abs().amax(-1, keepdim=True)
        near(q, ref, turn[:, :Hq] + half_step(BF) * ref.abs(), f"layer {n}: queries")
        k, v = (t.cpu() for t in cache.read(dtype=F32))
        for cached, new, what in ((k, rotate(heads[:, Hq:Hq + H], pos, freq, False), "keys"), (v, heads[:, Hq + H:], "values")):
            got = torch.stack([cached[b, :, lengths[b]:lengths[b] + T] for b in range(B)])
            top = new.abs().amax(-1, keepdim=True)
            half = (new.amax(-1, keepdim=True) - new.amin(-1, keepdim=True)) / 2 + 2.0 ** -8 * top   # furthest from the middle, in bf16
            near(got, new, half * (1 + 2.0 ** -7) / 16 + 2.0 ** -16 * top, f"layer {n}: cached {what}")   # half a step; |value - new|
        a = torch.empty(B, T, Hq, D, dtype=BF, device=DEV)
        attention_kv4(q, cache, out=a.transpose(1, 2), valid_len=valid, tree=tree)
        seen = [slice(0, int(m)) for m in valid]
        for b in range(B):   # (what no one has written yet reads as NaN)
            kb, vb = k[b:b + 1, :, seen[b]], v[b:b + 1, :, seen[b]]
            qb = q[b:b + 1].cpu()
            ref = attend_see(qb, kb, vb, see[b:b + 1, :, seen[b]])
            dx = 24 * 2.0 ** -24 / 8 * float(qb.double().abs().sum(-1).max()) * float(kb.abs().max()) * 6
            rel = 2 * (dx + 2.0 ** -22) + 2.0 ** -16 + (32 + 128 / 32) * 2.0 ** -24 * 16
            near(a[b:b + 1].transpose(1, 2), ref, rel * float(vb.abs().max()) + half_step(BF) * ref.abs(), f"layer {n}: attention {b}")
        was = x.cpu().double()
        rows = a.reshape(B * T, -1)
        ref, tol = product(rows, *out)
        kernels.gemm_i8(rows, *out, out=x, accumulate=True)
        near(x, was + ref, tol + 2.0 ** -24 * (was + ref).abs(), f"layer {n}: sum")
    h = normed(x, "head: norm")
    logits = kernels.gemm_i8(h, *dec.head, out_dtype=F32)
    ref, tol = product(h, *dec.head)
    near(logits, ref, tol, "logits")
    again = dec.verify(tree, drafted, lengths, torch.full((B * T,), 0.3, device=DEV))[3]
    assert torch.equal(again.reshape(B * T, -1), logits)
