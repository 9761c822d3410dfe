"""Trees of drafted tokens: their tables, attention of their nodes over the 4-bit
cache, the confirmed path and the cache with that path alone, against plain forms.

Tables, paths and kept tokens are whole numbers or bytes, and equal.  Attention:
the tolerance of test_kv4_gpu, without its part for values in fp16, which a tree's
rows never take."""
import math

import pytest
import torch

from servoflow_amd import kernels
from servoflow_amd.attention import DraftTree, Kv4Cache, accept_tree, attention_kv4, draft_tree

from _drafts import accept, ancestors, attend_see, random_parents, tree_sees
from _quant4 import half_step, kv4_levels

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


def _randn(seed, *shape, dtype=F32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def _int(t):
    return torch.as_tensor(t, dtype=torch.int32).to(DEV)


def _bits(masks, T):
    """[n, T, words] -> bool [n, T, 32 words]."""
    m = masks.cpu().long() & 0xffffffff
    return ((m[..., None] >> torch.arange(32)) & 1).bool().flatten(-2)


@pytest.mark.parametrize("T", [1, 2, 31, 32, 33, 64, 100, 1024])
@pytest.mark.parametrize("n", [1, 3])
def test_tables(T, n):
    parents = torch.stack([random_parents(T, 10 * T + i, back=3 if i == 1 else 8) for i in range(n)])
    tree = draft_tree(_int(parents))
    bits = _bits(tree.masks, T)
    for b in range(n):
        see = ancestors(parents[b])
        assert torch.equal(bits[b, :, :T], see) and not bits[b, :, T:].any()
        assert torch.equal(tree.depth[b].cpu().long(), see.sum(1) - 1)


def test_chain_star_and_bad_parents():
    T = 70
    chain, star = torch.arange(T) - 1, torch.zeros(T, dtype=torch.long)
    bad = random_parents(T, 1).long()
    bad[[0, 5, 9, 30, 40]] = torch.tensor([0, 5, 69, 2 ** 31 - 1, -2 ** 31])   # itself, a later node, no node
    parents = torch.stack([chain, star, bad]).to(torch.int32)
    tree = draft_tree(_int(parents))
    for b in range(3):
        see = ancestors(parents[b])
        assert torch.equal(_bits(tree.masks, T)[b, :, :T], see)
        assert torch.equal(tree.depth[b].cpu().long(), see.sum(1) - 1)
    one = draft_tree(_int(chain))
    assert one.parents.shape == (1, T) and torch.equal(one.depth[0].cpu().long(), torch.arange(T))


def test_a_tree_made_by_hand_is_checked():
    tree = draft_tree(_int(torch.stack([random_parents(40, i) for i in range(3)])))
    one = DraftTree(tree.parents[1:2], tree.masks[1:2], tree.depth[1:2])
    want = draft_tree(tree.parents[1])
    assert torch.equal(one.masks, want.masks) and torch.equal(one.depth, want.depth)
    for parents, masks, depth in ((tree.parents, tree.masks[:1], tree.depth), (tree.parents, tree.masks[..., :1], tree.depth),
                                  (tree.parents, tree.masks.long(), tree.depth), (tree.parents, tree.masks, tree.depth[:, :39]),
                                  (tree.parents[:, ::2], tree.masks[:, ::2, :1], tree.depth[:, ::2]),
                                  (tree.parents.cpu(), tree.masks, tree.depth)):
        with pytest.raises(ValueError):
            DraftTree(parents, masks, depth)


# --- attention ----------------------------------------------------------------


def _filled(B, H, Sk, D, dtype, seed, cap=None):
    c = Kv4Cache(B, H, cap or Sk, D, DEV)
    c.data.fill_(0xff)
    k, v = _randn(seed, B, H, Sk, D, dtype=dtype), _randn(seed + 1, B, H, Sk, D, dtype=dtype)
    c.write(k.to(DEV), v.to(DEV))
    return c, kv4_levels(k), kv4_levels(v)


def _near(got, q, k, v, see, dtype, what=""):
    ref = attend_see(q, k, v, see)
    D, Sk = q.shape[-1], k.shape[2]
    dx = 24 * 2.0 ** -24 / math.sqrt(D) * float(q.double().abs().sum(-1).max()) * float(k.abs().max()) * 6
    rel = 2 * (dx + 2.0 ** -22) + 2.0 ** -16 + (32 + Sk / 32) * 2.0 ** -24 * 16
    tol = rel * float(v.abs().max()) + half_step(dtype) * ref.abs() + (2.0 ** -25 if dtype == FP else 0)
    assert torch.isfinite(got).all(), what
    err = (got.cpu().double() - ref).abs()
    assert (err <= tol).all(), f"{what}: {float((err / tol).max())} of the tolerance"
    empty = ~see.any(-1)
    if empty.any():
        assert (got.cpu().transpose(1, 2)[empty] == 0).all(), what


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype,out_dtype", [(BF, BF), (FP, FP), (BF, F32)])
@pytest.mark.parametrize("Hq,H,T,Sq", [(4, 4, 1, 1), (8, 2, 4, 4), (4, 2, 16, 16), (8, 4, 33, 33), (4, 1, 64, 20), (2, 2, 130, 130),
                                       (16, 1, 5, 1), (24, 1, 6, 1)])
@pytest.mark.parametrize("extra", [0, 1, 31, 250])
def test_attention(D, dtype, out_dtype, Hq, H, T, Sq, extra):
    B, Sk = 2, T + extra
    c, k, v = _filled(B, H, Sk, D, dtype, 5, cap=Sk + 3)
    parents = [random_parents(T, 3)]
    q = _randn(9, B, Hq, Sq, D, dtype=dtype)
    out = attention_kv4(q.to(DEV), c, keys=Sk, out_dtype=out_dtype, tree=draft_tree(_int(parents[0])))
    _near(out, q, k, v, tree_sees(parents, Sq, Sk, [Sk] * B), out_dtype)


@pytest.mark.parametrize("D,Hq,H", [(64, 4, 2), (128, 2, 2), (64, 16, 2)])
@pytest.mark.parametrize("T,Sq", [(7, 7), (40, 40), (100, 37)])
@pytest.mark.parametrize("splits", [0, 1, 3, 64])
def test_lengths_masks_and_splits(D, Hq, H, T, Sq, splits):
    """A tree for each sequence; lengths of none, fewer than the nodes, a little more and all; a byte mask."""
    Sk, valid = T + 180, [0, T // 2, T, T + 33, T + 180, T + 400]
    B = len(valid)
    c, k, v = _filled(B, H, Sk, D, BF, 7)
    parents = [random_parents(T, 20 + b, back=2 + b) for b in range(B)]
    tree = draft_tree(_int(torch.stack(parents)))
    q = _randn(8, B, Hq, Sq, D, dtype=BF)
    mask = torch.rand(B, Sk, generator=torch.Generator().manual_seed(4)) < 0.7
    mask[4] = False
    for m in (None, mask):
        out = attention_kv4(q.to(DEV), c, valid_len=_int(valid), kv_mask=None if m is None else m.to(DEV), num_splits=splits,
                            tree=tree)
        _near(out, q, k, v, tree_sees(parents, Sq, Sk, valid, m), BF, f"mask {m is not None}")


@pytest.mark.parametrize("D", [64, 128])
def test_a_chain_is_causal(D):
    """Nodes in a chain see what causal queries see."""
    B, H, Hq, T, Sk = 2, 2, 8, 21, 333
    c, _, _ = _filled(B, H, Sk, D, BF, 3)
    q = _randn(4, B, Hq, T, D, dtype=BF).to(DEV)
    valid = _int([Sk, Sk - 60])
    tree = draft_tree(_int(torch.arange(T) - 1))
    for od in (BF, F32):
        a = attention_kv4(q, c, valid_len=valid, tree=tree, out_dtype=od)
        b = attention_kv4(q, c, valid_len=valid, is_causal=True, out_dtype=od)
        assert torch.equal(a, b)


@pytest.mark.parametrize("D,Hq,H,Sk", [(64, 64, 64, 8200), (128, 64, 32, 4700), (64, 128, 32, 8200)])
@pytest.mark.parametrize("out_dtype", [BF, F32])
def test_long_streams_of_few_rows(D, Hq, H, Sk, out_dtype):
    """The form that takes several blocks of keys at a time, trees across its blocks' borders."""
    B, T = 4, 2
    c, k, v = _filled(B, H, Sk, D, BF, 3)
    parents = [torch.tensor([-1, p], dtype=torch.int32) for p in (0, -1, 0, -1)]
    valid = [Sk, Sk - 31, 33, 1]
    q = _randn(6, B, Hq, T, D, dtype=BF)
    out = attention_kv4(q.to(DEV), c, valid_len=_int(valid), out_dtype=out_dtype, tree=draft_tree(_int(torch.stack(parents))))
    _near(out, q, k, v, tree_sees(parents, T, Sk, valid), out_dtype)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hq,Sq", [(2, 6), (8, 24)])
@pytest.mark.parametrize("out_dtype", [BF, F32])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_another_branch_is_not_felt(D, Hq, Sq, out_dtype, bad):
    """A NaN or an infinity in one node's key and value reaches its descendants and no other row."""
    B, H, T, Sk = 1, 2, 24, 200
    parents = (torch.arange(T, dtype=torch.int32) - 2).clamp_min(0)   # two chains from the root
    k, v = _randn(1, B, H, Sk, D, dtype=BF), _randn(2, B, H, Sk, D, dtype=BF)
    node = 9
    k[:, :, Sk - T + node, 3] = bad
    v[:, :, Sk - T + node, 5] = bad
    c = Kv4Cache(B, H, Sk, D, DEV)
    c.write(k.to(DEV), v.to(DEV))
    q = _randn(3, B, Hq, Sq, D, dtype=BF)
    out = attention_kv4(q.to(DEV), c, out_dtype=out_dtype, tree=draft_tree(_int(parents))).cpu()
    hit = ancestors(parents)[T - Sq:, node]
    assert hit.any() and not hit.all()
    assert torch.isnan(out[:, :, hit]).any(-1).all()
    k[:, :, Sk - T + node], v[:, :, Sk - T + node] = 0, 0
    see = tree_sees([parents], Sq, Sk, [Sk])
    _near(out[:, :, ~hit], q[:, :, ~hit], kv4_levels(k), kv4_levels(v), see[:, ~hit], out_dtype)


def test_strides_and_in_place():
    B, H, Hq, T, Sk, D = 2, 2, 4, 12, 90, 64
    c, k, v = _filled(B, H, Sk, D, BF, 3)
    parents = random_parents(T, 2)
    tree = draft_tree(_int(parents))
    rows = _randn(4, B, T, Hq * D + 24, dtype=BF).to(DEV)
    q = rows[..., 8:8 + Hq * D].unflatten(2, (Hq, D)).transpose(1, 2)
    want = attention_kv4(q.contiguous(), c, tree=tree)
    was = rows.clone()
    got = attention_kv4(q, c, out=q, tree=tree)
    assert torch.equal(got, want)
    assert torch.equal(rows[..., :8], was[..., :8]) and torch.equal(rows[..., 8 + Hq * D:], was[..., 8 + Hq * D:])
    _near(want, was[..., 8:8 + Hq * D].unflatten(2, (Hq, D)).transpose(1, 2).cpu(), k, v, tree_sees([parents], T, Sk, [Sk] * B), BF)


def test_front_end_refusals():
    c, _, _ = _filled(2, 2, 40, 64, BF, 3)
    q = _randn(4, 2, 4, 6, 64, dtype=BF).to(DEV)
    tree = draft_tree(_int(random_parents(6, 1)))
    for kw in ({"tree": draft_tree(_int(random_parents(5, 1)))}, {"tree": tree, "is_causal": True},
               {"tree": draft_tree(_int(torch.stack([random_parents(6, i) for i in range(3)])))}):
        with pytest.raises(ValueError):
            attention_kv4(q, c, **kw)
    with pytest.raises(ValueError):
        draft_tree(_int(torch.zeros(2, 6)).t())
    with pytest.raises(ValueError):
        accept_tree(tree, _int(torch.zeros(2, 5)), _int(torch.zeros(2, 5)))
    with pytest.raises(ValueError):
        c.keep(_int(torch.zeros(3, 6)), _int([0, 0]))


# --- the confirmed path -----------------------------------------------------------


@pytest.mark.parametrize("T", [1, 2, 17, 64, 65, 130, 1024])
@pytest.mark.parametrize("each", [False, True])
def test_accept(T, each):
    B = 5
    g = torch.Generator().manual_seed(T)
    trees = [random_parents(T, 30 + b, back=2 + 3 * b) for b in range(B if each else 1)]
    drafted, sampled = (torch.randint(0, 4, (B, T), generator=g, dtype=torch.int32) for _ in range(2))
    for b in range(B):   # long paths: most nodes sample a child's token
        p = trees[b if each else 0].tolist()
        for j in range(1, T):
            if torch.rand((), generator=g) < 0.9:
                sampled[b, p[j]] = drafted[b, j]
    nodes, count, tokens = (t.cpu() for t in accept_tree(draft_tree(_int(torch.stack(trees))), drafted.to(DEV), sampled.to(DEV)))
    for b in range(B):
        want, toks = accept(trees[b if each else 0], drafted[b].tolist(), sampled[b].tolist())
        n = len(want)
        assert count[b] == n and nodes[b, :n].tolist() == want and tokens[b, :n].tolist() == toks
        assert (nodes[b, n:] == -1).all() and (tokens[b, n:] == -1).all()


def test_accept_chain_star_and_bad_parents():
    T = 200
    chain = torch.arange(T) - 1
    star = torch.zeros(T, dtype=torch.long)
    loop = torch.tensor([0] + [(j * 7) % T for j in range(1, T)])   # later nodes and itself among the parents
    parents = torch.stack([chain, star, loop]).to(torch.int32)
    same = torch.zeros(3, T, dtype=torch.int32)   # every token the same
    nodes, count, _ = accept_tree(draft_tree(_int(parents)), same.to(DEV), same.to(DEV))
    for b in range(3):
        want, _ = accept(parents[b], [0] * T, [0] * T)
        assert count[b] == len(want) and nodes[b, :len(want)].tolist() == want
    assert count[0] == T and count[1] == 2 and nodes[1, 1] == 1


# --- the cache with the path alone ------------------------------------------------


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n,first", [(1, [0, 3]), (5, [30, 31]), (40, [0, 90]), (1024, [7, 1000])])
def test_keep(D, n, first):
    B, H = 2, 3
    cap = max(first) + n + 20
    c, _, _ = _filled(B, H, cap, D, BF, 11)
    raw = c.read(dtype=F32)
    k, v = (t.cpu().clone() for t in raw)
    nodes = torch.full((B, n), -1, dtype=torch.int32)
    for b in range(B):   # a path that skips, then nothing
        path = [0]
        while path[-1] < n - 1 and len(path) < n:
            path.append(path[-1] + 1 + (len(path) * (b + 2)) % 3)
        path = [j for j in path if j < n]
        nodes[b, :len(path)] = torch.tensor(path, dtype=torch.int32)
    wk, wv = k.clone(), v.clone()
    for b in range(B):
        for i, j in enumerate(nodes[b].tolist()):
            if j >= 0:
                wk[b, :, first[b] + i], wv[b, :, first[b] + i] = k[b, :, first[b] + j], v[b, :, first[b] + j]
    c.keep(nodes.to(DEV), _int(first))
    gk, gv = (t.cpu() for t in c.read(dtype=F32))
    assert torch.equal(gk, wk) and torch.equal(gv, wv)


def test_keep_any_order_holes_and_places_outside():
    """Sources in any order, more than once, behind holes; slots and places outside the cache are left out."""
    B, H, D, cap, n = 4, 2, 64, 50, 12
    c, _, _ = _filled(B, H, cap, D, BF, 13)
    k, v = (t.cpu().clone() for t in c.read(dtype=F32))
    nodes = torch.tensor([[11, 10, 9, 8, 7, 6, 5, 4, 3, 2, 1, 0],
                          [3, 3, 3, -1, 0, -7, 2, 40, 2 ** 31 - 1, -2 ** 31, 1, 11],
                          [0, 2, 4, 6, 8, 10, 1, 3, 5, 7, 9, 11],
                          [6, 5, 4, 3, 2, 1, 0, 9, 9, 9, 9, 9]], dtype=torch.int32)
    first = [4, 20, 45, -5]
    wk, wv = k.clone(), v.clone()
    for b in range(B):
        for i, j in enumerate(nodes[b].tolist()):
            src, dst = first[b] + j, first[b] + i
            if j >= 0 and 0 <= src < cap and 0 <= dst < cap:
                wk[b, :, dst], wv[b, :, dst] = k[b, :, src], v[b, :, src]
    c.keep(nodes.to(DEV), _int(first))
    gk, gv = (t.cpu() for t in c.read(dtype=F32))
    assert torch.equal(gk, wk) and torch.equal(gv, wv)
    far = _int([2 ** 31 - 1, -2 ** 31, 2 ** 31 - 6, 60])
    c.keep(nodes.to(DEV), far)
    assert all(torch.equal(a.cpu(), b) for a, b in zip(c.read(dtype=F32), (wk, wv)))


@pytest.mark.parametrize("D,Hq,H,T,splits", [(128, 32, 8, 8, 0), (128, 8, 2, 16, 5), (64, 8, 8, 64, 0), (64, 16, 4, 3, 7)])
@pytest.mark.parametrize("out_dtype", [BF, F32])
def test_runs_are_equal(D, Hq, H, T, splits, out_dtype):
    """Bit for bit, with other work and other memory between them."""
    B, Sk = 3, 1500
    c, _, _ = _filled(B, H, Sk, D, BF, 3)
    q = _randn(4, B, Hq, T, D, dtype=BF).to(DEV)
    tree, valid = draft_tree(_int(random_parents(T, 5))), _int([Sk, Sk // 2, T])
    first = attention_kv4(q, c, valid_len=valid, tree=tree, num_splits=splits, out_dtype=out_dtype)
    for i in range(6):
        torch.full((1 << 22,), float(i), device=DEV)
        assert torch.equal(attention_kv4(q, c, valid_len=valid, tree=tree, num_splits=splits, out_dtype=out_dtype), first)
