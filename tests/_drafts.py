"""Plain forms, on the CPU, of the operators of a step that verifies drafted tokens."""
import math

import torch


def random_parents(T, seed, back=8):
    g = torch.Generator().manual_seed(seed)
    at = torch.arange(T)
    step = (torch.rand(T, generator=g).square() * back).long() + 1
    return torch.where(at > 0, (at - step).clamp_min(0), -1).to(torch.int32)


def ancestors(parents):
    """see[j, i]: node i is node j or one of its ancestors (a parent that does not come before its node is none)."""
    T = len(parents)
    see = torch.zeros(T, T, dtype=torch.bool)
    for j, p in enumerate(parents.tolist()):
        if 0 <= p < j:
            see[j] = see[p]
        see[j, j] = True
    return see


def tree_sees(parents, Sq, Sk, valid, mask=None):
    """[B, Sq, Sk]: which slots the queries see; parents a list of one or B trees."""
    out = torch.zeros(len(valid), Sq, Sk, dtype=torch.bool)
    for b, n in enumerate(valid):
        n = min(max(n, 0), Sk)
        see = ancestors(parents[b if len(parents) > 1 else 0])
        T = len(see)
        for s in range(Sq):
            j = T - Sq + s
            if n - T + j < 0:
                continue
            out[b, s, :max(0, n - T)] = True
            for i in range(max(0, T - n), T):
                out[b, s, n - T + i] = see[j, i]
        if mask is not None:
            out[b] &= mask[b]
    return out


def attend_see(q, k, v, see, scale=0.0):
    """softmax(q k^T scale) v in 64 bits over the slots see [B, Sq, Sk]; rows that see nothing are zeros."""
    G = q.shape[1] // k.shape[1]
    k, v = (t.double().repeat_interleave(G, 1) for t in (k, v))
    x = torch.matmul(q.double(), k.transpose(2, 3)) * (scale or 1 / math.sqrt(q.shape[-1]))
    x = x.masked_fill(~see[:, None], -math.inf)
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(m > -math.inf, m, 0.0))
    t = p.sum(-1, keepdim=True)
    return torch.matmul(p, torch.where(see.any(1)[:, None, :, None], v, 0.0)) / torch.where(t > 0, t, 1.0)


def accept(parents, drafted, sampled):
    """(nodes, tokens) of one tree."""
    p, nodes = parents.tolist(), [0]
    while True:
        kids = [j for j in range(nodes[-1] + 1, len(p)) if p[j] == nodes[-1] and drafted[j] == sampled[nodes[-1]]]
        if not kids:
            return nodes, [int(sampled[j]) for j in nodes]
        nodes.append(kids[0])


def sample(logits, u, t=1.0, k=0, p=1.0, mp=0.0):
    """(token, logprob) of one row, in 64 bits."""
    l = logits.double()
    if torch.isnan(l).any() or not (l > -math.inf).any():
        return -1, math.nan
    if not t > 0:
        t, k = 1.0, 1
    order = torch.argsort(-l, stable=True)
    l = l[order][:int((l > -math.inf).sum())]
    lw = torch.where(l == l[0], 0.0, l - l[0]) / t
    lw = torch.where(torch.isnan(lw), -math.inf, lw)
    w = torch.exp(lw)
    n = len(l) if k <= 0 else min(k, len(l))
    if p < 1:
        n = min(n, 1 + int((torch.cumsum(w[:n], 0) < p * w[:n].sum()).sum()))
    n = max(1, min(n, int((w >= mp).sum())))
    run = torch.cumsum(w[:n], 0)
    j = min(int((run <= u * run[-1]).sum()), int((w[:n] > 0).sum()) - 1)
    return int(order[j]), float(lw[j] - torch.log(run[-1]))


def quant(x):
    """Codes and scale of rows x, the quotient and its rounding in 64 bits."""
    s = (x.float().abs().amax(1).numpy() / __import__("numpy").float32(127)).astype("float32")
    s = torch.from_numpy(s)
    q = x.double() / torch.where(s > 0, s, 1.0).double()[:, None]
    return torch.where(s[:, None] > 0, torch.round(q), 0.0).clamp(-127, 127), s
