"""The 4-bit operators together, as a program that decodes token by token uses
them: 4-bit projection -> head norm + rotation into the cache -> attention over
it -> 4-bit projection, a prompt first, then single tokens; each stage against
its 64-bit form on the stage's own inputs (the tolerances of test_w4_gpu and
test_kv4_gpu).  Then the same step on another stream, captured into a graph and
replayed, and at offsets beyond 32 bits."""
import pytest
import torch

from servoflow_amd import kernels
from servoflow_amd.attention import Kv4Cache, attention_kv4

from _quant4 import rms, rotate, w4_bytes, w4_random
from test_kv4_gpu import _attn_check, _freq, _randn, _rope_check
from test_w4_gpu import _check as _w4_check

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


class Layer:
    """Attention of one decoder layer in 4 bits."""

    def __init__(self, Hq, H, D, hidden, B, cap, dtype, seed):
        self.Hq, self.H, self.D, self.dtype = Hq, H, D, dtype
        self.w, self.packed = {}, {}
        for j, (name, N, K) in enumerate((("qkv", (Hq + 2 * H) * D, hidden), ("out", hidden, Hq * D))):
            codes, scales, zeros, w = w4_random(N, K, 64, dtype, True, seed + j)
            self.w[name] = (w, scales, zeros)
            self.packed[name] = kernels.w4_pack(w4_bytes(codes).to(DEV), scales.to(DEV), zeros.to(DEV), group=64)
        self.gq, self.gk = (1 + 0.2 * _randn(seed + 5 + j, D) for j in range(2))
        self.gq, self.gk, self.freq = self.gq.to(DEV), self.gk.to(DEV), _freq(D).to(DEV)
        self.cache = Kv4Cache(B, H, cap, D, DEV)
        self.cache.data.fill_(0xff)

    def step(self, x, S, pos, valid, keys=None, workspace=None):
        """x [B * S, hidden], pos [B * S], valid [B]: (projection, q, attention, output)."""
        p = kernels.gemm_w4(x, self.packed["qkv"])
        q, _, _ = kernels.heads_rope(p, S, (self.Hq, self.H, self.H), self.D, (self.gq, self.gk), pos, self.freq,
                                     cache=self.cache)
        B = valid.numel()
        a = torch.empty(B, S, self.Hq, self.D, dtype=self.dtype, device=DEV)
        attention_kv4(q, self.cache, out=a.transpose(1, 2), is_causal=True, valid_len=valid, keys=keys, workspace=workspace)
        return p, q, a, kernels.gemm_w4(a.reshape(B * S, -1), self.packed["out"])

    def check_w4(self, got, x, name):
        w, scales, zeros = self.w[name]
        x = x.cpu()
        big = x.double().abs() @ ((47 + zeros.double()) * scales.double()).repeat_interleave(64, 1).t()
        _w4_check(got, x.double() @ w.t(), big, w.shape[1], self.dtype, what=name)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("Hq,H,D", [(4, 2, 64), (8, 1, 128), (3, 3, 64)])
def test_prompt_and_steps(dtype, Hq, H, D):
    B, hidden, S0, cap = 2, 256, 43, 64
    L = Layer(Hq, H, D, hidden, B, cap, dtype, 7)
    lens = torch.tensor([S0, S0 - 11])           # a padded batch: the second prompt is shorter
    done = torch.zeros(B, dtype=torch.long)
    for step in range(6):
        S = S0 if step == 0 else 1
        x = _randn(20 + step, B * S, hidden, dtype=dtype).to(DEV)
        n = lens if step == 0 else torch.ones(B, dtype=torch.long)
        at = torch.arange(S)
        # a causal chunk ends at valid_len: the shorter prompt's padding comes first
        pos = done[:, None] + at - (S - n)[:, None]
        pos = torch.where(at >= (S - n)[:, None], pos, -1).to(torch.int32)
        done = done + n
        valid = done.to(torch.int32).to(DEV)
        p, q, a, y = L.step(x, S, pos.to(DEV), valid)
        L.check_w4(p, x, "qkv")
        real = (pos >= 0)[:, None, :, None]
        part = rms(p.cpu().double().reshape(B, S, -1, D).transpose(1, 2)[:, :Hq], L.gq.cpu(), 1e-6)
        ref = rotate(part, pos.clamp_min(0), L.freq.cpu(), False)
        keep = real.expand_as(ref)
        qd = torch.where(keep, q.cpu().double(), torch.zeros(()).double())   # rows of padding are not written
        _rope_check(qd, torch.where(keep, ref, torch.zeros(()).double()), part, dtype)
        k, v = (t.cpu().double() for t in L.cache.read(dtype=F32))
        for b in range(B):
            m = int(done[b])
            rows = real[b, 0, :, 0].nonzero()[:, 0]
            _attn_check(a.transpose(1, 2)[b:b + 1, :, rows], q[b:b + 1, :, rows].cpu(), k[b:b + 1, :, :m], v[b:b + 1, :, :m],
                        dtype, causal=True, what=f"step {step}")
        rows = real[:, 0, :, 0].reshape(-1)
        L.check_w4(y[rows.to(DEV)], a.reshape(B * S, -1)[rows.to(DEV)], "out")


def _inputs(B, hidden, n):
    return [_randn(60 + i, B, hidden, dtype=BF).to(DEV) for i in range(n)]


def _eager(B, cap, xs, first):
    L = Layer(8, 2, 64, 256, B, cap, BF, 9)
    out = []
    for i, x in enumerate(xs):
        pos = torch.full((B,), first + i, dtype=torch.int32, device=DEV)
        out.append(L.step(x, 1, pos, pos + 1)[3].clone())
    return out, L.cache.read(torch.arange(first, first + len(xs), dtype=torch.int32, device=DEV).expand(B, -1).contiguous())


def test_graph_replays_match_eager():
    """A captured step whose positions and lengths move on the device, with eager work and waits between replays."""
    B, cap, first = 3, 1100, 0
    xs = _inputs(B, 256, 6)
    ref, kv = _eager(B, cap, xs, first)
    L = Layer(8, 2, 64, 256, B, cap, BF, 9)
    x = torch.zeros_like(xs[0])
    pos = torch.full((B,), first, dtype=torch.int32, device=DEV)
    valid = pos + 1
    L.step(xs[0], 1, pos, valid)   # the kernels are loaded before the capture
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = L.step(x, 1, pos, valid)[3]
        pos += 1
        valid += 1
    pos.fill_(first)
    valid.fill_(first + 1)
    L.cache.data.fill_(0xff)
    for i, xi in enumerate(xs):
        x.copy_(xi)
        g.replay()
        assert torch.equal(y, ref[i]), i
        (torch.randn(512, 512, device=DEV) @ torch.randn(512, 512, device=DEV)).sum().item()
    got = L.cache.read(torch.arange(first, first + 6, dtype=torch.int32, device=DEV).expand(B, -1).contiguous())
    assert torch.equal(got[0], kv[0]) and torch.equal(got[1], kv[1])


def test_streams_with_their_own_workspaces():
    """Two programs at once on two streams, each with its cache and its workspace (key splits and a merge)."""
    B, H, Hq, Sk, D = 1, 2, 8, 3000, 128
    ks = [_randn(70 + i, B, H, Sk, D, dtype=BF).to(DEV) for i in range(2)]
    q = _randn(75, B, Hq, 1, D, dtype=BF).to(DEV)
    caches = [Kv4Cache(B, H, Sk, D, DEV) for _ in ks]
    ref = []
    for c, k in zip(caches, ks):
        c.write(k, k)
        ref.append(attention_kv4(q, c, num_splits=6))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ks]
    ws = [torch.empty(6 * B * Hq * (D + 2) * 4, dtype=torch.uint8, device=DEV) for _ in ks]
    outs = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(attention_kv4(q, caches[i], num_splits=6, workspace=ws[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, ref[i]) for o in outs[i])


def test_cache_beyond_32_bits():
    """4.5 GiB of cache: the last head's last tokens, the only ones the mask leaves."""
    B, H, D, cap = 4, 4, 64, 1 << 22
    c = Kv4Cache(B, H, cap, D, DEV)
    assert c.data.numel() > 1 << 32
    c.data.fill_(0xff)
    S = 40
    slots = torch.arange(cap - S, cap, dtype=torch.int32).expand(B, S).contiguous()
    k, v = _randn(80, B, H, S, D, dtype=BF), _randn(81, B, H, S, D, dtype=BF)
    c.write(k.to(DEV), v.to(DEV), slots.to(DEV))
    rk, rv = c.read(slots.to(DEV), F32)
    mask = torch.zeros(B, cap, dtype=torch.bool, device=DEV)
    mask[:, -S:] = True
    q = _randn(82, B, H, 2, D, dtype=BF)
    got = attention_kv4(q.to(DEV), c, kv_mask=mask, out_dtype=F32)
    _attn_check(got, q, rk.cpu().double(), rv.cpu().double(), F32)


def test_weights_beyond_32_bits():
    """4.3 GB of codes: the columns at the end against their rows."""
    N, K, M = (1 << 18) + 24, 1 << 15, 3
    assert N * K // 2 > 1 << 32
    codes = torch.randint(0, 256, (N, K // 2), dtype=torch.uint8, device=DEV)
    scales = torch.full((N, K // 128), 0.01, dtype=FP, device=DEV)
    w = kernels.w4_pack(codes, scales)
    a = _randn(83, M, K, dtype=FP)
    y = kernels.gemm_w4(a.to(DEV), w, out_dtype=F32)[:, -40:]
    tail = codes[-40:].cpu()
    c = torch.stack((tail & 15, tail >> 4), -1).flatten(1).double()
    s = scales[0, 0].double().item()
    big = (a.double().abs().sum(1, keepdim=True) * 55 * s).expand(M, 40)
    _w4_check(y, a.double() @ ((c - 8) * s).t(), big, K, F32)
