"""Plain 64-bit forms of the 4-bit operators, on the CPU, for the tests."""
import math

import torch


def half_step(dtype):
    """The largest relative error of one rounding to dtype."""
    return torch.finfo(dtype).eps / 2


def w4_random(N, K, group, scale_dtype, zeros, seed):
    """Codes [N, K] (uint8), scales, zeros or None, and the weights in 64 bits."""
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 16, (N, K), generator=g, dtype=torch.uint8)
    scales = (torch.rand(N, K // group, generator=g) * 0.02 + 1e-3).to(scale_dtype)
    z = torch.randint(0, 16, (N, K // group), generator=g, dtype=torch.uint8) if zeros else None
    zz = z.double() if zeros else torch.full((N, K // group), 8.0, dtype=torch.float64)
    w = (codes.double().reshape(N, -1, group) - zz[..., None]) * scales.double()[..., None]
    return codes, scales, z, w.reshape(N, K)


def w4_bytes(codes):
    return codes[:, 0::2] | (codes[:, 1::2] << 4)


def kv4_levels(x):
    """What the cache's format makes of x [..., D] (fp32 or narrower, finite), in 64 bits."""
    y = x.double().unflatten(-1, (-1, 64))
    hi, lo = y.amax(-1, keepdim=True), y.amin(-1, keepdim=True)
    mid = (0.5 * hi + 0.5 * lo).to(torch.bfloat16).double()
    a = torch.maximum(hi - mid, mid - lo).float()   # exact: both are of 24 bits at most here
    s = (((a.view(torch.int32) + 0xffff) & -65536).view(torch.float32) * 0.125).double()
    s = torch.where(s < 2.0 ** -126, 0.0, s)
    c = torch.floor((y - mid) / torch.where(s > 0, s, 1.0)).clamp(-8, 7)
    c = torch.where(s > 0, c, 0.0)
    return (s * (c + 0.5) + mid).flatten(-2)


def rotate(x, pos, inv_freq, interleaved):
    """x [B, H, S, D], pos [B, S], inv_freq [rot / 2] (64 bits throughout)."""
    half = inv_freq.numel()
    i = torch.arange(half)
    i, j = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    ang = pos.double()[:, None, :, None] * inv_freq.double()
    c, s = torch.cos(ang), torch.sin(ang)
    out = x.clone()
    out[..., i] = x[..., i] * c - x[..., j] * s
    out[..., j] = x[..., j] * c + x[..., i] * s
    return out


def rms(x, gamma, eps):
    return x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * gamma.double()


def attend(q, k, v, scale=0.0, valid=None, mask=None, causal=False):
    """softmax(q k^T scale) v in 64 bits; q [B, Hq, Sq, D], k, v [B, H, Sk, D]; rows that see nothing are zeros."""
    B, Hq, Sq, D = q.shape
    H, Sk = k.shape[1], k.shape[2]
    k, v = (t.double().repeat_interleave(Hq // H, 1) for t in (k, v))
    x = torch.matmul(q.double(), k.transpose(2, 3)) * (scale or 1 / math.sqrt(D))
    n = torch.full((B,), Sk) if valid is None else valid.long().clamp(0, Sk)
    at = torch.arange(Sk)
    see = (at < n[:, None]) if mask is None else (at < n[:, None]) & mask.bool()
    see = see[:, None, None, :].expand(B, 1, Sq, Sk)
    if causal:
        see = see & (at <= (n[:, None, None, None] - Sq + torch.arange(Sq)[:, None]))
    x = x.masked_fill(~see, -math.inf)
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(m > -math.inf, m, 0.0))
    t = p.sum(-1, keepdim=True)
    v = torch.where(see.any(2).transpose(1, 2)[:, None], v, 0.0)   # what no row sees may hold anything
    return torch.matmul(p, v) / torch.where(t > 0, t, 1.0)
