"""Head norm + rotation, the 4-bit key / value cache and the attention over it
against plain forms in 64 bits.

Tolerances, from the arithmetic.
  norm + rotation: fp32; a norm takes D / 8 + 4 additions, a root, a division
  and two products (24 roundings), a rotation 3 and an angle whose fraction of
  a turn is held to 2^-26 (2 pi 2^-26 radians) with sine and cosine to 2 units:
  40 roundings of 2^-24 of |x1| + |x2| cover both; then half a step of the
  output type.
  cache: keys and values as given are quantised exactly as the format says, so
  the read values are equal.
  attention, against the values that the cache stands for: a score is off by
  the roundings of its sums (24 of 2^-24 of scale * sum |q| (|k| + 40 s)); p by
  that and by exp2's 2^-22; the (hi, lo) pair by 2^-17; sums over tokens by
  (32 + tokens / 32) 2^-24 of 55 s / max |v| <= 16 times the largest value.  A
  bf16 output of more than 16 rows to a key head takes p and V in fp16 instead
  of the pair: p, its sum and V round by 2^-12 each, and mid - 7.5 s, of which
  V is formed, by 2^-12 of itself, which is at most |v| + 8 s <= twice the
  largest value (16 s is at most a row's spread, twice its largest): 5 2^-12 of
  the largest value together."""
import math

import pytest
import torch

from servoflow_amd import kernels
from servoflow_amd.attention import Kv4Cache, attention_kv4

from _quant4 import attend, half_step, kv4_levels, rms, rotate

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


def _randn(seed, *shape, dtype=F32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def _freq(rot, base=10000.0):
    return base ** (-torch.arange(rot // 2, dtype=torch.float64) / (rot // 2))


def _rope_check(got, ref, x, dtype, what=""):
    """x: the normed values before the rotation, 64 bits."""
    tol = 40 * 2.0 ** -24 * (x.abs().amax(-1, keepdim=True) * 2 + 1e-30) + half_step(dtype) * ref.abs()
    if dtype == FP:
        tol = tol + 2.0 ** -25
    err = (got.cpu().double() - ref).abs()
    assert torch.isfinite(got).all(), what
    assert (err <= tol).all(), f"{what}: {float((err / tol).max())} of the tolerance"


# --- norm + rotation -------------------------------------------------------


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype,out_dtype", [(BF, BF), (FP, FP), (F32, F32), (BF, F32), (F32, BF)])
@pytest.mark.parametrize("rot,interleaved", [(0, False), (16, False), (16, True), (48, False), (48, True), ("D", False),
                                             ("D", True)])
def test_heads_rope(D, dtype, out_dtype, rot, interleaved):
    rot = D if rot == "D" else rot
    B, S, Hq, Hk = 2, 5, 6, 3
    p = _randn(1, B * S, (Hq + 2 * Hk) * D, dtype=dtype)
    gq, gk = 1 + 0.2 * _randn(2, D), 1 + 0.2 * _randn(3, D)
    pos = torch.tensor([[0, 1, 7, 1000, 999999], [3, 2 ** 31 - 1, 65536, 12, 1]], dtype=torch.int32)
    f = _freq(rot) if rot else None
    q, k, v = kernels.heads_rope(p.to(DEV), S, (Hq, Hk, Hk), D, (gq.to(DEV), gk.to(DEV)), pos.to(DEV),
                                 None if f is None else f.to(DEV), interleaved, 1e-6, out_dtype)
    x = p.double().reshape(B, S, -1, D).transpose(1, 2)
    for name, got, part, gm in (("q", q, x[:, :Hq], gq), ("k", k, x[:, Hq:Hq + Hk], gk)):
        n = rms(part, gm, 1e-6)
        _rope_check(got, rotate(n, pos, f, interleaved) if rot else n, n, out_dtype, name)
    assert torch.equal(v.cpu(), x[:, Hq + Hk:].to(dtype).to(out_dtype))


@pytest.mark.parametrize("B,S,Hq,Hk,Hv", [(1, 1, 1, 0, 0), (1, 1, 0, 1, 1), (3, 1, 0, 0, 2), (1, 2049, 3, 1, 1),
                                          (2049, 1, 5, 0, 0), (7, 9, 33, 2, 1)])
def test_heads_rope_shapes(B, S, Hq, Hk, Hv):
    D, dtype = 64, FP
    p = _randn(4, B * S, (Hq + Hk + Hv) * D, dtype=dtype)
    out = kernels.heads_rope(p.to(DEV), S, (Hq, Hk, Hv), D, inv_freq=_freq(D).to(DEV))
    x = p.double().reshape(B, S, -1, D).transpose(1, 2)
    pos = torch.arange(S).expand(B, S)
    for got, part, turn in ((out[0], x[:, :Hq], True), (out[1], x[:, Hq:Hq + Hk], True), (out[2], x[:, Hq + Hk:], False)):
        assert (got is None) == (part.shape[1] == 0)
        if got is not None:
            _rope_check(got, rotate(part, pos, _freq(D), False) if turn else part, part, dtype)


def test_padding_rows_and_strided_in_place():
    """Padding tokens stay as they were; rows rotated where they lie, behind other columns."""
    B, S, H, D = 2, 6, 4, 64
    wide = _randn(5, B * S, 3 * H * D + 40, dtype=BF).to(DEV)
    was = wide.clone()
    x = wide[:, 16:16 + H * D].unflatten(0, (B, S)).unflatten(2, (H, D)).transpose(1, 2)
    pos = torch.tensor([[0, 1, 2, 3, -1, -5], [9, -1, 11, 12, 13, 14]], dtype=torch.int32)
    ref = rotate(x.cpu().double(), pos.clamp_min(0), _freq(D), True)
    before = x.cpu().double()
    kernels.heads_rope_strided((x, None, None), (x, None, None), positions=pos.to(DEV), inv_freq=_freq(D).to(DEV),
                               interleaved=True)
    real = (pos >= 0)[:, None, :, None]
    _rope_check(x, torch.where(real, ref, before), before, BF)
    assert torch.equal(torch.masked_select(x.cpu().double(), ~real), torch.masked_select(before, ~real))
    same = torch.ones(wide.shape[1], dtype=torch.bool)
    same[16:16 + H * D] = False
    assert torch.equal(wide[:, same], was[:, same])


# --- the cache --------------------------------------------------------------


def _levels(x):
    return kv4_levels(x.cpu())


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("S", [1, 31, 32, 33, 100])
def test_cache_round_trip(D, dtype, S):
    B, H = 2, 3
    k, v = (_randn(6 + i, B, H, S, D, dtype=dtype) * (1 + 3 * i) + 0.3 for i in range(2))
    c = Kv4Cache(B, H, S, D, DEV)
    c.write(k.to(DEV), v.to(DEV))
    rk, rv = c.read(dtype=F32)
    assert torch.equal(rk.cpu(), _levels(k).float()) and torch.equal(rv.cpu(), _levels(v).float())


def test_cache_slots_leave_the_rest():
    """Ragged slots, slots out of range, and what other slots held."""
    B, H, D, cap = 3, 2, 64, 70
    c = Kv4Cache(B, H, cap, D, DEV)
    k, v = _randn(8, B, H, cap, D, dtype=BF), _randn(9, B, H, cap, D, dtype=BF)
    c.write(k.to(DEV), v.to(DEV))
    nk, nv = _randn(10, B, H, 4, D, dtype=BF), _randn(11, B, H, 4, D, dtype=BF)
    slots = torch.tensor([[69, 0, 33, -1], [70, 5, 2 ** 31 - 1, 6], [31, 32, 63, 64]], dtype=torch.int32)
    c.write(nk.to(DEV), nv.to(DEV), slots.to(DEV))
    ek, ev = k.clone(), v.clone()
    for b in range(B):
        for j, s in enumerate(slots[b].tolist()):
            if 0 <= s < cap:
                ek[b, :, s], ev[b, :, s] = nk[b, :, j], nv[b, :, j]
    rk, rv = c.read(dtype=F32)
    assert torch.equal(rk.cpu(), _levels(ek).float()) and torch.equal(rv.cpu(), _levels(ev).float())
    gk, gv = c.read(slots.to(DEV), F32)
    inside = ((slots >= 0) & (slots < cap))[:, None, :, None]
    assert torch.equal(gk.cpu(), torch.where(inside, _levels(nk).float(), torch.zeros(())))
    assert torch.equal(gv.cpu(), torch.where(inside, _levels(nv).float(), torch.zeros(())))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("S", [32, 40, 64, 70, 95, 131])
@pytest.mark.parametrize("first", [0, 1, 10, 31, 33])
def test_cache_runs_of_tokens(D, S, first):
    """Prompts whose slots count up from anywhere in a block, whole blocks and ragged ends; one batch element with a
    gap, one that runs out of the cache, and what lay beside them."""
    B, H = 3, 5
    cap = first + S + 3
    c = Kv4Cache(B, H, cap, D, DEV)
    old = _randn(100, B, H, cap, D, dtype=BF)
    c.write(old.to(DEV), old.to(DEV))
    k, v = _randn(101, B, H, S, D, dtype=BF), _randn(102, B, H, S, D, dtype=BF)
    slots = (torch.arange(S) + torch.tensor([[first], [first], [first + 8]])).to(torch.int32)
    slots[1, S // 2:] += 2
    c.write(k.to(DEV), v.to(DEV), slots.to(DEV))
    ek, ev = old.clone(), old.clone()
    for b in range(B):
        for j, s in enumerate(slots[b].tolist()):
            if s < cap:
                ek[b, :, s], ev[b, :, s] = k[b, :, j], v[b, :, j]
    rk, rv = c.read(dtype=F32)
    assert torch.equal(rk.cpu(), _levels(ek).float()) and torch.equal(rv.cpu(), _levels(ev).float())


def test_rope_prompt_into_cache_at_an_offset():
    """A prompt's queries, keys and values together, behind cached tokens, with padding at its end."""
    B, S, Hq, H, D = 2, 77, 3, 2, 64
    p = _randn(110, B * S, (Hq + 2 * H) * D, dtype=FP)
    pos = (torch.arange(S) + torch.tensor([[19], [64]])).to(torch.int32)
    pos[0, 70:] = -1
    c = Kv4Cache(B, H, 150, D, DEV)
    q, _, _ = kernels.heads_rope(p.to(DEV), S, (Hq, H, H), D, positions=pos.to(DEV), inv_freq=_freq(D).to(DEV), cache=c)
    x = p.double().reshape(B, S, -1, D).transpose(1, 2)
    real = (pos >= 0)[:, None, :, None]
    ref = rotate(x[:, :Hq], pos.clamp_min(0), _freq(D), False)
    keep = real.expand_as(ref)
    _rope_check(torch.where(keep, q.cpu().double(), 0.0), torch.where(keep, ref, 0.0), x[:, :Hq], FP)
    _, rv = c.read(pos.to(DEV), F32)
    assert torch.equal(rv.cpu().double(), torch.where(real, kv4_levels(x[:, Hq + H:].float()), torch.zeros(()).double()))


def test_cache_extreme_values():
    """Constant groups, outliers, the largest and smallest numbers; an infinity or NaN spoils its group alone."""
    D = 128
    x = _randn(12, 1, 1, 12, D)
    x[0, 0, 0] = 0
    x[0, 0, 1] = -3.25
    x[0, 0, 2, 5] = 3e38
    x[0, 0, 3] *= 1e-37
    x[0, 0, 4] *= 1e-30
    x[0, 0, 5, :] = 3.3895e38
    x[0, 0, 5, 1::2] = -3.3895e38
    x[0, 0, 6, 70] = 1e5
    x[0, 0, 7, 3] = float("inf")
    x[0, 0, 8, 100] = float("nan")
    x[0, 0, 9] = 2.0 ** torch.arange(D).remainder(16).float()
    c = Kv4Cache(1, 1, 12, D, DEV)
    c.write(x.to(DEV), x.to(DEV))
    bad = torch.zeros(12, 2, dtype=torch.bool)
    bad[7, 0] = bad[8, 1] = True
    y = x.clone()
    y[0, 0].unflatten(-1, (2, 64))[bad] = 0
    ref = _levels(y).float()[0, 0].unflatten(-1, (2, 64))
    for got in c.read(dtype=F32):
        got = got.cpu()[0, 0].unflatten(-1, (2, 64))
        assert torch.isnan(got[bad]).all()
        keep = ~bad
        keep[3] = False   # steps near the normal range's end: only how far they are from the input
        assert torch.equal(got[keep], ref[keep])
        assert ((got[3] - x[0, 0, 3].unflatten(-1, (2, 64))).abs() <= 1e-37).all()


def test_cache_of_the_largest_numbers():
    """Numbers above bf16's largest (3.3895e38): it is their middle, the step an eighth of what is left (1.34e36)."""
    x = torch.full((1, 1, 3, 64), 3.4028e38)
    x[0, 0, 1, ::3] = 3.395e38
    x[0, 0, 2] = -3.4028e38
    c = Kv4Cache(1, 1, 3, 64, DEV)
    c.write(x.to(DEV), x.to(DEV))
    for got in c.read(dtype=F32):
        assert ((got.cpu().double() - x.double()).abs() <= 0.5 * 1.35e36 / 8).all()


def test_rope_into_cache():
    """Normed, rotated keys and plain values at given slots; queries to a tensor."""
    B, S, Hq, H, D = 2, 37, 4, 2, 128
    p = _randn(13, B * S, (Hq + 2 * H) * D, dtype=BF)
    gk = 1 + 0.2 * _randn(14, D)
    pos = (torch.arange(S) + torch.tensor([[5], [60]])).to(torch.int32)
    pos[1, 3] = -1
    c = Kv4Cache(B, H, 100, D, DEV)
    c.data.zero_()
    q, k, v = kernels.heads_rope(p.to(DEV), S, (Hq, H, H), D, (None, gk.to(DEV)), pos.to(DEV), _freq(D).to(DEV),
                                 cache=c)
    assert k is None and v is None
    x = p.double().reshape(B, S, -1, D).transpose(1, 2)
    n = rms(x[:, Hq:Hq + H], gk, 1e-6)
    ref = rotate(n, pos.clamp_min(0), _freq(D), False)
    rk, rv = (t.cpu().double() for t in c.read(pos.to(DEV), F32))
    real = pos >= 0
    assert torch.equal(rv, torch.where(real[:, None, :, None], kv4_levels(x[:, Hq + H:]), torch.zeros((), dtype=rv.dtype)))
    # a key's code may fall on the other side of a border by the rounding before it: half a step more
    step = (ref.unflatten(-1, (2, 64)).amax(-1) - ref.unflatten(-1, (2, 64)).amin(-1)) / 16 * 1.02
    err = (rk - ref).abs().unflatten(-1, (2, 64)).amax(-1)
    assert (err <= torch.where(real[:, None, :, None], step * 0.5 + 1e-4, math.inf)).all()
    same = (rk - kv4_levels(ref.float())).abs() < 1e-6
    assert same[real[:, None, :, None].expand_as(same)].float().mean() > 0.999


# --- attention ----------------------------------------------------------------


def _filled(B, H, Sk, D, dtype, seed, cap=None):
    k = _randn(seed, B, H, Sk, D, dtype=dtype) + 0.5 * _randn(seed + 1, 1, H, 1, D).to(dtype)
    v = _randn(seed + 2, B, H, Sk, D, dtype=dtype)
    c = Kv4Cache(B, H, cap or Sk, D, DEV)
    c.data.fill_(0xff)   # NaN parameters everywhere: what is not written must not be seen
    c.write(k.to(DEV), v.to(DEV))
    return c, kv4_levels(k), kv4_levels(v)


def _attn_check(got, q, k, v, dtype, scale=0.0, what="", **kw):
    ref = attend(q, k, v, scale=scale, **kw)
    D, Sk = q.shape[-1], k.shape[2]
    sc = scale or 1 / math.sqrt(D)
    # |k| + 40 s: s is at most a sixteenth of a row's spread, itself at most twice its largest value
    dx = 24 * 2.0 ** -24 * sc * float(q.double().abs().sum(-1).max()) * float(k.abs().max()) * 6 if k.numel() else 0.0
    rel = 2 * (dx + 2.0 ** -22) + 2.0 ** -16 + (32 + Sk / 32) * 2.0 ** -24 * 16
    if dtype == BF and q.shape[1] // k.shape[1] * q.shape[2] > 16:
        rel += 5 * 2.0 ** -12
    tol = rel * float(v.abs().max()) + half_step(dtype) * ref.abs()
    if dtype == FP:
        tol = tol + 2.0 ** -25
    err = (got.cpu().double() - ref).abs()
    assert torch.isfinite(got).all(), what
    assert (err <= tol).all(), f"{what}: {float((err / tol).max())} of the tolerance"
    return ref


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("Hq,H,Sq", [(1, 1, 1), (8, 2, 1), (4, 4, 1), (6, 2, 5), (2, 2, 16), (4, 2, 17), (2, 2, 67),
                                     (8, 1, 33)])
@pytest.mark.parametrize("Sk", [1, 31, 32, 33, 257, 700])
def test_attention(D, dtype, Hq, H, Sq, Sk):
    B = 2
    c, k, v = _filled(B, H, Sk, D, dtype, 20)
    q = _randn(23, B, Hq, Sq, D, dtype=dtype)
    for out_dtype in (F32, dtype):
        got = attention_kv4(q.to(DEV), c, out_dtype=out_dtype)
        _attn_check(got, q, k, v, out_dtype, what=f"out {out_dtype}")


@pytest.mark.parametrize("splits", [1, 2, 7, 64])
@pytest.mark.parametrize("Sq,causal", [(1, False), (3, True), (40, True), (200, True)])
def test_splits_and_causal(splits, Sq, causal):
    B, Hq, H, Sk, D = 3, 4, 2, 190, 64
    c, k, v = _filled(B, H, Sk, D, BF, 30, cap=201)
    q = _randn(33, B, Hq, Sq, D, dtype=BF)
    valid = torch.tensor([190, 0, 77], dtype=torch.int32)
    got = attention_kv4(q.to(DEV), c, keys=Sk, is_causal=causal, valid_len=valid.to(DEV), num_splits=splits,
                        out_dtype=F32)
    ref = _attn_check(got, q, k, v, F32, valid=valid, causal=causal)
    assert (ref[1] == 0).all() and (got[1] == 0).all()   # no key at all
    if causal and Sq == 200:
        assert (got[2, :, :123] == 0).all()               # rows before the first token


@pytest.mark.parametrize("Sq", [1, 67])
def test_masks(Sq):
    """Masks with rows of nothing, lengths out of range, and a NaN key behind the mask."""
    B, Hq, H, Sk, D = 4, 4, 2, 150, 128
    c, k, v = _filled(B, H, Sk, D, FP, 40, cap=160)
    mask = torch.rand(B, Sk, generator=torch.Generator().manual_seed(4)) < 0.6
    mask[0] = False
    mask[1, :64] = False
    mask[2, 77] = False
    bad = torch.full((B, H, 1, D), float("nan"), dtype=FP, device=DEV)
    c.write(bad, bad, torch.tensor([[-1], [3], [77], [159]], dtype=torch.int32, device=DEV))
    valid = torch.tensor([150, 1000, 149, -3], dtype=torch.int32)
    q = _randn(43, B, Hq, Sq, D, dtype=FP)
    for dt in (torch.bool, torch.uint8):
        got = attention_kv4(q.to(DEV), c, keys=Sk, valid_len=valid.to(DEV), kv_mask=mask.to(dt).to(DEV), out_dtype=FP)
        _attn_check(got, q, k, v, FP, valid=valid, mask=mask)
        assert (got[0] == 0).all() and (got[3] == 0).all()


def test_causal_nan_is_seen_by_later_rows_only():
    B, H, Sk, D = 1, 1, 40, 64
    c, k, v = _filled(B, H, Sk, D, BF, 50)
    bad = torch.full((1, 1, 1, D), float("nan"), dtype=BF, device=DEV)
    c.write(bad, bad, torch.tensor([[30]], dtype=torch.int32, device=DEV))
    q = _randn(53, B, H, Sk, D, dtype=BF)
    got = attention_kv4(q.to(DEV), c, is_causal=True, out_dtype=F32)
    _attn_check(got[:, :, :30], q[:, :, :30], k[:, :, :30], v[:, :, :30], F32, causal=True)
    assert torch.isnan(got[:, :, 30:]).all()


@pytest.mark.parametrize("scale", [0.02, 1.0, 8.0])
def test_scales_and_peaks(scale):
    """Nearly uniform weights up to one key's taking all, with maxima that rise along the keys."""
    B, H, Sk, D = 1, 2, 300, 64
    k = _randn(60, B, H, Sk, D, dtype=BF) * torch.linspace(0.1, 3, Sk)[:, None].to(BF)
    v = _randn(61, B, H, Sk, D, dtype=BF)
    c = Kv4Cache(B, H, Sk, D, DEV)
    c.write(k.to(DEV), v.to(DEV))
    q = _randn(62, B, H, 3, D, dtype=BF)
    got = attention_kv4(q.to(DEV), c, scale=scale, out_dtype=F32)
    _attn_check(got, q, kv4_levels(k), kv4_levels(v), F32, scale=scale)


def test_values_of_unequal_size():
    """Tokens whose values differ by 2^40, the large ones all but unseen."""
    B, H, Sk, D = 1, 1, 96, 64
    k = _randn(63, B, H, Sk, D, dtype=BF)
    v = _randn(64, B, H, Sk, D, dtype=BF)
    v[:, :, ::7] *= 2.0 ** 20
    v[:, :, 1::7] *= 2.0 ** -20
    c = Kv4Cache(B, H, Sk, D, DEV)
    c.write(k.to(DEV), v.to(DEV))
    q = _randn(65, B, H, 2, D, dtype=BF)
    _attn_check(attention_kv4(q.to(DEV), c, out_dtype=F32), q, kv4_levels(k), kv4_levels(v), F32)


def test_strides_and_neighbours():
    """Queries as columns of a projection's rows, output as rows [B, S, H * D] inside a wider buffer."""
    B, Hq, H, Sq, Sk, D = 2, 6, 3, 9, 65, 64
    c, k, v = _filled(B, H, Sk, D, BF, 70)
    rows = _randn(73, B, Sq, 2 * Hq * D, dtype=BF).to(DEV)
    q = rows[..., Hq * D:].unflatten(2, (Hq, D)).transpose(1, 2)
    wide = torch.full((B, Sq, Hq * D + 16), 7.0, dtype=F32, device=DEV)
    out = wide[..., 8:8 + Hq * D].unflatten(2, (Hq, D)).transpose(1, 2)
    attention_kv4(q, c, out=out)
    _attn_check(out, q.cpu(), k, v, F32)
    assert (wide[..., :8] == 7).all() and (wide[..., 8 + Hq * D:] == 7).all()


def test_runs_are_equal_and_splits_agree():
    B, Hq, H, Sk, D = 2, 8, 2, 3000, 128
    c, k, v = _filled(B, H, Sk, D, BF, 80)
    q = _randn(83, B, Hq, 1, D, dtype=BF).to(DEV)
    one = attention_kv4(q, c, out_dtype=F32)
    for _ in range(3):
        assert torch.equal(one, attention_kv4(q, c, out_dtype=F32))
    _attn_check(attention_kv4(q, c, num_splits=5, out_dtype=F32), q.cpu(), k, v, F32)


@pytest.mark.parametrize("D", [64, 128])
def test_bf16_rows_of_many_tiles(D):
    """Many query rows with a bf16 output: V in fp16 under a common power of two, p in fp16 (5 2^-12 together)."""
    B, Hq, H, Sq, Sk = 2, 4, 2, 67, 333
    k = _randn(90, B, H, Sk, D, dtype=BF)
    v = _randn(91, B, H, Sk, D, dtype=BF)
    v[0] *= 2.0 ** 100          # beyond fp16's range, a head at a time
    v[1, 1] *= 2.0 ** -100
    v[0, 0, ::5] *= 2.0 ** -20  # and within one
    v[1, 0, 200:] *= 2.0 ** 30  # a common power that has to move
    c = Kv4Cache(B, H, Sk, D, DEV)
    c.write(k.to(DEV), v.to(DEV))
    q = _randn(92, B, Hq, Sq, D, dtype=BF)
    got = attention_kv4(q.to(DEV), c).cpu().double()
    lk, lv = kv4_levels(k), kv4_levels(v)
    ref = attend(q, lk, lv)
    for b in range(B):
        for h in range(Hq):
            tol = 2.0 ** -9 * float(lv[b, h // 2].abs().max()) + half_step(BF) * ref[b, h].abs()
            assert ((got[b, h] - ref[b, h]).abs() <= tol).all(), (b, h)


@pytest.mark.parametrize("D", [64, 128])
def test_causal_nan_with_bf16_output(D):
    B, H, Sk = 1, 1, 70
    c, k, v = _filled(B, H, Sk, D, BF, 93)
    good = _randn(94, 1, 1, 1, D, dtype=BF)
    bad = good.clone()
    bad[..., 5] = float("inf")
    c.write(good.to(DEV), bad.to(DEV), torch.tensor([[30]], dtype=torch.int32, device=DEV))
    q = _randn(95, B, H, Sk, D, dtype=BF)
    got = attention_kv4(q.to(DEV), c, is_causal=True)
    ref = attend(q[:, :, :30], k[:, :, :30], v[:, :, :30], causal=True)
    assert ((got[:, :, :30].cpu().double() - ref).abs() <= 2.0 ** -9 * 5 + half_step(BF) * ref.abs()).all()
    assert torch.isnan(got[:, :, 30:, :64]).all()


@pytest.mark.parametrize("kind", ["plain", "causal", "mask"])
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("B,Hq,H,Sq,Sk", [(4, 32, 32, 67, 150), (4, 64, 64, 64, 150), (4, 64, 64, 67, 150), (8, 64, 32, 33, 97)])
def test_many_heads(B, Hq, H, Sq, Sk, dtype, kind):
    """Enough heads that a workgroup takes three, four or five tiles of rows, with rows left over in the last."""
    D = 64
    c, k, v = _filled(B, H, Sk, D, dtype, 120)
    q = _randn(123, B, Hq, Sq, D, dtype=dtype)
    kw = {}
    if kind == "causal":
        kw["valid"] = torch.tensor([Sk, 0, 30, Sk - 1][:B] + [Sk] * (B - 4), dtype=torch.int32)
    if kind == "mask":
        kw["mask"] = torch.rand(B, Sk, generator=torch.Generator().manual_seed(9)) < 0.5
        kw["mask"][1] = False
        kw["mask"][2, :70] = False
    got = attention_kv4(q.to(DEV), c, is_causal=kind == "causal",
                        valid_len=kw["valid"].to(DEV) if "valid" in kw else None,
                        kv_mask=kw["mask"].to(DEV) if "mask" in kw else None)
    _attn_check(got, q, k, v, dtype, what=kind, causal=kind == "causal", **kw)
    if kind != "plain":
        assert (got[1] == 0).all()


@pytest.mark.parametrize("kind", ["plain", "causal", "ragged", "mask"])
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("D,Hq,Sq,Sk", [(64, 64, 1, 512), (64, 128, 2, 497), (64, 64, 7, 500), (128, 64, 1, 481), (128, 128, 4, 512)])
def test_long_streams_of_few_rows(D, Hq, Sq, Sk, dtype, kind):
    """Blocks of keys enough that the tile's columns take several at a time; blocks left over at the end, splits,
    masked rows and NaN keys among them.  The reference runs on the device, in 64 bits."""
    B, H = 16, 64
    k = _randn(130, 1, H, Sk, D, dtype=dtype).to(DEV).repeat(B, 1, 1, 1) + torch.linspace(-1, 1, B, device=DEV).to(dtype)[:, None, None, None]
    v = (k * 0.75).flip(2)
    c = Kv4Cache(B, H, Sk + 9, D, DEV)
    c.data.fill_(0xff)
    c.write(k, v)
    lk, lv = kv4_levels(k), kv4_levels(v)
    q = _randn(133, B, Hq, Sq, D, dtype=dtype).to(DEV)
    valid = mask = None
    if kind in ("causal", "ragged"):
        valid = (torch.arange(B, device=DEV, dtype=torch.int32) * 41 + 3).clamp_max(Sk)
        valid[5] = 0
    if kind == "mask":
        mask = torch.rand(B, Sk, generator=torch.Generator().manual_seed(9)).to(DEV) < 0.5
        mask[1] = False
        mask[:, 40] = False
        bad = torch.full((B, H, 1, D), float("nan"), dtype=dtype, device=DEV)
        c.write(bad, bad, torch.full((B, 1), 40, dtype=torch.int32, device=DEV))
    causal = kind == "causal"
    sc = 1 / math.sqrt(D)
    for splits in (0, 3):
        got = attention_kv4(q, c, keys=Sk, is_causal=causal, valid_len=valid, kv_mask=mask, num_splits=splits)
        for b in range(B):
            n = Sk if valid is None else int(valid[b])
            kk, vv = (t[b, :, :n].repeat_interleave(Hq // H, 0) for t in (lk, lv))
            x = torch.matmul(q[b].double(), kk.transpose(1, 2).contiguous()) * sc
            if mask is not None:
                x[..., ~mask[b, :n]] = -math.inf
            if causal:
                x = x.masked_fill(torch.arange(n, device=DEV) > torch.arange(Sq, device=DEV)[:, None] + n - Sq, -math.inf)
            w = torch.softmax(x, -1)
            ref = torch.matmul(torch.where(torch.isnan(w), 0.0, w), vv) if n else torch.zeros_like(q[b]).double()
            dx = 24 * 2.0 ** -24 * sc * float(q.double().abs().sum(-1).max()) * float(lk.abs().max()) * 6
            rel = 2 * (dx + 2.0 ** -22) + 2.0 ** -16 + (32 + Sk / 32) * 2.0 ** -24 * 16 + (7 * 2.0 ** -12 if Hq // H * Sq > 16 and dtype == BF else 0)
            tol = rel * float(lv.abs().max()) + half_step(dtype) * ref.abs() + (2.0 ** -25 if dtype == FP else 0)
            assert ((got[b].double() - ref).abs() <= tol).all(), (splits, b)


@pytest.mark.parametrize("kind", ["causal", "mask"])
@pytest.mark.parametrize("dtype,out_dtype", [(BF, BF), (FP, FP), (BF, F32)])
@pytest.mark.parametrize("splits", [1, 3, 64])
def test_many_rows_of_128_channels(splits, dtype, out_dtype, kind):
    """Several blocks to a wave, splits with nothing to read, lengths of zero and below the rows' number."""
    B, Hq, H, Sq, Sk, D = 4, 6, 2, 19, 1100, 128
    c, k, v = _filled(B, H, Sk, D, dtype, 140, cap=1111)
    q = _randn(143, B, Hq, Sq, D, dtype=dtype)
    kw = {"valid": torch.tensor([1100, 0, 7, 513], dtype=torch.int32)}
    if kind == "mask":
        kw["mask"] = torch.rand(B, Sk, generator=torch.Generator().manual_seed(5)) < 0.4
        kw["mask"][0, 64:900] = False
    got = attention_kv4(q.to(DEV), c, keys=Sk, is_causal=kind == "causal", valid_len=kw["valid"].to(DEV), num_splits=splits,
                        kv_mask=kw["mask"].to(DEV) if "mask" in kw else None, out_dtype=out_dtype)
    _attn_check(got, q, k, v, out_dtype, what=kind, causal=kind == "causal", **kw)
    assert (got[1] == 0).all()


@pytest.mark.parametrize("Sq", [1, 40])
def test_no_keys_and_in_place(Sq):
    B, Hq, H, Sk, D = 2, 8, 2, 90, 64
    c, k, v = _filled(B, H, Sk, D, BF, 150)
    q = _randn(153, B, Hq, Sq, D, dtype=BF).to(DEV)
    assert (attention_kv4(q, c, keys=0) == 0).all()
    assert (attention_kv4(q, c, keys=0, is_causal=True, num_splits=2) == 0).all()
    assert attention_kv4(q[:, :, :0], c).shape == (B, Hq, 0, D)
    ref = attention_kv4(q, c)
    for splits in (0, 3):   # the output in the queries' place
        x = q.clone()
        attention_kv4(x, c, out=x, num_splits=splits)
        assert ((x.double() - ref.double()).abs() <= 2 * half_step(BF) * ref.double().abs() + 2.0 ** -9 * float(v.abs().max())).all()
        assert splits or torch.equal(x, ref)


def test_two_tokens_at_one_slot():
    """They leave a mixture there; what lies beside is as written."""
    B, H, S, D = 1, 3, 40, 64
    c = Kv4Cache(B, H, 64, D, DEV)
    old = _randn(160, B, H, 64, D, dtype=BF)
    c.write(old.to(DEV), old.to(DEV))
    new = _randn(161, B, H, S, D, dtype=BF)
    slots = torch.arange(S, dtype=torch.int32)[None].clone()
    slots[0, 7] = 20
    c.write(new.to(DEV), new.to(DEV), slots.to(DEV))
    want = old.clone()
    want[:, :, :S] = new
    want[:, :, 7] = old[:, :, 7]
    keep = torch.arange(64) != 20
    for got in c.read(dtype=F32):
        assert torch.equal(got.cpu()[:, :, keep], _levels(want).float()[:, :, keep])


@pytest.mark.parametrize("B,Hq,H,Sq,Sk,D", [(2, 8, 2, 1, 300, 128), (1, 2, 1, 40, 5000, 64), (1, 4, 2, 20, 5000, 128),
                                            (4, 32, 32, 1, 4096, 64), (2, 64, 64, 6, 4096, 128), (1, 8, 8, 16, 8192, 128)])
def test_fp32_outputs_are_near(B, Hq, H, Sq, Sk, D):
    """Within 1e-6 of the output's norm, over values whose mean is small beside them.  The reference runs on the
    device, in 64 bits."""
    k, v = _randn(170, B, H, Sk, D, dtype=BF).to(DEV), _randn(171, B, H, Sk, D, dtype=BF).to(DEV)
    c = Kv4Cache(B, H, Sk, D, DEV)
    c.write(k, v)
    q = _randn(172, B, Hq, Sq, D, dtype=BF).to(DEV)
    got = attention_kv4(q, c, out_dtype=F32)
    off = norm = 0.0
    for b in range(B):
        kk, vv = (kv4_levels(t[b]).repeat_interleave(Hq // H, 0) for t in (k, v))
        w = torch.softmax(torch.matmul(q[b].double(), kk.transpose(1, 2).contiguous()) / math.sqrt(D), -1)
        ref = torch.matmul(w, vv)
        off += float((got[b].double() - ref).square().sum())
        norm += float(ref.square().sum())
    assert math.sqrt(off / norm) <= 1e-6


def _near_the_largest(got, q, lk, lv, what="", causal=False, **kw):
    """A bf16 output of many rows: 7 2^-12 of the largest value that a row sees, and its own rounding.

    To the first order: p, its sum taken over the rounded p, and the value rounds by 2^-11 each, as does mid - 7.5 s
    (at most the largest value; s itself is exact), which comes to 5.2 2^-12 where they add up worst; values far
    below the largest, and weights, stand on fp16's last step, 0.5 and 1 2^-12 more (4096 keys of a wave)."""
    ref = attend(q, lk, lv, causal=causal, **kw)
    G, Sq, Sk = q.shape[1] // lk.shape[1], q.shape[2], lk.shape[2]
    top = lv.abs().amax(-1).repeat_interleave(G, 1)[:, :, None].expand(-1, -1, Sq, -1)
    if causal:
        seen = torch.arange(Sk) <= torch.arange(Sq)[:, None] + Sk - Sq
        top = torch.where(seen, top, 0.0)
    tol = 7 * 2.0 ** -12 * top.amax(-1, keepdim=True) + half_step(BF) * ref.abs()
    err = (got.cpu().double() - ref).abs()
    assert torch.isfinite(got).all(), what
    assert (err <= tol).all(), f"{what}: {float((err / tol.clamp_min(1e-300)).max())} of the tolerance"


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("first,then", [(-60, 60), (-100, 30), (-100, 100), (-126, 0), (60, -60)])
def test_values_that_grow_along_the_keys(D, first, then):
    """Every wave's first block of keys holds values by a factor 2^(then - first) away from its later ones'."""
    H, Sk = 2, 600
    k, v = _randn(180, 1, H, Sk, D, dtype=BF), _randn(181, 1, H, Sk, D)
    v[:, :, :256] *= 2.0 ** first
    v[:, :, 256:] *= 2.0 ** then
    c = Kv4Cache(1, H, Sk, D, DEV)
    c.write(k.to(DEV), v.to(BF).to(DEV))
    q = _randn(182, 1, H, 40, D, dtype=BF)
    got = attention_kv4(q.to(DEV), c, num_splits=1)
    _near_the_largest(got, q, kv4_levels(k), kv4_levels(v.to(BF)))


@pytest.mark.parametrize("kind", ["causal", "mask", "plain"])
@pytest.mark.parametrize("bad", [5, 100])
@pytest.mark.parametrize("out_dtype", [BF, FP, F32])
def test_bad_values_stay_in_their_channels(kind, bad, out_dtype):
    """An infinity among the values of a token: its 64 channels are NaN in the rows that see it, the others right."""
    H, Sk, D = 2, 75, 128
    _, k, v = _filled(1, H, Sk, D, BF, 183)
    c, _, _ = _filled(1, H, Sk, D, BF, 183)
    one = _randn(184, 1, H, 1, D, dtype=BF)
    spoilt = one.clone()
    spoilt[0, 0, 0, bad] = float("inf")
    c.write(one.to(DEV), spoilt.to(DEV), torch.tensor([[30]], dtype=torch.int32, device=DEV))
    k[:, :, 30:31] = v[:, :, 30:31] = kv4_levels(one)
    q = _randn(185, 1, H, Sk, D, dtype=BF)
    mask = None
    if kind == "mask":
        mask = torch.ones(1, Sk, dtype=torch.bool)
        mask[0, 3] = False
    got = attention_kv4(q.to(DEV), c, is_causal=kind == "causal", kv_mask=None if mask is None else mask.to(DEV),
                        out_dtype=out_dtype)
    sees = torch.arange(Sk) >= (30 if kind == "causal" else 0)
    part = slice(0, 64) if bad < 64 else slice(64, 128)
    assert torch.isnan(got[0, 0, sees, part]).all()
    got = got.cpu()
    # what is NaN for certain is given the right value, so that all the rest is compared
    ref = attend(q, k, v, causal=kind == "causal", mask=mask)
    got[0, 0, sees, part] = ref[0, 0, sees, part].to(got.dtype)
    _attn_check(got, q, k, v, out_dtype, causal=kind == "causal", mask=mask)


@pytest.mark.parametrize("D,Hq,H,Sq", [(64, 2, 1, 96), (64, 2, 2, 96), (128, 2, 1, 96), (128, 1, 1, 33), (64, 8, 1, 20)])
@pytest.mark.parametrize("up", [8, 16, 20, 60, -20])
def test_rows_do_not_feel_later_values(D, Hq, H, Sq, up):
    """Causal rows with a bf16 output: tokens 2^up as large behind a row leave its accuracy as it is."""
    Sk = 128
    k, v = _randn(186, 1, H, Sk, D, dtype=BF), _randn(187, 1, H, Sk, D)
    for at in (Sk - Sq + 7, Sk - Sq + 15, Sk - 5):   # several in one block, one in the last
        v[:, :, at] *= 2.0 ** up
    v = v.to(BF)
    v[:, :, Sk - 3] = 0
    c = Kv4Cache(1, H, Sk, D, DEV)
    c.write(k.to(DEV), v.to(DEV))
    q = _randn(188, 1, Hq, Sq, D, dtype=BF)
    lk, lv = kv4_levels(k), kv4_levels(v)
    _near_the_largest(attention_kv4(q.to(DEV), c, is_causal=True), q, lk, lv, causal=True)
    mask = torch.rand(1, Sk, generator=torch.Generator().manual_seed(6)) < 0.8
    mask[0, 0] = True
    _near_the_largest(attention_kv4(q.to(DEV), c, is_causal=True, kv_mask=mask.to(DEV), num_splits=2), q, lk,
                      torch.where(mask[:, None, :, None], lv, 0.0), causal=True, mask=mask)


@pytest.mark.parametrize("D", [64, 128])
def test_one_strong_key_before_a_million(D):
    """A million keys of 2^-25.2 of the first one's weight each, 1/38 of it together: no wave may round its own away.
    Keys and values are constants, which the cache holds exactly."""
    Sk, R = 1 << 20, 20
    c = Kv4Cache(1, 1, Sk, D, DEV)
    k = torch.zeros(1, 1, Sk, D, dtype=BF, device=DEV)
    v = torch.ones(1, 1, Sk, D, dtype=BF, device=DEV)
    k[:, :, 0] = 2.1875 * 8 / math.sqrt(D)
    v[:, :, 0] = -1 / 32
    c.write(k, v)
    q = torch.ones(1, 1, R, D, dtype=BF, device=DEV)
    x = float(k[0, 0, 0].double().sum()) / math.sqrt(D)
    assert 2.0 ** -25.5 < math.exp(-x) < 2.0 ** -25.05
    w = (Sk - 1) * math.exp(-x)
    ref = (w - 1 / 32) / (w + 1)
    for splits in (0, 1, 3):
        got = attention_kv4(q, c, num_splits=splits).double()
        assert ((got - ref).abs() <= 7 * 2.0 ** -12 + half_step(BF) * abs(ref)).all(), splits


@pytest.mark.parametrize("D,Sk", [(64, 400), (64, 4374), (128, 2000)])
def test_exact_pv(D, Sk):
    """exact_pv: a bf16 output of many rows is the fp32 output rounded, but for sums that lie 2^-14 of the output's
    norm or less from a border between two numbers (the pair is off by about 2^-16 of it; fp16 weights by 2^-11)."""
    B, H, Sq = 2, 4, 67
    c, _, _ = _filled(B, H, Sk, D, BF, 190)
    q = _randn(193, B, H, Sq, D, dtype=BF).to(DEV)
    fine = attention_kv4(q, c, out_dtype=F32)
    got = attention_kv4(q, c, exact_pv=True)
    rms = float(fine.double().square().mean().sqrt())
    # a sum moves by at most 2^-14 rms: it may then round to a neighbour, and not further
    lo, hi = (fine + 2.0 ** -14 * rms).to(BF), (fine - 2.0 ** -14 * rms).to(BF)
    assert (torch.minimum(lo, hi) <= got).all() and (got <= torch.maximum(lo, hi)).all()
    for dt in (FP, F32):   # nothing changes where there is no fp16 form
        assert torch.equal(attention_kv4(q, c, out_dtype=dt), attention_kv4(q, c, out_dtype=dt, exact_pv=True))
    one = q[:, :, :1]
    assert torch.equal(attention_kv4(one, c), attention_kv4(one, c, exact_pv=True))


def test_a_workspace_is_one_piece():
    """A view that names a place more than once has fewer bytes behind its pointer than elements."""
    c, k, v = _filled(1, 2, 300, 64, BF, 210)
    q = _randn(213, 1, 4, 1, 64, dtype=BF).to(DEV)
    n = 3 * 4 * 66   # floats: three splits of four rows
    with pytest.raises(ValueError):
        attention_kv4(q, c, num_splits=3, workspace=torch.zeros(1, dtype=F32, device=DEV).expand(n))
    with pytest.raises(ValueError):
        attention_kv4(q, c, num_splits=3, workspace=torch.zeros(2 * n, dtype=F32, device=DEV)[::2])
    with pytest.raises(RuntimeError):
        attention_kv4(q, c, num_splits=3, workspace=torch.zeros(n - 1, dtype=F32, device=DEV))
    room = torch.full((n + 8,), 7.0, dtype=F32, device=DEV)
    _attn_check(attention_kv4(q, c, num_splits=3, workspace=room[4:-4], out_dtype=F32), q.cpu(), k, v, F32)
    assert (room[:4] == 7).all() and (room[-4:] == 7).all()


@pytest.mark.parametrize("D,H,Hq,Sq,Sk,kind", [(64, 8, 8, 67, 404, "plain"), (64, 32, 32, 67, 4374, "plain"), (64, 4, 8, 130, 1537, "causal"),
                                               (64, 8, 8, 67, 4374, "mask"), (128, 8, 8, 67, 4374, "plain"), (128, 4, 16, 33, 2000, "causal"),
                                               (128, 2, 8, 268, 3000, "mask"), (128, 4, 16, 1, 16384, "plain"), (64, 4, 4, 4, 8192, "mask")])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_outputs_of_16_bits_in_the_norm(D, H, Hq, Sq, Sk, kind, dtype):
    """The 2-norm of the error over the output's.  Rounding the output adds at most half_step / sqrt(3) of it (an error
    spread evenly over its step).  The pair adds below 2^-15.  fp16 weights and values add, for values with a mean of
    zero, three errors that are independent from key to key: of p and of V, 2^-11 / sqrt(3) each, and of mid - 7.5 s,
    the same of a number about 2.5 times the values' own size: at most 2.9 2^-11 / sqrt(3).  The reference runs on the
    device, in 64 bits."""
    B = 2
    c = Kv4Cache(B, H, Sk, D, DEV)
    k, v = (_randn(s, B, H, Sk, D, dtype=dtype).to(DEV) for s in (194, 195))
    c.write(k, v)
    q = _randn(196, B, Hq, Sq, D, dtype=dtype).to(DEV)
    mask = torch.rand(B, Sk, generator=torch.Generator().manual_seed(8)).to(DEV) < 0.7 if kind == "mask" else None
    got = attention_kv4(q, c, is_causal=kind == "causal", kv_mask=mask)
    off = norm = 0.0
    for b in range(B):
        kk, vv = (kv4_levels(t[b]).repeat_interleave(Hq // H, 0) for t in (k, v))
        x = torch.matmul(q[b].double(), kk.transpose(1, 2).contiguous()) / math.sqrt(D)
        if mask is not None:
            x[..., ~mask[b]] = -math.inf
        if kind == "causal":
            x = x.masked_fill(torch.arange(Sk, device=DEV) > torch.arange(Sq, device=DEV)[:, None] + Sk - Sq, -math.inf)
        ref = torch.matmul(torch.softmax(x, -1), vv)
        off += float((got[b].double() - ref).square().sum())
        norm += float(ref.square().sum())
    half = dtype == BF and Hq // H * Sq > 16
    own = 2.9 * 2.0 ** -11 / math.sqrt(3) if half else 2.0 ** -15
    assert math.sqrt(off / norm) <= math.hypot(half_step(dtype) / math.sqrt(3), own)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hq,Sq,out_dtype", [(2, 2, F32), (2, 2, BF), (2, 2, FP), (2, 33, F32), (2, 33, FP), (64, 1, F32), (64, 1, FP)])
def test_large_values_of_unseen_weight(D, Hq, Sq, out_dtype):
    """Tokens whose values are 2^20 larger and whose weights are below 2^-45 of the rest: what a row is off by goes by
    the products of both, not by the values.  Many heads take several blocks of keys in one tile."""
    B, H, Sk = (8, 64, 1024) if Hq == 64 else (1, 2, 200)
    base = _randn(198, 1, 1, 1, D)
    k, v = _randn(199, 1, H, Sk, D, dtype=BF), _randn(200, 1, H, Sk, D, dtype=BF)
    # against rows near base a score of -44 (2^-63)
    far = (base * (-44.0 * math.sqrt(D) / float(base.square().sum()))).to(BF).expand(1, H, 1, D)
    k[:, :, ::9] = far
    v[:, :, ::9] *= 2.0 ** 20
    q = (base + _randn(201, 1, Hq, Sq, D) / 16).to(BF)
    c = Kv4Cache(B, H, Sk, D, DEV)
    c.write(*(t.expand(B, -1, -1, -1).contiguous().to(DEV) for t in (k, v)))
    got = attention_kv4(q.expand(B, -1, -1, -1).contiguous().to(DEV), c, out_dtype=out_dtype)
    lk, lv = kv4_levels(k), kv4_levels(v)
    x = torch.matmul(q.double(), lk.repeat_interleave(Hq // H, 1).transpose(2, 3)) / math.sqrt(D)
    p = torch.softmax(x, -1)
    assert float(p[..., ::9].max()) < 2.0 ** -45
    vv = lv.repeat_interleave(Hq // H, 1)
    ref, size = torch.matmul(p, vv), torch.matmul(p, vv.unflatten(-1, (-1, 64)).abs().amax(-1, keepdim=True).expand(*vv.shape[:-1], -1, 64).flatten(-2))
    # of the sum of p |v| (the largest of the 64 channels): the tolerance of _attn_check, its parts as there
    dx = 24 * 2.0 ** -24 / math.sqrt(D) * float(q.double().abs().sum(-1).max()) * float(lk.abs().max()) * 6
    rel = 2 * (dx + 2.0 ** -22) + 2.0 ** -16 + (32 + Sk / 32) * 2.0 ** -24 * 16
    tol = rel * size + half_step(out_dtype) * ref.abs() + (2.0 ** -25 if out_dtype == FP else 0)
    for b in range(B):
        assert ((got[b].cpu().double() - ref[0]).abs() <= tol[0]).all(), b


@pytest.mark.parametrize("kind", ["plain", "causal", "ragged", "mask"])
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("D,Hq,Sq,Sk", [(64, 64, 1, 512), (64, 128, 2, 497), (64, 64, 7, 500), (128, 64, 1, 481), (128, 128, 4, 512)])
def test_long_streams_of_few_rows_to_fp32(D, Hq, Sq, Sk, dtype, kind):
    """The three-term form of several blocks of keys in one tile, as test_long_streams_of_few_rows has the pair's."""
    B, H = 16, 64
    k = _randn(202, 1, H, Sk, D, dtype=dtype).to(DEV).repeat(B, 1, 1, 1) + torch.linspace(-1, 1, B, device=DEV).to(dtype)[:, None, None, None]
    v = (k * 0.75).flip(2)
    c = Kv4Cache(B, H, Sk + 9, D, DEV)
    c.data.fill_(0xff)
    c.write(k, v)
    lk, lv = kv4_levels(k), kv4_levels(v)
    q = _randn(203, B, Hq, Sq, D, dtype=dtype).to(DEV)
    valid = mask = None
    if kind in ("causal", "ragged"):
        valid = (torch.arange(B, device=DEV, dtype=torch.int32) * 41 + 3).clamp_max(Sk)
        valid[5] = 0
    if kind == "mask":
        mask = torch.rand(B, Sk, generator=torch.Generator().manual_seed(9)).to(DEV) < 0.5
        mask[1] = False
        mask[:, 40] = False
        bad = torch.full((B, H, 1, D), float("nan"), dtype=dtype, device=DEV)
        c.write(bad, bad, torch.full((B, 1), 40, dtype=torch.int32, device=DEV))
    sc = 1 / math.sqrt(D)
    for splits in (0, 3):
        got = attention_kv4(q, c, keys=Sk, is_causal=kind == "causal", valid_len=valid, kv_mask=mask, num_splits=splits,
                            out_dtype=F32)
        for b in range(B):
            n = Sk if valid is None else int(valid[b])
            kk, vv = (t[b, :, :n].repeat_interleave(Hq // H, 0) for t in (lk, lv))
            x = torch.matmul(q[b].double(), kk.transpose(1, 2).contiguous()) * sc
            if mask is not None:
                x[..., ~mask[b, :n]] = -math.inf
                vv = torch.where(mask[b, :n, None], vv, 0.0)
            if kind == "causal":
                x = x.masked_fill(torch.arange(n, device=DEV) > torch.arange(Sq, device=DEV)[:, None] + n - Sq, -math.inf)
            w = torch.softmax(x, -1)
            ref = torch.matmul(torch.where(torch.isnan(w), 0.0, w), vv) if n else torch.zeros_like(q[b]).double()
            dx = 24 * 2.0 ** -24 * sc * float(q.double().abs().sum(-1).max()) * float(lk.abs().max()) * 6
            rel = 2 * (dx + 2.0 ** -22) + 2.0 ** -16 + (32 + Sk / 32) * 2.0 ** -24 * 16
            assert ((got[b].double() - ref).abs() <= rel * float(lv.abs().max())).all(), (splits, b)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Sq", [1, 3, 40])
@pytest.mark.parametrize("out_dtype,causal", [(BF, False), (BF, True), (FP, False), (F32, False), (F32, True)])
def test_a_bad_query_stays_alone(D, Sq, out_dtype, causal):
    """An infinity and a NaN in two query rows: those are NaN, the tiles' other rows are right."""
    Hq, H, Sk = 4, 1, 333
    c, k, v = _filled(1, H, Sk, D, BF, 220)
    q = _randn(223, 1, Hq, Sq, D, dtype=BF)
    bad = q.clone()
    bad[0, 1, Sq - 1, 3], bad[0, 2, 0, D - 1] = float("inf"), float("nan")
    got = attention_kv4(bad.to(DEV), c, is_causal=causal, out_dtype=out_dtype)
    assert torch.isnan(got[0, 1, Sq - 1]).all() and torch.isnan(got[0, 2, 0]).all()
    ref = attend(q, k, v, causal=causal)
    got[0, 1, Sq - 1], got[0, 2, 0] = (ref[0, h, s].to(DEV, got.dtype) for h, s in ((1, Sq - 1), (2, 0)))
    _attn_check(got, q, k, v, out_dtype, causal=causal)


@pytest.mark.parametrize("D", [64, 128])
def test_a_causal_token_is_as_one_that_is_not(D):
    """One token's many heads see the same keys, causal or not: the same form, bit for bit."""
    B, Hq, H, Sk = 2, 64, 2, 700
    c, k, v = _filled(B, H, Sk, D, BF, 230)
    q = _randn(233, B, Hq, 1, D, dtype=BF)
    valid = torch.tensor([700, 331], dtype=torch.int32)
    got = [attention_kv4(q.to(DEV), c, is_causal=causal, valid_len=valid.to(DEV)) for causal in (True, False)]
    assert torch.equal(*got)
    _attn_check(got[0], q, k, v, BF, valid=valid, causal=True)
