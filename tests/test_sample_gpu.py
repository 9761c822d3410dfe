"""sf_sample against its definition in 64 bits.

Tokens are equal: weights are held to 2^-44 of the largest, and no case here puts
u within that (times the vocabulary) of a border but where the sums are exact on
both sides (equal logits).  A logprob is rounded to 32 bits once, from a value off by
2^-40 at most."""
import math

import pytest
import torch

from servoflow_amd import abi, kernels

from _drafts import sample as plain

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


def _logits(B, V, seed, dtype=F32, std=2.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, V, generator=g) * std
    x.scatter_add_(1, torch.randint(0, V, (B, 9), generator=g), 3 * torch.rand(B, 9, generator=g) + 4)
    return x.to(dtype)


def _u(B, seed):
    return torch.rand(B, generator=torch.Generator().manual_seed(seed + 99))


def _check(x, u, t=1.0, k=0, p=1.0, mp=0.0, what=""):
    """Every parameter a number or a list of one a row."""
    B = x.shape[0]
    dev = lambda v, dt: torch.tensor(v, dtype=dt, device=DEV) if isinstance(v, list) else v   # noqa: E731
    tok, lp = kernels.sample(x if x.is_cuda else x.to(DEV), u.to(DEV), dev(t, F32), dev(k, torch.int32), dev(p, F32), dev(mp, F32))
    x = x.cpu()
    for b in range(B):
        at = lambda v: float(torch.tensor(v[b] if isinstance(v, list) else v, dtype=F32))   # noqa: E731
        want, ref = plain(x[b], float(u[b]), at(t), int(k[b] if isinstance(k, list) else k), at(p), at(mp))
        assert int(tok[b]) == want, (what, b, int(tok[b]), want)
        got = float(lp[b])
        if math.isnan(ref):
            assert math.isnan(got)
        else:
            assert abs(got - ref) <= 2.0 ** -24 * abs(ref) + 2.0 ** -40, (what, b, got, ref)
    return tok


RULES = [{}, {"t": 0.7}, {"k": 50}, {"p": 0.9}, {"mp": 0.05}, {"t": 1.3, "k": 40, "p": 0.8, "mp": 0.02}, {"k": 1}, {"t": 0.0},
         {"p": 0.999, "t": 2.0}, {"k": 3000, "p": 0.95}]


@pytest.mark.parametrize("V", [1, 2, 7, 8, 63, 64, 65, 1000, 2047, 2049, 5001, 32000])
@pytest.mark.parametrize("dtype", [BF, FP, F32])
def test_rules(V, dtype):
    B = 3
    for i, r in enumerate(RULES):
        _check(_logits(B, V, V + i, dtype), _u(B, V + i), what=str(r), **r)


@pytest.mark.parametrize("V,dtype", [(131072, BF), (131073, FP), (200001, F32), (1 << 20, BF)])
def test_large_vocabularies(V, dtype):
    for i, r in enumerate(RULES):
        _check(_logits(2, V, i, dtype), _u(2, i), what=str(r), **r)


def test_parameters_a_row():
    B = 12
    x, u = _logits(B, 4000, 5, BF), _u(B, 5)
    _check(x, u, t=[0.0, 1.0, 0.5, 2.0, -1.0, 1e-30, 1e30, math.inf, 1.0, 1.0, 1.0, 1.0],
           k=[0, 1, 5, 4000, 9, 0, 0, 0, -3, 2 ** 31 - 1, 4001, 7], p=[0.5, 1.0, 0.3, 0.99, 0.2, 1.0, 1.0, 1.0, 0.0, -1.0, 1.5, 0.6],
           mp=[0.0, 0.0, 0.1, 0.0, 0.5, 0.0, 0.0, 0.0, 0.0, 0.2, 1.0, 2.0])


def test_views_and_alignment():
    for dtype in (BF, F32):
        wide = _logits(5, 3011, 8, dtype).to(DEV)
        for at, V in ((0, 3000), (1, 3000), (3, 2999), (7, 3), (9, 1)):
            x = wide[:, at:at + V]
            _check(x, _u(5, at), k=30, what=f"{at} {V}")
    one = _logits(1, 500, 3, BF).to(DEV)
    _check(one[:, 1:], _u(1, 3))


@pytest.mark.parametrize("V", [3, 1000, 5000, 131072])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_equal_logits(V, dtype):
    """Ties go by index: token n of V is the one whose range of 1 / V holds u; sums are exact."""
    x = torch.full((6, V), -1.25, dtype=dtype)
    u = torch.tensor([0.0, 0.24, 0.5, 0.77, 0.9999, 1 - 2.0 ** -24])
    _check(x, u)
    _check(x, u, k=max(1, V // 3))
    _check(x, u, p=0.5)
    _check(x, u, t=0.0)
    x[:, V // 2] = 0.5   # one above, its own weight
    _check(x, u, t=0.5)
    _check(x, u, p=[0.1, 0.3, 0.61, 0.72, 0.9, 0.95])


@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("V,std", [(131072, 0.01), (131072, 0.3), (60000, 1e-4), (60000, 1e-6), (20000, 1e-3)])
def test_flat_rows(V, dtype, std):
    """Thousands of tokens in one bucket: parts of its keys, down to one value."""
    B = 4
    x = torch.randn(B, V, generator=torch.Generator().manual_seed(3)) * std + 1.0
    x = x.to(dtype)
    u = _u(B, 7)
    for r in ({}, {"p": 0.4}, {"k": V // 2}, {"k": V // 3, "p": 0.37}, {"k": 5000, "p": 0.9, "mp": 0.5}, {"t": 30.0}):
        _check(x, u, what=f"{r}", **r)


@pytest.mark.parametrize("V", [3000, 70000])   # of fp32: by one workgroup, in parts
@pytest.mark.parametrize("dtype", [BF, FP, F32])
def test_masked_and_special_logits(dtype, V):
    low = torch.finfo(dtype).min
    x = _logits(9, V, 4, dtype)
    x[0] = -math.inf                       # nothing
    x[1, 5:] = -math.inf
    x[2, torch.arange(V) != 1234] = -math.inf
    x[3, 17] = math.nan
    x[4, [40, 2000]] = math.inf            # the two share all the weight
    x[5, 100:] = low                       # masks of the type's lowest value
    x[6] = low                             # every token masked so: all the same
    x[7, ::2] = -math.inf
    x[8, :] = torch.where(torch.arange(V) % 3 == 0, 0.0, -0.0)   # equal
    for r in ({}, {"k": 10}, {"p": 0.7}, {"mp": 0.3}, {"t": 0.0}, {"t": 5.0, "k": 2000, "p": 0.9}):
        tok = _check(x, torch.tensor([0.3, 0.9, 0.5, 0.5, 0.75, 0.99, 0.3334, 0.6, 0.5]), what=str(r), **r)
        assert tok[0] == -1 and tok[3] == -1


@pytest.mark.parametrize("V", [1, 9, 3000, 70000])
@pytest.mark.parametrize("dtype", [BF, FP, F32])
def test_nan_of_either_sign(dtype, V):
    x = _logits(6, V, 5, dtype)
    bits = {BF: 0x7fc0, FP: 0x7e00, F32: 0x7fc00000}[dtype]
    whole = x.view(torch.int32 if dtype is F32 else torch.int16)
    sign = -2 ** (31 if dtype is F32 else 15)
    whole[0, V // 2] = bits
    whole[1, V // 2] = bits + sign
    whole[2, :] = bits + sign
    whole[3, 0] = -1                       # all bits set
    whole[4, V - 1] = bits + sign
    assert x[:5].isnan().any(1).all() and not x[5].isnan().any()
    tok = _check(x, _u(6, 1))
    assert (tok[:5] == -1).all() and tok[5] >= 0


@pytest.mark.parametrize("V", [40, 3000, 50001, 131072])   # of fp32: by one workgroup, in parts
@pytest.mark.parametrize("dtype", [BF, FP, F32])
def test_logprob_of_a_token_that_has_nearly_all(dtype, V):
    """-log(1 + what the others weigh), to 1e-6 of itself down to V 2^-75: for one token far above a bulk, for two, with each
    rule.  The sums of the others are in 64 bits apart from the largest here."""
    B = 7
    base = torch.randn(B, V, generator=torch.Generator().manual_seed(V)) * 2
    u = torch.full((B,), 0.5)
    for gap in (8.0, 14.0, 20.0, 27.0, 33.0, 40.0):
        x = base.clone()
        at = torch.arange(B) * 5 % V
        x[torch.arange(B), at] = base.max() + gap
        x[:3, V - 1] = base.max() + gap / 2
        x = x.to(dtype)
        for r in ({}, {"t": 0.5}, {"t": 1.5}, {"k": 2}, {"k": 39}, {"mp": 1e-12}, {"k": 30, "mp": 1e-9}, {"p": 1 - 2.0 ** -24},
                  {"t": 2.0, "k": 1000, "p": 1 - 2.0 ** -23}, {"k": 1}):
            tok, lp = kernels.sample(x.to(DEV), u.to(DEV), r.get("t", 1.0), r.get("k", 0), r.get("p", 1.0), r.get("mp", 0.0))
            for b in range(B):
                order = torch.argsort(-x[b].double(), stable=True)
                y = (x[b].double()[order] - x[b].double().max()) / r.get("t", 1.0)
                w = torch.exp(y)
                n = min(r.get("k", 0) or V, V)
                if "p" in r:
                    p = float(torch.tensor(r["p"], dtype=F32))
                    # reaches p of all: what is left behind is (1 - p) of it at most, summed from the smallest on; V weights
                    # held to 2^-44 leave the border undecided by V 2^-44
                    left = torch.flip(torch.cumsum(torch.flip(w[:n], [0]), 0), [0])
                    edge = (left[1:] / left[0] - (1 - p)).abs() < V * 2.0 ** -44
                    if edge.any():
                        continue
                    n = 1 + int((left[1:] / left[0] > 1 - p).sum())
                if "mp" in r:
                    n = min(n, int((w >= float(torch.tensor(r["mp"], dtype=F32))).sum()))
                rest = float(torch.flip(w[1:n], [0]).sum())
                if rest >= 0.5:
                    continue
                want = -math.log1p(rest)
                assert int(tok[b]) == int(order[0])
                # 16 bits: each weight is cut off to a multiple of 2^-75, from 2^-12 on of 2^-67.  fp32: V threads' sums
                # at most are cut off to 2^-70; what top-k leaves out below 2^-46 of the largest may be in; and k kept weights
                # are taken as held, to 2^-44, where they are k 2^-24 and more.
                cut = V * 2.0 ** -75
                if dtype is F32:
                    k = min(r.get("k", 0), V)
                    cut = V * 2.0 ** -70 + (V - k if k else 0) * 2.0 ** -46
                assert abs(float(lp[b]) - want) <= 1e-6 * abs(want) + cut, (gap, r, b, float(lp[b]), want)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_min_p_of_one_keeps_equal_weights(dtype):
    # Logits 1e-20 apart weigh the same in 64 bits (and 2^-44 of the largest, in which they are held, is more); those 1e-3 apart
    # do not.
    x = _logits(4, 500, 8) * 1e-20
    x[1] = x[1] * 1e17
    _check(x.to(dtype), _u(4, 8), mp=1.0)


def test_u_at_its_ends():
    x = _logits(6, 777, 9)
    u = torch.tensor([0.0, 1 - 2.0 ** -24, 2.0 ** -149, 0.5, 2.0 ** -24, 0.0])
    _check(x, u)
    a, _ = kernels.sample(x[:3].to(DEV), torch.tensor([1.0, -1.0, math.nan], device=DEV), top_k=20)
    b, _ = kernels.sample(x[:3].to(DEV), torch.tensor([1 - 2.0 ** -24, 0.0, 0.0], device=DEV), top_k=20)
    assert torch.equal(a, b)


@pytest.mark.parametrize("r", [{"t": 0.9}, {"k": 7}, {"p": 0.8}])
def test_frequencies(r):
    """u on a grid of N gives every token N times its share, but for one at each end."""
    N, V = 4096, 300
    row = _logits(1, V, 2, F32)
    u = (torch.arange(N) + 0.5) / N
    dev = {"t": "temperature", "k": "top_k", "p": "top_p"}
    tok, lp = kernels.sample(row.expand(N, V).contiguous().to(DEV), u.to(DEV), **{dev[a]: b for a, b in r.items()})
    share = torch.zeros(V, dtype=torch.float64)
    share[tok.cpu().long()] = torch.exp(lp.cpu().double())
    assert 1 - V / N < float(share.sum()) <= 1 + 1e-6   # a token that no u of the grid meets has less than 1 / N, V of them V / N
    got = torch.bincount(tok.cpu().long(), minlength=V).double()
    assert ((got - N * share).abs() <= 1.001).all()


def test_runs_are_equal():
    x, u = _logits(64, 50001, 6, BF).to(DEV), _u(64, 6).to(DEV)
    first = kernels.sample(x, u, temperature=1.5, top_p=0.97)
    for _ in range(5):
        again = kernels.sample(x, u, temperature=1.5, top_p=0.97)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
    alone = torch.cat([kernels.sample(x[i:i + 1], u[i:i + 1], temperature=1.5, top_p=0.97)[0] for i in range(64)])
    assert torch.equal(first[0], alone)


def test_workspace():
    """Rows in parts: a workspace given, used twice, too small, and the rows alone."""
    x, u = _logits(3, 100001, 6, F32).to(DEV), _u(3, 6).to(DEV)
    want = kernels.sample(x, u, top_p=0.95)
    ws = torch.full((3 * (2048 * 12 + 2 * 8 + 64 * 4),), 0xff, dtype=torch.uint8, device=DEV)
    for _ in range(3):
        got = kernels.sample(x, u, top_p=0.95, workspace=ws)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    with pytest.raises(abi.SfError):
        kernels.sample(x, u, workspace=ws[:-8])
    with pytest.raises(ValueError):
        kernels.sample(x, u, workspace=ws[::2])
    alone = torch.cat([kernels.sample(x[i:i + 1], u[i:i + 1], top_p=0.95)[0] for i in range(3)])
    assert torch.equal(alone, want[0])
    many = x.repeat(60, 1)   # so many rows go by one workgroup each
    assert torch.equal(kernels.sample(many, u.repeat(60), top_p=0.95)[0], want[0].repeat(60))


def test_no_rows_and_refusals():
    x, u = torch.zeros(2, 10, device=DEV), torch.zeros(2, device=DEV)
    tok, lp = kernels.sample(x[:0], u[:0])
    assert tok.shape == lp.shape == (0,)
    for kw in ({"u": u[:1]}, {"u": None}, {"temperature": u[:1]}, {"top_k": u}, {"top_p": u.double()}, {"logits": x.double()},
               {"logits": x.t()}, {"logits": x[0]}):
        with pytest.raises(ValueError):
            kernels.sample(**{"logits": x, "u": u, **kw})


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("V", [70000, 131072, 300001])
def test_many_equal_16_bit_logits(V, dtype):
    """More than 65535 tokens of one value: a mask's, the row's largest, zeros of both signs, or all of them; and many values."""
    g = torch.Generator().manual_seed(V)
    x = (torch.randn(8, V, generator=g) * 2).to(dtype)
    x[0, torch.rand(V, generator=g) < 0.99] = -math.inf
    x[1, torch.rand(V, generator=g) < 0.99] = torch.finfo(dtype).min
    x[2, torch.rand(V, generator=g) < 0.97] = -3.0
    x[3] = 0.0
    x[3, ::2] = -0.0
    x[4, torch.rand(V, generator=g) < 0.97] = 9.0
    x[5] = torch.randint(-32768, 32767, (V,), generator=g, dtype=torch.int16).view(dtype)   # any 16 bits
    x[5][torch.isnan(x[5])] = 1.0
    x[5][torch.isinf(x[5])] = 2.0
    x[6] = math.nan
    x[7, :65536] = -1.5
    u = torch.tensor([0.1, 0.999, 0.7, 0.3, 0.6, 0.5, 0.2, 0.97])
    for r in ({}, {"t": 3.0}, {"k": 1000}, {"p": 0.9}, {"t": 1e4, "p": 0.6}, {"k": 60000, "p": 0.99, "mp": 1e-3}, {"t": 0.0}):
        _check(x, u, what=str(r), **r)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("V", [1023, 1024, 5001, 70000, 200000])
def test_a_value_that_many_tokens_share(dtype, V):
    """It is counted apart where it is many tokens' (by itself, as 0 beside -0, beside -infinity); it is drawn as any other."""
    g = torch.Generator().manual_seed(V)
    x = _logits(8, V, 3, dtype)
    some = torch.rand(8, V, generator=g)
    x[0][some[0] < 0.97] = -1e4
    x[1][some[1] < 0.5] = 0.0
    x[2][some[2] < 0.5] = torch.where(torch.rand(V, generator=g) < 0.5, 0.0, -0.0).to(dtype)[some[2] < 0.5]
    x[3][some[3] < 0.4], x[3][some[3] > 0.6] = -math.inf, 2.0
    x[4][some[4] < 0.97] = -0.0
    x[5][some[5] < 0.2] = 1.5
    x[6, V // 3:] = torch.finfo(dtype).min
    x[7][some[7] < 0.9] = x[7].max()       # the largest
    u = torch.tensor([0.999, 0.5, 0.55, 0.8, 0.6, 0.3, 1 - 2.0 ** -24, 0.777])
    for r in ({}, {"k": V - 3}, {"p": 0.7}, {"mp": 0.3, "t": 3.0}, {"t": 1e6}, {"t": 5.0, "k": 2000, "p": 0.9}, {"t": 0.0}):
        _check(x, u, what=str(r), **r)


def test_only_lowest_numbers_are_left():
    """A row masked by the lowest number but for -infinity: its tokens share the weight."""
    for dtype in (BF, FP, F32):
        low = torch.finfo(dtype).min
        x = torch.full((3, 5000), -math.inf, dtype=dtype)
        x[0, 100:2000] = low
        x[1, 4999] = low
        x[2, ::3] = low
        x[2, 17] = low / 2
        for r in ({}, {"p": 0.5}, {"k": 7}, {"mp": 0.5}, {"t": math.inf}):
            _check(x, torch.tensor([0.77, 0.5, 0.3]), what=str(r), **r)


@pytest.mark.parametrize("V", [131072, 131073, 1 << 18, 300001, 1 << 20])
@pytest.mark.parametrize("rows", [2, 300])   # fp32: in parts, by one workgroup each
def test_logprob_beside_the_others_of_a_large_vocabulary(V, rows):
    """One token far above others that weigh up to more than V 2^-24 of it in all, where their sum is not taken any more: flat
    bulks and broad ones, with temperature alone, min-p that keeps all or some, and rules that keep all."""
    g = torch.Generator().manual_seed(V)
    shares = [2.0 ** -9, 2.0 ** -7, 1.02 * 2.0 ** -6, 0.03, 0.99 * V * 2.0 ** -24, 0.999 * V * 2.0 ** -24, 1.05 * V * 2.0 ** -24, 0.1]
    base = torch.empty(2 * len(shares), V)
    for i, share in enumerate(shares):
        base[2 * i] = math.log(share / (V - 1))
        base[2 * i + 1] = math.log(share / (V - 1)) - 0.125 + 0.5 * torch.randn(V, generator=g)   # exp(randn / 2) is 1.133 in the mean
    top = torch.randint(0, V, (len(base),), generator=g)
    base[torch.arange(len(base)), top] = 0.0
    base = base.to(DEV)
    w = torch.exp(base.double())
    w[torch.arange(len(base)), top] = 0.0
    cut = float(torch.tensor(0.03 / V, dtype=F32))
    for r, keep in (({}, w), ({"temperature": 0.5}, w), ({"min_p": 1e-12}, w), ({"min_p": cut}, torch.where(w >= cut, w, 0.0)),
                    ({"top_k": V, "top_p": 1.0}, w)):
        x = base * r.get("temperature", 1.0)   # (a half: exact)
        want = torch.log1p(keep.sum(1)).neg().cpu()
        for at in range(0, len(base), rows):
            pick = torch.arange(at, at + rows) % len(base)
            tok, lp = kernels.sample(x[pick.to(DEV)], torch.full((rows,), 0.5, device=DEV), **r)
            assert torch.equal(tok.cpu().long(), top[pick])
            # Rounded to fp32 once; the others' sum is cut off by V 2^-70 in all, or each of them is held to 2^-44 where they weigh
            # V 2^-24 and more (a few that weigh hardly less may be taken so).
            held = torch.where(torch.expm1(want[pick].neg()) >= 0.9999 * V * 2.0 ** -24, V * 2.0 ** -44, V * 2.0 ** -70)
            err = (lp.cpu().double() - want[pick]).abs()
            assert (err <= (2.0 ** -24 + 2.0 ** -40) * want[pick].abs() + held).all(), (r, at, float((err / want[pick].abs()).max()))


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("V", [300001, 1 << 20])
def test_logprob_beside_two_values_that_most_tokens_share(dtype, V):
    """Each of them more often than 16 bits count: 16-bit rows that go through the buckets."""
    shares = [2.0 ** -8, 1.02 * 2.0 ** -6, 0.9 * V * 2.0 ** -24]
    x = torch.empty(len(shares), V, dtype=dtype)
    for i, share in enumerate(shares):
        x[i] = math.log(share / V) - 0.2
        x[i, 1::2] -= 0.125   # a step of both types, or several
        x[i, 7 * i + 5] = 0.0
    w = torch.exp(x.double())
    w[torch.arange(len(shares)), 7 * torch.arange(len(shares)) + 5] = 0.0
    want = torch.log1p(w.sum(1)).neg()
    assert (torch.expm1(-want) < 0.999 * V * 2.0 ** -24).all()
    for r in ({}, {"min_p": 1e-12}):
        tok, lp = kernels.sample(x.to(DEV), torch.full((len(shares),), 0.5, device=DEV), **r)
        assert tok.tolist() == [5, 12, 19]
        assert ((lp.cpu().double() - want).abs() <= (2.0 ** -24 + 2.0 ** -40) * want.abs() + V * 2.0 ** -70).all(), (lp, want)


@pytest.mark.parametrize("V", [5, 500, 6000, 60000])   # of fp32: by one workgroup, in parts
@pytest.mark.parametrize("dtype", [BF, F32])
def test_smallest_logits_and_temperatures(dtype, V):
    """Logits of the smallest numbers there are: how far below the largest they weigh nothing is then less than a bucket of theirs
    takes apart."""
    unit = 2.0 ** -133 if dtype is BF else 2.0 ** -149
    x = torch.randint(-4, 5, (6, V), generator=torch.Generator().manual_seed(V)).double() * unit
    x[1] *= 2.0 ** 11
    x[2] = torch.where(torch.arange(V) % 3 == 0, 0.0, -unit)
    x[3, ::2] = -math.inf
    x[4] = torch.rand(V, generator=torch.Generator().manual_seed(V)).double() * 1e-36
    x[5] = torch.where(torch.arange(V) % 3 == 0, 0.0, -8e-39)   # a bucket of one value
    y = x.to(dtype)
    if dtype is BF:
        assert torch.equal(y[:4].double(), x[:4])
    u = torch.tensor([0.95, 0.5, 0.999, 0.3, 0.97, 0.999])
    for r in ({"t": 1.4e-39}, {"t": 7e-40}, {"t": 2.0 ** -149}, {"t": 1e-44, "k": 3}, {"t": 1e-40}, {"t": 2e-41, "p": 0.9}, {"t": 1e-38, "mp": 0.5}, {"t": 5e-37, "k": V}):
        _check(y, u, what=str(r), **r)
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("V", [400, 3000, 60000])   # of fp32: by one workgroup, in parts
def test_differences_beyond_the_largest_number(dtype, V):
    """Logits of both ends of the type: their difference has no fp32 value, its quotient by a large temperature has."""
    g = torch.Generator().manual_seed(V)
    x = ((torch.rand(4, V, generator=g) * 2 - 1) * 3.3e38).to(dtype)
    x[1] = torch.where(torch.rand(V, generator=g) < 0.5, -3.3e38, 3.3e38).to(dtype)
    x[2, ::3] = -math.inf
    x[3] = torch.finfo(dtype).min
    x[3, V // 2] = torch.finfo(dtype).max
    u = torch.tensor([0.95, 0.9, 0.99, 0.999])
    for r in ({"t": 1e38}, {"t": 3e37, "p": 0.99}, {"t": 2e38, "k": V - 5}, {"t": 3e38, "mp": 0.2}, {"t": math.inf}, {"t": 1.0}):
        _check(x, u, what=str(r), **r)


@pytest.mark.parametrize("V", [1500, 70000, 200001])
@pytest.mark.parametrize("dtype", [BF, FP, F32])
def test_one_of_many_largest(dtype, V):
    """A min-p above 1 leaves the first of thousands of equals, whose logprob is 0: nothing else weighs; beside lower ones, few and
    many, and as the whole row."""
    x = torch.full((4, V), 2.5, dtype=dtype)
    x[1, :7] = -3.0
    x[2, ::5] = 1.0
    x[3, :V // 2] = -math.inf
    first = [0, 7, 1, V // 2]
    for u in (0.0, 0.4, 1 - 2.0 ** -24):
        for r in ({"min_p": 2.0}, {"min_p": 1.5, "top_k": V - 1}, {"min_p": 3.0, "top_p": 0.9}):
            tok, lp = kernels.sample(x.to(DEV), torch.full((4,), u, device=DEV), **r)
            assert tok.tolist() == first and (lp == 0).all(), (u, r, tok, lp)


@pytest.mark.parametrize("V", [1, 2, 500, 50001])   # of fp32: by one workgroup, in parts
@pytest.mark.parametrize("dtype", [BF, FP, F32])
def test_the_first_in_order_alone_has_a_logprob_of_0(dtype, V):
    """Beside others that weigh from e^-60 to e^-1 of it."""
    x = torch.randn(5, V, generator=torch.Generator().manual_seed(V))
    for b, gap in enumerate((1.0, 20.0, 33.0, 40.0, 60.0)):
        x[b, (7 * b + V // 2) % V] = x[b].max() + gap
    x = x.to(dtype)
    for r in ({"t": 0.0}, {"k": 1}, {"t": -1.0, "k": 7, "mp": 1e-30}, {"k": 1, "p": 0.5}, {"t": 0.5, "k": 1, "mp": 0.1}):
        tok, lp = kernels.sample(x.to(DEV), _u(5, V).to(DEV), r.get("t", 1.0), r.get("k", 0), r.get("p", 1.0), r.get("mp", 0.0))
        assert torch.equal(tok.cpu().long(), x.float().argmax(1)) and (lp == 0).all(), (r, tok, lp)
