"""sf_quant_i8 and sf_gemm_i8 against the definition in 64 bits.

Codes and scales are equal.  The sum over k is exact; an output takes its conversion
to fp32, two products and the bias, each 2^-24 of |sum| s t + |bias|; activations have
slopes below 1.2 and add at most 2^-20 of that by their own evaluation; a 16-bit
output adds half a step of itself."""
import math

import pytest
import torch

from servoflow_amd import abi, kernels

from _drafts import quant
from _quant4 import half_step

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _codes(seed, *shape):
    return torch.randint(-128, 128, shape, generator=_gen(seed), dtype=torch.int8)


def _scales(seed, n):
    return torch.rand(n, generator=_gen(seed)) * 0.02 + 1e-3


def _act(act, x):
    if act == abi.SF_ACT_GELU_TANH:
        return 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)))
    return x * torch.sigmoid(x) if act == abi.SF_ACT_SILU else x


def _check(got, a, s, w, t, bias=None, act=0, was=None, what=""):
    y = torch.matmul(a.double(), w.double().t()) * s.double()[:, None] * t.double()
    big = y.abs() + (0 if bias is None else bias.double().abs())
    ref = _act(act, y if bias is None else y + bias.double())
    tol = 1.2 * 5 * 2.0 ** -24 * big + (2.0 ** -20 * big if act else 0)
    if was is not None:
        ref = ref + was.double()
        tol = tol + 2.0 ** -24 * ref.abs()
    tol = tol + half_step(got.dtype) * (ref.abs() + tol) + 1e-30 + (2.0 ** -25 if got.dtype == FP else 0)
    err = (got.cpu().double() - ref).abs()
    assert torch.isfinite(got).all(), what
    assert (err <= tol).all(), f"{what}: {float((err / tol).max())} of the tolerance"


# --- quantising ---------------------------------------------------------------


@pytest.mark.parametrize("K", [16, 48, 2048, 2064, 8192, 8208, 20000])
@pytest.mark.parametrize("dtype", [BF, FP, F32])
def test_quant(K, dtype):
    x = torch.randn(9, K, generator=_gen(K)).to(dtype)
    x[1] *= 100
    x[2] = 0
    x[3] = x[3] * 2.0 ** -14 if dtype == FP else x[3] * 1e-30
    x[4, 1:] = 0
    x[5] = torch.sign(x[5])
    codes, scale = kernels.quant_i8(x.to(DEV))
    want, s = quant(x)
    assert torch.equal(scale.cpu(), s)
    assert torch.equal(codes.cpu().double(), want)


@pytest.mark.parametrize("dtype", [BF, FP, F32])
def test_quant_next_to_borders(dtype):
    """Numbers around every half step of several scales, ties among them."""
    rows = []
    for big in (127.0, 254.0, 1.0, 0.3, 100.0, 2.0 ** -100 if dtype != FP else 2.0 ** -6, 3e4):
        b = torch.tensor(big).to(dtype).float()
        s = float(b) / 127
        n = torch.arange(-127, 127).double() + 0.5
        mid = (n * s).to(dtype).float()
        up, down = (torch.nextafter(mid.to(dtype), torch.full_like(mid, c).to(dtype)).float() for c in (1e4, -1e4))
        row = torch.cat((b[None], mid, up, down))
        rows.append(torch.nn.functional.pad(row.clamp(-float(b), float(b)), (0, 768 - len(row))))
    x = torch.stack(rows).to(dtype)
    codes, scale = kernels.quant_i8(x.to(DEV))
    want, s = quant(x)
    assert torch.equal(scale.cpu(), s) and torch.equal(codes.cpu().double(), want)


def test_quant_smallest_and_special_rows():
    x = torch.zeros(6, 64)
    x[0] = torch.arange(64) * 2.0 ** -149          # subnormal steps, or none at all
    x[1] = torch.arange(64) * 2.0 ** -140
    x[2] = torch.linspace(-1, 1, 64) * 3.4e38
    x[3, 7], x[4, 9], x[5, 3] = math.nan, math.inf, -math.inf
    x[3:, 1] = 5.0
    codes, scale = kernels.quant_i8(x.to(DEV))
    want, s = quant(x[:3])
    assert torch.equal(scale[:3].cpu(), s) and torch.equal(codes[:3].cpu().double(), want)
    assert torch.isnan(scale[3]) and torch.isinf(scale[4:]).all() and (codes[3:] == 0).all()
    w, t = _codes(1, 5, 64).to(DEV), _scales(1, 5).to(DEV)
    y = kernels.gemm_i8(x.to(DEV), w, t)
    assert torch.isnan(y[3:]).all() and torch.isfinite(y[:2]).all()


# --- products -----------------------------------------------------------------


@pytest.mark.parametrize("M", [1, 2, 15, 16, 17, 33, 64, 65, 67, 128, 129, 200, 257, 520])
@pytest.mark.parametrize("N,K", [(80, 512), (300, 208), (7, 16)])
def test_rows(M, N, K):
    a, w, s, t = _codes(M, M, K), _codes(M + 1, N, K), _scales(2, M), _scales(3, N)
    bias = torch.randn(N, generator=_gen(4))
    out = kernels.gemm_i8(a.to(DEV), w.to(DEV), t.to(DEV), s.to(DEV), bias.to(DEV), out_dtype=F32)
    _check(out, a, s, w, t, bias, what=f"M {M}")


@pytest.mark.parametrize("M,N,K", [(20, 300, 528), (20, 2050, 528), (67, 1000, 1040), (134, 1000, 528), (33, 4100, 1040),
                                   (20, 4100, 1040), (67, 8193, 2064), (67, 8193, 528), (400, 8193, 528), (200, 8193, 528),
                                   (4374, 1000, 2064), (1072, 8193, 528), (33, 70, 8208), (67, 2050, 8208), (134, 2050, 8176),
                                   (268, 1000, 4112), (268, 2050, 8208), (536, 1000, 2064), (67, 1000, 65536)])
def test_tile_shapes(M, N, K):
    """Of each shape of tile one product at least, ragged in rows, columns and inputs; sums equal those of whole numbers."""
    a, w = _codes(M, M, K), _codes(N, N, K)
    one = torch.ones(max(M, N), device=DEV)
    out = kernels.gemm_i8(a.to(DEV), w.to(DEV), one[:N], one[:M], out_dtype=F32)
    whole = torch.matmul(a.to(DEV).double(), w.to(DEV).double().t())   # exact: below 2^53
    assert torch.equal(out, whole.float())


@pytest.mark.parametrize("N", [1, 3, 15, 16, 17, 31, 33, 127, 128, 129, 257, 1031])
@pytest.mark.parametrize("K", [16, 64, 112, 128, 144, 256, 1152, 2064])
def test_columns_and_inputs(N, K):
    for M, od in ((5, BF), (100, FP)):
        a, w, s, t = _codes(N, M, K), _codes(K, N, K), _scales(2, M), _scales(3, N)
        out = kernels.gemm_i8(a.to(DEV), w.to(DEV), (0.01 * t).to(DEV), s.to(DEV), out_dtype=od)
        _check(out, a, s, w, 0.01 * t)


@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("act", [abi.SF_ACT_NONE, abi.SF_ACT_GELU_TANH, abi.SF_ACT_SILU])
def test_floats_and_activations(dtype, act):
    for M, N, K in ((3, 70, 160), (67, 260, 1152), (300, 513, 2048)):
        x = torch.randn(M, K, generator=_gen(M)).to(dtype)
        w, t, bias = _codes(5, N, K), _scales(3, N) * 0.01, torch.randn(N, generator=_gen(6)) * 0.1
        codes, s = quant(x)
        out = kernels.gemm_i8(x.to(DEV), w.to(DEV), t.to(DEV), bias=bias.to(DEV), act=act)
        assert out.dtype == dtype
        _check(out, codes, s, w, t, bias, act)


@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("M,K", [(1, 16), (1, 48), (1, 4096), (1, 8192), (1, 8208), (2, 4096), (3, 2064), (5, 1152), (8, 1024), (13, 624),
                                 (16, 512), (16, 528), (16, 16), (17, 480)])
def test_few_rows_quantised_on_the_way(M, K, dtype):
    """One launch or two, at the border between them; strided rows, zeros, and rows that are no numbers."""
    for N in (5, 16, 100, 8200):
        wide = torch.randn(M, K + 32, generator=_gen(M + K)).to(dtype)
        wide[M // 2] = 0 if M > 1 else wide[M // 2]
        x = wide[:, 16:16 + K]
        w, t = _codes(K, N, K), _scales(3, N) * 0.01
        out = kernels.gemm_i8(wide.to(DEV)[:, 16:16 + K], w.to(DEV), t.to(DEV), out_dtype=F32)
        codes, s = quant(x.contiguous())
        _check(out, codes, s, w, t, what=f"N {N}")
    x = x.clone()
    x[0, K // 2] = math.inf
    x[M - 1, 0] = math.nan
    out = kernels.gemm_i8(x.contiguous().to(DEV), w.to(DEV), t.to(DEV))
    assert torch.isnan(out[0]).all() and torch.isnan(out[M - 1]).all()
    if M > 2:
        _check(kernels.gemm_i8(x[1:-1].contiguous().to(DEV), w.to(DEV), t.to(DEV), out_dtype=F32), codes[1:-1], s[1:-1], w, t)


@pytest.mark.parametrize("M", [4, 90, 300])
def test_strides_accumulate_and_neighbours(M):
    """Views of wider rows, fp32 sums in place, and nothing written beside them."""
    N, K = 133, 272
    a_w, w_w, s, t = _codes(1, M, K + 48), _codes(2, N, K + 16), _scales(3, M), _scales(4, N)
    a, w = a_w.to(DEV)[:, 16:16 + K], w_w.to(DEV)[:, :K]
    for off in (0, 1, 4):
        c = torch.randn(M, N + 9, generator=_gen(5)).to(DEV)
        was = c.clone()
        kernels.gemm_i8(a, w, t.to(DEV), s.to(DEV), out=c[:, off:off + N], accumulate=True)
        _check(c[:, off:off + N], a.cpu(), s, w.cpu(), t, was=was[:, off:off + N].cpu())
        assert torch.equal(c[:, :off], was[:, :off]) and torch.equal(c[:, off + N:], was[:, off + N:])


@pytest.mark.parametrize("M,N", [(2, 33), (130, 300)])
def test_largest_sums(M, N):
    """65536 products of the largest codes: 2^30, exact."""
    K = 1 << 16
    a = torch.full((M, K), -128, dtype=torch.int8)
    w = torch.full((N, K), -128, dtype=torch.int8)
    w[1::2] = 127
    out = kernels.gemm_i8(a.to(DEV), w.to(DEV), torch.ones(N, device=DEV), torch.ones(M, device=DEV), out_dtype=F32)
    want = torch.where(torch.arange(N) % 2 == 0, 2.0 ** 30, -128.0 * 127 * K).expand(M, N)
    assert torch.equal(out.cpu().double(), want.double())


def test_many_tiles_are_each_computed_once():
    """More tiles than CUs, bands of columns that are not full, sums beyond one workgroup's share."""
    for M, N, K in ((2100, 2309, 256), (4374, 700, 128)):
        a, w, s, t = _codes(1, M, K), _codes(2, N, K), _scales(3, M), _scales(4, N)
        c = torch.zeros(M, N, device=DEV)
        kernels.gemm_i8(a.to(DEV), w.to(DEV), t.to(DEV), s.to(DEV), out=c, accumulate=True)
        _check(c, a, s, w, t, was=torch.zeros(M, N))


def test_runs_are_equal_and_rows_do_not_depend_on_others():
    M, N, K = 300, 520, 1024
    x, w, t = torch.randn(M, K, generator=_gen(1)).to(BF).to(DEV), _codes(2, N, K).to(DEV), _scales(3, N).to(DEV)
    y = kernels.gemm_i8(x, w, t)
    for _ in range(4):
        assert torch.equal(kernels.gemm_i8(x, w, t), y)
    for n in (1, 16, 40, 100):
        assert torch.equal(kernels.gemm_i8(x[:n], w, t), y[:n])
    ws = torch.empty(M * K + 16 + 4 * M, dtype=torch.uint8, device=DEV)
    assert torch.equal(kernels.gemm_i8(x, w, t, workspace=ws), y)
    codes, s = kernels.quant_i8(x)
    assert torch.equal(kernels.gemm_i8(codes, w, t, s), y)


def test_weights_beyond_32_bits():
    """4.3 GB of codes: the columns at the end."""
    N, K, M = (1 << 18) + 24, 1 << 14, 3
    w = torch.randint(-128, 128, (N, K), dtype=torch.int8, device=DEV)
    assert w.numel() > 1 << 32
    a, s, t = _codes(1, M, K), _scales(2, M), _scales(3, N)
    y = kernels.gemm_i8(a.to(DEV), w, t.to(DEV), s.to(DEV), out_dtype=F32)[:, -40:]
    _check(y, a, s, w[-40:].cpu(), t[-40:])


def test_no_rows_and_refusals():
    w, t = _codes(1, 8, 32).to(DEV), _scales(1, 8).to(DEV)
    assert kernels.gemm_i8(torch.zeros(0, 32, device=DEV), w, t).shape == (0, 8)
    codes, s = kernels.quant_i8(torch.zeros(0, 32, device=DEV))
    assert codes.shape == (0, 32) and s.shape == (0,)
    x = torch.zeros(2, 32, device=DEV)
    c = torch.zeros(2, 32, dtype=torch.int8, device=DEV)
    one = torch.ones(2, device=DEV)
    for args, kw in (((x, w, t, one), {}), ((c, w, t), {}), ((x[:, :16], w, t), {}), ((x, w, one), {}), ((x, w, None), {}),
                     ((x, w.float(), t), {}), ((x.double(), w, t), {}), ((x, w, t), {"bias": one}), ((x, w, t), {"accumulate": True}),
                     ((x, w, t), {"out": torch.zeros(2, 9, device=DEV)}),
                     ((x, w, t), {"workspace": torch.zeros(64, 2, device=DEV)[:, 0]})):
        with pytest.raises(ValueError):
            kernels.gemm_i8(*args, **kw)
    with pytest.raises(abi.SfError):
        kernels.gemm_i8(torch.zeros(40, 32, device=DEV), w, t, workspace=torch.empty(8, dtype=torch.uint8, device=DEV))
    with pytest.raises(abi.SfError):
        kernels.gemm_i8(x, w, t, out=torch.zeros(2, 8, dtype=BF, device=DEV), accumulate=True)
    with pytest.raises(abi.SfError):
        kernels.quant_i8(torch.zeros(2, 24, device=DEV))


@pytest.mark.parametrize("M", [3, 16, 40, 300])
@pytest.mark.parametrize("as_codes", [False, True])
def test_rows_of_the_largest_numbers(M, as_codes):
    """A row's sums times its scale have no fp32 value where the outputs have one; beside rows of 1 and of the smallest."""
    N, K = 130, 256
    x = torch.randn(M, K, generator=_gen(M))
    big = torch.tensor([1e36, 1.0, 3e38, 1e-36, 3e19, 5e18])[torch.arange(M) % 6]
    x = x / x.abs().amax(1, keepdim=True) * big[:, None]
    x[2, 1:] = 0.97 * x[2, 0].abs().clamp_min(1e38)   # sums of 2^22 and more
    w, t = _codes(K, N, K), _scales(3, N) * 1e-3
    w[3:7] = 127
    codes, s = quant(x)
    assert ((codes.abs() @ w.abs().double().t()).amax() * float(s.max())) > 3.4e38
    a = (kernels.quant_i8(x.to(DEV))) if as_codes else (x.to(DEV), None)
    out = kernels.gemm_i8(a[0], w.to(DEV), t.to(DEV), a[1], out_dtype=F32)
    y = (codes @ w.double().t()) * s.double()[:, None] * t.double()
    fits = y.abs() < 3.3e38
    assert fits.any(1).all()
    y, got = torch.where(fits, y, 0.0), torch.where(fits, out.cpu().double(), 0.0)
    assert torch.isfinite(got).all()
    assert ((got - y).abs() <= 5 * 2.0 ** -24 * y.abs() + 2.0 ** -149).all()


def test_a_sum_of_0_beside_large_scales():
    """A row of the largest step and a column of a large one: their zeros stay zeros, the bias stays."""
    M, N, K = 20, 40, 64
    x = torch.zeros(M, K)
    x[:, 0] = 3e38
    w = torch.zeros(N, K, dtype=torch.int8)
    w[:, 1:] = 5
    t, bias = torch.full((N,), 1e29), torch.arange(N).float()
    for rows in (3, M):
        out = kernels.gemm_i8(x[:rows].to(DEV), w.to(DEV), t.to(DEV), bias=bias.to(DEV), out_dtype=F32)
        assert torch.equal(out.cpu(), bias.expand(rows, N))
