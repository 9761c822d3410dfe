"""sf_w4_pack / sf_gemm_w4 against the product in 64 bits.

Tolerance, from the arithmetic: codes and activations multiply exactly, so an
output of fp32 is off by the accumulator's roundings alone.  A term passes at
most 32 additions inside one matrix instruction, 4 instructions of a group, 2
fused steps of the scale, K / 128 blocks, 8 waves and the bias, each 2^-24 of
what is summed, at most A = sum |a| |s| (31 + 16 + z); a 16-bit output adds
half a step of itself; GELU and SiLU have slopes below 1.2 and add at most
2^-20 of their argument by their own evaluation."""
import pytest
import torch

from servoflow_amd import abi, kernels

from _quant4 import half_step, w4_bytes, w4_random

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


def _case(M, N, K, group, dtype, zeros, seed=0):
    g = torch.Generator().manual_seed(seed + 1)
    codes, scales, z, w = w4_random(N, K, group, dtype, zeros, seed)
    a = torch.randn(M, K, generator=g).to(dtype)
    packed = kernels.w4_pack(w4_bytes(codes).to(DEV), scales.to(DEV), None if z is None else z.to(DEV), group=group)
    zz = 8.0 if z is None else z.double().repeat_interleave(group, 1)
    big = torch.matmul(a.double().abs(), ((47 + zz) * scales.double().repeat_interleave(group, 1)).t())
    return a, packed, w, big


def _depth(K):
    return 32 + 4 + 2 + (K + 127) // 128 + 8 + 2


def _check(got, ref, big, K, dtype, act=False, what=""):
    tol = 1.2 * _depth(K) * 2.0 ** -24 * big + (2.0 ** -20 * big if act else 0)
    tol = tol + (half_step(dtype) * (ref.abs() + tol) if dtype != F32 else 0) + 1e-30
    if dtype == FP:
        tol = tol + 2.0 ** -25
    err = (got.cpu().double() - ref).abs()
    assert torch.isfinite(got).all(), what
    worst = float((err / tol).max())
    assert worst <= 1, f"{what}: {worst} of the tolerance"


@pytest.mark.parametrize("M", [1, 2, 15, 16, 17, 33, 67, 80, 81, 161])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_rows(M, dtype):
    a, w, ref_w, big = _case(M, 80, 512, 128, dtype, True, M)
    out = kernels.gemm_w4(a.to(DEV), w, out_dtype=F32)
    _check(out, a.double() @ ref_w.t(), big, 512, F32, what=f"M {M}")


@pytest.mark.parametrize("N", [1, 3, 15, 16, 17, 33, 250, 1031])
@pytest.mark.parametrize("group,K", [(32, 32), (32, 96), (32, 1184), (64, 64), (64, 192), (128, 128), (128, 384),
                                     (128, 2176)])
def test_columns_and_groups(N, group, K):
    for zeros, dtype in ((False, BF), (True, FP)):
        a, w, ref_w, big = _case(5, N, K, group, dtype, zeros, N)
        out = kernels.gemm_w4(a.to(DEV), w, out_dtype=dtype)
        _check(out, a.double() @ ref_w.t(), big, K, dtype, what=f"N {N} K {K} group {group}")


@pytest.mark.parametrize("M,N", [(5, 4113), (20, 4113), (40, 4113), (90, 2100), (321, 3300)])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_many_columns(M, N, group):
    """More tiles of columns and rows than one shape of workgroup takes."""
    K, dtype = 384, BF if M & 1 else FP
    a, w, ref_w, big = _case(M, N, K, group, dtype, True, M)
    _check(kernels.gemm_w4(a.to(DEV), w, out_dtype=F32), a.double() @ ref_w.t(), big, K, F32, what=f"{M} x {N}")


@pytest.mark.parametrize("M,N", [(33, 8200), (45, 6100), (67, 6111), (150, 16500)])
@pytest.mark.parametrize("group,K", [(32, 32), (64, 64), (32, 96), (128, 128), (64, 192), (128, 640), (64, 1088),
                                     (32, 1184), (128, 2176)])
def test_tiles_of_rows(M, N, group, K):
    """Three to five tiles of rows, one or two column tiles to an activation block, fewer blocks than waves, a last
    block that is not full; rows that are not packed tightly, followed by NaN."""
    dtype = BF if K % 128 else FP
    a, w, ref_w, big = _case(M, N, K, group, dtype, True, M + K)
    wide = torch.full((M, K + 8), float("nan"), dtype=dtype, device=DEV)
    wide[:, :K] = a.to(DEV)
    _check(kernels.gemm_w4(wide[:, :K], w, out_dtype=F32), a.double() @ ref_w.t(), big, K, F32, what=f"{M} x {N} x {K}")


@pytest.mark.parametrize("M", [1, 67])
@pytest.mark.parametrize("out_dtype", [F32, BF, FP])
@pytest.mark.parametrize("act", [abi.SF_ACT_NONE, abi.SF_ACT_GELU_TANH, abi.SF_ACT_SILU])
def test_epilogue(M, out_dtype, act):
    K, N = 256, 48
    a, w, ref_w, big = _case(M, N, K, 64, BF, True, act)
    bias = torch.randn(N, generator=torch.Generator().manual_seed(9))
    y = a.double() @ ref_w.t() + bias.double()
    if act == abi.SF_ACT_GELU_TANH:
        y = 0.5 * y * (1 + torch.tanh(0.7978845608028654 * (y + 0.044715 * y ** 3)))
    elif act == abi.SF_ACT_SILU:
        y = y / (1 + torch.exp(-y))
    out = kernels.gemm_w4(a.to(DEV), w, bias.to(DEV), act=act, out_dtype=out_dtype)
    _check(out, y, big + bias.double().abs(), K, out_dtype, act != abi.SF_ACT_NONE)


def test_accumulate_and_strides():
    M, N, K = 19, 40, 384
    a, w, ref_w, big = _case(M, N, K, 128, FP, False)
    wide = torch.full((M, K + 24), float("nan"), dtype=FP, device=DEV)
    wide[:, 8:8 + K] = a.to(DEV)
    c = torch.randn(M, N + 3, generator=torch.Generator().manual_seed(3)).to(DEV)
    was = c.clone()
    out = kernels.gemm_w4(wide[:, 8:8 + K], w, out=c[:, 1:1 + N], accumulate=True)
    assert out.data_ptr() == c[:, 1:].data_ptr()
    _check(c[:, 1:1 + N], was[:, 1:1 + N].cpu().double() + a.double() @ ref_w.t(), big + was[:, 1:1 + N].cpu().double().abs(), K, F32)
    assert torch.equal(c[:, 0], was[:, 0]) and torch.equal(c[:, 1 + N:], was[:, 1 + N:])


@pytest.mark.parametrize("N", [48, 6150])
def test_rows_far_apart(N):
    """The widest row stride: a workgroup's rows span 1.3 GB."""
    M, K, ld = 83, 320, 1 << 23
    a, w, ref_w, big = _case(M, N, K, 64, BF, True, 7)
    wide = torch.empty(M, ld, dtype=BF, device=DEV)
    wide[:, K:K + 64] = float("nan")
    wide[:, :K] = a.to(DEV)
    _check(kernels.gemm_w4(wide[:, :K], w, out_dtype=F32), a.double() @ ref_w.t(), big, K, F32)


def test_rows_are_independent_of_a_bad_one():
    a, w, ref_w, big = _case(20, 32, 128, 32, BF, True)
    a[7, 5], a[18, 3] = float("nan"), float("inf")
    out = kernels.gemm_w4(a.to(DEV), w, out_dtype=F32)
    good = [i for i in range(20) if i not in (7, 18)]
    _check(out[good], a[good].double() @ ref_w.t(), big[good], 128, F32)
    assert not torch.isfinite(out[[7, 18]]).any()


def test_large_activations_and_small_scales():
    """fp16's largest activations against every code; scales in fp16's subnormals."""
    N, K = 16, 128
    codes = (torch.arange(K, dtype=torch.int64) % 16).to(torch.uint8).expand(N, K).contiguous()
    scales = torch.full((N, 1), 2.0 ** -24).to(FP)
    a = torch.full((3, K), 65504.0).to(FP)
    w = kernels.w4_pack(w4_bytes(codes).to(DEV), scales.to(DEV), group=128)
    ref = a.double() @ ((codes.double() - 8) * 2.0 ** -24).t()
    big = a.double().abs() @ torch.full((K, N), 55 * 2.0 ** -24, dtype=torch.float64)
    _check(kernels.gemm_w4(a.to(DEV), w, out_dtype=F32), ref, big, K, F32)


def test_strided_checkpoint():
    """Codes, scales and zeros as columns of wider matrices."""
    N, K, group = 21, 256, 64
    codes, scales, z, w = w4_random(N, K, group, BF, True, 4)
    wide = torch.zeros(N, K // 2 + 5, dtype=torch.uint8, device=DEV)
    wide[:, 3:3 + K // 2] = w4_bytes(codes).to(DEV)
    s2 = torch.zeros(N, 9, dtype=BF, device=DEV)
    s2[:, 2:6] = scales.to(DEV)
    z2 = torch.zeros(N, 7, dtype=torch.uint8, device=DEV)
    z2[:, 1:5] = z.to(DEV)
    one = kernels.w4_pack(wide[:, 3:3 + K // 2], s2[:, 2:6], z2[:, 1:5], group=group)
    two = kernels.w4_pack(w4_bytes(codes).to(DEV), scales.to(DEV), z.to(DEV), group=group)
    assert torch.equal(one.data, two.data)


def test_empty_rows():
    _, w, _, _ = _case(1, 16, 128, 128, BF, False)
    assert kernels.gemm_w4(torch.empty(0, 128, dtype=BF, device=DEV), w).shape == (0, 16)


@pytest.mark.parametrize("M,N", [(3, 48), (20, 4113), (67, 6111), (90, 8200)])
@pytest.mark.parametrize("group,K", [(32, 32), (32, 160), (64, 64)])
def test_largest_sums_in_a_last_block_that_is_not_full(M, N, group, K):
    """31 times a group's sum of |A| is just finite (2^127.96): nothing of it may be added up more than once."""
    codes, scales, z, w = w4_random(N, K, group, BF, True, 11)
    a = torch.zeros(M, K, dtype=BF)
    a[:, K - 1] = 2.0 ** 123
    ref = a.double() @ w.t()
    packed = kernels.w4_pack(w4_bytes(codes).to(DEV), scales.to(DEV), z.to(DEV), group=group)
    big = a.double() @ ((47 + z.double().repeat_interleave(group, 1)) * scales.double().repeat_interleave(group, 1)).t()
    _check(kernels.gemm_w4(a.to(DEV), packed, out_dtype=F32), ref, big, K, F32)
