"""The 4-bit operators' refusals and layouts that need no GPU."""
import ctypes
import os
import shutil
import subprocess

import pytest
import torch

from servoflow_amd import abi, kernels
from servoflow_amd.attention import Kv4Cache, attention_kv4

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_ctypes_mirrors_match_the_c_layout(tmp_path):
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    mirrors = {"sf_w4_pack_desc": abi.W4PackDesc, "sf_gemm_w4_desc": abi.GemmW4Desc, "sf_kv4_cache": abi.Kv4CacheDesc,
               "sf_heads_rope_desc": abi.HeadsRopeDesc, "sf_attn_kv4_desc": abi.AttnKv4Desc}
    lines = ["#include <stdio.h>", '#include "sf_hip.h"', "int main(void) {"]
    for c, py in mirrors.items():
        lines.append(f'  printf("{c} size %zu\\n", sizeof({c}));')
        lines += [f'  printf("{c} {f} %zu\\n", offsetof({c}, {f}));' for f, *_ in py._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["  return 0;", "}"]) + "\n")
    subprocess.run([cc, "-std=c11", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = {}
    for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines():
        c, f, val = line.split()
        got[c, f] = int(val)
    for c, py in mirrors.items():
        assert got[c, "size"] == ctypes.sizeof(py), c
        for f, *_ in py._fields_:
            assert got[c, f] == getattr(py, f).offset, (c, f)


def test_sizes():
    L = abi.lib()
    # codes in blocks of 16 x 128 with a dword a group and row
    assert L.sf_w4_bytes(16, 128, 128) == 1024 + 64
    assert L.sf_w4_bytes(17, 160, 32) == 2 * (2 * 1024 + 8 * 64)
    assert L.sf_w4_bytes(1 << 20, 1 << 14, 64) == (1 << 16) * ((1 << 17) + (1 << 8) * 64)
    for bad in ((0, 128, 128), (16, 0, 128), (16, 128, 48), (16, 160, 128), (16, 16, 16), (-1, 128, 128)):
        assert L.sf_w4_bytes(*bad) == 0
    assert L.sf_kv4_bytes(2, 3, 33, 64) == 2 * 3 * 2 * 2304
    assert L.sf_kv4_bytes(1, 1, 1, 128) == 4608
    assert L.sf_kv4_bytes(64, 32, 1 << 20, 128) == 64 * 32 * (1 << 15) * 4608   # beyond 32 bits
    for bad in ((0, 1, 1, 64), (1, 0, 1, 64), (1, 1, 0, 64), (1, 1, 1, 96), (1, -1, 1, 64)):
        assert L.sf_kv4_bytes(*bad) == 0


def _pack(**kw):
    d = abi.W4PackDesc()
    d.N, d.K, d.group, d.codes, d.ldc, d.scales, d.lds, d.scale_dtype = 16, 256, 64, 256, 128, 256, 4, abi.SF_F16
    out = kw.pop("out", 256)
    for k, v in kw.items():
        setattr(d, k, v)
    return abi.lib().sf_w4_pack(ctypes.byref(d), out, None)


def test_w4_pack_refusals():
    assert abi.lib().sf_w4_pack(None, 256, None) == abi.SF_EINVAL
    for kw in ({"group": 48}, {"K": 200}, {"N": 0}, {"codes": None}, {"scales": None}, {"out": None}, {"out": 264},
               {"ldc": 127}, {"lds": 3}, {"scales": 257}, {"zeros": 256, "ldz": 3}):
        assert _pack(**kw) == abi.SF_EINVAL, kw
    assert _pack(scale_dtype=abi.SF_F32) == abi.SF_ENOTSUP


def _gemm(**kw):
    d = abi.GemmW4Desc()
    d.M, d.N, d.K, d.group, d.A, d.lda, d.a_dtype = 4, 16, 256, 64, 256, 256, abi.SF_BF16
    d.W, d.scale_dtype, d.C, d.ldc, d.c_dtype = 256, abi.SF_BF16, 256, 16, abi.SF_BF16
    for k, v in kw.items():
        setattr(d, k, v)
    return abi.lib().sf_gemm_w4(ctypes.byref(d), None)


def test_gemm_w4_refusals():
    assert abi.lib().sf_gemm_w4(None, None) == abi.SF_EINVAL
    for kw in ({"M": -1}, {"N": 0}, {"K": 32}, {"group": 16}, {"A": None}, {"W": None}, {"C": None}, {"A": 264},
               {"W": 264}, {"lda": 248}, {"lda": 260}, {"ldc": 15}, {"C": 257}, {"c_dtype": abi.SF_F32, "C": 258},
               {"bias": 258}):
        assert _gemm(**kw) == abi.SF_EINVAL, kw
    for kw in ({"a_dtype": abi.SF_F32}, {"scale_dtype": abi.SF_F32}, {"c_dtype": abi.SF_I8}, {"act": 3}, {"act": -1},
               {"accumulate": 1}, {"M": (1 << 31) - 1}):
        assert _gemm(**kw) == abi.SF_ENOTSUP, kw
    assert _gemm(M=0) == abi.SF_OK


def _rope(cache=None, **kw):
    d = abi.HeadsRopeDesc()
    d.B, d.S, d.D, d.in_dtype, d.out_dtype, d.rot, d.inv_freq = 2, 3, 64, abi.SF_BF16, abi.SF_BF16, 64, 256
    for j in range(3):
        d.heads[j], d.src[j], d.out[j] = 4, 256, 1 << 20
        d.src_stride[j][:] = d.out_stride[j][:] = (768, 64, 256)
    if cache:
        for f, v in zip(("data", "B", "H", "capacity", "D"), cache):
            setattr(d.cache, f, v)
    for k, v in kw.items():
        if isinstance(v, tuple):
            at = getattr(d, k)
            at[v[0]] = v[1] if not isinstance(v[1], tuple) else at[v[0]].__class__(*v[1])
        else:
            setattr(d, k, v)
    return abi.lib().sf_heads_rope(ctypes.byref(d), None)


def test_heads_rope_refusals():
    assert abi.lib().sf_heads_rope(None, None) == abi.SF_EINVAL
    for kw in ({"B": -1}, {"S": -1}, {"heads": (0, -1)}, {"rot": 8}, {"rot": 80}, {"rot": -16}, {"inv_freq": None},
               {"inv_freq": 260}, {"src": (1, None)}, {"src": (0, 264)}, {"out": (2, None)}, {"out": (1, 8)},
               {"src_stride": (0, (768, 64, 252))}, {"out_stride": (1, (-8, 64, 256))}, {"gamma": (1, 2)},
               {"slots": 256}):
        assert _rope(**kw) == abi.SF_EINVAL, kw
    for kw in ({"D": 96}, {"in_dtype": abi.SF_I8}, {"out_dtype": abi.SF_I32}):
        assert _rope(**kw) == abi.SF_ENOTSUP, kw
    assert _rope(S=0) == abi.SF_OK and _rope(B=0) == abi.SF_OK
    good = (256, 2, 4, 100, 64)
    for cache in ((264, 2, 4, 100, 64), (256, 1, 4, 100, 64), (256, 2, 5, 100, 64), (256, 2, 4, 0, 64),
                  (256, 2, 4, 100, 128)):
        assert _rope(cache) == abi.SF_EINVAL, cache
    assert _rope((256, 2, 4, 100, 32)) == abi.SF_ENOTSUP
    assert _rope(good, heads=(2, 3)) == abi.SF_EINVAL       # as many value heads as key heads
    assert _rope(good, S=0) == abi.SF_OK


def test_heads_rope_refuses_no_heads():
    d = abi.HeadsRopeDesc()
    d.B, d.S, d.D = 1, 1, 64
    assert abi.lib().sf_heads_rope(ctypes.byref(d), None) == abi.SF_EINVAL


def _read(cache=(256, 2, 4, 100, 64), S=3, k=256, v=256, st=(768, 192, 64), dt=abi.SF_F32, slots=None):
    c = abi.Kv4CacheDesc(*cache)
    s = (ctypes.c_int64 * 3)(*st) if st else None
    return abi.lib().sf_kv4_read(ctypes.byref(c), slots, S, k, s, v, s, dt, None)


def test_kv4_read_refusals():
    s = (ctypes.c_int64 * 3)(768, 192, 64)
    assert abi.lib().sf_kv4_read(None, None, 1, 256, s, 256, s, abi.SF_F32, None) == abi.SF_EINVAL
    for kw in ({"cache": (None, 2, 4, 100, 64)}, {"cache": (256, 0, 4, 100, 64)}, {"S": -1}, {"k": None}, {"v": 8},
               {"st": None}, {"st": (768, 192, 60)}, {"st": (768, -8, 64)}):
        assert _read(**kw) == abi.SF_EINVAL, kw
    for kw in ({"cache": (256, 2, 4, 100, 80)}, {"dt": abi.SF_I8}):
        assert _read(**kw) == abi.SF_ENOTSUP, kw
    assert _read(S=0) == abi.SF_OK


def _attn_desc(**kw):
    d = abi.AttnKv4Desc()
    d.B, d.Hq, d.Sq, d.Sk, d.in_dtype, d.out_dtype = 2, 8, 1, 100, abi.SF_BF16, abi.SF_BF16
    d.q_stride[:] = d.o_stride[:] = (512, 64, 64)
    d.cache = abi.Kv4CacheDesc(256, 2, 4, 100, 64)
    for k, v in kw.items():
        if k == "cache":
            d.cache = abi.Kv4CacheDesc(*v)
        elif isinstance(v, tuple):
            getattr(d, k)[v[0]] = v[1]
        else:
            setattr(d, k, v)
    return d


def _attn(q=256, out=256, ws=None, n=0, **kw):
    return abi.lib().sf_attn_kv4(ctypes.byref(_attn_desc(**kw)), q, out, ws, n, None)


def test_attn_kv4_refusals():
    assert abi.lib().sf_attn_kv4(None, 256, 256, None, 0, None) == abi.SF_EINVAL
    for kw in ({"B": 3}, {"B": -1}, {"Hq": 6}, {"Sq": -1}, {"Sk": 101}, {"Sk": -1}, {"num_splits": -1},
               {"num_splits": 65}, {"q": None}, {"out": None}, {"q": 264}, {"out": 264}, {"q_stride": (1, 60)},
               {"o_stride": (0, -8)}, {"cache": (None, 2, 4, 100, 64)}, {"cache": (264, 2, 4, 100, 64)},
               {"cache": (256, 2, 0, 100, 64)}, {"kv_mask": 256, "kv_mask_stride": -1}):
        assert _attn(**kw) == abi.SF_EINVAL, kw
    for kw in ({"cache": (256, 2, 4, 100, 32)}, {"in_dtype": abi.SF_F32}, {"out_dtype": abi.SF_I8}, {"scale": -1.0}):
        assert _attn(**kw) == abi.SF_ENOTSUP, kw
    assert _attn(num_splits=2) == abi.SF_EWORKSPACE
    need = abi.lib().sf_attn_kv4_workspace_bytes(ctypes.byref(_attn_desc(num_splits=2)))
    assert need == 2 * 2 * 8 * 66 * 4
    assert _attn(num_splits=2, ws=256, n=need - 1) == abi.SF_EWORKSPACE
    assert _attn(num_splits=2, ws=258, n=need) == abi.SF_EINVAL
    for kw in ({"Hq": 0}, {"Sq": 0}):
        assert _attn(**kw) == abi.SF_OK, kw


def test_sizes_beyond_a_launch_are_refused():
    for kw in ({"lda": (1 << 23) + 8}, {"N": (1 << 25) + 1, "ldc": 1 << 26}, {"M": (1 << 21) + 1}):
        assert _gemm(**kw) == abi.SF_ENOTSUP, kw
    assert _pack(N=1 << 25, K=2048, ldc=1024, lds=64, zeros=None) == abi.SF_ENOTSUP
    assert _rope(B=1 << 12, S=1 << 11) == abi.SF_ENOTSUP
    assert _read(S=1 << 22) == abi.SF_ENOTSUP
    big = (256, 2, 2, (1 << 30) + 1, 64)
    assert _attn(cache=big, Sk=(1 << 30) + 1) == abi.SF_ENOTSUP
    assert _attn(Sq=(1 << 28) + 1) == abi.SF_ENOTSUP                  # 4 heads to a key head
    many = (256, 1 << 22, 2, 100, 64)
    assert _attn(B=1 << 22, cache=many) == abi.SF_ENOTSUP


def test_front_ends_refuse_host_tensors_and_shapes():
    a = torch.zeros(2, 128, dtype=torch.bfloat16)
    codes, scales = torch.zeros(16, 64, dtype=torch.uint8), torch.zeros(16, 1, dtype=torch.float16)
    with pytest.raises(ValueError):
        kernels.w4_pack(codes, scales)
    with pytest.raises(ValueError):
        kernels.gemm_w4(a, kernels.W4(codes, 16, 128, 128, torch.float16))
    with pytest.raises(ValueError):
        kernels.heads_rope(a, 1, (1, 1, 0), 64)
    for bad in ((0, 1, 1, 64), (1, 1, 1, 80)):
        with pytest.raises(ValueError):
            Kv4Cache(*bad, device="cpu")
    c = Kv4Cache(1, 2, 5, 64, device="cpu")
    for q in (torch.zeros(1, 3, 1, 64), torch.zeros(2, 2, 1, 64), torch.zeros(1, 2, 1, 128), torch.zeros(1, 2, 64),
              torch.zeros(1, 2, 1, 64)):
        with pytest.raises(ValueError):
            attention_kv4(q, c)


def test_no_key_splits_that_the_merge_cannot_take():
    """The choice of splits knows the merge's limit of rows (it refused what it had chosen itself)."""
    L = abi.lib()
    for D in (64, 128):
        d = _attn_desc(B=1 << 16, Hq=256, Sk=4096, cache=(256, 1 << 16, 16, 4096, D))
        assert L.sf_attn_kv4_workspace_bytes(ctypes.byref(d)) == 0
    d = _attn_desc(B=1 << 14, Hq=64, Sk=4096, cache=(256, 1 << 14, 16, 4096, 64))   # few enough rows
    assert L.sf_attn_kv4_workspace_bytes(ctypes.byref(d)) == 2 * (1 << 20) * 66 * 4


def test_nan_is_honoured_where_it_is_promised():
    """The 4-bit operators' sources are not compiled under the assumption that no NaN is met."""
    make = shutil.which("make")
    if make is None:
        pytest.skip("no make")
    out = subprocess.run([make, "-n", "-B", "-C", os.path.join(ROOT, "servoflow_amd"), "lib/libsf_hip_kernels.so"],
                         check=True, capture_output=True, text=True).stdout
    for name in ("sf_heads_rope", "sf_kv4_attn", "sf_w4"):
        flags = next(line for line in out.splitlines() if f"-c csrc/{name}.hip" in line).split()
        assert flags.index("-fhonor-nans") > flags.index("-fno-honor-nans"), name
