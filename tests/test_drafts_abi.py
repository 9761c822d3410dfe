"""Layouts and refusals of the operators of a step that verifies drafted tokens, without a GPU."""
import ctypes
import os
import shutil
import subprocess

import pytest
import torch

from servoflow_amd import abi, kernels
from servoflow_amd.attention import DraftTree, Kv4Cache, accept_tree, attention_kv4, draft_tree

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_ctypes_mirrors_match_the_c_layout(tmp_path):
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    mirrors = {"sf_draft_tree": abi.DraftTreeDesc, "sf_sample_desc": abi.SampleDesc, "sf_gemm_i8_desc": abi.GemmI8Desc}
    lines = ["#include <stdio.h>", '#include "sf_hip.h"', "int main(void) {",
             '  printf("max %d %d\\n", SF_TREE_MAX_NODES, SF_SAMPLE_MAX_VOCAB);']
    for c, py in mirrors.items():
        lines.append(f'  printf("{c} size %zu\\n", sizeof({c}));')
        lines += [f'  printf("{c} {f} %zu\\n", offsetof({c}, {f}));' for f, *_ in py._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["  return 0;", "}"]) + "\n")
    subprocess.run([cc, "-std=c11", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines()
    assert out[0] == f"max {abi.SF_TREE_MAX_NODES} {abi.SF_SAMPLE_MAX_VOCAB}"
    got = {tuple(line.split()[:2]): int(line.split()[2]) for line in out[1:]}
    for c, py in mirrors.items():
        assert got[c, "size"] == ctypes.sizeof(py), c
        for f, *_ in py._fields_:
            assert got[c, f] == getattr(py, f).offset, (c, f)


def test_tree_refusals():
    L = abi.lib()
    build = lambda p=256, n=2, T=5, m=256, d=256: L.sf_tree_build(p, n, T, m, d, None)   # noqa: E731
    for kw in ({"p": None}, {"p": 258}, {"m": None}, {"d": 2}, {"T": 0}, {"T": -1}, {"n": -1}):
        assert build(**kw) == abi.SF_EINVAL, kw
    assert build(T=1025) == abi.SF_ENOTSUP and build(n=65536) == abi.SF_ENOTSUP
    assert build(n=0) == abi.SF_OK
    acc = lambda p=256, e=1, d=256, s=256, B=2, T=5, n=256, c=256, t=256: L.sf_tree_accept(p, e, d, s, B, T, n, c, t, None)   # noqa: E731
    for kw in ({"p": None}, {"d": None}, {"s": 257}, {"n": None}, {"c": None}, {"t": 6}, {"T": 0}, {"B": -1}):
        assert acc(**kw) == abi.SF_EINVAL, kw
    assert acc(T=1025) == abi.SF_ENOTSUP and acc(B=1 << 24) == abi.SF_ENOTSUP
    assert acc(B=0) == abi.SF_OK

    def keep(cache=(256, 2, 4, 100, 64), nodes=256, n=3, first=256):
        return L.sf_kv4_keep(ctypes.byref(abi.Kv4CacheDesc(*cache)), nodes, n, first, None)

    assert L.sf_kv4_keep(None, 256, 3, 256, None) == abi.SF_EINVAL
    for kw in ({"cache": (None, 2, 4, 100, 64)}, {"cache": (264, 2, 4, 100, 64)}, {"cache": (256, 0, 4, 100, 64)},
               {"cache": (256, 2, 4, 0, 64)}, {"nodes": None}, {"nodes": 258}, {"first": None}, {"n": -1}):
        assert keep(**kw) == abi.SF_EINVAL, kw
    for kw in ({"cache": (256, 2, 4, 100, 96)}, {"n": 1025}, {"cache": (256, 65536, 4, 100, 64)},
               {"cache": (256, 1 << 12, 1 << 11, 100, 64)}):
        assert keep(**kw) == abi.SF_ENOTSUP, kw
    assert keep(n=0) == abi.SF_OK


def _attn(tree=(256, 8, 0), no_tree=False, **kw):
    d = abi.AttnKv4Desc()
    d.B, d.Hq, d.Sq, d.Sk, d.in_dtype, d.out_dtype = 2, 8, 5, 100, abi.SF_BF16, abi.SF_BF16
    d.q_stride[:] = d.o_stride[:] = (512, 64, 64)
    d.cache = abi.Kv4CacheDesc(256, 2, 4, 100, 64)
    for k, v in kw.items():
        setattr(d, k, v)
    t = None if no_tree else ctypes.byref(abi.DraftTreeDesc(*tree))
    need = abi.lib().sf_attn_kv4_tree_workspace_bytes(ctypes.byref(d), t)
    return abi.lib().sf_attn_kv4_tree(ctypes.byref(d), t, 256, 256, None, 0, None), need


def test_attention_refusals():
    for kw in ({"no_tree": True}, {"tree": (None, 8, 0)}, {"tree": (258, 8, 0)}, {"tree": (256, 0, 0)}, {"tree": (256, 4, 0)},
               {"is_causal": 1}, {"Hq": 6}, {"Sk": 101}, {"num_splits": 65}):
        assert _attn(**kw)[0] == abi.SF_EINVAL, kw
    assert _attn(tree=(256, 1025, 0))[0] == abi.SF_ENOTSUP
    assert _attn(num_splits=2) == (abi.SF_EWORKSPACE, 2 * 2 * 8 * 5 * 66 * 4)
    assert _attn(Sq=0) == (abi.SF_OK, 0)


def _sample(ws=None, n=0, **kw):
    d = abi.SampleDesc()
    d.rows, d.V, d.logits, d.ld, d.dtype, d.u, d.token = 2, 100, 256, 100, abi.SF_BF16, 256, 256
    for k, v in kw.items():
        setattr(d, k, v)
    return abi.lib().sf_sample(ctypes.byref(d), ws, n, None)


def test_sample_refusals():
    assert abi.lib().sf_sample(None, None, 0, None) == abi.SF_EINVAL
    for kw in ({"rows": -1}, {"V": 0}, {"logits": None}, {"logits": 257}, {"dtype": abi.SF_F32, "logits": 258}, {"u": None},
               {"u": 2}, {"token": None}, {"token": 258}, {"ld": 99}, {"temperature": 2}, {"top_k": 1}, {"top_p": 258},
               {"min_p": 3}, {"logprob": 6}):
        assert _sample(**kw) == abi.SF_EINVAL, kw
    for kw in ({"dtype": abi.SF_I8}, {"V": (1 << 20) + 1, "ld": 1 << 21}, {"rows": 1 << 22}):
        assert _sample(**kw) == abi.SF_ENOTSUP, kw
    assert _sample(rows=0) == abi.SF_OK
    long = {"dtype": abi.SF_F32, "V": 40000, "ld": 40000}
    need = abi.lib().sf_sample_workspace_bytes(ctypes.byref(abi.SampleDesc(rows=2, V=40000, dtype=abi.SF_F32)))
    assert need == 2 * (2048 * 12 + 2 * 8 + 64 * 4)
    assert _sample(**long) == abi.SF_EWORKSPACE and _sample(ws=256, n=need - 1, **long) == abi.SF_EWORKSPACE
    assert _sample(ws=260, n=need, **long) == abi.SF_EINVAL
    for kw in ({"rows": 2, "V": 1000, "dtype": abi.SF_F32}, {"rows": 300, "V": 40000, "dtype": abi.SF_F32},
               {"rows": 2, "V": 40000, "dtype": abi.SF_F16}, {"rows": 0, "V": 40000}):
        assert abi.lib().sf_sample_workspace_bytes(ctypes.byref(abi.SampleDesc(**kw))) == 0


def _quant(x=256, ldx=64, dt=abi.SF_BF16, rows=2, cols=64, codes=256, ldc=64, scale=256):
    return abi.lib().sf_quant_i8(x, ldx, dt, rows, cols, codes, ldc, scale, None)


def _gemm(ws=None, n=0, **kw):
    d = abi.GemmI8Desc()
    d.M, d.N, d.K, d.A, d.lda, d.a_dtype, d.a_scale = 4, 16, 256, 256, 256, abi.SF_I8, 256
    d.W, d.ldw, d.w_scale, d.C, d.ldc, d.c_dtype = 256, 256, 256, 256, 16, abi.SF_BF16
    for k, v in kw.items():
        setattr(d, k, v)
    return abi.lib().sf_gemm_i8(ctypes.byref(d), ws, n, None), abi.lib().sf_gemm_i8_workspace_bytes(ctypes.byref(d))


def test_int8_refusals():
    for kw in ({"x": None}, {"x": 264}, {"codes": None}, {"codes": 260}, {"scale": None}, {"scale": 2}, {"rows": -1},
               {"cols": 0}, {"cols": 40}, {"ldx": 56}, {"ldx": 68}, {"ldc": 56}, {"ldc": 68}):
        assert _quant(**kw) == abi.SF_EINVAL, kw
    for kw in ({"dt": abi.SF_I8}, {"cols": (1 << 16) + 16}, {"rows": (1 << 22) + 1}):
        assert _quant(**kw) == abi.SF_ENOTSUP, kw
    assert _quant(rows=0) == abi.SF_OK
    assert abi.lib().sf_gemm_i8(None, None, 0, None) == abi.SF_EINVAL
    for kw in ({"M": -1}, {"N": 0}, {"K": 0}, {"K": 24}, {"A": None}, {"A": 264}, {"W": None}, {"W": 264}, {"C": None},
               {"C": 257}, {"a_scale": None}, {"a_scale": 2}, {"w_scale": None}, {"w_scale": 2}, {"bias": 2}, {"lda": 240},
               {"lda": 264}, {"ldw": 240}, {"ldw": 264}, {"ldc": 15}, {"a_dtype": abi.SF_F32, "lda": 258}):
        assert _gemm(**kw)[0] == abi.SF_EINVAL, kw
    for kw in ({"a_dtype": abi.SF_I32}, {"c_dtype": abi.SF_I8}, {"act": 3}, {"act": -1}, {"accumulate": 1},
               {"M": (1 << 22) + 1}, {"N": (1 << 25) + 1, "ldc": 1 << 26}, {"K": (1 << 16) + 16},
               {"lda": (1 << 22) + 16}, {"ldw": (1 << 22) + 16}, {"M": 1 << 20, "N": 1 << 20, "ldc": 1 << 20}):
        assert _gemm(**kw)[0] == abi.SF_ENOTSUP, kw
    assert _gemm(M=0)[0] == abi.SF_OK
    assert _gemm()[1] == 0
    need = 100 * 256 + 100 * 4
    assert _gemm(a_dtype=abi.SF_BF16, M=100) == (abi.SF_EWORKSPACE, need)
    assert _gemm(a_dtype=abi.SF_BF16, M=100, ws=256, n=need - 1)[0] == abi.SF_EWORKSPACE
    assert _gemm(a_dtype=abi.SF_BF16, M=100, ws=264, n=need)[0] == abi.SF_EINVAL
    for M, K, want in ((16, 512, 0), (1, 1 << 13, 0), (16, 528, 16 * 528 + 64), (17, 16, 17 * 16 + 68), (1, 8208, 8208 + 4)):
        d = abi.GemmI8Desc(M=M, N=8, K=K, a_dtype=abi.SF_F16)   # few inputs are quantised where they are multiplied
        assert abi.lib().sf_gemm_i8_workspace_bytes(ctypes.byref(d)) == want


def test_front_ends_refuse_host_tensors_and_shapes():
    p = torch.zeros(2, 5, dtype=torch.int32)
    for bad in (p, p.long(), p[None]):
        with pytest.raises(ValueError):
            draft_tree(bad)
    tree = DraftTree(p, p[..., None], p)
    with pytest.raises(ValueError):
        accept_tree(tree, p, p)
    with pytest.raises(ValueError):
        accept_tree(tree, p[:1].expand(3, 5), p)
    c = Kv4Cache(2, 2, 8, 64, device="cpu")
    with pytest.raises(ValueError):
        c.keep(p, p[:, 0])
    with pytest.raises(ValueError):
        attention_kv4(torch.zeros(2, 2, 5, 64, dtype=torch.bfloat16), c, tree=tree)
    with pytest.raises(ValueError):
        kernels.sample(torch.zeros(2, 8), torch.zeros(2))
    with pytest.raises(ValueError):
        kernels.quant_i8(torch.zeros(2, 16))
    with pytest.raises(ValueError):
        kernels.gemm_i8(torch.zeros(2, 16), torch.zeros(4, 16, dtype=torch.int8), torch.zeros(4))


def test_nan_is_honoured_where_it_is_promised():
    make = shutil.which("make")
    if make is None:
        pytest.skip("no make")
    out = subprocess.run([make, "-n", "-B", "-C", os.path.join(ROOT, "servoflow_amd"), "lib/libsf_hip_kernels.so"],
                         check=True, capture_output=True, text=True).stdout
    for name in ("sf_i8", "sf_sample"):
        flags = next(line for line in out.splitlines() if f"-c csrc/{name}.hip" in line).split()
        assert flags.index("-fhonor-nans") > flags.index("-fno-honor-nans"), name
