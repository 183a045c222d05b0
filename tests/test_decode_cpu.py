"""Decode operators without a GPU: struct layouts, exports and the refusals that need no device."""

import ctypes as C
import os
import struct
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

FUNCTIONS = ("add_rmsnorm_fp8", "gemm_fp8", "append_kv", "paged_attention", "attention_workspace")
SYMBOLS = ("hv_decode_error", "hv_add_rmsnorm_fp8", "hv_gemm_fp8", "hv_append_kv", "hv_paged_attention",
           "hv_paged_attention_workspace")


@pytest.fixture(scope="module")
def library():
    from heatvit_b200 import build
    build.build()
    from heatvit_b200 import _lib
    return _lib.lib()


# hv_norm_args, hv_gemm_fp8_args, hv_append_args and hv_attention_args of the header
NORM, GEMM = struct.Struct("@6P7q2if"), struct.Struct("@5P10qi")
APPEND, ATTEND = struct.Struct("@10P16q12i"), struct.Struct("@8P14q8if")


def test_packed_structs_match_the_header(tmp_path):
    fields = {"hv_norm_args": ("rows", "scale_strides", "dim", "eps"),
              "hv_gemm_fp8_args": ("m", "a_scale_strides", "out_dtype"),
              "hv_append_args": ("d_positions", "q_strides", "rope_stride", "tokens", "rope_rows"),
              "hv_attention_args": ("workspace_bytes", "page_table_stride", "seqs", "scale")}
    terms = [f"sizeof({t})" for t in fields] + [f"offsetof({t}, {f})" for t, fs in fields.items() for f in fs]
    prog = tmp_path / "sz.c"
    prog.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "heatvit_b200.h"\nint main(){'
                    + "".join(f'printf("%zu ", {t});' for t in terms) + 'return 0;}\n')
    exe = tmp_path / "sz"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(prog), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True).stdout.split()]
    sizes = [-(-s.size // 8) * 8 for s in (NORM, GEMM, APPEND, ATTEND)]
    offsets = [struct.calcsize(f) for f in (
        "@6P", "@6P5q", "@6P7q", "@6P7q2i", "@5P", "@5P6q", "@5P10q", "@9P", "@10P", "@10P14q", "@10P16q", "@10P16q11i",
        "@8P", "@8P13q", "@8P14q", "@8P14q8i")]
    assert got == sizes + offsets


def test_every_symbol_has_a_signature(library):
    from heatvit_b200 import _lib
    for name in SYMBOLS:
        assert name in _lib._SIGNATURES and getattr(library, name)


def test_c_entries_refuse_before_they_touch_a_device(library):
    """Status codes of mistakes that are visible on the host."""
    from heatvit_b200 import abi

    def norm(rows=1, dim=64, dtype=0, eps=1e-6, x=16, res=0, out=0):
        return library.hv_add_rmsnorm_fp8(NORM.pack(x, res, 16, out, 16, 16, rows, *[64] * 6, dim, dtype, eps),
                                          None)
    assert norm(dtype=7) == abi.HV_ERR_TYPE
    assert norm(dim=0) == abi.HV_ERR_VALUE and norm(dim=32769) == abi.HV_ERR_VALUE
    assert norm(rows=-1) == abi.HV_ERR_VALUE and norm(x=0) == abi.HV_ERR_VALUE
    assert norm(eps=-1.0) == abi.HV_ERR_VALUE and norm(eps=float("nan")) == abi.HV_ERR_VALUE
    assert norm(res=16) == abi.HV_ERR_VALUE and b"together" in library.hv_last_error()
    assert norm(rows=0) == abi.HV_OK

    def gemm(m=1, n=1, k=16, a=16, lda=16, dtype=0):
        return library.hv_gemm_fp8(GEMM.pack(a, 16, 16, 16, 16, m, n, k, lda, 16, n, 1, 1, 1, 1, dtype), None)
    assert gemm(dtype=3) == abi.HV_ERR_TYPE
    assert gemm(k=0) == abi.HV_ERR_VALUE and gemm(m=-1) == abi.HV_ERR_VALUE and gemm(a=0) == abi.HV_ERR_VALUE
    assert gemm(m=1 << 31) == abi.HV_ERR_VALUE and gemm(k=1 << 31) == abi.HV_ERR_VALUE
    assert gemm(a=24) == abi.HV_ERR_VALUE and b"16 bytes" in library.hv_last_error()
    assert gemm(m=2, lda=24) == abi.HV_ERR_VALUE and gemm(m=2, k=32, lda=16) == abi.HV_ERR_VALUE
    assert gemm(m=0) == abi.HV_OK and gemm(n=0) == abi.HV_OK

    def append(tokens=1, heads=0, kv=1, dim=8, rot=0, dtype=0, pages=1, page=1, k=16):
        return library.hv_append_kv(APPEND.pack(0, k, 16, 0, 16, 16, 0, 16, 0, 16, *[8] * 16, tokens, heads, kv,
                                                        dim, rot, 0, dtype, pages, page, 1, 1, 0), None)
    assert append(dtype=2) == abi.HV_ERR_TYPE
    for bad in (dict(tokens=-1), dict(kv=0), dict(dim=0), dict(rot=3), dict(rot=16), dict(rot=2), dict(page=0),
                dict(heads=1), dict(k=0), dict(pages=-1)):
        assert append(**bad) == abi.HV_ERR_VALUE, bad
    assert append(tokens=0) == abi.HV_OK

    def attend(seqs=1, heads=1, kv=1, dim=64, dtype=0, pages=1, page=1, ws=256, wsb=0, stride=8, q=16):
        return library.hv_paged_attention(ATTEND.pack(q, 16, 0, 16, 16, 16, 16, ws, wsb, *[8] * 6,
                                                              *[stride] * 6, 1, seqs, heads, kv, dim, dtype, pages,
                                                              page, 1, 1.0), None)
    assert attend(dtype=2) == abi.HV_ERR_TYPE
    for bad in (dict(seqs=-1), dict(heads=3, kv=2), dict(kv=0), dict(dim=80), dict(page=0), dict(q=0)):
        assert attend(**bad) == abi.HV_ERR_VALUE, bad
    assert library.hv_paged_attention(None, None) == abi.HV_ERR_VALUE
    assert library.hv_append_kv(None, None) == abi.HV_ERR_VALUE
    assert library.hv_add_rmsnorm_fp8(None, None) == abi.HV_ERR_VALUE
    assert library.hv_gemm_fp8(None, None) == abi.HV_ERR_VALUE
    assert library.hv_decode_error(None) == abi.HV_ERR_VALUE
    assert library.hv_paged_attention_workspace(80, C.byref(C.c_int64())) == abi.HV_ERR_VALUE
    assert library.hv_paged_attention_workspace(64, None) == abi.HV_ERR_VALUE


def test_native_module_loads_and_refuses_wrong_arguments(library):
    """Without a device: it imports beside the installed torch, and what is no CUDA tensor is refused."""
    import importlib.util
    import torch
    from heatvit_b200 import build
    spec = importlib.util.spec_from_file_location("_decode_native", build.build_native())
    native = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(native)
    x, w = torch.zeros(2, 64), torch.zeros(64)
    for name in FUNCTIONS:
        with pytest.raises(TypeError, match="arguments"):
            getattr(native, name)()
    with pytest.raises(TypeError, match="x must be a torch.Tensor"):
        native.add_rmsnorm_fp8(None, w, 1e-6, None, None)
    with pytest.raises(ValueError, match="x must be a CUDA tensor"):
        native.add_rmsnorm_fp8(x, w, 1e-6, None, None)
    with pytest.raises(TypeError):
        native.add_rmsnorm_fp8(x, w, "small", None, None)
    with pytest.raises(ValueError, match="a must be a CUDA tensor"):
        native.gemm_fp8(x, w, x, w, None, None)
    with pytest.raises(ValueError, match="k must be a CUDA tensor"):
        native.append_kv(x, x, x, x, x, x, None, None, None, False, None)
    with pytest.raises(ValueError, match="q must be a CUDA tensor"):
        native.paged_attention(x, x, x, x, x, None, None, None, False)


def test_python_needs_a_device():
    import torch
    if torch.cuda.is_available():
        pytest.skip("a CUDA device is present")
    from heatvit_b200 import decode
    with pytest.raises(RuntimeError, match="CUDA"):
        decode.add_rmsnorm_fp8(torch.zeros(1, 8), torch.zeros(8))
