"""Chunk attention, the append with head norms, and sampling without a GPU: struct layouts and the refusals that need no device."""

import ctypes as C
import os
import struct
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# hv_norm_append_args, hv_chunk_args and hv_sample_args of the header
APPEND = "10P16q12i"
NORM_APPEND, CHUNK, SAMPLE = struct.Struct("@" + APPEND + "2Pf"), struct.Struct("@9P14q10if"), struct.Struct("@8Pq4i3f")


@pytest.fixture(scope="module")
def library():
    from heatvit_b200 import build
    build.build()
    from heatvit_b200 import _lib
    return _lib.lib()


def test_packed_structs_match_the_header(tmp_path):
    terms = ["sizeof(hv_norm_append_args)", "offsetof(hv_norm_append_args, d_q_weight)", "offsetof(hv_norm_append_args, eps)",
             "sizeof(hv_chunk_args)", "offsetof(hv_chunk_args, d_starts)", "offsetof(hv_chunk_args, workspace_bytes)",
             "offsetof(hv_chunk_args, page_table_stride)", "offsetof(hv_chunk_args, tokens)", "offsetof(hv_chunk_args, scale)",
             "sizeof(hv_sample_args)", "offsetof(hv_sample_args, d_logprobs)", "offsetof(hv_sample_args, rows)",
             "offsetof(hv_sample_args, top_k)", "offsetof(hv_sample_args, min_p)"]
    prog = tmp_path / "sz.c"
    prog.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "heatvit_b200.h"\nint main(){'
                    + "".join(f'printf("%zu ", {t});' for t in terms) + 'return 0;}\n')
    exe = tmp_path / "sz"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(prog), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True).stdout.split()]

    def size(f):
        return -(-struct.calcsize("@" + f) // 8) * 8
    at = struct.calcsize
    assert got == [size(APPEND + "2Pf"), at("@" + APPEND), at("@" + APPEND + "2P"),
                   size("9P14q10if"), at("@7P"), at("@9P"), at("@9P13q"), at("@9P14q"), at("@9P14q10i"),
                   size("8Pq4i3f"), at("@7P"), at("@8Pq"), at("@8Pq3i"), at("@8Pq4i2f")]


def test_c_entries_refuse_before_they_touch_a_device(library):
    from heatvit_b200 import abi
    VALUE, TYPE = abi.HV_ERR_VALUE, abi.HV_ERR_TYPE

    def append(tokens=1, heads=0, kv=1, dim=8, rot=0, dtype=0, pages=1, page=1, k=16, qw=0, kw=16, eps=1e-6):
        return library.hv_norm_append_kv(NORM_APPEND.pack(0, k, 16, 0, 16, 16, 0, 16, 0, 16, *[8] * 16, tokens, heads, kv, dim, rot, 0,
                                                          dtype, pages, page, 1, 1, 0, qw, kw, eps), None)
    assert append(dtype=2) == TYPE
    for bad in (dict(tokens=-1), dict(kv=0), dict(dim=0), dict(rot=3), dict(rot=2), dict(page=0), dict(heads=1), dict(k=0),
                dict(eps=-1.0), dict(eps=float("nan")), dict(qw=16)):
        assert append(**bad) == VALUE, bad
    assert append(tokens=0) == abi.HV_OK
    assert library.hv_norm_append_kv(None, None) == VALUE

    def chunk(tokens=1, seqs=1, heads=1, kv=1, dim=64, dtype=0, pages=1, page=1, q=16, starts=16, ws=256, wsb=0, stride=8):
        return library.hv_paged_chunk_attention(CHUNK.pack(q, 16, 0, 16, 16, 16, 16, starts, ws, wsb, *[8] * 6, *[stride] * 6, 1, tokens,
                                                           seqs, heads, kv, dim, dtype, 1, pages, page, 1, 1.0), None)
    assert chunk(dtype=2) == TYPE
    for bad in (dict(tokens=-1), dict(seqs=-1), dict(heads=3, kv=2), dict(kv=0), dict(heads=0), dict(dim=80), dict(page=0), dict(q=0),
                dict(starts=0), dict(pages=-1), dict(tokens=1 << 30, heads=4)):
        assert chunk(**bad) == VALUE, bad
    assert chunk(seqs=0) == abi.HV_OK and chunk(tokens=0) == abi.HV_OK
    assert library.hv_paged_chunk_attention(None, None) == VALUE
    assert library.hv_paged_chunk_attention_workspace(80, C.byref(C.c_int64())) == VALUE
    assert library.hv_paged_chunk_attention_workspace(64, None) == VALUE

    def sample(rows=1, vocab=10, dtype=0, z=16, u=16, out=16):
        return library.hv_sample_tokens(SAMPLE.pack(z, u, 0, 0, 0, 0, out, 0, 10, rows, vocab, dtype, 0, 1.0, 1.0, 0.0), None)
    assert sample(dtype=5) == TYPE
    for bad in (dict(rows=-1), dict(vocab=0), dict(vocab=(1 << 30) + 1), dict(z=0), dict(u=0), dict(out=0)):
        assert sample(**bad) == VALUE, bad
    assert sample(rows=0) == abi.HV_OK
    assert library.hv_sample_tokens(None, None) == VALUE


def test_symbols_have_signatures_and_bits_match_the_header(library):
    from heatvit_b200 import _lib, abi
    for name in ("hv_norm_append_kv", "hv_paged_chunk_attention", "hv_paged_chunk_attention_workspace", "hv_sample_tokens"):
        assert name in _lib._SIGNATURES and getattr(library, name)
    src = open(os.path.join(ROOT, "include", "heatvit_b200.h")).read()
    for name in ("HV_DECODE_BAD_LOGITS", "HV_DECODE_BAD_START"):
        assert f"#define {name} {getattr(abi, name)} " in src


def test_native_module_refuses_what_is_no_cuda_tensor(library):
    import importlib.util
    import torch
    from heatvit_b200 import build
    spec = importlib.util.spec_from_file_location("_decode_native", build.build_native())
    native = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(native)
    x = torch.zeros(2, 64)
    for name in ("norm_append_kv", "paged_chunk_attention", "sample_tokens", "chunk_attention_workspace"):
        with pytest.raises(TypeError, match="arguments"):
            getattr(native, name)()
    with pytest.raises(ValueError, match="k must be a CUDA tensor"):
        native.norm_append_kv(x, x, x, x, x, x, None, None, None, False, None, x, x, 1e-6)
    with pytest.raises(ValueError, match="q must be a CUDA tensor"):
        native.paged_chunk_attention(x, x, x, x, x, x, True, None, None, None, False)
    with pytest.raises(ValueError, match="logits must be a CUDA tensor"):
        native.sample_tokens(x, x, None, None, None, None, None, False)
    with pytest.raises(TypeError, match="logits must be a torch.Tensor"):
        native.sample_tokens(None, x, None, None, None, None, None, False)


@pytest.mark.parametrize("chunks,maker", [(False, "attention_workspace"), (True, "chunk_attention_workspace")])
def test_workspace_of_either_kind(monkeypatch, chunks, maker):
    import types
    import torch
    from heatvit_b200 import decode
    made = []
    cuda = types.SimpleNamespace(current_device=lambda: 3, current_stream=lambda device: types.SimpleNamespace(synchronize=lambda: None))
    monkeypatch.setattr(decode, "_torch", lambda: types.SimpleNamespace(cuda=cuda, device=torch.device))
    monkeypatch.setattr(decode, "_load", lambda: types.SimpleNamespace(**{maker: made.append}))
    assert decode.AttentionWorkspace(chunks=chunks).device == torch.device("cuda", 3) and made == [3]
