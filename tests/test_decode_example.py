"""examples/describe_images.py: every call that it makes of the operators, as they follow one
another, against the 64-bit forms and bounds of test_decode_gpu."""

import os
import subprocess
import sys

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
for p in (os.path.join(ROOT, "examples"), os.path.join(ROOT, "tests")):
    if p not in sys.path:
        sys.path.insert(0, p)

import test_decode_gpu as G  # noqa: E402


def checked(decode, monkeypatch, seen):
    """Each operator with its result checked on the inputs that it was given."""
    norm, gemm, append, attend = (decode.add_rmsnorm_fp8, decode.gemm_fp8, decode.append_kv, decode.paged_attention)

    def add_rmsnorm_fp8(x, weight, eps=1e-6, residual=None, residual_out=None):
        before = None if residual is None else residual.clone()
        r = norm(x, weight, eps, residual, residual_out)
        G.check_norm(r, x, weight, eps, before)
        assert residual_out is None or r.residual is residual_out
        seen.append("norm")
        return r

    def gemm_fp8(a, a_scale, b, b_scale):
        out = gemm(a, a_scale, b, b_scale)
        G.check_gemm(out, a, a_scale, b, b_scale)
        seen.append("gemm")
        return out

    def append_kv(k, v, k_cache, v_cache, page_table, positions, seq_ids=None, rope=None, q=None):
        want_k, want_v = k_cache.double(), v_cache.double()
        out = append(k, v, k_cache, v_cache, page_table, positions, seq_ids=seq_ids, rope=rope, q=q)
        ids = seq_ids.long() if seq_ids is not None else torch.arange(len(positions), device="cuda")
        page = k_cache.shape[1]
        at = positions.long()
        slot = page_table[ids, at // page].long(), at % page
        want_k[slot] = G.rotate64(k.double(), rope, at, rope.shape[1], False)
        want_v[slot] = v.double()
        size = float(k.abs().max()) * 2
        G.near(k_cache, want_k, size)
        assert torch.equal(v_cache.double(), want_v)
        if q is not None:
            G.near(out, G.rotate64(q.double(), rope, at, rope.shape[1], False), float(q.abs().max()) * 2)
        seen.append("append")
        return out

    def paged_attention(q, k_cache, v_cache, page_table, lens):
        out = attend(q, k_cache, v_cache, page_table, lens)
        want, _, bound = G.plain_attention(q, k_cache, v_cache, page_table, lens.tolist(), q.shape[2] ** -0.5)
        assert bool(((out.double() - want).abs() <= bound).all())
        seen.append("attend")
        return out

    for f in (add_rmsnorm_fp8, gemm_fp8, append_kv, paged_attention):
        monkeypatch.setattr(decode, f.__name__, f)


def test_describe_images_operator_by_operator(cuda, monkeypatch):
    import describe_images as E
    from heatvit_b200 import decode, synth
    images = torch.from_numpy(synth.baseline_images(synth.SEED, 5)).cuda()
    tokens, counts = E.encode(images)
    counts = counts.tolist()
    assert len(set(counts)) > 1 and sum(counts) == tokens.shape[0]
    seen = []
    checked(decode, monkeypatch, seen)
    d = E.Decoder(layers=2)
    d.start(tokens, counts, 4)
    ids = torch.arange(5, device="cuda") * 7
    for _ in range(3):
        logits = d.step(ids)
        assert logits.shape == (5, 1000) and bool(logits.isfinite().all())
        ids = logits.argmax(1)
    assert d.lens.tolist() == [n + 3 for n in counts]
    assert {k: seen.count(k) for k in ("norm", "gemm", "append", "attend")} == {
        "norm": 2 + 3 * (4 * 2 + 1), "gemm": 3 + 3 * (4 * 2 + 1), "append": 2 + 3 * 2, "attend": 3 * 2}
    assert decode.device_error() == 0


def test_describe_images_runs_from_the_command_line(cuda):
    out = subprocess.run([sys.executable, os.path.join(ROOT, "examples", "describe_images.py"), "--images", "3",
                          "--steps", "4"], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stderr
    assert out.stdout.count("tokens ->") == 3
