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


def test_describe_images_with_prompt_attention(cuda, monkeypatch):
    """The prompt through every layer, norms of q and k, and sampling: the new calls checked as they follow one another."""
    import describe_images as E
    import test_chunk_attention_gpu as A
    import test_head_norms_gpu as H
    import test_sample_gpu as S
    from heatvit_b200 import decode, synth
    images = torch.from_numpy(synth.baseline_images(synth.SEED, 5)).cuda()
    tokens, counts = E.encode(images)
    counts = counts.tolist()
    seen = []
    append, chunk, attend = decode.append_kv, decode.paged_chunk_attention, decode.paged_attention

    def append_kv(k, v, k_cache, v_cache, page_table, positions, seq_ids=None, rope=None, q=None, q_weight=None, k_weight=None):
        want_k = k_cache.double()
        out = append(k, v, k_cache, v_cache, page_table, positions, seq_ids=seq_ids, rope=rope, q=q, q_weight=q_weight, k_weight=k_weight)
        ids = seq_ids.long() if seq_ids is not None else torch.arange(len(positions), device="cuda")
        at = positions.long()
        slot = page_table[ids, at // k_cache.shape[1]].long(), at % k_cache.shape[1]
        turned = [H.normed64(t, w, 1e-6) for t, w in ((k, k_weight), (q, q_weight))]
        size = [float(t.abs().max()) * 2 for t in turned]
        turned = [G.rotate64(t, rope, at, rope.shape[1], False) for t in turned]
        want_k[slot] = turned[0]
        H.near(k_cache, want_k, size[0])
        H.near(out, turned[1], size[1])
        assert torch.equal(v_cache[slot], v)
        seen.append("append")
        return out

    def paged_chunk_attention(q, k_cache, v_cache, page_table, lens, starts, causal=True):
        out = chunk(q, k_cache, v_cache, page_table, lens, starts, causal=causal)
        want, _, bound = A.plain(q, k_cache, v_cache, page_table, lens.tolist(), starts.tolist(), causal, q.shape[2] ** -0.5)
        assert bool(((out.double() - want).abs() <= bound).all())
        seen.append("chunk")
        return out

    def paged_attention(q, k_cache, v_cache, page_table, lens):
        out = attend(q, k_cache, v_cache, page_table, lens)
        want, _, bound = G.plain_attention(q, k_cache, v_cache, page_table, lens.tolist(), q.shape[2] ** -0.5)
        assert bool(((out.double() - want).abs() <= bound).all())
        seen.append("attend")
        return out

    for f in (append_kv, paged_chunk_attention, paged_attention):
        monkeypatch.setattr(decode, f.__name__, f)
    d = E.Decoder(layers=2, sees_prompt=True, head_norms=True)
    d.start(tokens, counts, 4)
    ids = torch.arange(5, device="cuda") * 7
    for i in range(3):
        logits = d.step(ids)
        ids = S.check(logits, S.uniform(i, 5), temperature=0.8, top_p=0.9, top_k=200)
    assert {k: seen.count(k) for k in ("append", "chunk", "attend")} == {"append": 2 + 3 * 2, "chunk": 2, "attend": 3 * 2}
    assert decode.device_error() == 0


def test_describe_images_options_from_the_command_line(cuda):
    out = subprocess.run([sys.executable, os.path.join(ROOT, "examples", "describe_images.py"), "--images", "3", "--steps", "4",
                          "--prompt-attention", "--temperature", "0.8", "--top-p", "0.9"], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stderr
    assert out.stdout.count("tokens ->") == 3


def test_prompt_in_chunks_and_a_sampled_step_in_a_graph(cuda):
    """A prompt appended and attended to in pieces gives what it gives whole; then a step of append, attention and
    sampling that a graph holds, replayed over growing sequences."""
    from heatvit_b200 import decode
    gen = torch.Generator(device="cuda").manual_seed(3)

    def rand(*shape, scale=1.0):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale).bfloat16()
    heads, kv, dim, page, n = 8, 2, 64, 16, 300
    rope, w = decode.rope_table(512, dim), (1 + rand(dim).float() * 0.2).bfloat16()
    table = torch.arange(2 * 20, dtype=torch.int32, device="cuda").view(2, 20)
    q, k, v = rand(2 * n, heads, dim), rand(2 * n, kv, dim), rand(2 * n, kv, dim)

    def run(pieces):
        kc, vc = (torch.zeros(40, page, kv, dim, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        got = torch.zeros_like(q)
        for a, b in pieces:
            rows = torch.cat([torch.arange(a, b), torch.arange(n + a, n + b)]).cuda()
            ids = torch.tensor([0] * (b - a) + [1] * (b - a), dtype=torch.int32, device="cuda")
            pos = torch.arange(a, b, dtype=torch.int32, device="cuda").repeat(2)
            turned = decode.append_kv(k[rows], v[rows], kc, vc, table, pos, seq_ids=ids, rope=rope, q=q[rows], q_weight=w, k_weight=w)
            ends = torch.tensor([b, b], dtype=torch.int32, device="cuda")
            starts = torch.tensor([0, b - a, 2 * (b - a)], dtype=torch.int32, device="cuda")
            got[rows] = decode.paged_chunk_attention(turned, kc, vc, table, ends, starts)
        return got, kc, vc
    whole, kc, vc = run([(0, n)])
    parts, kc2, vc2 = run([(0, 1), (1, 130), (130, 131), (131, n)])
    assert torch.equal(kc, kc2) and torch.equal(vc, vc2)
    # other cuts of the same sums: each within its rounding of weights and of the result (bf16: 2^-8 of |v| <= 5 or so)
    assert bool(((whole.float() - parts.float()).abs() <= 2.0 ** -6 + whole.float().abs() * 2.0 ** -6).all())

    head = rand(1000, heads * dim, scale=0.3)
    ws = decode.AttentionWorkspace(chunks=True)
    nq, nk, nv = rand(2, heads, dim), rand(2, kv, dim), rand(2, kv, dim)
    lens = torch.tensor([n, n], dtype=torch.int32, device="cuda")
    u = torch.rand(2, generator=gen, device="cuda")

    def step():
        pos = lens.clone()
        lens.add_(1)
        turned = decode.append_kv(nk, nv, kc, vc, table, pos, rope=rope, q=nq, q_weight=w, k_weight=w)
        out = decode.paged_attention(turned, kc, vc, table, lens, workspace=ws)
        logits = out.view(2, -1) @ head.t()
        return decode.sample_tokens(logits, u, temperature=0.9, top_k=100, top_p=0.95), logits
    before = lens.clone()
    eager = [step()[0].tolist() for _ in range(3)]
    lens.copy_(before)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ids, _ = step()
    lens.copy_(before)
    got = []
    for _ in range(3):
        g.replay()
        got.append(ids.tolist())
    assert got == eager
    assert decode.device_error() == 0
