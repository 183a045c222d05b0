"""The cache append with a norm of each query and key head, on the GPU against a plain 64-bit form."""

import math
import os
import sys

import pytest

torch = pytest.importorskip("torch")

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))

from test_decode_gpu import BF, HF, U, clean, make_cache, make_table, rand, rotate64  # noqa: E402,F401

pytestmark = pytest.mark.gpu


def normed64(x, weight, eps):
    x = x.double()
    return x if weight is None else x * torch.rsqrt((x * x).mean(2, keepdim=True) + eps) * weight.double()


def near(got, want, size):
    """One rounding of what 32-bit steps give: a sum of dim squares (in a chain of 16 and a tree above it, halved by
    the root), the root, two products and a rotation, under 32 * 2^-24 of the largest normed value `size`."""
    bound = want.abs() * U[got.dtype] * (1 + 2.0 ** -10) + size * 2.0 ** -19 + 2.0 ** -25
    assert bool(((got.double() - want).abs() <= bound).all())


def run(dtype, layout, interleaved, heads, kv, dim, rot, page, q_norm=True, k_norm=True, eps=1e-6, off=0):
    from heatvit_b200 import decode
    past, new = [0, 3, 40, 17], [9, 1, 30, 0]
    lens = [p + n for p, n in zip(past, new)]
    table, pages = make_table(1, lens, page, spare=1)
    seq = torch.tensor(sum([[i] * n for i, n in enumerate(new)], []), dtype=torch.int32, device="cuda")
    pos = torch.tensor(sum([list(range(p, p + n)) for p, n in zip(past, new)], []), dtype=torch.int32, device="cuda")
    pos[4] = -1  # a padding token
    qkv = rand(2, pos.numel(), (heads + 2 * kv) * dim + off, dtype=dtype, scale=2.0)[:, off:]
    q = qkv[:, :heads * dim].view(-1, heads, dim)
    k = qkv[:, heads * dim:(heads + kv) * dim].view(-1, kv, dim)
    v = qkv[:, (heads + kv) * dim:].view(-1, kv, dim)
    qw, kw = ((1 + rand(s, dim, scale=0.3)).to(dtype) for s in (6, 7))
    qw, kw = qw if q_norm else None, kw if k_norm else None
    kc, vc = (make_cache(s, pages, page, kv, dim, dtype, layout) for s in (3, 4))
    want_k, want_v = kc.double(), vc.double()
    rope = decode.rope_table(80, rot) if rot else None
    q_out = decode.append_kv(k, v, kc, vc, table, pos, seq_ids=seq, rope=rope, q=q, interleaved=interleaved, q_weight=qw,
                             k_weight=kw, eps=eps)
    live = pos >= 0
    ids, at = seq[live].long(), pos[live].long()
    pg, slot = table[ids, at // page].long(), at % page
    turned = [normed64(k[live], kw, eps), normed64(q[live], qw, eps)]
    size = [float(t.abs().max()) * 2 for t in turned]
    if rot:
        turned = [rotate64(t, rope, at, rot, interleaved) for t in turned]
    want_k[pg, slot] = turned[0]
    want_v[pg, slot] = v[live].double()
    near(kc, want_k, size[0])
    assert torch.equal(vc.double(), want_v)
    untouched = torch.ones(pages, page, dtype=torch.bool, device="cuda")
    untouched[pg, slot] = False
    assert torch.equal(kc.double()[untouched], want_k[untouched])
    near(q_out[live], turned[1], size[1])
    assert bool((q_out[4] == 0).all())


@pytest.mark.parametrize("dtype,layout", [(BF, "nhd"), (HF, "hnd")])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("heads,kv,dim,rot,page", [(4, 2, 64, 64, 16), (6, 3, 64, 32, 5), (8, 1, 128, 128, 1), (3, 3, 96, 96, 16),
                                                   (2, 2, 40, 24, 7), (3, 3, 63, 62, 16), (2, 1, 33, 10, 16), (4, 4, 96, 0, 16),
                                                   (5, 1, 192, 64, 16), (2, 2, 256, 256, 16), (2, 1, 320, 320, 16),
                                                   (1, 1, 8, 0, 16), (3, 1, 16, 16, 4), (1, 1, 1, 0, 2)])
def test_norm_append(dtype, layout, interleaved, heads, kv, dim, rot, page):
    run(dtype, layout, interleaved, heads, kv, dim, rot, page)


@pytest.mark.parametrize("q_norm,k_norm", [(True, False), (False, True)])
@pytest.mark.parametrize("dim,rot", [(64, 64), (63, 30)])
def test_norm_of_one_alone(q_norm, k_norm, dim, rot):
    run(BF, "nhd", False, 4, 2, dim, rot, 16, q_norm, k_norm, eps=0.1)


def test_norm_append_off_16_bytes():
    run(HF, "nhd", False, 4, 2, 64, 64, 16, off=3)
    run(BF, "nhd", True, 4, 2, 64, 64, 16, off=1)


@pytest.mark.parametrize("interleaved,rot", [(False, 128), (True, 64)])
@pytest.mark.parametrize("heads,kv", [(31, 1), (8, 8)])
def test_norm_append_many_tokens(heads, kv, interleaved, rot):
    from heatvit_b200 import decode
    lens, dim, page = [3000, 1, 2049], 128, 64
    table, pages = make_table(1, lens, page)
    seq = torch.tensor(sum([[i] * n for i, n in enumerate(lens)], []), dtype=torch.int32, device="cuda")
    pos = torch.cat([torch.arange(n, dtype=torch.int32) for n in lens]).cuda()
    q, k, v = (rand(s, pos.numel(), n, dim, dtype=BF) for s, n in ((2, heads), (3, kv), (4, kv)))
    qw, kw = ((1 + rand(s, dim, scale=0.3)).to(BF) for s in (8, 9))
    kc, vc = (make_cache(s, pages, page, kv, dim, BF, "hnd") for s in (5, 6))
    rope = decode.rope_table(3000, rot)
    got = decode.append_kv(k, v, kc, vc, table, pos, seq_ids=seq, rope=rope, q=q, interleaved=interleaved, q_weight=qw, k_weight=kw)
    pg, slot = table[seq.long(), pos.long() // page].long(), pos.long() % page
    want_k, want_q = (rotate64(normed64(x, w, 1e-6), rope, pos.long(), rot, interleaved) for x, w in ((k, kw), (q, qw)))
    near(kc[pg, slot], want_k, 16.0)
    near(got, want_q, 16.0)
    assert torch.equal(vc[pg, slot], v)


@pytest.mark.parametrize("dtype,interleaved,rot", [(BF, False, 128), (HF, True, 64)])
@pytest.mark.parametrize("heads,kv", [(31, 1), (8, 3)])
@pytest.mark.parametrize("tokens", [700, 1400, 6000])
def test_norm_append_is_the_same_whatever_comes_with_it(tokens, heads, kv, dtype, interleaved, rot):
    """A token's bits do not depend on how many heads a thread takes: calls of few, of some and of many tokens."""
    from heatvit_b200 import decode
    dim, page = 128, 64
    table, pages = make_table(1, [tokens], page)
    pos = torch.arange(tokens, dtype=torch.int32, device="cuda")
    seq = torch.zeros_like(pos)
    q, k, v = (rand(s, tokens, n, dim, dtype=dtype) for s, n in ((2, heads), (3, kv), (4, kv)))
    qw, kw = ((1 + rand(s, dim, scale=0.3)).to(dtype) for s in (8, 9))
    rope = decode.rope_table(tokens, rot)
    results = []
    for step in (tokens, 64):
        kc, vc = (make_cache(s, pages, page, kv, dim, dtype, "nhd") for s in (5, 6))
        parts = [decode.append_kv(k[i:i + step], v[i:i + step], kc, vc, table, pos[i:i + step], seq_ids=seq[i:i + step], rope=rope,
                                  q=q[i:i + step], interleaved=interleaved, q_weight=qw, k_weight=kw) for i in range(0, tokens, step)]
        results.append((torch.cat(parts), kc, vc))
    for whole, pieces in zip(*results):
        assert torch.equal(whole, pieces)
    near(results[0][0], rotate64(normed64(q, qw, 1e-6), rope, pos.long(), rot, interleaved), 16.0)


@pytest.mark.parametrize("dim", [64, 36])
def test_norm_append_in_place_without_q_and_extreme_heads(dim):
    """q_out = q; no q; heads of zeros, of the type's largest values, and with a NaN, which stays its head's."""
    from heatvit_b200 import decode
    lens = [5, 1, 33]
    table, pages = make_table(1, lens, 16)
    pos = torch.tensor([n - 1 for n in lens], dtype=torch.int32, device="cuda")
    k, v, q = (rand(s, 3, 2, dim, dtype=BF) for s in (1, 2, 3))
    w = (1 + rand(4, dim, scale=0.3)).to(BF)
    rope = decode.rope_table(64, dim)
    kc, vc, kc2, vc2 = (make_cache(5, pages, 16, 2, dim, BF, "nhd") for _ in range(4))
    got = decode.append_kv(k, v, kc, vc, table, pos, rope=rope, q=q, q_weight=w, k_weight=w)
    same = q.clone()
    assert decode.append_kv(k, v, kc2, vc2, table, pos, rope=rope, q=same, q_out=same, q_weight=w, k_weight=w) is same
    assert torch.equal(same, got) and torch.equal(kc, kc2)
    kc2.zero_()
    assert decode.append_kv(k, v, kc2, vc2, table, pos, rope=rope, k_weight=w) is None
    at = table[torch.arange(3), pos.long() // 16].long(), pos.long() % 16
    assert torch.equal(kc2[at], kc[at])
    q[0, 0], q[1, 1, 7], q[2, 0] = 0, math.nan, 1e30
    out = decode.append_kv(k, v, kc, vc, table, pos, rope=rope, q=q, q_weight=w, k_weight=w)
    assert bool((out[0, 0] == 0).all()) and bool(out[1, 1].isnan().all())
    # squares past 32 bits: the mean is infinite there, as in the plain form in 32 bits
    assert bool((out[2, 0] == 0).all())
    for i, h in ((0, 1), (1, 0), (2, 1)):
        assert torch.equal(out[i, h], got[i, h])


def test_norm_append_reports_what_only_the_device_sees():
    from heatvit_b200 import abi, decode
    i32 = dict(dtype=torch.int32, device="cuda")
    position, page = abi.HV_DECODE_BAD_POSITION, abi.HV_DECODE_BAD_PAGE
    for dim in (64, 36):
        k, v = (rand(s, 1, 1, dim, dtype=BF) for s in (1, 2))
        w = torch.ones(dim, dtype=BF, device="cuda")
        kc, vc = (make_cache(s, 2, 4, 1, dim, BF, "nhd") for s in (5, 6))
        before = kc.clone(), vc.clone()
        rope = decode.rope_table(3, dim)
        for table, pos, seq, bit in (([[0, 1]], 8, 0, position), ([[0, 1]], 3, 0, position), ([[0, 1]], 0, 1, position),
                                     ([[0, 1]], 0, -1, position), ([[2, 1]], 0, 0, page), ([[-1, 1]], 0, 0, page)):
            decode.append_kv(k, v, kc, vc, torch.tensor(table, **i32), torch.tensor([pos], **i32),
                             seq_ids=torch.tensor([seq], **i32), rope=rope, k_weight=w)
            assert decode.device_error() == bit
            assert torch.equal(kc, before[0]) and torch.equal(vc, before[1])


def test_norm_append_in_a_graph():
    from heatvit_b200 import decode
    lens = [5, 1, 33]
    table, pages = make_table(1, lens, 16)
    pos = torch.tensor([n - 1 for n in lens], dtype=torch.int32, device="cuda")
    k, v, q = (rand(s, 3, 2, 128, dtype=BF) for s in (1, 2, 3))
    w = (1 + rand(4, 128, scale=0.3)).to(BF)
    rope = decode.rope_table(64, 128)
    kc, vc = (make_cache(5, pages, 16, 2, 128, BF, "nhd") for _ in range(2))
    decode.append_kv(k, v, kc, vc, table, pos, rope=rope, q=q, q_weight=w, k_weight=w)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = decode.append_kv(k, v, kc, vc, table, pos, rope=rope, q=q, q_weight=w, k_weight=w)
    q.copy_(rand(8, 3, 2, 128))
    pos -= 1
    pos.clamp_(min=0)
    g.replay()
    near(out, rotate64(normed64(q, w, 1e-6), rope, pos.long(), 128, False), 16.0)


def test_norm_append_refusals():
    from heatvit_b200 import decode
    table, pages = make_table(1, [5, 1], 16)
    pos = torch.zeros(2, dtype=torch.int32, device="cuda")
    k, v, q = (rand(s, 2, 2, 64, dtype=BF) for s in (1, 2, 3))
    kc, vc = (make_cache(5, pages, 16, 2, 64, BF, "nhd") for _ in range(2))
    w = torch.ones(64, dtype=BF, device="cuda")

    def bad(kind, match, **kw):
        with pytest.raises(kind, match=match):
            decode.append_kv(k, v, kc, vc, table, pos, **kw)
    bad(ValueError, "without q", q_weight=w)
    bad(ValueError, "channels", q=q, q_weight=w[:63])
    bad(ValueError, "channels", k_weight=torch.ones(65, dtype=BF, device="cuda"))
    bad(TypeError, "k's type", k_weight=w.float())
    bad(ValueError, "live on", k_weight=w.cpu())
    bad(ValueError, "1-dimensional", k_weight=w[None])
    bad(ValueError, "eps", k_weight=w, eps=-1e-6)
    bad(ValueError, "eps", k_weight=w, eps=math.nan)
    bad(TypeError, None, k_weight=w, eps="small")
    bad(TypeError, "Tensor", k_weight=1.0)
