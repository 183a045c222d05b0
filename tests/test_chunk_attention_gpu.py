"""Attention of a chunk of new tokens over a paged cache on the GPU, against a plain 64-bit form."""

import math
import os
import sys

import pytest

torch = pytest.importorskip("torch")

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))

import test_decode_gpu as G  # noqa: E402
from test_decode_gpu import BF, HF, U, clean, make_cache, make_table, rand  # noqa: E402,F401

pytestmark = pytest.mark.gpu


def plain(q, kc, vc, table, lens, starts, causal, scale):
    """Outputs, log-sum-exps and the error bound, in 64 bits; NaN in rows of no sequence."""
    t, h, d = q.shape
    page, kv = kc.shape[1:3]
    out = torch.full((t, h, d), math.nan, dtype=torch.float64, device="cuda")
    bound = torch.zeros_like(out)
    lse = torch.full((t, h), math.nan, dtype=torch.float64, device="cuda")
    for i, n in enumerate(lens):
        rows = slice(starts[i], starts[i + 1])
        m = starts[i + 1] - starts[i]
        if m == 0:
            continue
        out[rows], lse[rows] = 0, -math.inf
        if n <= 0:
            continue
        pg = table[i, :-(-n // page)].long()
        k, v = (c[pg].reshape(-1, kv, d)[:n].double().repeat_interleave(h // kv, 1) for c in (kc, vc))
        x = q[rows].double()
        s = torch.einsum("mhd,nhd->mhn", x, k) * scale
        size = torch.einsum("mhd,nhd->mhn", x.abs(), k.abs()) * abs(scale)
        seen = torch.full((m,), n, device="cuda")
        if causal:
            seen = (n - m + 1 + torch.arange(m, device="cuda")).clamp(min=0)
        hidden = torch.arange(n, device="cuda")[None, :] >= seen[:, None]
        s = s.masked_fill(hidden[:, None], -math.inf)
        size = size.masked_fill(hidden[:, None], 0.0)
        some = seen > 0
        p = torch.softmax(s[some], 2)
        # what a row does not see is no part of its sum, whatever its value
        vz = v.nan_to_num(0.0, 0.0, 0.0)
        o = torch.einsum("mhn,nhd->mhd", p, vz)
        out[rows][some] = o
        lse[rows][some] = torch.logsumexp(s[some], 2)
        # The scores' 32-bit error is at most 2^-20 of the sum of absolute products, and moves a weight by that; the
        # exponential is within 2^-20.  A weight is rounded to q's type and the sum is that of the rounded ones: U of
        # the sum of absolute terms, and U of the result.  fp16 weights stand beside a reference of 2^9 at least and have
        # steps of 2^-24: 2^-34 of the largest for each token.  Then one rounding of the result.
        shift = size[some].amax(2, keepdim=True) * 2.0 ** -20
        terms = torch.einsum("mhn,nhd->mhd", p, vz.abs())
        bound[rows][some] = (terms + o.abs()) * (U[q.dtype] + 2 * shift + 2.0 ** -16) + o.abs() * U[q.dtype] + 2.0 ** -24
        if q.dtype == HF:
            bound[rows][some] += p.amax(2, keepdim=True) * 2.0 ** -34 * (vz.abs().sum(0)[None] + n * o.abs())
    return out, lse, bound


def chunk_case(seed, new, past, heads, kv, dim, page, dtype, layout="nhd", spare=0, rest=0, poison=True):
    """q (with `rest` rows behind the last sequence), caches, page table, lengths and starts."""
    lens = [a + b for a, b in zip(new, past)]
    table, pages = make_table(seed, [max(n, 0) for n in lens], page, spare)
    kc, vc = (make_cache(seed + s, pages + 1, page, kv, dim, dtype, layout) for s in (1, 2))
    if poison:  # what no sequence owns, and the slots past each length, must not be read into the result
        live = torch.zeros(pages + 1, page, dtype=torch.bool, device="cuda")
        for i, n in enumerate(lens):
            if n > 0:
                t = torch.arange(n, device="cuda")
                live[table[i, t // page].long(), t % page] = True
        kc[~live] = math.nan
        vc[~live] = math.inf
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    q = rand(seed + 3, starts[-1] + rest, heads, dim, dtype=dtype, scale=1.5)
    return q, kc, vc, table, lens, starts


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def check(q, kc, vc, table, lens, starts, causal=True, scale=None, **kw):
    from heatvit_b200 import decode
    out, lse = decode.paged_chunk_attention(q, kc, vc, table, ints(lens), ints(starts), causal=causal, scale=scale,
                                            return_lse=True, **kw)
    want, want_lse, bound = plain(q, kc, vc, table, lens, starts, causal, q.shape[2] ** -0.5 if scale is None else scale)
    some = ~want_lse.isnan()
    off = (out.double() - want).abs()[some]
    assert bool((off <= bound[some]).all()), float((off / bound[some]).nan_to_num(9e9).max())
    none = want_lse == -math.inf
    assert bool((lse[none] == -math.inf).all()) and bool((out[none] == 0).all())
    near = some & ~none
    # the sum of the rounded weights is within U of the sum
    assert bool(((lse.double() - want_lse).abs()[near] <= U[q.dtype] + 2.0 ** -12 + want_lse.abs()[near] * 2.0 ** -20).all())
    return out, lse


@pytest.mark.parametrize("dim", [32, 64, 96, 128, 192, 256])
@pytest.mark.parametrize("dtype,layout,page", [(BF, "nhd", 16), (HF, "hnd", 64), (BF, "hnd", 24), (HF, "nhd", 1), (BF, "nhd", 256)])
@pytest.mark.parametrize("causal", [True, False])
def test_chunk_dims_and_pages(dim, dtype, layout, page, causal):
    check(*chunk_case(1, [5, 0, 130, 1, 300], [7, 9, 0, 200, 261], 4, 2, dim, page, dtype, layout), causal=causal)


@pytest.mark.parametrize("heads,kv", [(1, 1), (3, 3), (8, 1), (6, 2), (5, 1), (12, 4), (48, 2), (7, 7), (130, 1), (300, 1)])
def test_chunk_head_layouts(heads, kv):
    check(*chunk_case(2, [33, 1, 90], [100, 260, 0], heads, kv, 64, 16, BF))


@pytest.mark.parametrize("new,past", [([1], [0]), ([1], [126]), ([127], [0]), ([128], [0]), ([129], [0]), ([2], [127]), ([1000], [0]),
                                      ([1], [5000]), ([3], [20000]), ([257], [4000]), ([1] * 40, list(range(0, 400, 10))),
                                      ([0, 0, 3, 0], [0, 50, 0, 0]), ([2000, 1], [0, 3000]), ([17, 600, 5, 1], [900, 1, 4000, 0])])
@pytest.mark.parametrize("dim,dtype", [(64, HF), (128, BF), (256, BF)])
def test_chunk_lengths(new, past, dim, dtype):
    check(*chunk_case(3, new, past, 4, 2, dim, 16, dtype))
    check(*chunk_case(4, new, past, 3, 3, dim, 16, dtype), causal=False)


def test_chunk_many_items():
    """More items than resident blocks, of every length."""
    check(*chunk_case(5, [(i * 37) % 200 for i in range(60)], [(i * 91) % 500 for i in range(60)], 16, 8, 64, 32, BF))


def test_chunk_rows_that_see_nothing():
    """A sequence shorter than what it brings (its first rows stand before its first token), or of no length."""
    q, kc, vc, table, lens, starts = chunk_case(6, [40, 10, 5], [0, 0, 8], 4, 2, 128, 16, BF)
    lens = [25, 0, 13]
    check(q, kc, vc, table, lens, starts)
    check(q, kc, vc, table, lens, starts, causal=False)
    check(q, kc, vc, table, [25, -3, 13], starts)


@pytest.mark.parametrize("rest", [1, 200])
def test_chunk_rows_of_no_sequence_stay(rest):
    q, kc, vc, table, lens, starts = chunk_case(7, [30, 131], [10, 0], 4, 2, 64, 16, BF, rest=rest)
    out = torch.full_like(q, 7.0)
    check(q, kc, vc, table, lens, starts, out=out)
    assert bool((out[starts[-1]:] == 7).all())
    # and ahead of the first
    out.fill_(7.0)
    got, _ = check(q, kc, vc, table[1:], lens[1:], starts[1:], out=out)
    assert got is out and bool((out[:starts[1]] == 7).all()) and bool((out[starts[-1]:] == 7).all())


def test_chunk_strided_q_and_out():
    """q as a slice of a projection's output (rows off 16 bytes as well), out with strides of its own."""
    for pad, dtype in ((0, BF), (8, HF), (1, BF), (3, HF)):
        q, kc, vc, table, lens, starts = chunk_case(8, [70, 3, 150], [5, 300, 0], 4, 2, 64, 16, dtype)
        wide = torch.zeros(q.shape[0], 4 * 64 + 100 + pad, dtype=dtype, device="cuda")
        view = wide[:, pad:pad + 256].view(-1, 4, 64)
        view.copy_(q)
        out = torch.zeros(4, q.shape[0], 64 + pad, dtype=dtype, device="cuda")[:, :, :64].transpose(0, 1)
        got, _ = check(view, kc, vc, table, lens, starts, out=out)
        assert got is out
        plain_out, _ = check(q, kc, vc, table, lens, starts)
        assert torch.equal(plain_out, out)


@pytest.mark.parametrize("heads,kv,dim,dtype", [(4, 2, 64, HF), (5, 1, 128, BF), (8, 1, 256, BF)])
def test_chunk_out_may_be_q(heads, kv, dim, dtype):
    """Whole items and items that many shares cut, rows behind the last sequence, and a sequence of no rows."""
    q, kc, vc, table, lens, starts = chunk_case(28, [300, 0, 2, 90], [50, 10, 9000, 0], heads, kv, dim, 16, dtype, rest=3)
    want, _ = check(q, kc, vc, table, lens, starts)
    got, _ = check_in_place(q, kc, vc, table, lens, starts)
    assert got is q and torch.equal(got[:starts[-1]], want[:starts[-1]])


def check_in_place(q, *rest):
    from heatvit_b200 import decode
    kc, vc, table, lens, starts = rest
    behind = q[starts[-1]:].clone()
    result = decode.paged_chunk_attention(q, kc, vc, table, ints(lens), ints(starts), out=q, return_lse=True)
    assert torch.equal(q[starts[-1]:], behind)
    return result


def test_chunk_scale_and_wide_scores():
    q, kc, vc, table, lens, starts = chunk_case(9, [50, 200], [300, 0], 4, 2, 128, 16, BF)
    for scale in (0.0, 0.5, -0.25):
        check(q, kc, vc, table, lens, starts, scale=scale)
    for scale, dtype in ((10.0, BF), (3.0, HF)):  # nearly one-hot rows: maxima that move late and far
        check(*chunk_case(10, [50, 200], [3000, 0], 4, 2, 64, 16, dtype), scale=scale)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_chunk_rising_scores(dim, dtype):
    """Scores that rise along the sequence, by a little a token and by much between tiles, so that the sums are rescaled
    in every one; and falling ones, whose late weights are small."""
    n = 1500
    q, kc, vc, table, lens, starts = chunk_case(11, [200], [n - 200], 2, 1, dim, 16, dtype, poison=False)
    at = torch.arange(n, device="cuda")
    for slope in (0.05, 0.005, -0.005, -0.05):
        q.zero_()
        q[:, :, 0] = 1
        kc.zero_()
        kc[table[0, at // 16].long(), at % 16, :, 0] = (slope * at.float()).to(dtype)[:, None]
        check(q, kc, vc, table, lens, starts, scale=1.0)


@pytest.mark.parametrize("dtype,dim", [(BF, 64), (HF, 128), (BF, 256)])
@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("new,past,bad", [(300, 0, [5, 137, 290]), (40, 100, [120]), (3, 2000, [2001]), (129, 383, [400, 511])])
def test_chunk_masked_values_stay_out(dtype, dim, value, new, past, bad):
    """A key or value that is infinite or not a number is no part of the rows that do not see it, and a NaN or an
    infinity in those that do."""
    from heatvit_b200 import decode
    q, kc, vc, table, lens, starts = chunk_case(12, [new, 20], [past, 50], 4, 2, dim, 16, dtype)
    at = torch.tensor(bad, device="cuda")
    sees = (past + torch.arange(new, device="cuda") >= bad[0])
    pg = table[0, at // 16].long()
    clean_v = vc.clone()
    vc[pg, at % 16, :, 3] = value
    out = decode.paged_chunk_attention(q, kc, vc, table, ints(lens), ints(starts))
    want, _, bound = plain(q, kc, clean_v, table, lens, starts, True, dim ** -0.5)
    fine = torch.ones_like(out, dtype=torch.bool)
    fine[:new, :, 3][sees] = False
    assert bool(((out.double() - want).abs() <= bound)[fine].all())
    assert not bool(out[~fine].isfinite().any())
    kc = kc.clone()
    kc[pg, at % 16, :, 5] = value
    out = decode.paged_chunk_attention(q, kc, clean_v, table, ints(lens), ints(starts))
    fine = torch.ones_like(out, dtype=torch.bool)
    fine[:new][sees] = False
    assert bool(((out.double() - want).abs() <= bound)[fine].all())
    if math.isnan(value):
        assert bool(out[~fine].isnan().all())


def test_chunk_nan_in_q_stays_in_its_row():
    from heatvit_b200 import decode
    q, kc, vc, table, lens, starts = chunk_case(13, [50], [300], 4, 2, 64, 16, BF)
    good = decode.paged_chunk_attention(q, kc, vc, table, ints(lens), ints(starts))
    q[17, 2, 9] = math.nan
    bad = decode.paged_chunk_attention(q, kc, vc, table, ints(lens), ints(starts))
    assert bool(bad[17, 2].isnan().all())
    bad[17, 2] = good[17, 2]
    assert torch.equal(bad, good)


def test_chunk_of_one_token_is_paged_attention():
    """To a rounding: the same sequences with one new token each, and a mixed batch beside its parts."""
    from heatvit_b200 import decode
    q, kc, vc, table, lens, starts = chunk_case(14, [1] * 9, [0, 1, 15, 16, 127, 128, 300, 2000, 5000], 8, 2, 128, 16, BF)
    one, lse = decode.paged_attention(q, kc, vc, table, ints(lens), return_lse=True)
    got, got_lse = check(q, kc, vc, table, lens, starts)
    assert bool(((one.float() - got.float()).abs() <= one.float().abs() * 2.0 ** -6 + 2.0 ** -7).all())
    assert bool(((lse - got_lse).abs() <= 2.0 ** -7).all())


def test_chunk_is_deterministic_and_shares_a_workspace():
    from heatvit_b200 import decode
    ws = decode.AttentionWorkspace(chunks=True)
    big = chunk_case(15, [9, 300, 3], [20000, 100, 7000], 8, 2, 128, 16, BF)
    small = chunk_case(16, [5], [700], 4, 4, 64, 16, HF)
    first, _ = check(*big, workspace=ws)
    one = chunk_case(17, [1, 1], [900, 5000], 4, 4, 64, 16, HF)
    step = decode.paged_attention(one[0], *one[1:4], ints(one[4]))
    for _ in range(3):
        check(*small, workspace=ws)
        assert torch.equal(step, decode.paged_attention(one[0], *one[1:4], ints(one[4]), workspace=ws))
        again, _ = check(*big, workspace=ws)
        assert torch.equal(first, again)


def test_chunk_cache_offsets_past_32_bits():
    page, kv, dim = 64, 8, 128
    pages = (1 << 31) // (page * kv * dim) + 40
    kc, vc = (torch.empty(pages, page, kv, dim, dtype=BF, device="cuda") for _ in range(2))
    table = torch.arange(pages - 20, pages, dtype=torch.int32, device="cuda").view(2, 10)
    for i, c in enumerate((kc, vc)):
        c[-20:].copy_(rand(20 + i, 20, page, kv, dim))
    q = rand(22, 140, 16, dim, dtype=BF)
    check(q, kc, vc, table, [600, 400], [0, 40, 140])


def test_chunk_reports_what_only_the_device_sees():
    from heatvit_b200 import abi, decode
    q, kc, vc, table, lens, starts = chunk_case(18, [50, 60], [100, 300], 4, 2, 64, 16, BF)
    good = decode.paged_chunk_attention(q, kc, vc, table, ints(lens), ints(starts))
    # a length past the page table's row is taken as what that can name
    room = table.shape[1] * 16
    long = decode.paged_chunk_attention(q, kc, vc, table[1:], ints([room + 5]), ints([50, 110]), out=torch.zeros_like(q))
    assert decode.device_error() == abi.HV_DECODE_BAD_LENGTH
    whole = decode.paged_chunk_attention(q, kc, vc, table[1:], ints([room]), ints([50, 110]))
    # (the slots past its 360 tokens are NaN and infinite, and live now: bits are compared)
    assert torch.equal(long[50:].view(torch.int16), whole[50:].view(torch.int16))
    # pages outside the cache are not read: the other sequence is as it was
    for page in (-1, kc.shape[0], 1 << 30, -(1 << 31)):
        bad = table.clone()
        bad[0, 3] = page
        out = decode.paged_chunk_attention(q, kc, vc, bad, ints(lens), ints(starts))
        assert decode.device_error() == abi.HV_DECODE_BAD_PAGE
        assert torch.equal(out[50:], good[50:]) and bool(out.isfinite().all())
    # starts that fall or lie outside: the nearest that do not
    for wrong, right in (([-5, 50, 110], [0, 50, 110]), ([0, 50, 500], [0, 50, 110]), ([0, 60, 50], [0, 60, 60])):
        out = decode.paged_chunk_attention(q, kc, vc, table, ints(lens), ints(wrong), out=torch.zeros_like(q))
        assert decode.device_error() == abi.HV_DECODE_BAD_START
        assert torch.equal(out, decode.paged_chunk_attention(q, kc, vc, table, ints(lens), ints(right), out=torch.zeros_like(q)))
    assert decode.device_error() == 0


def test_chunk_streams_and_graphs():
    """Another stream than the tensors' own; two captured graphs that are replayed with new inputs, in turn."""
    from heatvit_b200 import decode
    a = chunk_case(19, [40, 200], [3000, 0], 8, 2, 128, 16, BF)
    b = chunk_case(23, [7], [9000], 4, 1, 64, 16, HF)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        check(*a)
    torch.cuda.current_stream().wait_stream(side)
    ws = decode.AttentionWorkspace(chunks=True)
    graphs = []
    for case, w in ((a, None), (b, ws), (a, ws)):
        q, kc, vc, table, lens, starts = case
        n, s = ints(lens), ints(starts)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = decode.paged_chunk_attention(q, kc, vc, table, n, s, workspace=w)
        graphs.append((g, out, n, s, case))
    for _ in range(2):
        for g, out, n, s, case in graphs:
            q, kc, vc, table, lens, starts = case
            g.replay()
            want, _, bound = plain(q, kc, vc, table, lens, starts, True, q.shape[2] ** -0.5)
            assert bool(((out.double() - want).abs() <= bound).all())
        # shorter lengths and other inputs in the same memory
        for g, out, n, s, case in graphs[:2]:
            case[0].mul_(0.7)
            for i in range(len(case[4])):
                case[4][i] -= 33 if case[4][i] > 1000 else 0
            n.copy_(ints(case[4]))
        graphs[2][2].copy_(ints(a[4]))


def test_chunk_empty_calls():
    from heatvit_b200 import decode
    q, kc, vc, table, lens, starts = chunk_case(24, [4], [4], 2, 2, 64, 16, BF)
    assert decode.paged_chunk_attention(q[:0], kc, vc, table, ints(lens), ints([0, 0])).shape == (0, 2, 64)
    out = torch.ones_like(q)
    assert decode.paged_chunk_attention(q, kc, vc, table[:0], ints([]), ints([0]), out=out) is out
    assert bool((out == 1).all())
    assert bool((decode.paged_chunk_attention(q, kc, vc, table[:, :0], ints([0]), ints(starts)) == 0).all())


def test_chunk_refusals():
    from heatvit_b200 import decode
    q, kc, vc, table, lens, starts = chunk_case(25, [4, 3], [4, 0], 4, 2, 64, 16, BF, poison=False)
    n, s = ints(lens), ints(starts)
    good = (q, kc, vc, table, n, s)

    def bad(kind, match, *args, **kw):
        with pytest.raises(kind, match=match):
            decode.paged_chunk_attention(*args, **kw)

    def with_(i, t):
        return good[:i] + (t,) + good[i + 1:]
    bad(ValueError, "CUDA", *with_(0, q.cpu()))
    bad(ValueError, "live on", *with_(4, n.cpu()))
    bad(TypeError, "float16", *with_(0, q.float()))
    bad(TypeError, "same type", *with_(0, q.half()))
    bad(TypeError, "int32", *with_(5, s.long()))
    bad(TypeError, "int32", *with_(4, n.long()))
    bad(ValueError, "one more entry", *with_(5, s[:2]))
    bad(ValueError, "one row", *with_(3, table[:1]))
    bad(ValueError, "multiple", *with_(0, q[:, :3]))
    bad(ValueError, "3-dimensional", *with_(0, q[:, 0]))
    bad(ValueError, "contiguous", *with_(0, q.transpose(1, 2)))
    bad(ValueError, "dimension", *with_(0, q[:, :, :32]))
    bad(ValueError, "dim must be", q[:, :, :40], kc[..., :40], vc[..., :40], table, n, s)
    bad(ValueError, "16 bytes", q[:, :, :32], kc[..., 1:33], vc[..., 1:33], table, n, s)
    bad(ValueError, "share memory", *good, out=torch.zeros(1, 4, 64, dtype=BF, device="cuda").expand(7, 4, 64))
    bad(ValueError, "shape", *good, out=torch.zeros(6, 4, 64, dtype=BF, device="cuda"))
    bad(TypeError, None, *good, scale="large")
    v = q._version
    out = torch.zeros_like(q)
    decode.paged_chunk_attention(*good, out=out)
    assert out._version == 1 + 0 and q._version == v


def test_chunk_workspace_is_large_enough():
    from heatvit_b200 import decode
    case = chunk_case(16, [5], [700], 4, 4, 64, 16, HF)
    for small in (decode.AttentionWorkspace(),):
        with pytest.raises(ValueError, match="workspace"):
            check(*case, workspace=small)
    check(*case, workspace=decode.AttentionWorkspace(chunks=True))


@pytest.fixture
def stall():
    from heatvit_b200 import _lib, decode
    assert _lib.lib().hv_test_decode_stall(-1) == 0
    yield _lib.lib().hv_test_decode_stall
    _lib.lib().hv_test_decode_stall(-1)
    decode.device_error()


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("new,past", [(600, 0), (3, 40000)])
@pytest.mark.parametrize("copy", [0, 1, 3])
def test_chunk_wait_runs_out_reports_and_recovers(stall, dim, new, past, copy):
    """A tile of keys or values that is not reported (in a workspace that is used on): the error word, then the same
    call right."""
    from heatvit_b200 import abi, decode
    q, kc, vc, table, lens, starts = chunk_case(26, [new, 10], [past, 300], 4, 2, dim, 16, BF)
    ws = decode.AttentionWorkspace(chunks=True)
    assert stall(copy) == 0
    decode.paged_chunk_attention(q, kc, vc, table, ints(lens), ints(starts), workspace=ws)
    assert stall(-1) == 0
    assert decode.device_error() == abi.HV_DECODE_STALLED
    assert int(ws.buffer[:12288].max()) == 0
    check(q, kc, vc, table, lens, starts, workspace=ws)
