"""Chunk attention on the GPU where values are infinite or not numbers, against the plain 64-bit form."""

import math
import os
import sys

import pytest

torch = pytest.importorskip("torch")

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))

from test_chunk_attention_gpu import chunk_case, ints, plain  # noqa: E402
from test_decode_gpu import BF, HF, clean  # noqa: E402,F401

pytestmark = pytest.mark.gpu


def hidden_values_stay_out(case, past, hidden, value):
    """Values of the tokens `hidden` (from a sequence's first new token on) are `value` in every sequence: rows that do not see
    the first of them are as if they were not there, the others are no numbers; three calls give the same bits."""
    from heatvit_b200 import decode
    q, kc, vc, table, lens, starts = case
    want, _, bound = plain(q, kc, vc, table, lens, starts, True, q.shape[2] ** -0.5)
    page = kc.shape[1]
    row = torch.arange(q.shape[0], device="cuda")
    for b in range(len(lens)):
        t = torch.tensor([past[b] + h for h in hidden], device="cuda")
        vc[table[b, t // page].long(), t % page] = value
        row[starts[b]:starts[b + 1]] -= starts[b]
    sees = row >= hidden[0]
    first = None
    for _ in range(3):
        out = decode.paged_chunk_attention(q, kc, vc, table, ints(lens), ints(starts))
        assert bool(((out.double() - want).abs() <= bound)[~sees].all())
        assert not bool(out[sees].isfinite().any())
        first = out if first is None else first
        assert torch.equal(first.view(torch.int16), out.view(torch.int16))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("page", [1, 12, 16])
@pytest.mark.parametrize("dim", [32, 64, 96, 128, 192, 256])
@pytest.mark.parametrize("group", [1, 2])
def test_hidden_values_late_in_a_segment(dim, page, dtype, group):
    """The border of what rows see lies in the last but one tile of keys, long after the maxima have settled, and the values in
    its second half; there are more items than shares, so that segments are of up to all nine steps."""
    seqs, kv = 24, 8
    case = chunk_case(40, [40] * seqs, [1000] * seqs, kv * group, kv, dim, page, dtype)
    hidden_values_stay_out(case, [1000] * seqs, [7, 20, 39], math.nan)


@pytest.mark.parametrize("dim,dtype", [(64, BF), (128, HF), (192, BF), (256, BF), (256, HF)])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("new,past,hidden", [(300, 700, [70, 200]), (130, 1987, [1, 60]), (5, 4000, [3])])
def test_hidden_values_in_cut_items(dim, dtype, value, new, past, hidden):
    """The same of a few sequences, whose items many shares cut, and of a border that crosses several tiles."""
    case = chunk_case(41, [new] * 3, [past] * 3, 4, 2, dim, 16, dtype)
    hidden_values_stay_out(case, [past] * 3, hidden, value)


@pytest.mark.parametrize("dtype", [HF, BF])
@pytest.mark.parametrize("heads,kv,dim", [(4, 2, 64), (8, 1, 128), (2, 2, 256), (9, 1, 64), (20, 1, 192)])
@pytest.mark.parametrize("new,n,equal", [(1, 1, True), (3, 70, True), (70, 70, False), (5, 3000, False), (200, 3000, False)])
def test_infinite_values_that_are_seen(dtype, heads, kv, dim, new, n, equal):
    """An infinity among the values that a row sees is its output, as in the formula, whatever its weight rounds
    to (one and halves among them); two of either sign make a NaN."""
    from heatvit_b200 import decode
    q, kc, vc, table, lens, starts = chunk_case(42, [new] * 4, [n - new] * 4, heads, kv, dim, 16, dtype)
    if equal:
        q.zero_()
    q[:, :, :8] *= 0.25
    at = lambda b, t: (table[b, t // 16].long(), t % 16)  # noqa: E731
    vc[at(0, (n - new) // 2)] = math.inf
    vc[at(1, n - new)] = -math.inf  # the first row's own, which all see
    vc[at(2, 0)], vc[at(2, n - 1)] = math.inf, -math.inf
    if n == 1:
        vc[at(2, 0)] = math.nan
    out = decode.paged_chunk_attention(q, kc, vc, table, ints(lens), ints(starts), scale=0.02).unflatten(0, (4, new))
    assert bool((out[0] == math.inf).all()) and bool((out[1] == -math.inf).all()) and bool(out[2, -1].isnan().all())
    assert bool((out[2, :-1] == math.inf).all()) and bool(out[3].isfinite().all())


@pytest.mark.parametrize("dim", [32, 64, 128, 192, 256])
@pytest.mark.parametrize("new,past,causal", [(3, 1021, False), (40, 1000, True), (260, 780, True)])
def test_large_values_keep_their_sums(dim, new, past, causal):
    """bf16 values whose sum, each times a weight of one at most, is a number in 32 bits: also where the scores rise, after a
    row's first steps, by a little less than what its maximum has to be passed by to move."""
    from heatvit_b200 import decode
    n, seqs = new + past, 24  # items enough that segments are of many steps
    q, kc, vc, table, lens, starts = chunk_case(43, [new] * seqs, [past] * seqs, 8, 8, dim, 16, BF)
    q.zero_()
    q[:, :, 0] = 1
    at = torch.arange(n, device="cuda")
    v = torch.rand(n, 8, dim, generator=torch.Generator("cuda").manual_seed(44), device="cuda")
    for b in range(seqs):
        place = table[b, at // 16].long(), at % 16
        kc[place] = 0
        kc[place[0][256:], place[1][256:], :, 0] = 4.0  # 5.8 powers of two above the first ones
        vc[place] = ((v + 1) * 2.0 ** (126 - math.ceil(math.log2(n)))).to(BF)
    want, _, bound = plain(q, kc, vc, table, lens, starts, causal, 1.0)
    out = decode.paged_chunk_attention(q, kc, vc, table, ints(lens), ints(starts), causal=causal, scale=1.0)
    assert bool(out.isfinite().all()) and bool(((out.double() - want).abs() <= bound).all())


@pytest.mark.parametrize("dim,dtype", [(64, HF), (128, BF), (256, BF)])
def test_scale_that_is_no_number(dim, dtype):
    """A NaN for a scale is every row's, as in attention of one token; rows that see nothing are zeros all the same."""
    from heatvit_b200 import decode
    q, kc, vc, table, lens, starts = chunk_case(45, [40, 1, 150], [0, 700, 20], 4, 2, dim, 16, dtype)
    lens[0] = 30  # the first ten rows stand before the first token
    out, lse = decode.paged_chunk_attention(q, kc, vc, table, ints(lens), ints(starts), scale=math.nan, return_lse=True)
    assert bool((out[:10] == 0).all()) and bool((lse[:10] == -math.inf).all())
    assert bool(out[10:].isnan().all()) and bool(lse[10:].isnan().all())
    one = decode.paged_attention(q[40:41], kc, vc, table[1:2], ints(lens[1:2]), scale=math.nan)
    assert bool(one.isnan().all())
