"""Decode operators on the GPU where they can go quietly wrong: small weights, equal weights, workspaces.

Bounds are derived as in test_decode_gpu, whose helpers are used."""

import math
import os
import sys
import time

import pytest

torch = pytest.importorskip("torch")

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))

import test_decode_gpu as G  # noqa: E402
from test_decode_gpu import BF, FF, HF, clean, rand  # noqa: E402,F401

pytestmark = pytest.mark.gpu


# ---- attention: weights -------------------------------------------------------------

def scored(scores, v, dtype, heads, kv, dim, seqs, scale=1.0):
    """Attention over tokens of the given scores (before `scale`) and values [tokens, dim], the same for every
    head and sequence: enough items that none is cut, over one set of pages.  -> out, lse, 64-bit out, lse, bound."""
    from heatvit_b200 import decode
    n = len(scores)
    page = 16
    kc, vc = (torch.zeros(-(-n // page), page, kv, dim, dtype=dtype, device="cuda") for _ in range(2))
    kc.view(-1, kv, dim)[:n, :, 0] = scores.to(dtype)[:, None]
    vc.view(-1, kv, dim)[:n] = v.to(dtype)[:, None]
    q = torch.zeros(seqs, heads, dim, dtype=dtype, device="cuda")
    q[:, :, 0] = 1
    table = torch.arange(kc.shape[0], dtype=torch.int32, device="cuda").expand(seqs, -1)
    out, lse = decode.paged_attention(q, kc, vc, table, torch.full((seqs,), n, dtype=torch.int32, device="cuda"),
                                      scale=scale, return_lse=True)
    s, x = kc.view(-1, kv, dim)[:n, 0, 0].double() * scale, vc.view(-1, kv, dim)[:n, 0].double()
    p = torch.softmax(s, 0)
    want = p @ x
    # A score is one exact product, scaled in 32 bits, and its exponential within 2^-21 (2^-20 of a score); a
    # weight is held in two numbers of the cache's type, within 2^-16, in fp16 also to 2^-34 of the largest weight
    # (2^-25 beside a reference of 2^9); a warp adds n / 32 products in a chain of 2^-23 each.
    rel = float(s.abs().max()) * 2.0 ** -20 + 2.0 ** -16 + 2.0 ** -21 + n / 32 * 2.0 ** -23
    error = p @ x.abs() * 2 * rel
    if dtype == HF:
        error = error + 2.0 ** -34 * p.max() * x.abs().sum(0)
    # One rounding to nearest of what is within `error` of `want`: no farther from that than the number of the
    # type nearest to `want` is, so no farther from `want` than that number's distance and twice `error`.
    bound = (want.to(dtype).double() - want).abs() + 2 * error
    return out, lse, want, torch.logsumexp(s, 0), bound


@pytest.mark.parametrize("dtype", [HF, BF])
@pytest.mark.parametrize("heads,kv,dim", [(4, 4, 64), (8, 4, 128), (4, 4, 256), (64, 4, 64), (36, 4, 128)])
@pytest.mark.parametrize("nats", [11.5755, 12.0, 14.0, 16.0])
def test_attention_long_tail_under_one_weight(dtype, heads, kv, dim, nats):
    """One early token takes nearly all the weight and has a value of zero: the output is the tail's, whose weights
    are 12 to 16 nats smaller each (11.5755: all of them exactly 16.7 bits)."""
    n = 8192
    tail = torch.zeros(n, device="cuda") if nats == 11.5755 else rand(1, n, scale=0.3)
    tail[0] = nats
    v = 1 + rand(2, n, dim)
    v[0] = 0
    out, lse, want, want_lse, bound = scored(tail, v, dtype, heads, kv, dim, 112)
    assert bool(((out.double() - want).abs() <= bound).all()), float(((out.double() - want).abs() / bound).max())
    assert bool(((lse.double() - want_lse).abs() <= 1e-4 + 2.0 ** -18 * want_lse.abs()).all())


@pytest.mark.parametrize("dtype,step", [(BF, 2.0 ** -8), (HF, 2.0 ** -11)])
@pytest.mark.parametrize("heads,kv,dim", [(4, 4, 64), (8, 4, 128), (4, 4, 256), (64, 4, 64), (36, 4, 128)])
def test_attention_equal_weights_between_two_numbers(dtype, step, heads, kv, dim):
    """Weights of 1 + half a step of the cache's type, after a tile of ones: were each rounded alone, the output
    would be half a step off as a whole."""
    n = 4096
    scores = torch.ones(n, device="cuda")
    scores[:128] = 0
    v = torch.ones(n, dim, device="cuda")
    v[:, 1] = rand(3, n)
    out, lse, want, want_lse, bound = scored(scores, v, dtype, heads, kv, dim, 112, scale=math.log1p(step))
    assert bool(((out.double() - want).abs() <= bound).all()), float(((out.double() - want).abs() / bound).max())
    assert bool(((lse.double() - want_lse).abs() <= 1e-4 + 2.0 ** -18 * want_lse.abs()).all())


@pytest.mark.parametrize("dtype", [HF, BF])
@pytest.mark.parametrize("heads,kv,dim", [(8, 2, 64), (12, 1, 128), (4, 1, 256)])
@pytest.mark.parametrize("where", ["first", "middle", "none"])
def test_attention_long_tail_over_many_parts(dtype, heads, kv, dim, where):
    """One sequence over every SM: the parts, one of which holds a token that outweighs its tail 1000 times, have
    references of their own."""
    n = 100000
    scores = rand(1, n, scale=0.5)
    v = 1 + rand(2, n, dim)
    if where != "none":
        at = 0 if where == "first" else n // 2 + 5
        scores[at] = math.log(n) + math.log(1000.0)
        v[at] = 0
    out, lse, want, want_lse, bound = scored(scores, v, dtype, heads, kv, dim, 1)
    assert bool(((out.double() - want).abs() <= bound).all()), float(((out.double() - want).abs() / bound).max())
    assert bool(((lse.double() - want_lse).abs() <= 1e-4 + 2.0 ** -18 * want_lse.abs()).all())


@pytest.mark.parametrize("lens", [[100000, 3], [40000, 0, 777, 12345]])
def test_attention_long_fp16(lens):
    q, kc, vc, table = G.attend_case(3, lens, 4, 1, 128, 32, HF, "hnd", poison=False)
    G.check_attention(q, kc, vc, table, lens)


@pytest.mark.parametrize("dtype", [HF, BF])
@pytest.mark.parametrize("heads,kv,dim", [(4, 2, 64), (8, 1, 128), (2, 2, 256), (9, 1, 64), (32, 2, 128), (20, 1, 256)])
@pytest.mark.parametrize("n,equal", [(1, True), (70, True), (70, False), (3000, False)])
def test_attention_infinite_values(dtype, heads, kv, dim, n, equal):
    """An infinity among the values of live tokens is the output's, as in the formula, whatever its weight rounds
    to (one and halves among them); two of either sign, or a NaN, make a NaN."""
    from heatvit_b200 import decode
    q, kc, vc, table = G.attend_case(9, [n] * 4, heads, kv, dim, 16, dtype, "nhd")
    if equal:
        q.zero_()
    q[:, :, :8] *= 0.25
    at = lambda b, t: (table[b, t // 16].long(), t % 16)  # noqa: E731
    vc[at(0, n // 2)] = math.inf
    vc[at(1, n - 1)] = -math.inf
    vc[at(2, 0)], vc[at(2, n - 1)] = math.inf, -math.inf
    if n == 1:
        vc[at(2, 0)] = math.nan
    out = decode.paged_attention(q, kc, vc, table, torch.full((4,), n, dtype=torch.int32, device="cuda"), scale=0.02)
    assert bool((out[0] == math.inf).all()) and bool((out[1] == -math.inf).all()) and bool(out[2].isnan().all())
    assert bool(out[3].isfinite().all())


@pytest.mark.parametrize("n", [(1 << 31) - 256, (1 << 31) - 1])
def test_attention_length_at_the_end_of_its_type(n):
    """The longest cache that lengths can name, on one page that the table repeats; above 2^31 - 256, that, reported."""
    from heatvit_b200 import abi, decode
    page, dim, most = 1 << 16, 32, (1 << 31) - 256
    kc = rand(1, 1, page, 1, dim, dtype=BF)
    vc = torch.randint(-1, 3, (1, page, 1, dim), generator=torch.Generator().manual_seed(2)).cuda().to(BF)
    table = torch.zeros(1, 1 << 15, dtype=torch.int32, device="cuda")
    q = torch.zeros(1, 2, dim, dtype=BF, device="cuda")  # equal weights: every warp's sums are whole numbers under 2^24
    out, lse = decode.paged_attention(q, kc, vc, table, torch.tensor([n], dtype=torch.int32, device="cuda"),
                                      return_lse=True)
    assert decode.device_error() == (abi.HV_DECODE_BAD_LENGTH if n > most else 0)
    v = vc.view(page, dim).double()
    want = (v.sum(0) * (most // page) + v[:most % page].sum(0)) / most
    # warps' sums joined in 32 bits (a few hundred additions), then one rounding
    error = 2.0 ** -14 * 2
    assert bool(((out[0].double() - want).abs() <= (want.to(BF).double() - want).abs() + 2 * error).all())
    assert bool(((lse.double() - math.log(most)).abs() <= 1e-4).all())


# ---- attention: workspaces ----------------------------------------------------------

def test_new_workspace_zeroes_its_counters_alone():
    """The rest of the 5 MB is written before it is read: a captured call makes a workspace of its own, and a
    graph would fill it at every replay."""
    from heatvit_b200 import decode
    size = decode.AttentionWorkspace().buffer.numel()
    torch.cuda.empty_cache()
    block = torch.full((size,), 255, dtype=torch.uint8, device="cuda")
    at = block.data_ptr()
    del block
    ws = decode.AttentionWorkspace()  # the allocator gives the block that has just come free
    assert ws.buffer.data_ptr() == at
    counters = 12288  # HV_ATTENTION_COUNTER_BYTES
    assert bool((ws.buffer[:counters] == 0).all()) and bool((ws.buffer[counters:] == 255).all())
    case = G.attend_case(6, [50000, 7, 30000], 8, 1, 128, 16, BF, "nhd", poison=False)
    for _ in range(2):  # parts are joined, and nothing of what was there before (NaN) is in them
        G.check_attention(*case, [50000, 7, 30000], workspace=ws)
    assert bool((ws.buffer[:counters] == 0).all())


def test_workspace_dropped_while_another_stream_uses_it():
    """Its memory goes to nobody before the call on the other stream is through."""
    from heatvit_b200 import decode
    lens = [9000, 300]
    q, kc, vc, table = G.attend_case(6, lens, 8, 1, 128, 16, BF, "nhd")
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    want = decode.paged_attention(q, kc, vc, table, n)
    ws = decode.AttentionWorkspace()
    at, size = ws.buffer.data_ptr(), ws.buffer.numel()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)  # the call is still ahead of the device when the workspace goes
        got = decode.paged_attention(q, kc, vc, table, n, workspace=ws)
    del ws
    other = torch.empty(size, dtype=torch.uint8, device="cuda")
    assert other.data_ptr() != at
    side.synchronize()
    assert torch.equal(got, want)


def test_workspace_in_a_graph():
    """One workspace through a captured step of several calls, replayed on another stream, and then dropped."""
    from heatvit_b200 import decode
    ws = decode.AttentionWorkspace()
    cases = [(*G.attend_case(seed, lens, 8, 1, 128, 16, BF, "nhd"), torch.tensor(lens, dtype=torch.int32, device="cuda"))
             for seed, lens in ((6, [9000, 300]), (7, [40, 0, 20000]))]
    want = [decode.paged_attention(*c) for c in cases]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = [decode.paged_attention(*c, workspace=ws) for c in cases * 2]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            graph.replay()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want * 2))
    del graph, ws
    torch.cuda.empty_cache()


def test_workspace_refusals():
    """One that is too small, not on 256 bytes, not contiguous bytes, or not on a device at all."""
    from types import SimpleNamespace
    from heatvit_b200 import decode
    q, kc, vc, table = G.attend_case(1, [20, 5], 4, 2, 64, 16, BF, "nhd")
    n = torch.tensor([20, 5], dtype=torch.int32, device="cuda")
    size = decode.AttentionWorkspace().buffer.numel()
    room = torch.zeros(2 * size, dtype=torch.uint8, device="cuda")
    for kind, buffer in ((ValueError, room[:4096]), (ValueError, room[16:16 + size]), (TypeError, room[::2]),
                         (TypeError, room.view(torch.int32)), (ValueError, room.cpu()), (TypeError, "workspace")):
        with pytest.raises(kind):
            decode.paged_attention(q, kc, vc, table, n, workspace=SimpleNamespace(buffer=buffer))
    assert bool((room == 0).all())


# ---- append -------------------------------------------------------------------------

def test_append_refuses_more_elements_than_threads():
    """Rows off 16 bytes take a thread an element: too many are a ValueError, as with aligned rows, and not a CUDA error."""
    from heatvit_b200 import decode
    tokens, dim = 1 << 20, 4096
    k = torch.zeros(dim + 1, dtype=BF, device="cuda")[1:].view(1, 1, dim).expand(tokens, 1, dim)
    cache = torch.zeros(1, 1, 1, dim, dtype=BF, device="cuda")
    nowhere = torch.full((tokens,), -1, dtype=torch.int32, device="cuda")  # padding tokens
    table = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="too many elements"):
        decode.append_kv(k, k, cache, cache.clone(), table, nowhere, seq_ids=nowhere)


# ---- autograd -----------------------------------------------------------------------

def a_step(make):
    """One call of each operator into the caller's tensors, which `make` allocates -> those tensors."""
    from heatvit_b200 import decode
    x, w = rand(1, 5, 512, dtype=BF), rand(3, 512, dtype=BF)
    residual, out = make(5, 512, dtype=BF), make(5, 256, dtype=BF)
    rows = decode.add_rmsnorm_fp8(x, w, residual=residual, residual_out=residual)
    wq, ws = decode.quantize_weight_fp8(rand(4, 256, 512, scale=0.05))
    decode.gemm_fp8(rows.q, rows.scale, wq, ws, out=out)
    kc, vc, q, attended = (make(*size, dtype=BF) for size in ((5, 16, 1, 64), (5, 16, 1, 64), (5, 2, 64), (5, 2, 64)))
    h = out.view(5, 4, 64)
    table = torch.arange(5, dtype=torch.int32, device="cuda")[:, None]
    pos = torch.zeros(5, dtype=torch.int32, device="cuda")
    decode.append_kv(h[:, 2:3], h[:, 3:], kc, vc, table, pos, q=h[:, :2], q_out=q)
    decode.paged_attention(q, kc, vc, table, pos + 1, out=attended)
    return residual, out, kc, vc, q, attended


def test_written_tensors_count_their_versions():
    """What a call writes of the caller's, and nothing else, is newer to autograd than what it saved before."""
    made = {}

    def make(*size, dtype):
        t = torch.zeros(*size, dtype=dtype, device="cuda")
        made[t] = t._version
        return t
    for t in a_step(make):
        assert t._version == made[t] + 1
    with torch.inference_mode():
        frozen = []

        def make_frozen(*size, dtype):
            frozen.append(torch.zeros(*size, dtype=dtype, device="cuda"))
            return frozen[-1]
        a_step(make_frozen)
    a_step(lambda *size, dtype, held=iter(frozen): next(held))  # inference tensors outside that mode are taken too


def test_inputs_that_ask_for_gradients_are_read_as_values():
    from heatvit_b200 import decode
    x, w = rand(1, 5, 512, dtype=BF), rand(3, 512, dtype=BF)
    plain = decode.add_rmsnorm_fp8(x, w, residual=x)
    r = decode.add_rmsnorm_fp8(x, torch.nn.Parameter(w), residual=x.clone().requires_grad_())
    assert torch.equal(r.residual, plain.residual) and torch.equal(r.scale, plain.scale)
    assert not (r.residual.requires_grad or r.scale.requires_grad or r.q.requires_grad)


# ---- refusals -----------------------------------------------------------------------

def test_written_tensors_do_not_share_memory():
    """An expanded tensor is read where it is an input, and refused where rows would race to write it."""
    from heatvit_b200 import decode
    x, w = rand(1, 5, 512, dtype=BF), rand(3, 512, dtype=BF)
    one = rand(2, 1, 512, dtype=BF)
    many = one.expand(5, 512)
    r = decode.add_rmsnorm_fp8(x, w, residual=many)
    assert torch.equal(r.residual, decode.add_rmsnorm_fp8(x, w, residual=many.clone()).residual)
    wq, ws = decode.quantize_weight_fp8(rand(4, 256, 512, scale=0.05))
    kc, vc = (torch.zeros(5, 16, 1, 64, dtype=BF, device="cuda") for _ in range(2))
    table = torch.arange(5, dtype=torch.int32, device="cuda")[:, None]
    pos = torch.zeros(5, dtype=torch.int32, device="cuda")
    h = rand(5, 5, 1, 64, dtype=BF)
    for call in (lambda: decode.add_rmsnorm_fp8(x, w, residual=x, residual_out=many),
                 lambda: decode.gemm_fp8(r.q, r.scale, wq, ws, out=one[:, :256].expand(5, 256)),
                 lambda: decode.append_kv(h, h, kc[:1].expand(5, 16, 1, 64), vc, table, pos),
                 lambda: decode.append_kv(h, h, kc, vc[:, :1].expand(5, 16, 1, 64), table, pos),
                 lambda: decode.append_kv(h, h, kc, vc, table, pos, q=h, q_out=h[:1].expand(5, 1, 64)),
                 lambda: decode.paged_attention(h, kc, vc, table, pos, out=h[:1].expand(5, 1, 64))):
        with pytest.raises(ValueError, match="share memory"):
            call()
    # one page read by every sequence is no such thing
    shared = decode.paged_attention(h, kc[:1].expand(5, 16, 1, 64), vc[:1].expand(5, 16, 1, 64), table, pos + 1)
    assert torch.equal(shared, torch.zeros_like(shared))


# ---- bounded waits ------------------------------------------------------------------

@pytest.fixture
def stall():
    """Sets a copy that each CTA leaves out (-1: none); normal operation again at the end."""
    from heatvit_b200 import _lib
    hook = _lib.lib().hv_test_decode_stall
    yield lambda copy: _lib.check(hook(copy))
    _lib.check(hook(-1))


@pytest.mark.parametrize("copy", [0, 1, 2])
@pytest.mark.parametrize("m,n,k", [(1, 4096, 4096), (30, 300, 300), (128, 4096, 4096), (300, 600, 300), (2048, 4096, 384)])
def test_gemm_wait_runs_out_reports_and_recovers(stall, m, n, k, copy):
    """A copy that never comes, in each shape of work (few tokens split and whole, tiles split and whole, wide tiles
    one after another): the call returns and says so, and the next one is as it was."""
    from heatvit_b200 import abi, decode
    a, b = G.e4m3(1, m, k), G.e4m3(2, n, k)
    sa, sb = G.scales(3, m, -(-k // 128)), G.scales(4, -(-n // 128), -(-k // 128))
    good = decode.gemm_fp8(a, sa, b, sb)
    assert decode.device_error() == 0
    stall(copy)
    start = time.monotonic()
    decode.gemm_fp8(a, sa, b, sb)
    assert decode.device_error() == abi.HV_DECODE_STALLED
    assert time.monotonic() - start < 5
    assert decode.device_error() == 0  # reading clears the word
    stall(-1)
    for _ in range(2):
        assert torch.equal(decode.gemm_fp8(a, sa, b, sb), good)
        assert decode.device_error() == 0


@pytest.mark.parametrize("dtype,rows,dim,residual", [(BF, 1300, 2048, True), (FF, 700, 5000, True), (HF, 1300, 8192, False),
                                                     (BF, 600, 16384, True)])
def test_norm_wait_runs_out_reports_and_recovers(stall, dtype, rows, dim, residual):
    """Rows that never come into the ring whole: the call returns and says so, and the next one is as it was."""
    from heatvit_b200 import abi, decode
    x, w = rand(1, rows, dim, dtype=dtype), rand(3, dim, dtype=dtype)
    res = rand(2, rows, dim, dtype=dtype) if residual else None
    good = decode.add_rmsnorm_fp8(x, w, residual=res)
    assert decode.device_error() == 0
    stall(0)
    start = time.monotonic()
    decode.add_rmsnorm_fp8(x, w, residual=res)
    assert decode.device_error() == abi.HV_DECODE_STALLED
    assert time.monotonic() - start < 5
    stall(-1)
    for _ in range(2):
        r = decode.add_rmsnorm_fp8(x, w, residual=res)
        assert torch.equal(r.q.view(torch.uint8), good.q.view(torch.uint8)) and torch.equal(r.scale, good.scale)
        assert not residual or torch.equal(r.residual, good.residual)
        assert decode.device_error() == 0


def test_stall_hook_rejects_a_bad_copy():
    from heatvit_b200 import _lib, abi
    assert _lib.lib().hv_test_decode_stall(-2) == abi.HV_ERR_VALUE
