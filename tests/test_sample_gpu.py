"""Sampling on the GPU against the definition in 64 bits."""

import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

BF, HF, FF = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def clean(cuda):
    from heatvit_b200 import decode
    decode.device_error()
    yield
    assert decode.device_error() == 0


def rand(seed, *shape, dtype=FF, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def uniform(seed, rows):
    return torch.rand(rows, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def column(v, rows, dtype=torch.float64):
    return torch.as_tensor(v, device="cuda").to(dtype).expand(rows)


def plain(z, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """Each row's kept tokens (a mask), its weights in the vocabulary's order, and the token."""
    rows, vocab = z.shape
    z = z.double()
    t, p, m, u = (column(v, rows) for v in (temperature, top_p, min_p, u))
    k = column(top_k, rows, torch.long)
    top = z.amax(1, keepdim=True)
    w = torch.where(z == top, 1.0, ((z - top) / torch.where(t > 0, t, 1.0)[:, None]).exp())
    order = torch.sort(z, dim=1, descending=True, stable=True).indices
    sorted_w = w.gather(1, order)
    rank = torch.arange(vocab, device="cuda")[None]
    keep = (rank < torch.where((k > 0), k, vocab)[:, None]) & (sorted_w >= m.clamp(max=1)[:, None])
    mass = (sorted_w * keep).cumsum(1)
    ahead = mass - sorted_w * keep
    keep &= (p >= 1)[:, None] | (ahead < p[:, None] * mass[:, -1:]) | (rank == 0)
    keep &= (t > 0)[:, None] | (rank == 0)
    kept = torch.zeros_like(keep).scatter_(1, order, keep)
    w = w * kept
    cdf = w.cumsum(1)
    token = (cdf <= u[:, None] * cdf[:, -1:]).sum(1).clamp(max=vocab - 1)
    return kept, w, token


def check(z, u, **kw):
    from heatvit_b200 import decode
    token, logprob = decode.sample_tokens(z, u, return_logprob=True, **kw)
    kw = {k: v for k, v in kw.items() if v is not None and k != "out"}
    _, w, want = plain(z, u, **kw)
    assert token.dtype == torch.int64 and token.shape == u.shape
    assert torch.equal(token, want), (token != want).nonzero().flatten().tolist()[:5]
    share = (w.gather(1, want[:, None]) / w.sum(1, keepdim=True)).log().squeeze(1)
    # in 64 bits of sums of which each term is off by 2^-39 and 2^-46 at most; one rounding
    assert bool(((logprob.double() - share).abs() <= share.abs() * 2.0 ** -23 + 2.0 ** -24).all())
    return token


@pytest.mark.parametrize("dtype", [BF, HF, FF])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (5, 31), (2, 255), (4, 256), (3, 1000), (7, 8191), (2, 32768), (3, 50021),
                                        (2, 131073), (1, 300007)])
def test_sample(dtype, rows, vocab):
    z = rand(1, rows, vocab, dtype=dtype, scale=3.0)
    for i, kw in enumerate((dict(), dict(temperature=0.7, top_k=50), dict(temperature=1.3, top_p=0.9), dict(min_p=0.05),
                            dict(temperature=0.8, top_k=200, top_p=0.95, min_p=0.01), dict(temperature=0.0),
                            dict(top_p=0.3, top_k=7), dict(top_k=1), dict(top_p=0.0), dict(min_p=1.0))):
        check(z, uniform(10 + i, rows), **kw)


@pytest.mark.parametrize("dtype", [BF, FF])
def test_sample_flat_rows(dtype):
    """Hundreds of thousands of tokens of alike weights: borders of 2^-18 of the total, hundreds of draws each."""
    z = rand(2, 64, 200000, dtype=dtype, scale=0.3)
    check(z, uniform(3, 64))
    check(z, uniform(4, 64), top_p=0.9)
    check(z, uniform(5, 64), top_p=0.5, top_k=150000, temperature=2.0)


def test_sample_ties():
    """Equal logits everywhere or at the border of what is kept: the lowest indices are the first."""
    z = torch.zeros(6, 5000, device="cuda")
    u = torch.tensor([0.0, 0.2, 0.4999999, 0.5, 0.75, 1 - 2.0 ** -24], device="cuda")
    assert check(z, u).tolist() == [0, 1000, 2499, 2500, 3750, 4999]
    assert check(z, u, top_k=10).tolist() == [0, 2, 4, 5, 7, 9]
    assert check(z, u, top_p=0.5).tolist() == [0, 500, 1249, 1250, 1875, 2499]
    assert check(z, u, temperature=0.0).tolist() == [0] * 6
    z[:, 4000] = 1.0
    check(z, u, top_k=1500, temperature=0.9)
    check(z, u, top_p=0.25, temperature=0.9)
    # few values, each thousands of times, the cut within one
    z = (rand(6, 8, 60000) * 2).round().to(BF)
    for kw in (dict(top_k=30000), dict(top_p=0.8), dict(top_p=0.8, top_k=20001), dict(min_p=0.1), dict(top_k=1025)):
        check(z, uniform(7, 8), **kw)


def test_sample_settings_of_each_row():
    from heatvit_b200 import decode
    rows = 24
    z = rand(8, rows, 20000, scale=3.0)
    u = uniform(9, rows)
    i = torch.arange(rows, device="cuda")
    t = torch.where(i % 5 == 0, 0.0, 0.5 + i / 10).float()
    k = torch.where(i % 3 == 0, 0, i * 40).int()
    p = torch.where(i % 4 == 0, 1.0, 0.5 + i / 50).float()
    m = torch.where(i % 2 == 0, 0.0, i / 400).float()
    all_rows = check(z, u, temperature=t, top_k=k, top_p=p, min_p=m)
    for r in (0, 1, 7, 23):
        one = decode.sample_tokens(z[r:r + 1], u[r:r + 1], float(t[r]), int(k[r]), float(p[r]), float(m[r]))
        assert int(one) == int(all_rows[r])


def test_sample_infinite_and_lowest_logits():
    """Masks by -inf and by the type's lowest value weigh nothing; +inf takes all."""
    for dtype in (BF, HF, FF):
        z = rand(10, 6, 3000, dtype=dtype)
        z[0, 100:] = -math.inf
        z[1, 7:] = torch.finfo(dtype).min
        z[2, :2999] = -math.inf
        z[3] = torch.finfo(dtype).min
        z[4, 5], z[4, 77] = math.inf, math.inf
        z[5, ::2] = -math.inf
        for kw in (dict(), dict(top_k=50), dict(top_p=0.9), dict(temperature=0.0), dict(min_p=0.2), dict(top_k=2000, top_p=0.99)):
            token = check_no_nan(z, kw)
            assert int(token[2]) == 2999 and int(token[4]) in (5, 77) and int(token[5]) % 2 == 1
            assert int(token[0]) < 100 and int(token[1]) < 7


def check_no_nan(z, kw):
    """plain() by rows, with an infinite row as the definition has it: weight 1 for +inf, 0 for the others."""
    clean_z = z.clone()
    full = (z == math.inf).any(1)
    clean_z[full] = torch.where(z[full] == math.inf, 0.0, -math.inf).to(z.dtype)
    from heatvit_b200 import decode
    token = decode.sample_tokens(z, uniform(11, z.shape[0]), **kw)
    assert torch.equal(token, plain(clean_z, uniform(11, z.shape[0]), **kw)[2])
    return token


def test_sample_rows_without_a_distribution():
    from heatvit_b200 import abi, decode
    z = rand(12, 4, 700)
    z[1, 300] = math.nan
    z[2] = -math.inf
    good = decode.sample_tokens(z[[0, 3]], uniform(13, 4)[[0, 3]])
    token, logprob = decode.sample_tokens(z, uniform(13, 4), return_logprob=True)
    assert decode.device_error() == abi.HV_DECODE_BAD_LOGITS
    assert token.tolist() == [int(good[0]), 0, 0, int(good[1])]
    assert logprob.isnan().tolist() == [False, True, True, False]


def test_sample_extreme_settings():
    z = rand(14, 5, 4000, scale=2.0)
    u = uniform(15, 5)
    for kw in (dict(temperature=1e-6), dict(temperature=1e-40), dict(temperature=1e6), dict(top_p=1e-30), dict(top_p=1 - 2.0 ** -24),
               dict(top_k=-1), dict(top_k=4000), dict(top_k=3999), dict(top_k=1 << 30), dict(min_p=1e-30), dict(temperature=50.0, top_p=0.999)):
        check(z, u, **kw)
    from heatvit_b200 import decode
    greedy = z.argmax(1)
    assert torch.equal(decode.sample_tokens(z, u, min_p=2.0), greedy)
    assert torch.equal(decode.sample_tokens(z, u, temperature=-1.0), greedy)
    assert bool((decode.sample_tokens(z, u, temperature=math.inf) == (u.double() * 4000).long()).all())


@pytest.mark.parametrize("dtype", [BF, HF, FF])
def test_sample_strides(dtype):
    """Rows of a wider matrix, at odd starts and odd distances."""
    wide = rand(16, 9, 9001, dtype=dtype, scale=3.0)
    for at, n in ((0, 9001), (1, 8192), (8, 5000), (3, 4096), (16, 4001)):
        check(wide[:, at:at + n], uniform(17, 9), top_p=0.9, top_k=300)
    check(wide[::2, :1000], uniform(18, 5))
    check(wide[:1].expand(6, -1), uniform(19, 6), top_p=0.8)


def test_sample_out_and_determinism():
    from heatvit_b200 import decode
    z, u = rand(20, 33, 40000, scale=2.0), uniform(21, 33)
    out = torch.zeros(33, dtype=torch.int64, device="cuda")
    assert decode.sample_tokens(z, u, top_p=0.9, out=out) is out and out._version == 1
    for _ in range(3):
        assert torch.equal(decode.sample_tokens(z, u, top_p=0.9), out)
    assert decode.sample_tokens(z[:0], u[:0]).shape == (0,)


def test_sample_draws_what_the_weights_say():
    """Many draws from one row: each token as often as its share, within 5 standard deviations."""
    rows = 40000
    z = torch.tensor([2.0, 0.0, 1.0, -1.0, 1.5, 0.5], device="cuda")
    from heatvit_b200 import decode
    token = decode.sample_tokens(z.expand(rows, -1), uniform(22, rows), top_k=5)
    p = torch.softmax(z.double(), 0)
    p[3] = 0
    p /= p.sum()
    n = torch.bincount(token, minlength=6).double()
    assert int(n[3]) == 0
    assert bool(((n - rows * p).abs() <= 5 * (rows * p * (1 - p)).sqrt()).all())


def test_sample_streams_and_graphs():
    from heatvit_b200 import decode
    z, u = rand(23, 6, 30000, dtype=BF, scale=3.0), uniform(24, 6)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        check(z, u, top_p=0.9)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        token = decode.sample_tokens(z, u, top_p=0.9, top_k=1000)
    for seed in (25, 26):
        z.copy_(rand(seed, 6, 30000, scale=3.0))
        u.copy_(uniform(seed, 6))
        g.replay()
        assert torch.equal(token, plain(z, u, top_p=0.9, top_k=1000)[2])


def test_sample_refusals():
    from heatvit_b200 import decode
    z, u = rand(27, 4, 100), uniform(28, 4)

    def bad(kind, match, *args, **kw):
        with pytest.raises(kind, match=match):
            decode.sample_tokens(*args, **kw)
    bad(ValueError, "CUDA", z.cpu(), u)
    bad(ValueError, "live on", z, u.cpu())
    bad(TypeError, "bfloat16", z.double(), u)
    bad(TypeError, "float32", z, u.double())
    bad(ValueError, "one uniform", z, u[:3])
    bad(ValueError, "2-dimensional", z[0], u)
    bad(ValueError, "contiguous", z.t().contiguous().t(), u)
    bad(ValueError, "vocab", z[:, :0], u)
    bad(TypeError, "int32", z, u, top_k=torch.ones(4, dtype=torch.int64, device="cuda"))
    bad(TypeError, "float32", z, u, top_p=torch.ones(4, dtype=torch.float64, device="cuda"))
    bad(ValueError, "one entry", z, u, temperature=torch.ones(3, device="cuda"))
    bad(ValueError, "live on", z, u, temperature=torch.ones(4))
    bad(TypeError, None, z, u, temperature="hot")
    bad(TypeError, None, z, u, top_k=1.5)
    bad(TypeError, "int64", z, u, out=torch.zeros(4, dtype=torch.int32, device="cuda"))
    bad(ValueError, "one entry", z, u, out=torch.zeros(5, dtype=torch.int64, device="cuda"))
    bad(ValueError, "contiguous", z, u, out=torch.zeros(1, dtype=torch.int64, device="cuda").expand(4))


@pytest.mark.parametrize("dtype", [BF, FF])
def test_sample_cut_around_zero(dtype):
    """Logits of both zeros and of the smallest numbers about them, where the search's intervals end."""
    tiny = 2.0 ** -133 if dtype == BF else 2.0 ** -149
    z = torch.zeros(4, 20000, device="cuda", dtype=dtype)
    z[:, ::3] = -0.0
    z[:, 1::7] = tiny
    z[:, 2::11] = -tiny
    z[:, 5::13] = -1.0
    z[:, 3] = 0.5
    for kw in (dict(top_p=0.3), dict(top_p=0.8), dict(top_k=2000), dict(top_k=6000), dict(top_k=15000), dict(top_k=19990, top_p=0.9)):
        check(z, uniform(29, 4), **kw)


@pytest.mark.parametrize("dtype,vocab", [(FF, 500009), (BF, 1000003)])
def test_sample_rows_past_shared_memory(dtype, vocab):
    """Rows that a cluster's shared memory does not hold."""
    z = rand(30, 2, vocab, dtype=dtype, scale=2.0)
    for kw in (dict(), dict(top_p=0.9), dict(top_k=3000, top_p=0.7), dict(temperature=0.0), dict(min_p=0.1)):
        check(z, uniform(31, 2), **kw)
