"""Decode operators on the GPU against plain 64-bit forms.

Tolerances are bounds on the roundings that each operator makes: U[dtype] is the
unit roundoff of a type; 32-bit steps count 2^-24 each."""

import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
BF, HF, FF = torch.bfloat16, torch.float16, torch.float32
FLOOR = 2.0 ** -100


@pytest.fixture(autouse=True)
def clean(cuda):
    from heatvit_b200 import decode
    decode.device_error()
    yield
    assert decode.device_error() == 0


def rand(seed, *shape, dtype=FF, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


# ---- norm ---------------------------------------------------------------------------

def check_norm(r, x, w, eps, residual):
    h = x.double() + (residual.double() if residual is not None else 0.0)
    if residual is not None:
        # a rounding of the 32-bit sum; fp16 has subnormals of 2^-24
        assert bool(((r.residual.double() - h).abs() <= h.abs() * (U[x.dtype] + 2.0 ** -23) + 2.0 ** -25).all())
    y = h * torch.rsqrt((h * h).mean(1, keepdim=True) + eps) * w.double()
    rows, dim = y.shape
    g = -(-dim // 128)
    assert r.q.shape == x.shape and r.scale.shape == (rows, g)
    padded = torch.nn.functional.pad(y, (0, g * 128 - dim)).view(rows, g, 128)
    scale = padded.abs().amax(2).clamp(min=FLOOR) / 448.0
    # the sum of squares: at most 32 terms in a chain and a tree above it, halved by the root,
    # then about eight roundings: under 64 * 2^-24
    assert bool(((r.scale.double() - scale).abs() <= scale * 2.0 ** -18).all())
    s = r.scale.double().repeat_interleave(128, 1)[:, :dim]
    got = r.q.double() * s
    # half a step of e4m3: 2^-4 of a normal value, 2^-10 of a scale below
    assert bool(((got - y).abs() <= torch.maximum(y.abs() * 2.0 ** -4, s * 2.0 ** -10) * (1 + 2.0 ** -10)).all())


@pytest.mark.parametrize("dtype", [BF, HF, FF])
@pytest.mark.parametrize("rows,dim", [(1, 1), (1, 192), (3, 127), (9, 129), (197, 192), (5, 257), (7, 520), (2, 1000),
                                      (33, 1024), (4, 1025), (5, 2056), (3, 4096), (2, 4099), (2, 8192), (3, 12000),
                                      (2, 16392), (1, 32768)])
def test_norm(dtype, rows, dim):
    from heatvit_b200 import decode
    x, res = rand(1, rows, dim, dtype=dtype), rand(2, rows, dim, dtype=dtype, scale=3.0)
    w = (1 + rand(3, dim, scale=0.2)).to(dtype)
    check_norm(decode.add_rmsnorm_fp8(x, w, 1e-6), x, w, 1e-6, None)
    check_norm(decode.add_rmsnorm_fp8(x, w, 1e-5, residual=res), x, w, 1e-5, res)


@pytest.mark.parametrize("dtype,rows,dim", [(HF, 20011, 192), (BF, 5003, 512), (BF, 1500, 1000), (BF, 1183, 1032),
                                            (HF, 777, 2048), (FF, 1000, 3000), (BF, 601, 4104), (FF, 640, 8192),
                                            (BF, 593, 16384), (FF, 600, 16384), (HF, 650, 16392), (BF, 900, 2001)])
def test_norm_many_rows(dtype, rows, dim):
    """More rows than resident warps or CTAs: those that go on to further rows, and the ring."""
    from heatvit_b200 import decode
    x, res = rand(1, rows, dim, dtype=dtype), rand(2, rows, dim, dtype=dtype, scale=3.0)
    w = (1 + rand(3, dim, scale=0.2)).to(dtype)
    check_norm(decode.add_rmsnorm_fp8(x, w, 1e-6), x, w, 1e-6, None)
    before = res.clone()
    check_norm(decode.add_rmsnorm_fp8(x, w, 1e-6, residual=res, residual_out=res), x, w, 1e-6, before)


@pytest.mark.parametrize("dtype", [BF, FF])
def test_norm_strides_and_in_place(dtype):
    """Rows of a wider matrix at odd starts (element by element), and residual_out = residual."""
    from heatvit_b200 import decode
    wide, w = rand(1, 37, 1300, dtype=dtype), rand(2, 601, dtype=dtype)[1:]
    x = wide[:, 3:603]
    res = rand(3, 37, 600, dtype=dtype)
    before = res.clone()
    r = decode.add_rmsnorm_fp8(x, w, 1e-6, residual=res, residual_out=res)
    assert r.residual is res
    check_norm(r, x, w, 1e-6, before)
    assert decode.add_rmsnorm_fp8(x[:0], w).q.shape == (0, 600)


def test_norm_extreme_rows():
    """Zero rows, tiny rows, blocks of zeros, and a row with a NaN or an infinity, which stays its own."""
    from heatvit_b200 import decode
    x = rand(1, 6, 384)
    x[0] = 0
    x[1] *= 1e-30
    x[2, 128:256] = 0
    w = torch.ones(384, device="cuda")
    clean_rows = decode.add_rmsnorm_fp8(x, w, 1e-6)
    check_norm(clean_rows, x, w, 1e-6, None)
    assert bool((clean_rows.q[0].float() == 0).all()) and bool((clean_rows.scale > 0).all())
    x[3, 5], x[4, 6] = math.nan, math.inf
    r = decode.add_rmsnorm_fp8(x, w, 1e-6)
    assert bool(r.q[3].float().isnan().all())
    assert bool(r.q[4, 6].float().isnan())
    for i in (0, 1, 2, 5):
        assert torch.equal(r.q[i].view(torch.uint8), clean_rows.q[i].view(torch.uint8))
        assert torch.equal(r.scale[i], clean_rows.scale[i])


@pytest.mark.parametrize("rows,dim", [(6, 384), (5, 1500), (700, 2048)])
def test_norm_nan_reaches_scale(rows, dim):
    """As in the formula, a NaN makes its block's scale and every q of the block a NaN, and no other block's."""
    from heatvit_b200 import decode
    x, w = rand(1, rows, dim), torch.ones(dim, device="cuda")
    x[3, 5], x[4, 6] = math.nan, math.inf
    w[300] = math.nan
    r = decode.add_rmsnorm_fp8(x, w, 1e-6)
    y = x.double() * torch.rsqrt((x.double() ** 2).mean(1, keepdim=True) + 1e-6) * w.double()
    g = -(-dim // 128)
    amax = torch.nn.functional.pad(y, (0, g * 128 - dim)).view(rows, g, 128).abs().amax(2)
    assert torch.equal(r.scale.isnan(), amax.isnan())
    assert torch.equal(r.q.float().isnan(), amax.isnan().repeat_interleave(128, 1)[:, :dim])


# ---- GEMM ---------------------------------------------------------------------------

def e4m3(seed, rows, k, pad=0):
    t = torch.empty(rows, -(-k // 16) * 16 + pad, dtype=torch.float8_e4m3fn, device="cuda")
    t.copy_(rand(seed, *t.shape, scale=100.0).clamp_(-448, 448))
    return t[:, :k]


def scales(seed, rows, groups):
    return rand(seed, rows, groups).exp_() * 0.01


def check_gemm(out, a, sa, b, sb):
    k = a.shape[1]
    fa = a.double() * sa.double().repeat_interleave(128, 1)[:, :k]
    fb = b.double() * sb.double().repeat_interleave(128, 0)[:b.shape[0]].repeat_interleave(128, 1)[:, :k]
    want, size = fa @ fb.t(), fa.abs() @ fb.abs().t()
    # four accumulations of a group in the tensor core (2^-22 of the running sum each), a chain
    # over the groups, scales, and the joining of up to eight parts; then the output's rounding
    groups = -(-k // 128)
    bound = size * (4 * 2.0 ** -22 + (groups + 10) * 2.0 ** -24) + want.abs() * U[out.dtype] * (1 + 2.0 ** -10) + 2.0 ** -25
    assert bool(((out.double() - want).abs() <= bound).all()), float(((out.double() - want).abs() / bound).max())


@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 128, 128), (2, 129, 127), (7, 64, 300), (16, 576, 192), (17, 200, 4096),
                                   (32, 1000, 1024), (33, 130, 16), (64, 4096, 2048), (65, 64, 129), (127, 384, 640),
                                   (129, 257, 192), (197, 576, 192), (1, 192, 16384), (40, 96, 5000), (200, 192, 8192),
                                   (1576, 768, 192), (2048, 1111, 384), (3000, 3333, 512)])
@pytest.mark.parametrize("dtype", [BF, HF, FF])
def test_gemm(m, n, k, dtype):
    from heatvit_b200 import decode
    a, b = e4m3(1, m, k), e4m3(2, n, k)
    sa, sb = scales(3, m, -(-k // 128)), scales(4, -(-n // 128), -(-k // 128))
    check_gemm(decode.gemm_fp8(a, sa, b, sb, out_dtype=dtype), a, sa, b, sb)


def test_gemm_many_tiles():
    """More tiles than resident CTAs, with ragged last tiles both ways."""
    from heatvit_b200 import decode
    m, n, k = 4099, 4500, 300
    a, b = e4m3(1, m, k), e4m3(2, n, k)
    sa, sb = scales(3, m, 3), scales(4, -(-n // 128), 3)
    check_gemm(decode.gemm_fp8(a, sa, b, sb), a, sa, b, sb)


@pytest.mark.parametrize("m", [5, 300])
def test_gemm_strides(m):
    """Padded operand rows, transposed scales, an output that is a slice at an odd place with its surroundings untouched."""
    from heatvit_b200 import decode
    n, k = 333, 260
    a, b = e4m3(1, m, k, pad=48), e4m3(2, n, k, pad=16)
    sa, sb = scales(3, 3, m).t(), scales(4, 3, 3)[:, ::1]
    whole = torch.full((m, n + 9), 7.0, dtype=BF, device="cuda")
    out = decode.gemm_fp8(a, sa, b, sb, out=whole[:, 5:5 + n])
    check_gemm(out, a, sa, b, sb)
    assert bool((whole[:, :5] == 7).all()) and bool((whole[:, 5 + n:] == 7).all())


def test_gemm_output_past_32_bits():
    """Rows of an output whose element offsets pass 2^31."""
    from heatvit_b200 import decode
    m, n, k, stride = 2100, 200, 128, 1 << 20
    a, b, sa, sb = e4m3(1, m, k), e4m3(2, n, k), scales(3, m, 1), scales(4, 2, 1)
    whole = torch.empty((m, stride), dtype=BF, device="cuda")
    check_gemm(decode.gemm_fp8(a, sa, b, sb, out=whole[:, :n]), a, sa, b, sb)


@pytest.mark.parametrize("m", [3, 260])
def test_gemm_nan_stays_in_its_row(m):
    from heatvit_b200 import decode
    a, b, sa, sb = e4m3(1, m, 256), e4m3(2, 140, 256), scales(3, m, 2), scales(4, 2, 2)
    before = decode.gemm_fp8(a, sa, b, sb)
    a.view(torch.uint8)[1, 200] = 0x7F
    out = decode.gemm_fp8(a, sa, b, sb)
    assert bool(out[1].isnan().all())
    keep = [i for i in range(m) if i != 1]
    assert torch.equal(out[keep], before[keep])


def test_quantize_weight():
    from heatvit_b200 import decode
    w = rand(1, 300, 200, dtype=BF)
    w[:128, :128] = 0
    q, s = decode.quantize_weight_fp8(w)
    assert q.shape == w.shape and q.stride(0) % 16 == 0 and s.shape == (3, 2)
    full = s.double().repeat_interleave(128, 0)[:300].repeat_interleave(128, 1)[:, :200]
    err = (q.double() * full - w.double()).abs()
    assert bool((err <= torch.maximum(w.double().abs() * 2.0 ** -4, full * 2.0 ** -10) * (1 + 2.0 ** -10)).all())


# ---- cache --------------------------------------------------------------------------

def make_cache(seed, pages, page, kv, dim, dtype, layout, fill=True):
    shape = (pages, page, kv, dim) if layout == "nhd" else (pages, kv, page, dim)
    t = rand(seed, *shape, dtype=dtype) if fill else torch.full(shape, math.nan, dtype=dtype, device="cuda")
    return t if layout == "nhd" else t.transpose(1, 2)


def make_table(seed, lens, page, spare=0):
    need = [-(-n // page) for n in lens]
    table = torch.full((len(lens), max(1, max(need) + spare)), -1, dtype=torch.int32)
    order = torch.randperm(sum(need), generator=torch.Generator().manual_seed(seed)).tolist()
    for i, n in enumerate(need):
        for j in range(n):
            table[i, j] = order.pop()
    return table.cuda(), max(1, sum(need))


def rotate64(x, table, pos, rot, interleaved):
    """x [tokens, heads, dim] float64, by the table's own values."""
    x = x.clone()
    half = rot // 2
    c, s = table[pos].double()[:, None, :half], table[pos].double()[:, None, half:]
    i = torch.arange(half, device=x.device)
    u, w = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    a, b = x[:, :, u], x[:, :, w]
    x[:, :, u], x[:, :, w] = a * c - b * s, a * s + b * c
    return x


def near(got, want, parts):
    """One rounding of a 32-bit sum of two products."""
    bound = want.abs() * U[got.dtype] * (1 + 2.0 ** -10) + parts * 2.0 ** -22 + 2.0 ** -25
    assert bool(((got.double() - want).abs() <= bound).all())


@pytest.mark.parametrize("dtype,layout", [(BF, "nhd"), (HF, "hnd")])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("heads,kv,dim,rot,page", [(4, 2, 64, 64, 16), (6, 3, 64, 32, 5), (8, 1, 128, 128, 1),
                                                   (2, 2, 40, 24, 7), (3, 3, 63, 62, 16), (2, 1, 33, 10, 16), (4, 4, 96, 0, 16)])
def test_append(dtype, layout, interleaved, heads, kv, dim, rot, page):
    from heatvit_b200 import decode
    past, new = [0, 3, 40, 17], [9, 1, 30, 0]
    lens = [p + n for p, n in zip(past, new)]
    table, pages = make_table(1, lens, page, spare=1)
    seq = torch.tensor(sum([[i] * n for i, n in enumerate(new)], []), dtype=torch.int32, device="cuda")
    pos = torch.tensor(sum([list(range(p, p + n)) for p, n in zip(past, new)], []), dtype=torch.int32, device="cuda")
    pos[4] = -1  # a padding token
    qkv = rand(2, pos.numel(), (heads + 2 * kv) * dim, dtype=dtype)
    q = qkv[:, :heads * dim].view(-1, heads, dim)
    k = qkv[:, heads * dim:(heads + kv) * dim].view(-1, kv, dim)
    v = qkv[:, (heads + kv) * dim:].view(-1, kv, dim)
    kc, vc = (make_cache(s, pages, page, kv, dim, dtype, layout) for s in (3, 4))
    want_k, want_v = kc.double(), vc.double()
    rope = decode.rope_table(80, rot) if rot else None
    q_out = decode.append_kv(k, v, kc, vc, table, pos, seq_ids=seq, rope=rope, q=q, interleaved=interleaved)
    live = pos >= 0
    ids, at = seq[live].long(), pos[live].long()
    pg, slot = table[ids, at // page].long(), at % page
    turned = [t[live].double() for t in (k, q)]
    if rot:
        turned = [rotate64(t, rope, at, rot, interleaved) for t in turned]
    want_k[pg, slot] = turned[0]
    want_v[pg, slot] = v[live].double()
    near(kc, want_k, 8.0)
    assert torch.equal(vc.double(), want_v)
    untouched = torch.ones(pages, page, dtype=torch.bool, device="cuda")
    untouched[pg, slot] = False
    assert torch.equal(kc.double()[untouched], want_k[untouched])
    near(q_out[live], turned[1], 8.0)
    assert bool((q_out[4] == 0).all())


@pytest.mark.parametrize("interleaved,rot", [(False, 128), (True, 128), (False, 64), (True, 0)])
@pytest.mark.parametrize("heads,kv", [(31, 1), (8, 8)])
def test_append_many_tokens(heads, kv, interleaved, rot):
    """Tokens enough for threads of several heads, head counts that leave some without."""
    from heatvit_b200 import decode
    lens, dim, page = [3000, 1, 2049], 128, 64
    table, pages = make_table(1, lens, page)
    seq = torch.tensor(sum([[i] * n for i, n in enumerate(lens)], []), dtype=torch.int32, device="cuda")
    pos = torch.cat([torch.arange(n, dtype=torch.int32) for n in lens]).cuda()
    q, k, v = (rand(s, pos.numel(), n, dim, dtype=BF) for s, n in ((2, heads), (3, kv), (4, kv)))
    kc, vc = (make_cache(s, pages, page, kv, dim, BF, "hnd") for s in (5, 6))
    rope = decode.rope_table(3000, rot) if rot else None
    got = decode.append_kv(k, v, kc, vc, table, pos, seq_ids=seq, rope=rope, q=q, interleaved=interleaved)
    pg, slot = table[seq.long(), pos.long() // page].long(), pos.long() % page
    turned = [t.double() for t in (k, q)]
    if rot:
        turned = [rotate64(t, rope, pos.long(), rot, interleaved) for t in turned]
    near(kc[pg, slot], turned[0], 8.0)
    near(got, turned[1], 8.0)
    assert torch.equal(vc[pg, slot], v)


def test_append_decode_step_in_place_and_without_q():
    from heatvit_b200 import decode
    lens = [5, 1, 33]
    table, pages = make_table(1, lens, 16)
    pos = torch.tensor([n - 1 for n in lens], dtype=torch.int32, device="cuda")
    k, v, q = (rand(s, 3, 2, 64, dtype=BF) for s in (1, 2, 3))
    rope = decode.rope_table(64, 64)
    kc, vc, kc2, vc2 = (make_cache(5, pages, 16, 2, 64, BF, "nhd") for _ in range(4))
    got = decode.append_kv(k, v, kc, vc, table, pos, rope=rope, q=q)
    same = q.clone()
    assert decode.append_kv(k, v, kc2, vc2, table, pos, rope=rope, q=same, q_out=same) is same
    assert torch.equal(same, got) and torch.equal(kc, kc2)
    kc2.zero_()
    assert decode.append_kv(k, v, kc2, vc2, table, pos, rope=rope) is None
    pg = table[torch.arange(3), pos.long() // 16].long()
    assert torch.equal(kc2[pg, pos.long() % 16], kc[pg, pos.long() % 16])
    assert decode.append_kv(k[:0], v[:0], kc, vc, table, pos[:0]) is None


def test_append_reports_what_only_the_device_sees():
    """Positions past the tables, sequences past the page table, pages past the cache: nothing is stored."""
    from heatvit_b200 import abi, decode
    k, v = (rand(s, 1, 1, 64, dtype=BF) for s in (1, 2))
    kc, vc = (make_cache(s, 2, 4, 1, 64, BF, "nhd") for s in (5, 6))
    before = kc.clone(), vc.clone()
    i32 = dict(dtype=torch.int32, device="cuda")
    rope = decode.rope_table(3, 64)
    position, page = abi.HV_DECODE_BAD_POSITION, abi.HV_DECODE_BAD_PAGE
    for table, pos, seq, bit in (([[0, 1]], 8, 0, position), ([[0, 1]], 3, 0, position), ([[0, 1]], 0, 1, position),
                                 ([[0, 1]], 0, -1, position), ([[2, 1]], 0, 0, page), ([[-1, 1]], 0, 0, page)):
        decode.append_kv(k, v, kc, vc, torch.tensor(table, **i32), torch.tensor([pos], **i32),
                         seq_ids=torch.tensor([seq], **i32), rope=rope)
        assert decode.device_error() == bit
        assert torch.equal(kc, before[0]) and torch.equal(vc, before[1])


# ---- attention ----------------------------------------------------------------------

def plain_attention(q, kc, vc, table, lens, scale):
    """Outputs, log-sum-exps and the error bound, in 64 bits."""
    b, h, d = q.shape
    page, kv = kc.shape[1:3]
    out = torch.zeros(b, h, d, dtype=torch.float64, device="cuda")
    bound = torch.zeros_like(out)
    lse = torch.full((b, h), -math.inf, dtype=torch.float64, device="cuda")
    for i, n in enumerate(lens):
        if n <= 0:
            continue
        pg = table[i, :-(-n // page)].long()
        k, v = (c[pg].reshape(-1, kv, d)[:n].double().repeat_interleave(h // kv, 1) for c in (kc, vc))
        s = torch.einsum("hd,nhd->hn", q[i].double(), k) * scale
        size = torch.einsum("hd,nhd->hn", q[i].double().abs(), k.abs()) * abs(scale)
        p = torch.softmax(s, 1)
        out[i], lse[i] = torch.einsum("hn,nhd->hd", p, v), torch.logsumexp(s, 1)
        # the scores' 32-bit error is at most 2^-20 of the sum of absolute products, and moves a
        # weight by that; weights are rounded to q's type; joining adds a few 2^-24; then one rounding
        shift = size.amax(1, keepdim=True) * 2.0 ** -20
        bound[i] = torch.einsum("hn,nhd->hd", p, v.abs()) * (U[q.dtype] + 2 * shift + 2.0 ** -16) \
            + out[i].abs() * U[q.dtype] + 2.0 ** -24
    return out, lse, bound


def attend_case(seed, lens, heads, kv, dim, page, dtype, layout, spare=0, poison=True):
    table, pages = make_table(seed, lens, page, spare)
    kc, vc = (make_cache(seed + s, pages + 1, page, kv, dim, dtype, layout) for s in (1, 2))
    if poison:  # what no sequence owns, and the slots past each length, must not be read into the result
        live = torch.zeros(pages + 1, page, dtype=torch.bool, device="cuda")
        for i, n in enumerate(lens):
            if n > 0:
                t = torch.arange(n, device="cuda")
                live[table[i, t // page].long(), t % page] = True
        kc[~live] = math.nan
        vc[~live] = math.inf
    return rand(seed + 3, len(lens), heads, dim, dtype=dtype, scale=1.5), kc, vc, table


def check_attention(q, kc, vc, table, lens, scale=None, **kw):
    from heatvit_b200 import decode
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out, lse = decode.paged_attention(q, kc, vc, table, n, scale=scale, return_lse=True, **kw)
    want, want_lse, bound = plain_attention(q, kc, vc, table, lens, q.shape[2] ** -0.5 if scale is None else scale)
    assert bool(((out.double() - want).abs() <= bound).all()), float(((out.double() - want).abs() / bound).nan_to_num(9e9).max())
    live = torch.tensor([v > 0 for v in lens], device="cuda")
    assert bool((lse[~live] == -math.inf).all())
    assert bool(((lse.double() - want_lse)[live].abs() <= 1e-4 + 2.0 ** -18 * want_lse[live].abs()).all())
    return out


@pytest.mark.parametrize("dim", [32, 64, 96, 128, 192, 256])
@pytest.mark.parametrize("dtype,layout,page", [(BF, "nhd", 16), (HF, "hnd", 24), (BF, "hnd", 1)])
def test_attention_dims(dim, dtype, layout, page):
    lens = [0, 1, 15, 16, 17, 63, 64, 65, 300, 1029]
    q, kc, vc, table = attend_case(1, lens, 8, 2, dim, page, dtype, layout, spare=2)
    check_attention(q, kc, vc, table, lens)


@pytest.mark.parametrize("heads,kv", [(1, 1), (3, 3), (5, 1), (16, 1), (17, 1), (40, 2), (64, 64), (96, 3)])
def test_attention_head_layouts(heads, kv):
    lens = [130, 0, 1, 700]
    q, kc, vc, table = attend_case(2, lens, heads, kv, 64, 16, BF, "nhd")
    check_attention(q, kc, vc, table, lens)


@pytest.mark.parametrize("lens", [[1], [0], [0, 0, 0], [20000], [100000, 3], [9000, 0, 0, 12345, 1, 64], [64] * 400,
                                  [(7 * i) % 90 for i in range(1000)], [-5, 70]])
def test_attention_lengths(lens):
    """One token to long caches, empty rows, more sequences than CTAs, one sequence over all of them."""
    q, kc, vc, table = attend_case(3, [max(0, n) for n in lens], 4, 1, 128, 32, BF, "nhd", poison=max(lens) < 20001)
    check_attention(q, kc, vc, table, lens)


@pytest.mark.parametrize("lens", [[512] * 32, [470, 0, 512, 449] * 11, [1024] * 40 + [0] * 5, [150] * 75 + [600]])
def test_attention_lengths_of_as_many_tiles(lens):
    """Items of one size, whose borders the cuts are moved to, among empty rows; one that differs."""
    q, kc, vc, table = attend_case(5, lens, 32, 8, 128, 16, BF, "nhd")
    out = check_attention(q, kc, vc, table, lens)
    assert bool((out[torch.tensor(lens, device="cuda") == 0] == 0).all())


def test_attention_scale_and_wide_scores():
    """Scores over hundreds: the running maximum moves, and weights underflow to zero."""
    lens = [777, 64]
    q, kc, vc, table = attend_case(4, lens, 4, 2, 64, 16, HF, "nhd")
    check_attention(q * 8, kc, vc, table, lens, scale=1.0)
    check_attention(q, kc, vc, table, lens, scale=-0.3)
    check_attention(q, kc, vc, table, lens, scale=0.0)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("n,dead", [(40, 33), (700, 640), (30000, 12000)])
def test_attention_scores_out_of_range(dim, n, dead):
    """Leading tokens whose scores are -inf weigh nothing, as in the formula; all of them: a NaN, and lse -inf.
    A NaN in q is its head's alone, in the output and lse."""
    from heatvit_b200 import decode
    lens = [n, n, n]
    q, kc, vc, table = attend_case(6, lens, 4, 2, dim, 16, BF, "nhd")
    t = torch.arange(n, device="cuda")
    for b, stop in ((0, dead), (1, n)):
        at = t[:stop]
        kc[table[b, at // 16].long(), at % 16] = -1e30
    q[:2], q[2, 1, 3] = 1e30, math.nan
    rest = torch.arange(dead, n, device="cuda")
    kc[table[0, rest // 16].long(), rest % 16] = 0.0  # scores of 0: the mean of the values
    out, lse = decode.paged_attention(q, kc, vc, table, torch.tensor(lens, dtype=torch.int32, device="cuda"),
                                      return_lse=True)
    v = vc[table[0, rest // 16].long(), rest % 16].double().repeat_interleave(2, 1)  # [tokens, heads, dim]
    want, size = v.mean(0), v.abs().mean(0)
    # equal weights of one are exact, their sum too; the product's sum and the one rounding are not
    assert bool(((out[0].double() - want).abs() <= want.abs() * 2.0 ** -8 + size * 2.0 ** -14).all())
    assert bool(((lse[0].double() - math.log(n - dead)).abs() <= 1e-5).all())
    assert bool(out[1].isnan().all()) and bool((lse[1] == -math.inf).all())
    assert bool(out[2, 1].isnan().all()) and bool(lse[2, 1].isnan())
    others = [0, 2, 3]
    assert bool(out[2, others].isfinite().all()) and bool(lse[2, others].isfinite().all())


def test_attention_strided_q_and_out():
    """q as a slice of a projection at an odd place, out as every other row of a larger buffer."""
    from heatvit_b200 import decode
    lens = [100, 5, 0]
    q, kc, vc, table = attend_case(5, lens, 6, 2, 64, 16, BF, "hnd")
    wide = torch.zeros(3, 6 * 64 + 131, dtype=BF, device="cuda")
    odd = wide[:, 3:3 + 384].view(3, 6, 64)
    odd.copy_(q)
    buf = torch.full((6, 6, 64), 9.0, dtype=BF, device="cuda")
    want = check_attention(q, kc, vc, table, lens)
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    got = decode.paged_attention(odd, kc, vc, table, n, out=buf[::2])
    assert torch.equal(got, want) and bool((buf[1::2] == 9).all())


def test_attention_is_deterministic_and_shares_a_workspace():
    """Split sequences give the same bits each time; calls of other sizes in between leave the counters clean."""
    from heatvit_b200 import decode
    ws = decode.AttentionWorkspace()
    a = attend_case(6, [50000, 7, 30000], 8, 1, 128, 16, BF, "nhd", poison=False)
    b = attend_case(7, [4000, 100], 6, 3, 256, 16, HF, "nhd")
    first = check_attention(*a, [50000, 7, 30000], workspace=ws)
    for _ in range(3):
        check_attention(*b, [4000, 100], workspace=ws)
        assert torch.equal(check_attention(*a, [50000, 7, 30000], workspace=ws), first)


def test_cache_offsets_past_32_bits():
    """Pages whose element offsets pass 2^31, appended to and read."""
    from heatvit_b200 import decode
    kv, dim, page = 8, 128, 64
    pages = (1 << 31) // (kv * dim * page) + 40
    kc, vc = (torch.empty(pages, page, kv, dim, dtype=BF, device="cuda") for _ in range(2))
    table = torch.tensor([[pages - 1, 2, pages - 7]], dtype=torch.int32, device="cuda")
    n = 150
    k, v = rand(1, n, kv, dim, dtype=BF), rand(2, n, kv, dim, dtype=BF)
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    decode.append_kv(k, v, kc, vc, table, pos, seq_ids=torch.zeros_like(pos))
    assert torch.equal(kc[table[0].long()].reshape(-1, kv, dim)[:n], k)
    q = rand(3, 1, 32, dim, dtype=BF)
    check_attention(q, kc, vc, table, [n])


def test_attention_reports_bad_lengths_and_pages():
    from heatvit_b200 import abi, decode
    lens = [30, 40]
    q, kc, vc, table = attend_case(8, lens, 2, 2, 64, 16, BF, "nhd", poison=False)
    n = torch.tensor([30, 49], dtype=torch.int32, device="cuda")  # 48 is what the table can name
    table[1] = torch.tensor([0, 1, 2])
    good = decode.paged_attention(q, kc, vc, table, torch.tensor([30, 48], dtype=torch.int32, device="cuda"))
    assert decode.device_error() == 0
    assert torch.equal(decode.paged_attention(q, kc, vc, table, n), good)
    assert decode.device_error() == abi.HV_DECODE_BAD_LENGTH
    table[1, 1] = kc.shape[0]
    got = decode.paged_attention(q, kc, vc, table, torch.tensor([30, 48], dtype=torch.int32, device="cuda"))
    assert decode.device_error() == abi.HV_DECODE_BAD_PAGE
    assert torch.equal(got[0], good[0])


# ---- together -----------------------------------------------------------------------

def test_streams_and_graphs():
    """The step on a side stream and replayed from a CUDA graph equals the step on the default stream."""
    from heatvit_b200 import decode
    heads, kv, dim, width = 8, 2, 64, 512
    x, res, w = rand(1, 5, width, dtype=BF), rand(2, 5, width, dtype=BF), rand(3, width, dtype=BF)
    wq, ws = decode.quantize_weight_fp8(rand(4, (heads + 2 * kv) * dim, width, scale=0.05))
    lens = [1, 2000, 31, 6000, 400]
    table, pages = make_table(1, lens, 16)
    pos = torch.tensor([n - 1 for n in lens], dtype=torch.int32, device="cuda")
    n = pos + 1
    kc, vc = (make_cache(s, pages, 16, kv, dim, BF, "nhd") for s in (5, 6))
    rope = decode.rope_table(6000, dim)

    def step():
        r = decode.add_rmsnorm_fp8(x, w, residual=res)
        qkv = decode.gemm_fp8(r.q, r.scale, wq, ws).view(5, heads + 2 * kv, dim)
        q = decode.append_kv(qkv[:, heads:heads + kv], qkv[:, heads + kv:], kc, vc, table, pos, rope=rope,
                             q=qkv[:, :heads])
        return r.residual, qkv, decode.paged_attention(q, kc, vc, table, n)

    want = step()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for _ in range(3):
        for t in held:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))


def test_refusals():
    from heatvit_b200 import decode
    x, w = rand(1, 4, 64, dtype=BF), rand(2, 64, dtype=BF)
    cases = [
        (TypeError, lambda: decode.add_rmsnorm_fp8(x.double(), w)),
        (TypeError, lambda: decode.add_rmsnorm_fp8(x, w.float())),
        (ValueError, lambda: decode.add_rmsnorm_fp8(x, w[:63])),
        (ValueError, lambda: decode.add_rmsnorm_fp8(x.t(), w[:4])),
        (ValueError, lambda: decode.add_rmsnorm_fp8(x, w, residual=x[:3])),
        (ValueError, lambda: decode.add_rmsnorm_fp8(x, w, residual_out=x)),
        (ValueError, lambda: decode.add_rmsnorm_fp8(x, w, eps=-1.0)),
        (ValueError, lambda: decode.add_rmsnorm_fp8(x, w.cpu())),
    ]
    a, b, sa, sb = e4m3(1, 4, 256), e4m3(2, 130, 256), scales(3, 4, 2), scales(4, 2, 2)
    cases += [
        (TypeError, lambda: decode.gemm_fp8(a.float(), sa, b, sb)),
        (TypeError, lambda: decode.gemm_fp8(a, sa.double(), b, sb)),
        (TypeError, lambda: decode.gemm_fp8(a, sa, b, sb, out_dtype=torch.float64)),
        (ValueError, lambda: decode.gemm_fp8(a, sa, b[:, :128], sb)),
        (ValueError, lambda: decode.gemm_fp8(a, sa[:, :1], b, sb)),
        (ValueError, lambda: decode.gemm_fp8(a, sa, b, sb[:1])),
        (ValueError, lambda: decode.gemm_fp8(a[:, 8:], sa, b[:, 8:], sb)),  # rows that start on 8 bytes
        (ValueError, lambda: decode.gemm_fp8(a[:, :0], sa[:, :0], b[:, :0], sb[:, :0])),
        (ValueError, lambda: decode.gemm_fp8(a, sa, b, sb, out=torch.empty(4, 131, dtype=BF, device="cuda"))),
    ]
    lens = [20, 5]
    q, kc, vc, table = attend_case(1, lens, 4, 2, 64, 16, BF, "nhd")
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    k = rand(5, 2, 2, 64, dtype=BF)
    rope = decode.rope_table(32, 64)
    cases += [
        (TypeError, lambda: decode.paged_attention(q.float(), kc, vc, table, n)),
        (TypeError, lambda: decode.paged_attention(q.half(), kc, vc, table, n)),
        (TypeError, lambda: decode.paged_attention(q, kc, vc, table, n.long())),
        (ValueError, lambda: decode.paged_attention(q[:, :3], kc, vc, table, n)),
        (ValueError, lambda: decode.paged_attention(q, kc, vc, table[:1], n)),
        (ValueError, lambda: decode.paged_attention(q, kc, vc, table, n[:1])),
        (ValueError, lambda: decode.paged_attention(q, kc, vc[:1], table, n)),
        (ValueError, lambda: decode.paged_attention(q[:, :, :32], kc, vc, table, n)),
        (ValueError, lambda: decode.paged_attention(q[..., :40], kc[..., :40], vc[..., :40], table, n)),
        (ValueError, lambda: decode.paged_attention(q[..., 4:36], kc[..., 4:36], vc[..., 4:36], table, n)),
        (ValueError, lambda: decode.paged_attention(q, kc, vc, table, n, out=q[:1])),
        (TypeError, lambda: decode.append_kv(k.float(), k.float(), kc, vc, table, n)),
        (TypeError, lambda: decode.append_kv(k, k, kc, vc, table.long(), n)),
        (TypeError, lambda: decode.append_kv(k, k, kc, vc, table, n, rope=rope.double())),
        (ValueError, lambda: decode.append_kv(k, k[:1], kc, vc, table, n)),
        (ValueError, lambda: decode.append_kv(k, k, kc, vc, table, n[:1])),
        (ValueError, lambda: decode.append_kv(k, k, kc, vc, table[:1], n)),
        (ValueError, lambda: decode.append_kv(k, k, kc, vc, table, n, seq_ids=n[:1])),
        (ValueError, lambda: decode.append_kv(k, k, kc, vc, table, n, rope=decode.rope_table(32, 66))),
        (ValueError, lambda: decode.append_kv(k, k, kc, vc, table, n, q_out=q)),
        (ValueError, lambda: decode.append_kv(k, k, kc[:, :, :1], vc[:, :, :1], table, n)),
        (ValueError, lambda: decode.rope_table(4, 3)),
    ]
    for i, (kind, call) in enumerate(cases):
        with pytest.raises(kind):
            call()
            pytest.fail(f"case {i} was taken")
