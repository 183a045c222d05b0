"""Cases that measure the decode operators: residual RMSNorm with an e4m3 output, the block-scaled e4m3 GEMM,
the rotating paged-cache append, and paged single-token attention.

``run`` computes a case with elementary torch operations in 32 bits, or, with ``own`` set, through
``heatvit_b200.decode``.  ``exact`` gives the same outputs from the definitions in 64 bits.
"""

import math

import torch

own = False

E4M3_MAX = 448.0
AMAX_FLOOR = 2.0 ** -100  # an all-zero block's scale stays a normal float32
EPS = 1e-6
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # one decode step of a few sequences: the launch is what costs
        dict(name="norm 8x4096", op="norm", rows=8, dim=4096, dtype="bf16", residual=True),
        # a packed ragged batch in float32, neither size a multiple of a block
        dict(name="norm 1999x5000 fp32", op="norm", rows=1999, dim=5000, dtype="fp32", residual=True),
        # a long prompt batch through a wide layer
        dict(name="norm 16384x8192", op="norm", rows=16384, dim=8192, dtype="bf16", residual=True),
        # a single token against a square projection: the weights' bytes
        dict(name="gemm 1x4096x4096", op="gemm", m=1, n=4096, k=4096, out="bf16"),
        # a decode batch against a wide up-projection
        dict(name="gemm 48x10240x4096", op="gemm", m=48, n=10240, k=4096, out="bf16"),
        # the tokens of eight unpruned images through the encoder's own FFN width, odd rows, K a block and a half
        dict(name="gemm 1576x768x192", op="gemm", m=1576, n=768, k=192, out="fp16"),
        # prompt processing: the tensor cores
        dict(name="gemm 8192x8192x8192", op="gemm", m=8192, n=8192, k=8192, out="bf16"),
        # one decode step: each sequence adds one token
        dict(name="append 64 seqs", op="append", seqs=64, new=1, past=1000, heads=32, kv_heads=8, dim=128, rot=128,
             page=16, interleaved=False, dtype="bf16", layout="nhd"),
        # a ragged prompt batch, half the head rotated in neighbouring pairs, head-major pages
        dict(name="append 24 prompts", op="append", seqs=24, new=2047, past=0, heads=24, kv_heads=6, dim=64, rot=32,
             page=64, interleaved=True, dtype="fp16", layout="hnd"),
        # the encoder's three heads over the tokens of one image
        dict(name="attend 1x197", op="attend", seqs=1, longest=197, heads=3, kv_heads=3, dim=64, page=16,
             spread="same", dtype="fp16", layout="nhd"),
        # a serving batch: lengths from an idle slot to the longest, shared key heads
        dict(name="attend 64 ragged", op="attend", seqs=64, longest=8192, heads=32, kv_heads=8, dim=128, page=16,
             spread="ragged", dtype="bf16", layout="nhd"),
        # two long contexts: the work has to be split over the cache's length
        dict(name="attend 2x131072", op="attend", seqs=2, longest=131071, heads=64, kv_heads=8, dim=128, page=64,
             spread="same", dtype="bf16", layout="hnd"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _size(rng, lo, hi):
    """A size of [lo, hi], as often a multiple of 128 as an odd one."""
    v = _log_int(rng, lo, hi)
    return min(hi, (v + 127) // 128 * 128) if rng.random() < 0.5 else v


def _draw_one(rng):
    op = rng.choice(["norm", "gemm", "append", "attend"])
    if op == "norm":
        return dict(op=op, rows=_log_int(rng, 1, 32768), dim=_size(rng, 64, 16384),
                    dtype=rng.choice(["bf16", "fp16", "fp32"]), residual=rng.random() < 0.7)
    if op == "gemm":
        return dict(op=op, m=_log_int(rng, 1, 16384), n=_size(rng, 64, 16384), k=_size(rng, 64, 16384),
                    out=rng.choice(["bf16", "fp16"]))
    kv = rng.choice([1, 2, 3, 4, 8, 16])
    dim = rng.choice([64, 96, 128, 256])
    case = dict(op=op, seqs=_log_int(rng, 1, 256), heads=kv * rng.choice([1, 2, 3, 4, 8]), kv_heads=kv, dim=dim,
                page=rng.choice([1, 16, 24, 64, 256]), dtype=rng.choice(["bf16", "fp16"]),
                layout=rng.choice(["nhd", "hnd"]))
    if op == "append":
        case.update(new=_log_int(rng, 1, 4096), past=_log_int(rng, 1, 4096), rot=rng.choice([dim, dim // 2]),
                    interleaved=rng.random() < 0.5)
    else:
        case.update(longest=_log_int(rng, 1, 131072), spread=rng.choice(["same", "ragged"]))
    return case


def draw(rng):
    most = {}
    for c in listed():
        w = work(c)
        most[c["op"]] = max(most.get(c["op"], 0), w["bytes"], w["flops"] / 50)
    while True:
        case = _draw_one(rng)
        w = work(case)
        if max(w["bytes"], w["flops"] / 50) > most[case["op"]]:
            continue
        if case["op"] == "append" and case["seqs"] * (case["new"] + case["past"]) * case["kv_heads"] * case["dim"] > 1 << 28:
            continue  # the caches alone would be what is prepared and compared
        return case


def _counts(case):
    """Tokens that each sequence appends: the same, or from half of ``new`` to all of it."""
    n, b = case["new"], case["seqs"]
    return [n - (n // 2) * i // max(1, b - 1) if b > 1 else n for i in range(b)]


def _lengths(case):
    """Cached tokens of each sequence: the same, or from an idle slot (0) to the longest in even steps."""
    b, n = case["seqs"], case["longest"]
    return [n] * b if case["spread"] == "same" or b == 1 else [n * i // (b - 1) for i in range(b)]


def work(case):
    if case["op"] == "norm":
        rows, dim, size = case["rows"], case["dim"], 4 if case["dtype"] == "fp32" else 2
        streams = 3 if case["residual"] else 1  # x, the residual, and their sum written back
        return {"bytes": rows * dim * (streams * size + 1) + rows * -(-dim // 128) * 4 + dim * size,
                "flops": 6 * rows * dim}
    if case["op"] == "gemm":
        m, n, k = case["m"], case["n"], case["k"]
        groups = -(-k // 128)
        return {"bytes": m * k + n * k + 2 * m * n + 4 * groups * (m + -(-n // 128)), "flops": 2 * m * n * k}
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "append":
        t = sum(_counts(case))
        return {"bytes": t * (4 * d * (h + 2 * kv) + 8) + 4 * min(t, case["new"]) * case["rot"],
                "flops": 3 * t * (h + kv) * case["rot"]}
    t = sum(_lengths(case))
    return {"bytes": 4 * t * kv * d + 4 * case["seqs"] * h * d + 4 * t // case["page"], "flops": 4 * t * h * d}


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(gen, *shape, scale=1.0, dtype=torch.float32):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32).mul_(scale).to(dtype)


def _quantized(gen, rows, k, block_rows, scale):
    """Random e4m3 rows of a stride that is a multiple of 16, with the scale of each (block_rows x 128) block."""
    groups = -(-k // 128)
    blocks = -(-rows // block_rows)
    # blocks of different magnitude, as outlier channels and rows give them
    scales = torch.rand(groups, blocks, generator=gen, device="cuda").mul_(2.0).sub_(1.0).exp_().mul_(scale / 128).t()
    stored = torch.empty(rows, -(-k // 16) * 16, device="cuda", dtype=torch.float8_e4m3fn)
    step = max(1, (1 << 27) // stored.shape[1])
    for r in range(0, rows, step):
        part = stored[r:r + step]
        part.copy_((torch.randn(part.shape, generator=gen, device="cuda") * 128).clamp_(-E4M3_MAX, E4M3_MAX))
    return stored[:, :k], scales


def _cache(gen, pages, case, filled):
    n, d, dtype = case["kv_heads"], case["dim"], TYPES[case["dtype"]]
    shape = (pages, case["page"], n, d) if case["layout"] == "nhd" else (pages, n, case["page"], d)
    t = torch.zeros(shape, dtype=dtype, device="cuda")
    if filled:
        step = max(1, (1 << 27) // (n * d * case["page"]))
        for p in range(0, pages, step):
            t[p:p + step].copy_(torch.randn(t[p:p + step].shape, generator=gen, device="cuda"))
    return t if case["layout"] == "nhd" else t.transpose(1, 2)  # [pages, page, kv_heads, dim] either way


def _page_table(gen, lengths, page):
    """Pages in random order; entries past a sequence's length are -1."""
    need = torch.tensor([-(-n // page) for n in lengths], device="cuda")
    total = int(need.sum())
    table = torch.full((len(lengths), max(1, int(need.max()))), -1, dtype=torch.int32, device="cuda")
    used = torch.arange(table.shape[1], device="cuda")[None, :] < need[:, None]
    table[used] = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
    return table, max(1, total)


def prepare(case, seed):
    gen = _generator(seed)
    s = dict(case=case, op=case["op"])
    if case["op"] == "norm":
        dtype = TYPES[case["dtype"]]
        rows, dim = case["rows"], case["dim"]
        s["x"] = _normal(gen, rows, dim, dtype=dtype)
        s["residual"] = _normal(gen, rows, dim, scale=3.0, dtype=dtype) if case["residual"] else None
        s["weight"] = (1 + _normal(gen, dim, scale=0.2)).to(dtype)
    elif case["op"] == "gemm":
        s["a"], s["a_scale"] = _quantized(gen, case["m"], case["k"], 1, 1.0)
        s["b"], s["b_scale"] = _quantized(gen, case["n"], case["k"], 128, 0.03)
        s["out"] = TYPES[case["out"]]
    elif case["op"] == "append":
        dtype = TYPES[case["dtype"]]
        h, kv, d = case["heads"], case["kv_heads"], case["dim"]
        order = torch.randperm(case["seqs"], generator=gen, device="cuda").tolist()
        counts = [_counts(case)[i] for i in order]
        past = [case["past"] * (i + 1) // case["seqs"] for i in order]
        s["page_table"], pages = _page_table(gen, [p + c for p, c in zip(past, counts)], case["page"])
        n = torch.tensor(counts, device="cuda")
        first = torch.cumsum(n, 0) - n
        s["seq_ids"] = torch.repeat_interleave(torch.arange(case["seqs"], device="cuda"), n).to(torch.int32)
        ids = s["seq_ids"].long()
        s["positions"] = (torch.arange(ids.numel(), device="cuda") - first[ids]
                          + torch.tensor(past, device="cuda")[ids]).to(torch.int32)
        # one token a sequence needs no map from tokens to sequences
        s["seq_ids"] = None if case["new"] == 1 else s["seq_ids"]
        qkv = _normal(gen, ids.numel(), (h + 2 * kv) * d, dtype=dtype)  # the projection's output, split in place
        s["q"] = qkv[:, :h * d].view(-1, h, d)
        s["k"] = qkv[:, h * d:(h + kv) * d].view(-1, kv, d)
        s["v"] = qkv[:, (h + kv) * d:].view(-1, kv, d)
        s["k_cache"], s["v_cache"] = _cache(gen, pages, case, False), _cache(gen, pages, case, False)
        half = case["rot"] // 2
        angle = torch.arange(case["past"] + case["new"], device="cuda", dtype=torch.float64)[:, None] * \
            10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
        s["rope"] = torch.cat([angle.cos(), angle.sin()], 1).float()  # [position, cosines then sines]
    else:
        lengths = _lengths(case)
        order = torch.randperm(case["seqs"], generator=gen, device="cuda").tolist()
        lengths = [lengths[i] for i in order]
        s["page_table"], pages = _page_table(gen, lengths, case["page"])
        s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        s["q"] = _normal(gen, case["seqs"], case["heads"], case["dim"], scale=1.5, dtype=TYPES[case["dtype"]])
        s["k_cache"], s["v_cache"] = _cache(gen, pages, case, True), _cache(gen, pages, case, True)
    return s


def _plain_norm(s):
    h = s["x"].float()
    if s["residual"] is not None:
        h = h + s["residual"].float()
    y = h * torch.rsqrt((h * h).mean(1, keepdim=True) + EPS) * s["weight"].float()
    rows, dim = y.shape
    groups = -(-dim // 128)
    y = torch.nn.functional.pad(y, (0, groups * 128 - dim)).view(rows, groups, 128)
    scale = y.abs().amax(2).clamp(min=AMAX_FLOOR) / E4M3_MAX
    q = (y / scale[:, :, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    summed = h.to(s["x"].dtype) if s["residual"] is not None else None
    return q.view(rows, -1)[:, :dim], scale, summed


def _spread(scale, rows, k, block_rows):
    """Each element's scale, from a scale for each (block_rows x 128) block."""
    if block_rows > 1:
        scale = scale.repeat_interleave(block_rows, 0)[:rows]
    return scale.repeat_interleave(128, 1)[:, :k]


def _plain_gemm(s):
    a, b = s["a"].float(), s["b"].float()
    a = a * _spread(s["a_scale"], a.shape[0], a.shape[1], 1)
    b = b * _spread(s["b_scale"], b.shape[0], b.shape[1], 128)
    return torch.matmul(a, b.t()).to(s["out"])


def _rotated(x, cos_sin, interleaved):
    """x [tokens, heads, dim] with its first 2 * half elements rotated; cos_sin [tokens, cosines then sines]."""
    half = cos_sin.shape[1] // 2
    cos, sin = cos_sin[:, None, :half], cos_sin[:, None, half:]
    turned, kept = x[:, :, :2 * half], x[:, :, 2 * half:]
    u, w = (turned[:, :, 0::2], turned[:, :, 1::2]) if interleaved else (turned[:, :, :half], turned[:, :, half:])
    pair = (u * cos - w * sin, u * sin + w * cos)
    turned = torch.stack(pair, 3).flatten(2) if interleaved else torch.cat(pair, 2)
    return torch.cat([turned, kept], 2)


def _slots(s):
    page = s["k_cache"].shape[1]
    pos = s["positions"].long()
    seq = s["seq_ids"].long() if s["seq_ids"] is not None else torch.arange(pos.numel(), device=pos.device)
    return pos, s["page_table"][seq, pos // page].long(), pos % page


def _plain_append(s):
    pos, page, slot = _slots(s)
    cos_sin, interleaved = s["rope"][pos], s["case"]["interleaved"]
    s["k_cache"][page, slot] = _rotated(s["k"].float(), cos_sin, interleaved).to(s["k"].dtype)
    s["v_cache"][page, slot] = s["v"]
    return s["k_cache"], s["v_cache"], _rotated(s["q"].float(), cos_sin, interleaved).to(s["q"].dtype)


def _plain_attend(s):
    page, kv, d = s["k_cache"].shape[1:]
    q = s["q"].float()
    b, h = q.shape[:2]
    table = s["page_table"].clamp(min=0).long()
    keys, values = (c[table].flatten(1, 2).float().transpose(1, 2) for c in (s["k_cache"], s["v_cache"]))
    scores = torch.matmul(q.view(b, kv, h // kv, d), keys.transpose(2, 3)) * d ** -0.5
    seen = torch.arange(scores.shape[3], device=q.device)[None, :] < s["lengths"][:, None]
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    top = scores.amax(3, keepdim=True).clamp(min=-3e38)  # an empty sequence has no largest score
    p = (scores - top).exp()
    total = p.sum(3, keepdim=True)
    out = torch.matmul(p, values) / torch.where(total > 0, total, 1.0)  # and zeros for its output
    return out.view(b, h, d).to(s["q"].dtype)


def run(s):
    if not own:
        return {"norm": _plain_norm, "gemm": _plain_gemm, "append": _plain_append, "attend": _plain_attend}[s["op"]](s)
    from heatvit_b200 import decode
    if s["op"] == "norm":
        r = decode.add_rmsnorm_fp8(s["x"], s["weight"], EPS, residual=s["residual"])
        return r.q, r.scale, r.residual
    if s["op"] == "gemm":
        return decode.gemm_fp8(s["a"], s["a_scale"], s["b"], s["b_scale"], out_dtype=s["out"])
    if s["op"] == "append":
        q = decode.append_kv(s["k"], s["v"], s["k_cache"], s["v_cache"], s["page_table"], s["positions"],
                             seq_ids=s["seq_ids"], rope=s["rope"], q=s["q"], interleaved=s["case"]["interleaved"])
        return s["k_cache"], s["v_cache"], q
    return decode.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["page_table"], s["lengths"])


def _exact_norm(s):
    q, scale, total = [], [], []
    dim = s["x"].shape[1]
    edges = list(range(0, dim, 128)) + [dim]
    for r in range(0, s["x"].shape[0], 2048):
        h = s["x"][r:r + 2048].double()
        if s["residual"] is not None:
            h = h + s["residual"][r:r + 2048].double()
            total.append(h)
        rms = torch.sqrt(h.pow(2).sum(1) / dim + EPS)
        y = h / rms[:, None] * s["weight"].double()
        tops = torch.stack([y[:, i:j].abs().max(1).values for i, j in zip(edges, edges[1:])], 1)
        tops = torch.clamp(tops, min=AMAX_FLOOR) / E4M3_MAX
        q.append(torch.cat([(y[:, i:j] / tops[:, n:n + 1]).float().to(torch.float8_e4m3fn)
                            for n, (i, j) in enumerate(zip(edges, edges[1:]))], 1))
        scale.append(tops)
    return torch.cat(q), torch.cat(scale), torch.cat(total) if total else None


def _exact_gemm(s):
    m, k = s["a"].shape
    out = torch.zeros(m, s["b"].shape[0], dtype=torch.float64, device="cuda")
    for g, i in enumerate(range(0, k, 128)):
        a = s["a"][:, i:i + 128].double() * s["a_scale"][:, g:g + 1].double()
        b = s["b"][:, i:i + 128].double()
        rows = torch.arange(b.shape[0], device="cuda") // 128
        out.addmm_(a, (b * s["b_scale"][rows, g].double()[:, None]).t())
    return out


def _exact_append(s):
    pos, page, slot = _slots(s)
    half = s["rope"].shape[1] // 2
    angle = s["rope"][pos].double()  # the table is an input: its float32 values are what is applied
    turn = torch.complex(angle[:, :half], angle[:, half:])[:, None, :]

    def rotate(x):
        x = x.double()
        if s["case"]["interleaved"]:
            pairs = torch.view_as_complex(x[:, :, :2 * half].unflatten(2, (half, 2)).contiguous())
            x[:, :, :2 * half] = torch.view_as_real(pairs * turn).flatten(2)
        else:
            z = torch.complex(x[:, :, :half].contiguous(), x[:, :, half:2 * half].contiguous()) * turn
            x[:, :, :half], x[:, :, half:2 * half] = z.real, z.imag
        return x

    k_cache, v_cache = s["k_cache"].double(), s["v_cache"].double()
    k_cache[page, slot] = rotate(s["k"])
    v_cache[page, slot] = s["v"].double()
    return k_cache, v_cache, rotate(s["q"])


def _exact_attend(s):
    kv, d = s["k_cache"].shape[2:]
    page = s["k_cache"].shape[1]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for i, n in enumerate(s["lengths"].tolist()):
        if not n:
            continue
        pages = s["page_table"][i, :-(-n // page)].long()
        k = s["k_cache"][pages].reshape(-1, kv, d)[:n].double()
        v = s["v_cache"][pages].reshape(-1, kv, d)[:n].double()
        q = s["q"][i].double().view(kv, -1, d)
        p = torch.softmax(torch.einsum("hgd,nhd->hgn", q, k) / math.sqrt(d), 2)
        out[i] = torch.einsum("hgn,nhd->hgd", p, v).reshape(-1, d)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "gemm": _exact_gemm, "append": _exact_append, "attend": _exact_attend}[case["op"]](s)
