"""Cases that measure the decode operators between a prompt and its next token: attention of a chunk of new
tokens over a paged cache, the cache append with a norm of each query and key head, and sampling.

``run`` computes a case with elementary torch operations in 32 bits (sampling in 64, since whole numbers come out of
comparisons of sums), or, with ``own`` set, through ``heatvit_b200.decode``.  ``exact`` gives the same outputs from
the definitions in 64 bits.
"""

import math

import torch

own = False

EPS = 1e-6
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # a few short continuations of short sequences, the example decoder's heads: the launch is what costs
        dict(name="chunk 4x5 over 300", op="chunk", seqs=4, new=5, past=300, spread="ragged", heads=8, kv_heads=2, dim=64,
             page=16, causal=True, dtype="bf16", layout="nhd"),
        # one unpruned image's tokens as a prompt that sees all of itself, the encoder's heads
        dict(name="chunk 1x197 whole", op="chunk", seqs=1, new=197, past=0, spread="same", heads=3, kv_heads=3, dim=64,
             page=16, causal=False, dtype="fp16", layout="nhd"),
        # drafted tokens of long sequences checked at once: the cache's bytes
        dict(name="chunk 16x6 over 32768", op="chunk", seqs=16, new=6, past=32768, spread="same", heads=32, kv_heads=8,
             dim=128, page=16, causal=True, dtype="bf16", layout="nhd"),
        # a ragged batch of prompts, an empty one among them
        dict(name="chunk 24 prompts", op="chunk", seqs=24, new=4001, past=0, spread="ragged", heads=24, kv_heads=6, dim=64,
             page=64, causal=True, dtype="fp16", layout="hnd"),
        # wide heads that share one key head, pages that end inside tiles
        dict(name="chunk 3x1499 wide", op="chunk", seqs=3, new=1499, past=2000, spread="ragged", heads=8, kv_heads=1,
             dim=256, page=24, causal=True, dtype="bf16", layout="nhd"),
        # a long prompt taken in chunks, one of the later ones: the tensor cores
        dict(name="chunk 8192 over 16384", op="chunk", seqs=1, new=8192, past=16384, spread="same", heads=32, kv_heads=8,
             dim=128, page=64, causal=True, dtype="bf16", layout="hnd"),
        # one decode step: each sequence adds one token
        dict(name="append 64 seqs", op="append", seqs=64, new=1, past=1000, heads=32, kv_heads=8, dim=128, rot=128, page=16,
             interleaved=False, dtype="bf16", layout="nhd"),
        # a ragged prompt batch, a part of the head rotated in neighbouring pairs, head-major pages
        dict(name="append 8 prompts", op="append", seqs=8, new=4001, past=0, heads=40, kv_heads=8, dim=96, rot=64, page=64,
             interleaved=True, dtype="fp16", layout="hnd"),
        # one token over the example decoder's vocabulary
        dict(name="sample 1x1000", op="sample", rows=1, vocab=1000, dtype="bf16", top_k=50, top_p=0.9, min_p=0.0,
             temperature=0.7, mixed=False),
        # a serving batch in which every request brings its own settings, an odd vocabulary
        dict(name="sample 48x50021 mixed", op="sample", rows=48, vocab=50021, dtype="fp32", top_k=40, top_p=0.95, min_p=0.05,
             temperature=1.0, mixed=True),
        # a large vocabulary, the usual nucleus
        dict(name="sample 256x131072 nucleus", op="sample", rows=256, vocab=131072, dtype="bf16", top_k=0, top_p=0.95,
             min_p=0.0, temperature=0.8, mixed=False),
        # rollouts from the whole distribution
        dict(name="sample 1024x65536 whole", op="sample", rows=1024, vocab=65536, dtype="fp32", top_k=0, top_p=1.0,
             min_p=0.0, temperature=1.0, mixed=False),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_one(rng):
    op = rng.choice(["chunk", "chunk", "append", "sample"])
    if op == "sample":
        top_k = rng.choice([0, 0, 1]) * _log_int(rng, 1, 1000)
        return dict(op=op, rows=_log_int(rng, 1, 1024), vocab=_log_int(rng, 1000, 262144), dtype=rng.choice(["bf16", "fp16", "fp32"]),
                    top_k=top_k, top_p=rng.choice([1.0, 0.5, 0.9, 0.95, 0.99]), min_p=rng.choice([0.0, 0.0, 0.02, 0.1]),
                    temperature=rng.choice([0.3, 0.7, 1.0, 1.5]), mixed=rng.random() < 0.3)
    kv = rng.choice([1, 2, 3, 4, 8, 16])
    case = dict(op=op, seqs=_log_int(rng, 1, 128), heads=kv * rng.choice([1, 2, 3, 4, 6, 8]), kv_heads=kv,
                dim=rng.choice([32, 64, 96, 128, 192, 256]), page=rng.choice([1, 16, 24, 64, 256]),
                dtype=rng.choice(["bf16", "fp16"]), layout=rng.choice(["nhd", "hnd"]))
    if op == "append":
        case.update(new=_log_int(rng, 1, 4096), past=_log_int(rng, 1, 4096), rot=rng.choice([case["dim"], case["dim"] // 2]),
                    interleaved=rng.random() < 0.5)
    else:
        case.update(new=_log_int(rng, 1, 8192), past=rng.choice([0, 1]) * _log_int(rng, 1, 65536),
                    spread=rng.choice(["same", "ragged"]), causal=rng.random() < 0.8)
    return case


def draw(rng):
    most = {}
    for c in listed():
        w = work(c)
        most[c["op"]] = max(most.get(c["op"], 0), w["bytes"], w["flops"] / 100)
    while True:
        case = _draw_one(rng)
        w = work(case)
        if max(w["bytes"], w["flops"] / 100) > most[case["op"]]:
            continue
        # what is prepared, and for an append compared, is no more than the largest caches listed
        if case["op"] != "sample" and sum(_past(case)) + sum(_counts(case)) > (1 << 29) // (case["kv_heads"] * case["dim"]):
            continue
        if case["op"] == "append" and sum(_past(case)) + sum(_counts(case)) > (1 << 28) // (case["kv_heads"] * case["dim"]):
            continue
        return case


def _counts(case):
    """New tokens of each sequence: an append from half of ``new`` to all of it; a chunk the same, or from none in even
    steps to ``new``."""
    n, b = case["new"], case["seqs"]
    if b == 1 or case.get("spread") == "same":
        return [n] * b
    if case["op"] == "append":
        return [n - (n // 2) * i // (b - 1) for i in range(b)]
    return [n * i // (b - 1) for i in range(b)]


def _past(case):
    """Tokens that each sequence already has in the cache."""
    p, b = case["past"], case["seqs"]
    if case.get("spread") == "same":
        return [p] * b
    return [p * (i + 1) // b for i in range(b)]


def work(case):
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * (4 if case["dtype"] == "fp32" else 2) + case["rows"] * 32, "flops": 4 * n}
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    counts, past = _counts(case), _past(case)
    t = sum(counts)
    if case["op"] == "append":
        return {"bytes": t * (4 * d * (h + 2 * kv) + 8) + 4 * min(t, case["past"] + case["new"]) * case["rot"] + 4 * d,
                "flops": t * (h + kv) * (4 * d + 3 * case["rot"])}
    cached = sum(p + n for p, n in zip(past, counts) if n)
    pairs = sum(n * (p + n) - (n * (n - 1) // 2 if case["causal"] else 0) for p, n in zip(past, counts))
    return {"bytes": 4 * t * h * d + 4 * cached * kv * d + 4 * cached // case["page"], "flops": 4 * pairs * h * d}


def _normal(gen, *shape, scale=1.0, dtype=torch.float32):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32).mul_(scale).to(dtype)


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
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case=case, op=case["op"])
    if case["op"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        # a broad bulk, and in every row some dozen likely tokens above it, the first far ahead in some rows and not in others
        z = _normal(gen, rows, vocab, scale=2.0)
        at = torch.randint(0, vocab, (rows, 40), generator=gen, device="cuda")
        lift = -torch.rand(rows, 40, generator=gen, device="cuda").log_() * 3 + torch.rand(rows, 1, generator=gen, device="cuda") * 8
        s["logits"] = z.scatter_add_(1, at, lift).to(TYPES[case["dtype"]])
        s["uniform"] = torch.rand(rows, generator=gen, device="cuda")
        for name, kind in (("temperature", torch.float32), ("top_k", torch.int32), ("top_p", torch.float32), ("min_p", torch.float32)):
            s[name] = torch.full((rows,), case[name], dtype=kind, device="cuda")
        if case["mixed"]:  # some requests leave a setting out, some are greedy
            i = torch.randperm(rows, generator=gen, device="cuda")
            s["temperature"] *= 0.5 + (i % 8) / 4
            s["temperature"][i % 7 == 3] = 0
            s["top_k"][i % 3 == 0] = 0
            s["top_p"][i % 4 == 1] = 1
            s["min_p"][i % 5 != 2] = 0
        return s
    dtype = TYPES[case["dtype"]]
    h, kv, d, seqs = case["heads"], case["kv_heads"], case["dim"], case["seqs"]
    order = torch.randperm(seqs, generator=gen, device="cuda").tolist()
    counts, past = [_counts(case)[i] for i in order], [_past(case)[i] for i in order]
    s["page_table"], pages = _page_table(gen, [p + c for p, c in zip(past, counts)], case["page"])
    n = torch.tensor(counts, device="cuda")
    if case["op"] == "chunk":
        s["counts"], s["past"] = counts, past
        s["starts"] = torch.nn.functional.pad(torch.cumsum(n, 0), (1, 0)).to(torch.int32)
        s["lens"] = (n + torch.tensor(past, device="cuda")).to(torch.int32)
        s["q"] = _normal(gen, sum(counts), h, d, scale=1.5, dtype=dtype)
        s["k_cache"], s["v_cache"] = _cache(gen, pages, case, True), _cache(gen, pages, case, True)
        return s
    first = torch.cumsum(n, 0) - n
    s["seq_ids"] = torch.repeat_interleave(torch.arange(seqs, device="cuda"), n).to(torch.int32)
    ids = s["seq_ids"].long()
    s["positions"] = (torch.arange(ids.numel(), device="cuda") - first[ids] + torch.tensor(past, device="cuda")[ids]).to(torch.int32)
    s["seq_ids"] = None if case["new"] == 1 else s["seq_ids"]  # one token a sequence needs no map
    qkv = _normal(gen, ids.numel(), (h + 2 * kv) * d, scale=2.0, dtype=dtype)  # the projection's output, split in place
    s["q"] = qkv[:, :h * d].view(-1, h, d)
    s["k"] = qkv[:, h * d:(h + kv) * d].view(-1, kv, d)
    s["v"] = qkv[:, (h + kv) * d:].view(-1, kv, d)
    s["q_weight"], s["k_weight"] = ((1 + _normal(gen, d, scale=0.2)).to(dtype) for _ in range(2))
    s["k_cache"], s["v_cache"] = _cache(gen, pages, case, False), _cache(gen, pages, case, False)
    half = case["rot"] // 2
    angle = torch.arange(case["past"] + case["new"], device="cuda", dtype=torch.float64)[:, None] * \
        10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
    s["rope"] = torch.cat([angle.cos(), angle.sin()], 1).float()  # [position, cosines then sines]
    return s


def _plain_chunk(s):
    page, kv, d = s["k_cache"].shape[1:]
    h = s["q"].shape[1]
    out = torch.empty_like(s["q"])
    first = 0
    for i, (n, past) in enumerate(zip(s["counts"], s["past"])):
        length = past + n
        if n == 0:
            continue
        pages = s["page_table"][i, :-(-length // page)].long()
        keys, values = (c[pages].flatten(0, 1)[:length].float().transpose(0, 1) for c in (s["k_cache"], s["v_cache"]))  # [kv, length, d]
        at = torch.arange(length, device="cuda")
        step = max(1, (1 << 30) // (h * length))  # rows whose scores are held at one time
        for r in range(0, n, step):
            q = s["q"][first + r:first + min(n, r + step)].float()
            m = q.shape[0]
            q = q.view(m, kv, h // kv, d).permute(1, 2, 0, 3).reshape(kv, -1, d)
            scores = torch.matmul(q, keys.transpose(1, 2)).mul_(d ** -0.5).view(kv, h // kv, m, length)
            if s["case"]["causal"]:
                seen = past + r + torch.arange(m, device="cuda")
                scores.masked_fill_(at[None, :] > seen[:, None], -math.inf)
            p = scores.sub_(scores.amax(3, keepdim=True)).exp_()
            total = p.sum(3, keepdim=True)
            o = torch.matmul(p.view(kv, -1, length), values).view(kv, h // kv, m, d) / total
            out[first + r:first + r + m] = o.permute(2, 0, 1, 3).reshape(m, h, d).to(out.dtype)
        first += n
    return out


def _normed(x, weight):
    x = x.float()
    return x * torch.rsqrt((x * x).mean(2, keepdim=True) + EPS) * weight.float()


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
    s["k_cache"][page, slot] = _rotated(_normed(s["k"], s["k_weight"]), cos_sin, interleaved).to(s["k"].dtype)
    s["v_cache"][page, slot] = s["v"]
    return s["k_cache"], s["v_cache"], _rotated(_normed(s["q"], s["q_weight"]), cos_sin, interleaved).to(s["q"].dtype)


def _plain_sample(s):
    # in 64 bits: a token comes of comparing sums, and next to a border the last bits decide
    z = s["logits"].double()
    rows, vocab = z.shape
    greedy = s["temperature"] <= 0
    t = (z - z.amax(1, keepdim=True)) / torch.where(greedy, 1.0, s["temperature"].double())[:, None]
    t, order = t.sort(dim=1, descending=True, stable=True)  # ties: the lowest index first
    w = t.exp()
    rank = torch.arange(vocab, device="cuda")[None, :]
    keep = (rank < torch.where(s["top_k"] > 0, s["top_k"], vocab)[:, None]) & (w >= s["min_p"].double()[:, None])
    keep &= ~greedy[:, None] | (rank == 0)
    w = w * keep
    before = w.cumsum(1) - w
    keep &= (before < s["top_p"].double()[:, None] * w.sum(1, keepdim=True)) | (s["top_p"] >= 1)[:, None]
    w = torch.zeros_like(w).scatter_(1, order, w * keep)  # in the vocabulary's order
    cdf = w.cumsum(1)
    token = (cdf <= s["uniform"].double()[:, None] * cdf[:, -1:]).sum(1, keepdim=True)
    return token.squeeze(1), (w.gather(1, token) / cdf[:, -1:]).log().squeeze(1).float()


def run(s):
    if own:
        from heatvit_b200 import decode
        if s["op"] == "chunk":
            return decode.paged_chunk_attention(s["q"], s["k_cache"], s["v_cache"], s["page_table"], s["lens"], s["starts"],
                                                causal=s["case"]["causal"])
        if s["op"] == "append":
            q = decode.append_kv(s["k"], s["v"], s["k_cache"], s["v_cache"], s["page_table"], s["positions"],
                                 seq_ids=s["seq_ids"], rope=s["rope"], q=s["q"], interleaved=s["case"]["interleaved"],
                                 q_weight=s["q_weight"], k_weight=s["k_weight"], eps=EPS)
            return s["k_cache"], s["v_cache"], q
        return decode.sample_tokens(s["logits"], s["uniform"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                                    min_p=s["min_p"], return_logprob=True)
    return {"chunk": _plain_chunk, "append": _plain_append, "sample": _plain_sample}[s["op"]](s)


def _exact_chunk(s):
    page, kv, d = s["k_cache"].shape[1:]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    starts = s["starts"].tolist()
    for i, length in enumerate(s["lens"].tolist()):
        at = torch.arange(length, device="cuda")
        rows = torch.arange(starts[i], starts[i + 1], device="cuda")
        if not rows.numel():
            continue
        where = s["page_table"][i][at // page].long(), at % page
        k, v = s["k_cache"][where].double(), s["v_cache"][where].double()
        for part in rows.split(max(1, (1 << 28) // (out.shape[1] * length))):
            q = s["q"][part].double().unflatten(1, (kv, -1))
            x = torch.einsum("nkgd,lkd->kgnl", q, k) / math.sqrt(d)
            if s["case"]["causal"]:
                newest = length - starts[i + 1] + part
                x = x + torch.where(at[None, :] <= newest[:, None], 0.0, -math.inf)
            out[part] = torch.einsum("kgnl,lkd->nkgd", torch.softmax(x, 3), v).flatten(1, 2)
    return out


def _exact_append(s):
    pos, page, slot = _slots(s)
    half = s["rope"].shape[1] // 2
    angle = s["rope"][pos].double()  # the table is an input: its float32 values are what is applied
    turn = torch.complex(angle[:, :half], angle[:, half:])[:, None, :]

    def turned(x, weight):
        x = x.double()
        x = x / torch.sqrt(torch.linalg.vector_norm(x, dim=2, keepdim=True) ** 2 / x.shape[2] + EPS) * weight.double()
        if s["case"]["interleaved"]:
            pairs = torch.view_as_complex(x[:, :, :2 * half].unflatten(2, (half, 2)).contiguous())
            x[:, :, :2 * half] = torch.view_as_real(pairs * turn).flatten(2)
        else:
            z = torch.complex(x[:, :, :half].contiguous(), x[:, :, half:2 * half].contiguous()) * turn
            x[:, :, :half], x[:, :, half:2 * half] = z.real, z.imag
        return x

    k_cache, v_cache = s["k_cache"].double(), s["v_cache"].double()
    k_cache[page, slot] = turned(s["k"], s["k_weight"])
    v_cache[page, slot] = s["v"].double()
    return k_cache, v_cache, turned(s["q"], s["q_weight"])


def _exact_sample(s):
    tokens, logprobs = [], []
    limits = zip(s["temperature"].tolist(), s["top_k"].tolist(), s["top_p"].tolist(), s["min_p"].tolist(), s["uniform"].tolist())
    for z, (temperature, top_k, top_p, min_p, u) in zip(s["logits"], limits):
        z = z.double()
        if temperature <= 0:
            tokens.append(int((z == z.max()).int().argmax()))
            logprobs.append(0.0)
            continue
        z = z / temperature
        kept = torch.argsort(-z, stable=True)[:top_k or None]
        p = torch.softmax(z, 0)
        kept = kept[p[kept] >= min_p * p.max()]
        if top_p < 1:
            mass = torch.cumsum(p[kept], 0)
            kept = kept[:int((mass < top_p * mass[-1]).sum()) + 1]
        kept = kept.sort().values
        mass = torch.cumsum(p[kept], 0)
        i = min(int(torch.searchsorted(mass, u * mass[-1], right=True)), kept.numel() - 1)
        tokens.append(int(kept[i]))
        logprobs.append(float((p[kept[i]] / mass[-1]).log()))
    return torch.tensor(tokens, device="cuda"), torch.tensor(logprobs, dtype=torch.float64, device="cuda")


def exact(case, seed):
    s = prepare(case, seed)
    return {"chunk": _exact_chunk, "append": _exact_append, "sample": _exact_sample}[case["op"]](s)
