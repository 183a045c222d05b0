"""Tokens of text from images: the integer encoder, then a small language decoder that reads
its pruned tokens, one new token a step.

    python examples/describe_images.py [--images 8] [--steps 16] [--prompt-attention] [--temperature 0.8 --top-p 0.9]

The encoder is the benchmark model with its selectors, so that each image keeps another number
of tokens.  Those, as the last block leaves them, become the first entries of a paged cache of
keys and values in every decoder layer; a step then runs each layer with the operators of
heatvit_b200.decode.  The decoder's weights are random: it shows the calls, not a caption.

By default the image's tokens do not see one another in the decoder: every layer's entries are
projections of what the first layer is given.  With --prompt-attention they go through the layers as a
prompt does, each seeing all of its image, and queries and keys have a norm of their own; with a
temperature above zero the next token is drawn, else it is the largest logit's.
"""

import argparse
import os
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import torch  # noqa: E402

from heatvit_b200 import abi, decode, synth  # noqa: E402

LAST_BLOCK = abi.ckpt_block(abi.BLOCKS)


class Linear:
    """A weight [out, in] in e4m3 with block scales, laid out once."""

    def __init__(self, out, inp, gen):
        self.q, self.scale = decode.quantize_weight_fp8(
            torch.randn(out, inp, generator=gen, device="cuda") * inp ** -0.5)

    def __call__(self, rows):
        return decode.gemm_fp8(rows.q, rows.scale, self.q, self.scale)


class Decoder:
    def __init__(self, layers=2, width=512, heads=8, kv_heads=2, vocab=1000, page=16, longest=512, seed=0,
                 sees_prompt=False, head_norms=False):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.layers, self.width, self.heads, self.kv, self.page = layers, width, heads, kv_heads, page
        self.dim, self.sees_prompt = width // heads, sees_prompt
        one = torch.ones(self.dim, device="cuda", dtype=torch.bfloat16)
        self.norms = dict(q_weight=one, k_weight=one) if head_norms else {}
        self.rope = decode.rope_table(longest, self.dim)
        self.embed = torch.randn(vocab, width, generator=gen, device="cuda").bfloat16()
        self.one = torch.ones(width, device="cuda", dtype=torch.bfloat16)
        self.wide_one = torch.ones(2 * width, device="cuda", dtype=torch.bfloat16)
        self.image = Linear(width, abi.EMBED, gen)
        self.image_one = torch.ones(abi.EMBED, device="cuda", dtype=torch.bfloat16)
        self.qkv = [Linear((heads + 2 * kv_heads) * self.dim, width, gen) for _ in range(layers)]
        self.proj = [Linear(width, width, gen) for _ in range(layers)]
        self.up = [Linear(2 * width, width, gen) for _ in range(layers)]
        self.down = [Linear(width, 2 * width, gen) for _ in range(layers)]
        self.head = Linear(vocab, width, gen)

    def start(self, tokens, counts, steps):
        """Caches with the images' tokens in them: tokens [sum(counts), 192] int8, image after image."""
        counts = torch.as_tensor(counts, device="cuda", dtype=torch.int32)
        need = (counts + steps + self.page - 1) // self.page
        self.table = torch.full((len(counts), int(need.max())), -1, dtype=torch.int32, device="cuda")
        used = torch.arange(self.table.shape[1], device="cuda")[None, :] < need[:, None]
        self.table[used] = torch.arange(int(need.sum()), dtype=torch.int32, device="cuda")
        shape = (self.layers, 2, int(need.sum()), self.page, self.kv, self.dim)
        self.cache = torch.zeros(shape, dtype=torch.bfloat16, device="cuda")
        self.lens = counts.clone()
        first = torch.cumsum(counts, 0) - counts
        ids = torch.repeat_interleave(torch.arange(len(counts), device="cuda"), counts.long())
        positions = (torch.arange(len(ids), device="cuda") - first[ids]).int()
        # the codes as plain numbers: the power of two that they all share goes out in the norm
        x = self.image(decode.add_rmsnorm_fp8(tokens.bfloat16(), self.image_one))
        if self.sees_prompt:
            starts = torch.nn.functional.pad(torch.cumsum(counts, 0), (1, 0)).int()
            return self._layers(x, torch.zeros_like(x), positions, dict(seq_ids=ids.int()), lambda q, i: decode.paged_chunk_attention(
                q, *self.cache[i], self.table, self.lens, starts, causal=False))
        rows = decode.add_rmsnorm_fp8(x, self.one)
        for i in range(self.layers):
            _, k, v = self._split(self.qkv[i](rows))
            kn = {name: w for name, w in self.norms.items() if name == "k_weight"}
            decode.append_kv(k, v, *self.cache[i], self.table, positions, seq_ids=ids.int(), rope=self.rope, **kn)

    def _split(self, qkv):
        h = qkv.view(-1, self.heads + 2 * self.kv, self.dim)
        return h[:, :self.heads], h[:, self.heads:self.heads + self.kv], h[:, self.heads + self.kv:]

    def step(self, ids):
        """Logits [images, vocab] after one more token of each image, ids [images]."""
        positions = self.lens.clone()
        self.lens += 1
        x = torch.zeros(len(ids), self.width, dtype=torch.bfloat16, device="cuda")
        residual = self.embed[ids]
        x = self._layers(x, residual, positions, {},
                         lambda q, i: decode.paged_attention(q, *self.cache[i], self.table, self.lens))
        return self.head(decode.add_rmsnorm_fp8(x, self.one, residual=residual, residual_out=residual))

    def _layers(self, x, residual, positions, append, attend):
        """All layers over new tokens: x and residual [tokens, width], attend(q, layer) over the cache."""
        for i in range(self.layers):
            rows = decode.add_rmsnorm_fp8(x, self.one, residual=residual, residual_out=residual)
            q, k, v = self._split(self.qkv[i](rows))
            q = decode.append_kv(k, v, *self.cache[i], self.table, positions, rope=self.rope, q=q, **append, **self.norms)
            seen = attend(q, i)
            x = self.proj[i](decode.add_rmsnorm_fp8(seen.view(-1, self.width), self.one))
            rows = decode.add_rmsnorm_fp8(x, self.one, residual=residual, residual_out=residual)
            wide = torch.nn.functional.silu(self.up[i](rows))
            x = self.down[i](decode.add_rmsnorm_fp8(wide, self.wide_one))
        return x


def encode(images, params=None):
    """The last block's tokens of each image [sum(counts), 192] int8, and their counts."""
    from heatvit_b200.engine import Engine
    out = Engine(params or synth.config3_params()).infer(images, checkpoints=True)
    counts = out["checkpoint_rows"][:, LAST_BLOCK]
    kept = torch.arange(abi.TOKENS, device=images.device)[None, :] < counts[:, None]
    return out["checkpoints"][:, LAST_BLOCK][kept], counts


def main():
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--images", type=int, default=8)
    ap.add_argument("--steps", type=int, default=16)
    ap.add_argument("--prompt-attention", action="store_true", help="the image's tokens see one another; norms of q and k")
    ap.add_argument("--temperature", type=float, default=0.0, help="0: the largest logit")
    ap.add_argument("--top-p", type=float, default=1.0)
    a = ap.parse_args()
    images = torch.from_numpy(synth.baseline_images(synth.SEED, a.images)).cuda()
    tokens, counts = encode(images)
    decoder = Decoder(sees_prompt=a.prompt_attention, head_norms=a.prompt_attention)
    decoder.start(tokens, counts, a.steps)
    ids = torch.zeros(a.images, dtype=torch.long, device="cuda")
    said = []
    draws = torch.rand(a.steps, a.images, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    for u in draws:
        ids = decode.sample_tokens(decoder.step(ids), u, temperature=a.temperature, top_p=a.top_p)
        said.append(ids)
    for i, (n, row) in enumerate(zip(counts.tolist(), torch.stack(said, 1).tolist())):
        print(f"image {i}: {n} tokens ->", *row)
    if decode.device_error():
        raise RuntimeError("a decode operator reported an error")


if __name__ == "__main__":
    main()
