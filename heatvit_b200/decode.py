"""What a language decoder that reads the encoder's tokens runs, from a prompt to its next token.

Operators that belong together, on torch CUDA tensors, on the caller's
current stream: the norm writes the e4m3 rows that the GEMM multiplies, the GEMM's
q, k and v are what the append norms, rotates and stores, the attentions (of a prompt's tokens, and of
one new token a sequence) read that cache, and a token is drawn from the last GEMM's logits.
Floating point, inference only, with no counterpart in the reference.

    rows = add_rmsnorm_fp8(x, weight, residual=r)          # 8 bits, a scale for each 128 channels
    qkv = gemm_fp8(rows.q, rows.scale, w, w_scale)         # [tokens, (heads + 2 kv_heads) * dim]
    q = append_kv(k, v, k_cache, v_cache, page_table, positions, rope=table, q=q, q_weight=qw, k_weight=kw)
    out = paged_chunk_attention(q, k_cache, v_cache, page_table, lens, starts)  # prompts, or pieces of them
    out = paged_attention(q, k_cache, v_cache, page_table, lens)                # one new token a sequence
    ids = sample_tokens(logits, uniform, temperature=0.8, top_p=0.95)

The last dimension of every tensor is contiguous; the others may have any stride
(a cache may be [pages, page, kv_heads, dim] in memory or a transposed view of
[pages, kv_heads, page, dim]), but a tensor that is written may not be an expanded one,
and rows of an e4m3 operand do not overlap.  Shape and type mistakes raise ValueError and
TypeError.  What only the device can see (a page number outside the cache, a
position past a table) faults nothing and is reported by ``device_error``.
Calls may be captured in a CUDA graph after one of each outside it.  There are no
gradients: an input that asks for them is read as its values, a result never does.
"""

import ctypes as C
import importlib.util
import os
from collections import namedtuple

from ._lib import check, lib
from .engine import _torch

GROUP = 128  # channels that share a scale
E4M3_MAX = 448.0
HEAD_DIMS = (32, 64, 96, 128, 192, 256)
NATIVE_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "_lib", "_decode_native.so")

Fp8Rows = namedtuple("Fp8Rows", "q scale residual")
Fp8Rows.__doc__ = "q [rows, dim] e4m3, scale [rows, ceil(dim / 128)] float32, residual [rows, dim] or None."

_native = None


def _load():
    """The native module that checks tensors and makes the calls (hv_decode_torch.cpp),
    once a CUDA device and the library are known to be there."""
    global _native
    if _native is None:
        _torch()
        lib()
        if not os.path.exists(NATIVE_PATH):
            raise RuntimeError(f"{NATIVE_PATH} is not built; run heatvit_b200.build.build()")
        spec = importlib.util.spec_from_file_location("_decode_native", NATIVE_PATH)
        module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(module)
        _native = module
    return _native


def _done(result):
    """A native call's result; raises on the status that it is when a C entry refused."""
    if type(result) is int:
        check(result)
    return result


def device_error(device=None):
    """Read and clear the decode error bits of a device (synchronises with it):
    abi.HV_DECODE_BAD_PAGE, _BAD_POSITION, _BAD_LENGTH, _STALLED, _BAD_LOGITS, _BAD_START; 0 when all
    went well."""
    torch = _torch()
    bits = C.c_int()
    with torch.cuda.device(device):
        check(lib().hv_decode_error(C.byref(bits)))
    return bits.value


def add_rmsnorm_fp8(x, weight, eps=1e-6, residual=None, residual_out=None):
    """Residual addition, RMSNorm and e4m3 output in one pass -> Fp8Rows.

    ``h = x + residual`` in 32 bits; ``y = h * rsqrt(mean(h^2) + eps) * weight``;
    for each 128 channels of a row ``scale = max(amax |y|, 2^-100) / 448`` and
    ``q = e4m3(y / scale)``.  x and residual [rows, dim] and weight [dim] share one of
    bfloat16, float16, float32; ``residual_out`` (a new tensor unless given, and it may
    be ``residual``) receives h rounded to that type.  q's row stride is a multiple of 16 and
    scale is stored group by group, both as ``gemm_fp8`` reads them best, and they share a
    storage; a new residual's row stride is a multiple of 8, since rows that start on 16
    bytes go faster."""
    q, scale, out = _done((_native or _load()).add_rmsnorm_fp8(x, weight, eps, residual, residual_out))
    return Fp8Rows(q, scale, out)


def quantize_weight_fp8(weight):
    """A weight [n, k] as e4m3 with a float32 scale for each 128 x 128 block, as
    ``gemm_fp8`` takes it -> (q [n, k] with 16-byte aligned rows, scale [ceil(n/128),
    ceil(k/128)]).  Done once, when weights are loaded."""
    torch = _torch()
    if weight.dim() != 2:
        raise ValueError("weight must be 2-dimensional")
    n, k = weight.shape
    nb, kb = -(-n // GROUP), -(-k // GROUP)
    w = torch.zeros((nb * GROUP, kb * GROUP), dtype=torch.float32, device=weight.device)
    w[:n, :k] = weight.detach()
    blocks = w.view(nb, GROUP, kb, GROUP)
    scale = blocks.abs().amax((1, 3)).clamp_(min=2.0 ** -100) / E4M3_MAX
    q = torch.empty((n, -(-k // 16) * 16), dtype=torch.float8_e4m3fn, device=weight.device)[:, :k]
    q.copy_((blocks / scale[:, None, :, None]).clamp_(-E4M3_MAX, E4M3_MAX).view_as(w)[:n, :k])
    return q, scale


def gemm_fp8(a, a_scale, b, b_scale, out_dtype=None, out=None):
    """``out[m, n] = sum_k a[m, k] b[n, k]`` of e4m3 operands, where a_scale [m, groups]
    scales each 128 channels of a row of a, and b_scale [ceil(n / 128), groups] each
    128 x 128 block of b; groups = ceil(k / 128).

    Operand rows start on 16 bytes (as ``add_rmsnorm_fp8`` and ``quantize_weight_fp8``
    lay them out); scales are float32 of any strides.  Sums in 32 bits, rounded once to
    ``out_dtype`` (bfloat16 unless given; float16, float32) or to ``out``'s type."""
    return _done((_native or _load()).gemm_fp8(a, a_scale, b, b_scale, out_dtype, out))


def rope_table(positions, rot, base=10000.0, device="cuda"):
    """Cosines, then sines, of ``position * base^(-2 i / rot)``: float32 [positions, rot],
    angles in 64 bits.  Built once and kept by the caller."""
    torch = _torch()
    if rot < 2 or rot % 2:
        raise ValueError("rot must be even and positive")
    i = torch.arange(rot // 2, dtype=torch.float64, device=device)
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * base ** (-2.0 * i / rot)
    return torch.cat([angle.cos(), angle.sin()], 1).float()


def append_kv(k, v, k_cache, v_cache, page_table, positions, seq_ids=None, rope=None, q=None, interleaved=False,
              q_out=None, q_weight=None, k_weight=None, eps=1e-6):
    """Store new keys and values in a paged cache, rotating q and k by position.

    k, v [tokens, kv_heads, dim], q [tokens, heads, dim] (views of one projection's
    output will do), caches [pages, page, kv_heads, dim], all bfloat16 or all float16.
    Token t of sequence ``seq_ids[t]`` (t itself without seq_ids) at ``positions[t]``
    goes to page ``page_table[seq, position // page]``; a negative position marks a
    padding token (nothing stored, zeros in q_out).  ``rope`` [positions, rot]
    float32 (see ``rope_table``) turns the first rot elements of each head in pairs
    (i, i + rot/2), or (2i, 2i + 1) when interleaved; v is stored as it is.  Returns the
    rotated q (a new tensor, or q_out, which may be q), None without q.

    ``q_weight``, ``k_weight`` [dim] of k's type: an RMS norm of each q or k head goes ahead of the
    rotation, ``x * rsqrt(mean(x^2) + eps) * weight`` over the head's elements, all in 32 bits and
    rounded once; where one is None its heads are as they come."""
    native = _native or _load()
    if q_weight is None and k_weight is None:
        return _done(native.append_kv(k, v, k_cache, v_cache, page_table, positions, seq_ids, rope, q, interleaved, q_out))
    return _done(native.norm_append_kv(k, v, k_cache, v_cache, page_table, positions, seq_ids, rope, q, interleaved, q_out,
                                       q_weight, k_weight, eps))


class AttentionWorkspace:
    """Device memory that ``paged_attention`` joins split sequences in, for one device
    (the current one unless named) and any sizes.  Calls that share one must not overlap
    in time (one per stream).  Waits for the device to have zeroed its counters, so that
    any stream may use it.  With ``chunks`` a larger one (5 MB become 40), which
    ``paged_chunk_attention`` can use as well."""

    def __init__(self, device=None, chunks=False):
        torch = _torch()
        device = torch.device("cuda" if device is None else device)
        if device.type != "cuda":
            raise ValueError("an attention workspace lives on a CUDA device")
        self.device = torch.device("cuda", torch.cuda.current_device() if device.index is None else device.index)
        make = _load().chunk_attention_workspace if chunks else _load().attention_workspace
        self.buffer = make(self.device.index)
        torch.cuda.current_stream(self.device).synchronize()


def paged_attention(q, k_cache, v_cache, page_table, lens, scale=None, workspace=None, out=None, return_lse=False):
    """Attention of one new token per sequence over a paged cache.

    q [seqs, heads, dim]; caches [pages, page, kv_heads, dim] of q's type (bfloat16 or
    float16), heads a multiple of kv_heads; page_table [seqs, max_pages] and lens [seqs]
    int32.  ``softmax(scale * q K^T) V`` over the first lens[i] cached tokens, scale
    ``dim^-0.5`` unless given; a sequence of no tokens gives zeros.  Returns out (a new
    tensor unless given), with ``return_lse`` also the log-sum-exp of the scaled scores,
    float32 [seqs, heads] (-inf for no tokens).

    ``workspace``: an AttentionWorkspace; by default the module keeps one per stream, and a call that
    a CUDA graph captures makes its own and zeroes 12 KB of it at every replay (about 1 us): pass one
    to a captured step."""
    return _done((_native or _load()).paged_attention(
        q, k_cache, v_cache, page_table, lens, scale, None if workspace is None else workspace.buffer, out,
        return_lse))


def paged_chunk_attention(q, k_cache, v_cache, page_table, lens, starts, causal=True, scale=None, workspace=None, out=None,
                          return_lse=False):
    """Attention of a chunk of new tokens of each sequence over a paged cache that holds them
    already (``append_kv`` comes first): a prompt, a piece of one, or drafted tokens.

    q [tokens, heads, dim], packed: rows ``starts[i]`` to ``starts[i + 1]`` (int32 [seqs + 1]) are
    the newest tokens of sequence i, of which the cache has ``lens[i]`` in all; a sequence may
    bring none.  ``causal``: a token sees those up to itself; otherwise each sees all
    ``lens[i]``.  A row that sees no token gives zeros (log-sum-exp -inf); rows of no sequence are not
    written, neither in ``out`` (which may be q) nor in a new tensor.  The rest as ``paged_attention``.

    ``workspace``: an AttentionWorkspace made with ``chunks=True`` (by default the module keeps one of
    40 MB per stream, beside that of ``paged_attention``)."""
    return _done((_native or _load()).paged_chunk_attention(
        q, k_cache, v_cache, page_table, lens, starts, causal, scale, None if workspace is None else workspace.buffer, out,
        return_lse))


def sample_tokens(logits, uniform, temperature=None, top_k=None, top_p=None, min_p=None, out=None, return_logprob=False):
    """Draw a token for each row of logits [rows, vocab] (bfloat16, float16, float32) with that
    row's number of ``uniform`` (float32 [rows], in [0, 1)) -> int64 [rows].

    With ``w = exp((logit - largest) / temperature)`` and tokens ordered by logit, equal ones by
    index: ``top_k`` keeps the first top_k (0: all), ``min_p`` those with w >= min_p, ``top_p`` the
    shortest prefix of what these keep whose weights reach top_p of their sum (at least one token).
    The token is the first, in the vocabulary's order, at which the kept weights add up to more than
    ``uniform`` of their total.  Sums are exact, so the same numbers give the same token on any device.
    Temperature 0 takes the largest logit, the first of equal ones.

    Each setting is None (temperature 1, all tokens), a number, or a tensor [rows] (float32; top_k
    int32), so that every row may have its own.  With ``return_logprob`` also the logarithm of the token's
    probability among what was kept, float32 [rows].  A row with a NaN, or with nothing
    above -inf, gives token 0 and a logprob of NaN, and ``device_error`` reports it."""
    return _done((_native or _load()).sample_tokens(logits, uniform, temperature, top_k, top_p, min_p, out, return_logprob))
