"""The serving step of a language decoder that reads the encoder's tokens.

Four operators that belong together, on torch CUDA tensors, on the caller's
current stream: the norm writes the e4m3 rows that the GEMM multiplies, the GEMM's
q, k and v are what the append rotates and stores, and the attention reads that
cache.  Floating point, inference only, with no counterpart in the reference.

    rows = add_rmsnorm_fp8(x, weight, residual=r)          # 8 bits, a scale for each 128 channels
    qkv = gemm_fp8(rows.q, rows.scale, w, w_scale)         # [tokens, (heads + 2 kv_heads) * dim]
    q = append_kv(k, v, k_cache, v_cache, page_table, positions, rope=table, q=q)
    out = paged_attention(q, k_cache, v_cache, page_table, lens)

The last dimension of every tensor is contiguous; the others may have any stride
(a cache may be [pages, page, kv_heads, dim] in memory or a transposed view of
[pages, kv_heads, page, dim]).  Shape and type mistakes raise ValueError and
TypeError.  What only the device can see (a page number outside the cache, a
position past a table) faults nothing and is reported by ``device_error``.
"""

import struct
from collections import namedtuple

from . import abi
from ._lib import check, lib
from .engine import _torch

GROUP = 128  # channels that share a scale
E4M3_MAX = 448.0
HEAD_DIMS = (32, 64, 96, 128, 192, 256)

Fp8Rows = namedtuple("Fp8Rows", "q scale residual")
Fp8Rows.__doc__ = "q [rows, dim] e4m3, scale [rows, ceil(dim / 128)] float32, residual [rows, dim] or None."

# hv_append_args and hv_attention_args of include/heatvit_b200.h
_APPEND = struct.Struct("@10P16q12i")
_ATTEND = struct.Struct("@8P14q8if")

_types = None


def _dtype_codes():
    global _types
    if _types is None:
        torch = _torch()
        _types = {torch.bfloat16: abi.HV_BF16, torch.float16: abi.HV_F16, torch.float32: abi.HV_F32}
    return _types


def _need(t, name, dims, device):
    if not t.is_cuda or t.device != device:
        raise ValueError(f"{name} must live on {device}")
    if t.dim() != dims:
        raise ValueError(f"{name} must be {dims}-dimensional")
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name}'s last dimension must be contiguous")


def _ints(t, name, dims, device):
    _need(t, name, dims, device)
    if t.dtype != _torch().int32:
        raise TypeError(f"{name} must be int32")


def _call(fn, device, *args):
    """fn(*args, stream) with `device` current; raises on a status."""
    torch = _torch()
    if torch.cuda.current_device() == device.index:
        status = fn(*args, torch.cuda.current_stream(device).cuda_stream)
    else:
        with torch.cuda.device(device):
            status = fn(*args, torch.cuda.current_stream(device).cuda_stream)
    if status:
        check(status)


def device_error(device=None):
    """Read and clear the decode error bits of a device (synchronises with it):
    abi.HV_DECODE_BAD_PAGE, _BAD_POSITION, _BAD_LENGTH, _STALLED; 0 when all went well."""
    import ctypes as C
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
    be ``residual``) receives h rounded to that type.  q's row stride is a multiple of 16,
    scale is stored group by group: both as ``gemm_fp8`` reads them best."""
    torch = _torch()
    dev = x.device
    _need(x, "x", 2, dev)
    _need(weight, "weight", 1, dev)
    code = _dtype_codes().get(x.dtype)
    if code is None:
        raise TypeError("x must be bfloat16, float16 or float32")
    rows, dim = x.shape
    if weight.shape[0] != dim:
        raise ValueError(f"weight has {weight.shape[0]} channels, x {dim}")
    if weight.dtype != x.dtype:
        raise TypeError("weight must have x's type")
    r_ptr = ro_ptr = None
    r_stride = ro_stride = 0
    if residual is not None:
        if residual_out is None:
            residual_out = torch.empty((rows, dim), dtype=x.dtype, device=dev)
        for t, name in ((residual, "residual"), (residual_out, "residual_out")):
            _need(t, name, 2, dev)
            if t.shape != x.shape:
                raise ValueError(f"{name} must have x's shape")
            if t.dtype != x.dtype:
                raise TypeError(f"{name} must have x's type")
        r_ptr, r_stride = residual.data_ptr(), residual.stride(0)
        ro_ptr, ro_stride = residual_out.data_ptr(), residual_out.stride(0)
    elif residual_out is not None:
        raise ValueError("residual_out without a residual")
    wide = -(-dim // 16) * 16
    q = torch.empty((rows, wide), dtype=torch.float8_e4m3fn, device=dev)
    scale = torch.empty((-(-dim // GROUP), rows), dtype=torch.float32, device=dev)
    _call(lib().hv_add_rmsnorm_fp8, dev, x.data_ptr(), x.stride(0), r_ptr, r_stride, weight.data_ptr(), rows, dim,
          code, eps, ro_ptr, ro_stride, q.data_ptr(), wide, scale.data_ptr(), 1, rows)
    return Fp8Rows(q if wide == dim else q[:, :dim], scale.t(), residual_out)


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
    w[:n, :k] = weight
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
    torch = _torch()
    dev = a.device
    fp8 = torch.float8_e4m3fn
    for t, name in ((a, "a"), (b, "b")):
        _need(t, name, 2, dev)
        if t.dtype != fp8:
            raise TypeError(f"{name} must be float8_e4m3fn")
    m, k = a.shape
    n = b.shape[0]
    if b.shape[1] != k:
        raise ValueError(f"K mismatch: a has {k}, b has {b.shape[1]}")
    if k < 1:
        raise ValueError("k must be positive")
    groups = -(-k // GROUP)
    for t, name, rows in ((a_scale, "a_scale", m), (b_scale, "b_scale", -(-n // GROUP))):
        if t.device != dev:
            raise ValueError(f"{name} must live on {dev}")
        if t.dtype != torch.float32:
            raise TypeError(f"{name} must be float32")
        if t.shape != (rows, groups):
            raise ValueError(f"{name} must be [{rows}, {groups}]")
    if out is None:
        out = torch.empty((m, n), dtype=out_dtype or torch.bfloat16, device=dev)
    else:
        _need(out, "out", 2, dev)
        if out.shape != (m, n):
            raise ValueError(f"out must be [{m}, {n}]")
        if out_dtype is not None and out.dtype != out_dtype:
            raise TypeError("out has another type than out_dtype")
    code = _dtype_codes().get(out.dtype)
    if code is None:
        raise TypeError("out must be bfloat16, float16 or float32")
    _call(lib().hv_gemm_fp8, dev, a.data_ptr(), a.stride(0), a_scale.data_ptr(), a_scale.stride(0), a_scale.stride(1),
          b.data_ptr(), b.stride(0), b_scale.data_ptr(), b_scale.stride(0), b_scale.stride(1), m, n, k, out.data_ptr(),
          out.stride(0), code)
    return out


def rope_table(positions, rot, base=10000.0, device="cuda"):
    """Cosines, then sines, of ``position * base^(-2 i / rot)``: float32 [positions, rot],
    angles in 64 bits.  Built once and kept by the caller."""
    torch = _torch()
    if rot < 2 or rot % 2:
        raise ValueError("rot must be even and positive")
    i = torch.arange(rot // 2, dtype=torch.float64, device=device)
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * base ** (-2.0 * i / rot)
    return torch.cat([angle.cos(), angle.sin()], 1).float()


def _cache_strides(k_cache, v_cache, device):
    _need(k_cache, "k_cache", 4, device)
    _need(v_cache, "v_cache", 4, device)
    if k_cache.shape != v_cache.shape:
        raise ValueError("k_cache and v_cache must have the same shape")
    if k_cache.dtype != v_cache.dtype:
        raise TypeError("k_cache and v_cache must have the same type")
    return (*k_cache.stride()[:3], *v_cache.stride()[:3])


def append_kv(k, v, k_cache, v_cache, page_table, positions, seq_ids=None, rope=None, q=None, interleaved=False,
              q_out=None):
    """Store new keys and values in a paged cache, rotating q and k by position.

    k, v [tokens, kv_heads, dim], q [tokens, heads, dim] (views of one projection's
    output will do), caches [pages, page, kv_heads, dim], all bfloat16 or all float16.
    Token t of sequence ``seq_ids[t]`` (t itself without seq_ids) at ``positions[t]``
    goes to page ``page_table[seq, position // page]``; a negative position marks a
    padding token (nothing stored, zeros in q_out).  ``rope`` [positions, rot]
    float32 (see ``rope_table``) turns the first rot elements of each head in pairs
    (i, i + rot/2), or (2i, 2i + 1) when interleaved; v is stored as it is.  Returns the
    rotated q (a new tensor, or q_out, which may be q), None without q."""
    torch = _torch()
    dev = k.device
    _need(k, "k", 3, dev)
    _need(v, "v", 3, dev)
    cache = _cache_strides(k_cache, v_cache, dev)
    _ints(page_table, "page_table", 2, dev)
    _ints(positions, "positions", 1, dev)
    code = _dtype_codes().get(k.dtype)
    if code not in (abi.HV_BF16, abi.HV_F16):
        raise TypeError("k must be bfloat16 or float16")
    if v.dtype != k.dtype or k_cache.dtype != k.dtype:
        raise TypeError("k, v and the caches must have the same type")
    tokens, kv_heads, dim = k.shape
    if v.shape != k.shape:
        raise ValueError("k and v must have the same shape")
    if k_cache.shape[2:] != (kv_heads, dim):
        raise ValueError("the caches hold other heads or another head dimension")
    if positions.shape[0] != tokens:
        raise ValueError("one position per token")
    ids = None
    if seq_ids is not None:
        _ints(seq_ids, "seq_ids", 1, dev)
        if seq_ids.shape[0] != tokens:
            raise ValueError("one sequence id per token")
        ids = seq_ids.data_ptr()
    elif page_table.shape[0] < tokens:
        raise ValueError("without seq_ids the page table has one row per token")
    heads, q_ptr, qo_ptr, q_str, qo_str = 0, 0, 0, (0, 0), (0, 0)
    if q is not None:
        if q_out is None:
            q_out = torch.empty(q.shape, dtype=q.dtype, device=dev)
        for t, name in ((q, "q"), (q_out, "q_out")):
            _need(t, name, 3, dev)
            if t.shape[0] != tokens or t.shape[2] != dim or t.shape != q.shape:
                raise ValueError(f"{name} must be [tokens, heads, dim]")
            if t.dtype != k.dtype:
                raise TypeError(f"{name} must have k's type")
        heads, q_ptr, qo_ptr = q.shape[1], q.data_ptr(), q_out.data_ptr()
        q_str, qo_str = q.stride()[:2], q_out.stride()[:2]
    elif q_out is not None:
        raise ValueError("q_out without q")
    rot, rope_ptr, rope_stride, rope_rows = 0, 0, 0, 0
    if rope is not None:
        _need(rope, "rope", 2, dev)
        if rope.dtype != torch.float32:
            raise TypeError("rope must be float32")
        rope_rows, rot = rope.shape
        rope_ptr, rope_stride = rope.data_ptr(), rope.stride(0)
    args = _APPEND.pack(q_ptr, k.data_ptr(), v.data_ptr(), qo_ptr, k_cache.data_ptr(), v_cache.data_ptr(), rope_ptr,
                        page_table.data_ptr(), ids or 0, positions.data_ptr(), *q_str, *k.stride()[:2],
                        *v.stride()[:2], *qo_str, *cache, rope_stride, page_table.stride(0), tokens, heads, kv_heads,
                        dim, rot, bool(interleaved), code, k_cache.shape[0], k_cache.shape[1], page_table.shape[0],
                        page_table.shape[1], rope_rows)
    _call(lib().hv_append_kv, dev, args)
    return q_out


class AttentionWorkspace:
    """Device memory that ``paged_attention`` joins split sequences in, for one device
    and any sizes.  Calls that share one must not overlap in time (one per stream)."""

    def __init__(self, device=None):
        import ctypes as C
        torch = _torch()
        self.device = torch.device("cuda", torch.cuda.current_device() if device is None else
                                   torch.device(device).index or 0)
        need, most = C.c_int64(), 0
        with torch.cuda.device(self.device):
            for dim in HEAD_DIMS:
                check(lib().hv_paged_attention_workspace(dim, C.byref(need)))
                most = max(most, need.value)
            self.buffer = torch.zeros(most, dtype=torch.uint8, device=self.device)
        self.bytes = most
        self.ptr = self.buffer.data_ptr()


_workspaces = {}  # (device index, stream handle) -> AttentionWorkspace


def _workspace(torch, device):
    """The current stream's own workspace, made at its first call; a fresh one while the
    stream is being captured, since a graph may be replayed on any stream."""
    if torch.cuda.is_current_stream_capturing():
        return AttentionWorkspace(device)
    key = (device.index, torch.cuda.current_stream(device).cuda_stream)
    ws = _workspaces.get(key)
    if ws is None:
        ws = _workspaces[key] = AttentionWorkspace(device)
    return ws


def paged_attention(q, k_cache, v_cache, page_table, lens, scale=None, workspace=None, out=None, return_lse=False):
    """Attention of one new token per sequence over a paged cache.

    q [seqs, heads, dim]; caches [pages, page, kv_heads, dim] of q's type (bfloat16 or
    float16), heads a multiple of kv_heads; page_table [seqs, max_pages] and lens [seqs]
    int32.  ``softmax(scale * q K^T) V`` over the first lens[i] cached tokens, scale
    ``dim^-0.5`` unless given; a sequence of no tokens gives zeros.  Returns out (a new
    tensor unless given), with ``return_lse`` also the log-sum-exp of the scaled scores,
    float32 [seqs, heads] (-inf for no tokens).

    ``workspace``: an AttentionWorkspace; by default the module keeps one per stream."""
    torch = _torch()
    dev = q.device
    _need(q, "q", 3, dev)
    cache = _cache_strides(k_cache, v_cache, dev)
    _ints(page_table, "page_table", 2, dev)
    _ints(lens, "lens", 1, dev)
    code = _dtype_codes().get(q.dtype)
    if code not in (abi.HV_BF16, abi.HV_F16):
        raise TypeError("q must be bfloat16 or float16")
    if k_cache.dtype != q.dtype:
        raise TypeError("q and the caches must have the same type")
    seqs, heads, dim = q.shape
    pages, page, kv_heads, cache_dim = k_cache.shape
    if cache_dim != dim:
        raise ValueError("the caches have another head dimension")
    if dim not in HEAD_DIMS:
        raise ValueError(f"dim must be one of {HEAD_DIMS}")
    if kv_heads < 1 or heads < 1 or heads % kv_heads:
        raise ValueError("heads must be a positive multiple of kv_heads")
    if page_table.shape[0] != seqs or lens.shape[0] != seqs:
        raise ValueError("page_table and lens have one row per sequence")
    if out is None:
        out = torch.empty((seqs, heads, dim), dtype=q.dtype, device=dev)
    else:
        _need(out, "out", 3, dev)
        if out.shape != q.shape:
            raise ValueError("out must have q's shape")
        if out.dtype != q.dtype:
            raise TypeError("out must have q's type")
    if workspace is None:
        workspace = _workspace(torch, dev)
    elif workspace.device != dev:
        raise ValueError(f"the workspace must live on {dev}")
    lse = torch.empty((seqs, heads), dtype=torch.float32, device=dev) if return_lse else None
    args = _ATTEND.pack(q.data_ptr(), out.data_ptr(), lse.data_ptr() if return_lse else 0, k_cache.data_ptr(),
                        v_cache.data_ptr(), page_table.data_ptr(), lens.data_ptr(), workspace.ptr, workspace.bytes,
                        *q.stride()[:2], *out.stride()[:2], heads, 1, *cache, page_table.stride(0), seqs, heads,
                        kv_heads, dim, code, pages, page, page_table.shape[1], dim ** -0.5 if scale is None else scale)
    _call(lib().hv_paged_attention, dev, args)
    return (out, lse) if return_lse else out
