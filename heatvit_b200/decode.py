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

import ctypes as C
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

# hv_norm_args, hv_gemm_fp8_args, hv_append_args and hv_attention_args of include/heatvit_b200.h
_NORM = struct.Struct("@6P7q2if")
_GEMM = struct.Struct("@5P10qi")
_APPEND = struct.Struct("@10P16q12i")
_ATTEND = struct.Struct("@8P14q8if")

_torch_module = None
_types = _raw_stream = _current_device = _c = None


def _ready():
    """torch, once a CUDA device and the library are known to be there; small calls cost
    what the host does, so the look-ups are made once."""
    global _torch_module, _types, _raw_stream, _current_device, _c
    if _torch_module is None:
        torch = _torch()
        _c = lib()
        _types = {torch.bfloat16: abi.HV_BF16, torch.float16: abi.HV_F16, torch.float32: abi.HV_F32}
        _raw_stream, _current_device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice
        _torch_module = torch
    return _torch_module


def _index(t, name):
    """The CUDA device of an operator's first tensor, which the others share."""
    i = t.get_device()
    if i < 0:
        raise ValueError(f"{name} must be a CUDA tensor")
    return i


def _strides(t, name, dims, index):
    """t's strides, after the checks that every operand passes."""
    if t.get_device() != index:
        raise ValueError(f"{name} must live on cuda:{index}")
    s = t.stride()
    if len(s) != dims:
        raise ValueError(f"{name} must be {dims}-dimensional")
    if s[-1] != 1 and t.shape[-1] > 1:
        raise ValueError(f"{name}'s last dimension must be contiguous")
    return s


def _int_strides(t, name, dims, index):
    if t.dtype is not _torch_module.int32:
        raise TypeError(f"{name} must be int32")
    return _strides(t, name, dims, index)


def _like(t, name, other, its_name, index):
    """t's strides; t has the shape and the type of another operand."""
    s = _strides(t, name, len(other.shape), index)
    if t.shape != other.shape:
        raise ValueError(f"{name} must have {its_name}'s shape")
    if t.dtype is not other.dtype:
        raise TypeError(f"{name} must have {its_name}'s type")
    return s


def _call(fn, index, args):
    """fn(args, stream) with the device current; raises on a status."""
    if _current_device() == index:
        status = fn(args, _raw_stream(index))
    else:
        with _torch_module.cuda.device(index):
            status = fn(args, _raw_stream(index))
    if status:
        check(status)


def device_error(device=None):
    """Read and clear the decode error bits of a device (synchronises with it):
    abi.HV_DECODE_BAD_PAGE, _BAD_POSITION, _BAD_LENGTH, _STALLED; 0 when all went well."""
    torch = _ready()
    bits = C.c_int()
    with torch.cuda.device(device):
        check(_c.hv_decode_error(C.byref(bits)))
    return bits.value


def add_rmsnorm_fp8(x, weight, eps=1e-6, residual=None, residual_out=None):
    """Residual addition, RMSNorm and e4m3 output in one pass -> Fp8Rows.

    ``h = x + residual`` in 32 bits; ``y = h * rsqrt(mean(h^2) + eps) * weight``;
    for each 128 channels of a row ``scale = max(amax |y|, 2^-100) / 448`` and
    ``q = e4m3(y / scale)``.  x and residual [rows, dim] and weight [dim] share one of
    bfloat16, float16, float32; ``residual_out`` (a new tensor unless given, and it may
    be ``residual``) receives h rounded to that type.  q's row stride is a multiple of 16 and
    scale is stored group by group, both as ``gemm_fp8`` reads them best; a new residual's
    row stride is a multiple of 8, since rows that start on 16 bytes go faster."""
    torch = _ready()
    dev = _index(x, "x")
    x_stride = _strides(x, "x", 2, dev)[0]
    _strides(weight, "weight", 1, dev)
    dtype = x.dtype
    code = _types.get(dtype)
    if code is None:
        raise TypeError("x must be bfloat16, float16 or float32")
    rows, dim = x.shape
    if weight.shape[0] != dim:
        raise ValueError(f"weight has {weight.shape[0]} channels, x {dim}")
    if weight.dtype is not dtype:
        raise TypeError("weight must have x's type")
    device = x.device
    r_ptr = ro_ptr = r_stride = ro_stride = 0
    if residual is not None:
        r_stride = _like(residual, "residual", x, "x", dev)[0]
        if residual_out is None:
            ro_stride = -(-dim // 8) * 8
            residual_out = torch.empty(rows, ro_stride, dtype=dtype, device=device)
            if ro_stride != dim:
                residual_out = residual_out[:, :dim]
        else:
            ro_stride = _like(residual_out, "residual_out", x, "x", dev)[0]
        r_ptr, ro_ptr = residual.data_ptr(), residual_out.data_ptr()
    elif residual_out is not None:
        raise ValueError("residual_out without a residual")
    wide = -(-dim // 16) * 16
    q = torch.empty(rows, wide, dtype=torch.float8_e4m3fn, device=device)
    scale = torch.empty_strided((rows, -(-dim // GROUP)), (1, rows), dtype=torch.float32, device=device)
    _call(_c.hv_add_rmsnorm_fp8, dev, _NORM.pack(x.data_ptr(), r_ptr, weight.data_ptr(), ro_ptr, q.data_ptr(),
                                                 scale.data_ptr(), rows, x_stride, r_stride, ro_stride, wide, 1, rows,
                                                 dim, code, eps))
    return Fp8Rows(q if wide == dim else q[:, :dim], scale, residual_out)


def quantize_weight_fp8(weight):
    """A weight [n, k] as e4m3 with a float32 scale for each 128 x 128 block, as
    ``gemm_fp8`` takes it -> (q [n, k] with 16-byte aligned rows, scale [ceil(n/128),
    ceil(k/128)]).  Done once, when weights are loaded."""
    torch = _ready()
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
    torch = _ready()
    dev = _index(a, "a")
    a_stride, b_stride = _strides(a, "a", 2, dev)[0], _strides(b, "b", 2, dev)[0]
    fp8 = torch.float8_e4m3fn
    if a.dtype is not fp8 or b.dtype is not fp8:
        raise TypeError("a and b must be float8_e4m3fn")
    m, k = a.shape
    n = b.shape[0]
    if b.shape[1] != k:
        raise ValueError(f"K mismatch: a has {k}, b has {b.shape[1]}")
    if k < 1:
        raise ValueError("k must be positive")
    groups = -(-k // GROUP)
    for t, name, rows in ((a_scale, "a_scale", m), (b_scale, "b_scale", -(-n // GROUP))):
        if t.get_device() != dev:
            raise ValueError(f"{name} must live on cuda:{dev}")
        if t.dtype is not torch.float32:
            raise TypeError(f"{name} must be float32")
        if t.shape != (rows, groups):
            raise ValueError(f"{name} must be [{rows}, {groups}]")
    if out is None:
        out = torch.empty(m, n, dtype=out_dtype or torch.bfloat16, device=a.device)
        out_stride = n
    else:
        out_stride = _strides(out, "out", 2, dev)[0]
        if out.shape != (m, n):
            raise ValueError(f"out must be [{m}, {n}]")
        if out_dtype is not None and out.dtype is not out_dtype:
            raise TypeError("out has another type than out_dtype")
    code = _types.get(out.dtype)
    if code is None:
        raise TypeError("out must be bfloat16, float16 or float32")
    _call(_c.hv_gemm_fp8, dev, _GEMM.pack(a.data_ptr(), b.data_ptr(), a_scale.data_ptr(), b_scale.data_ptr(),
                                          out.data_ptr(), m, n, k, a_stride, b_stride, out_stride, *a_scale.stride(),
                                          *b_scale.stride(), code))
    return out


def rope_table(positions, rot, base=10000.0, device="cuda"):
    """Cosines, then sines, of ``position * base^(-2 i / rot)``: float32 [positions, rot],
    angles in 64 bits.  Built once and kept by the caller."""
    torch = _ready()
    if rot < 2 or rot % 2:
        raise ValueError("rot must be even and positive")
    i = torch.arange(rot // 2, dtype=torch.float64, device=device)
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * base ** (-2.0 * i / rot)
    return torch.cat([angle.cos(), angle.sin()], 1).float()


def _cache_strides(k_cache, v_cache, index):
    ks = _strides(k_cache, "k_cache", 4, index)
    return (*ks[:3], *_like(v_cache, "v_cache", k_cache, "k_cache", index)[:3])


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
    torch = _ready()
    dev = _index(k, "k")
    k_str, v_str = _strides(k, "k", 3, dev), _like(v, "v", k, "k", dev)
    cache = _cache_strides(k_cache, v_cache, dev)
    table_stride = _int_strides(page_table, "page_table", 2, dev)[0]
    _int_strides(positions, "positions", 1, dev)
    dtype = k.dtype
    code = _types.get(dtype)
    if code not in (abi.HV_BF16, abi.HV_F16):
        raise TypeError("k must be bfloat16 or float16")
    if k_cache.dtype is not dtype:
        raise TypeError("k, v and the caches must have the same type")
    tokens, kv_heads, dim = k.shape
    pages, page, cache_heads, cache_dim = k_cache.shape
    if cache_heads != kv_heads or cache_dim != dim:
        raise ValueError("the caches hold other heads or another head dimension")
    if positions.shape[0] != tokens:
        raise ValueError("one position per token")
    seqs, max_pages = page_table.shape
    ids = 0
    if seq_ids is not None:
        _int_strides(seq_ids, "seq_ids", 1, dev)
        if seq_ids.shape[0] != tokens:
            raise ValueError("one sequence id per token")
        ids = seq_ids.data_ptr()
    elif seqs < tokens:
        raise ValueError("without seq_ids the page table has one row per token")
    heads, q_ptr, qo_ptr, q_str, qo_str = 0, 0, 0, (0, 0), (0, 0)
    if q is not None:
        q_str = _strides(q, "q", 3, dev)
        if q.shape[0] != tokens or q.shape[2] != dim:
            raise ValueError("q must be [tokens, heads, dim]")
        if q.dtype is not dtype:
            raise TypeError("q must have k's type")
        heads = q.shape[1]
        if q_out is None:
            q_out = torch.empty(tokens, heads, dim, dtype=dtype, device=q.device)
            qo_str = (heads * dim, dim)
        else:
            qo_str = _like(q_out, "q_out", q, "q", dev)
        q_ptr, qo_ptr = q.data_ptr(), q_out.data_ptr()
    elif q_out is not None:
        raise ValueError("q_out without q")
    rot, rope_ptr, rope_stride, rope_rows = 0, 0, 0, 0
    if rope is not None:
        rope_stride = _strides(rope, "rope", 2, dev)[0]
        if rope.dtype is not torch.float32:
            raise TypeError("rope must be float32")
        rope_rows, rot = rope.shape
        rope_ptr = rope.data_ptr()
    args = _APPEND.pack(q_ptr, k.data_ptr(), v.data_ptr(), qo_ptr, k_cache.data_ptr(), v_cache.data_ptr(), rope_ptr,
                        page_table.data_ptr(), ids, positions.data_ptr(), *q_str[:2], *k_str[:2], *v_str[:2],
                        *qo_str[:2], *cache, rope_stride, table_stride, tokens, heads, kv_heads, dim, rot,
                        bool(interleaved), code, pages, page, seqs, max_pages, rope_rows)
    _call(_c.hv_append_kv, dev, args)
    return q_out


class AttentionWorkspace:
    """Device memory that ``paged_attention`` joins split sequences in, for one device
    and any sizes.  Calls that share one must not overlap in time (one per stream)."""

    def __init__(self, device=None):
        torch = _ready()
        self.device = torch.device("cuda", torch.cuda.current_device() if device is None else
                                   torch.device(device).index or 0)
        need, most = C.c_int64(), 0
        with torch.cuda.device(self.device):
            for dim in HEAD_DIMS:
                check(_c.hv_paged_attention_workspace(dim, C.byref(need)))
                most = max(most, need.value)
            self.buffer = torch.zeros(most, dtype=torch.uint8, device=self.device)
        self.bytes = most
        self.ptr = self.buffer.data_ptr()


_workspaces = {}  # (device index, stream handle) -> AttentionWorkspace


def _workspace(torch, index):
    """The current stream's own workspace, made at its first call; a fresh one while the
    stream is being captured, since a graph may be replayed on any stream."""
    if torch.cuda.is_current_stream_capturing():
        return AttentionWorkspace(f"cuda:{index}")
    key = (index, _raw_stream(index))
    ws = _workspaces.get(key)
    if ws is None:
        ws = _workspaces[key] = AttentionWorkspace(f"cuda:{index}")
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
    torch = _ready()
    dev = _index(q, "q")
    q_str = _strides(q, "q", 3, dev)
    cache = _cache_strides(k_cache, v_cache, dev)
    table_stride = _int_strides(page_table, "page_table", 2, dev)[0]
    _int_strides(lens, "lens", 1, dev)
    dtype = q.dtype
    code = _types.get(dtype)
    if code not in (abi.HV_BF16, abi.HV_F16):
        raise TypeError("q must be bfloat16 or float16")
    if k_cache.dtype is not dtype:
        raise TypeError("q and the caches must have the same type")
    seqs, heads, dim = q.shape
    pages, page, kv_heads, cache_dim = k_cache.shape
    if cache_dim != dim:
        raise ValueError("the caches have another head dimension")
    if dim not in HEAD_DIMS:
        raise ValueError(f"dim must be one of {HEAD_DIMS}")
    if kv_heads < 1 or heads < 1 or heads % kv_heads:
        raise ValueError("heads must be a positive multiple of kv_heads")
    rows, max_pages = page_table.shape
    if rows != seqs or lens.shape[0] != seqs:
        raise ValueError("page_table and lens have one row per sequence")
    if out is None:
        out = torch.empty(seqs, heads, dim, dtype=dtype, device=q.device)
        out_str = (heads * dim, dim)
    else:
        out_str = _like(out, "out", q, "q", dev)
    if workspace is None:
        workspace = _workspace(torch, dev)
    elif workspace.device.index != dev:
        raise ValueError(f"the workspace must live on cuda:{dev}")
    lse = torch.empty(seqs, heads, dtype=torch.float32, device=q.device) if return_lse else None
    args = _ATTEND.pack(q.data_ptr(), out.data_ptr(), lse.data_ptr() if return_lse else 0, k_cache.data_ptr(),
                        v_cache.data_ptr(), page_table.data_ptr(), lens.data_ptr(), workspace.ptr, workspace.bytes,
                        *q_str[:2], *out_str[:2], heads, 1, *cache, table_stride, seqs, heads, kv_heads, dim, code,
                        pages, page, max_pages, dim ** -0.5 if scale is None else scale)
    _call(_c.hv_paged_attention, dev, args)
    return (out, lse) if return_lse else out
