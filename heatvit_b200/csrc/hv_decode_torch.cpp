// hv_decode_torch.cpp — the decode operators' calls from Python: tensors checked, outputs
// allocated, and the C entries of include/heatvit_b200.h called on the current stream.
//
// heatvit_b200/decode.py documents these functions and is what a user calls.  A decode step's
// operators run for two to ten microseconds, about what reading a dozen tensors' shapes and
// strides and allocating the outputs takes in Python, so that is done here.  Mistakes raise
// TypeError and ValueError; a status that a C entry returns comes back as an int.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <map>
#include <utility>

#include "../../include/heatvit_b200.h"

namespace {

using at::Tensor;

// A caller's mistake, to be raised as `kind`.
struct Mistake {
    PyObject *kind;
    char text[256];
};
__attribute__((format(printf, 2, 3))) Mistake mistake(PyObject *kind, const char *format, ...) {
    Mistake m{kind, ""};
    va_list args;
    va_start(args, format);
    vsnprintf(m.text, sizeof(m.text), format, args);
    va_end(args);
    return m;
}
#define TypeError(...) mistake(PyExc_TypeError, __VA_ARGS__)
#define ValueError(...) mistake(PyExc_ValueError, __VA_ARGS__)

const Tensor &tensor(PyObject *o, const char *name) {
    if (!THPVariable_Check(o)) throw TypeError("%s must be a torch.Tensor", name);
    return THPVariable_Unpack(o);
}

// The device of an operator's first tensor, which the others share.
int device_of(const Tensor &t, const char *name) {
    if (!t.is_cuda()) throw ValueError("%s must be a CUDA tensor", name);
    return t.get_device();
}

void on(const Tensor &t, const char *name, int dev) {
    if (!t.is_cuda() || t.get_device() != dev) throw ValueError("%s must live on cuda:%d", name, dev);
}

// What every operand passes: its device, its number of dimensions, a contiguous last one.
void need(const Tensor &t, const char *name, int64_t dims, int dev) {
    on(t, name, dev);
    if (t.dim() != dims) throw ValueError("%s must be %d-dimensional", name, (int)dims);
    if (dims && t.size(dims - 1) > 1 && t.stride(dims - 1) != 1)
        throw ValueError("%s's last dimension must be contiguous", name);
}

// An operand that is written: elements that share memory (an expanded tensor) would be a race.
void need_apart(const Tensor &t, const char *name) {
    for (int64_t i = 0; i < t.dim(); ++i)
        if (t.size(i) > 1 && t.stride(i) == 0) throw ValueError("%s is written, so its elements may not share memory", name);
}

void need_ints(const Tensor &t, const char *name, int64_t dims, int dev) {
    if (t.scalar_type() != at::kInt) throw TypeError("%s must be int32", name);
    need(t, name, dims, dev);
}

// An operand of another one's shape and type.
void need_like(const Tensor &t, const char *name, const Tensor &other, const char *its_name, int dev) {
    need(t, name, other.dim(), dev);
    if (t.sizes() != other.sizes()) throw ValueError("%s must have %s's shape", name, its_name);
    if (t.scalar_type() != other.scalar_type()) throw TypeError("%s must have %s's type", name, its_name);
}

// A caller's tensor has been written: autograd's check of saved tensors goes by this.  (Tensors
// made in inference mode have no versions.)
void written(const Tensor &t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

int type_code(at::ScalarType t) {
    return t == at::kBFloat16 ? HV_BF16 : t == at::kHalf ? HV_F16 : t == at::kFloat ? HV_F32 : -1;
}

int32_t int_of(int64_t v, const char *name) {
    if (v > INT32_MAX) throw ValueError("%s is above 2^31", name);
    return (int32_t)v;
}

Tensor empty(c10::IntArrayRef size, at::ScalarType type, const Tensor &like) {
    return at::detail::empty_cuda(size, type, like.device(), std::nullopt);
}

void *stream_of(int dev) { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream(); }

PyObject *none() { Py_RETURN_NONE; }

// Rows of `t` (its first dimension) that start a multiple of `by` elements apart.
Tensor padded_rows(int64_t rows, int64_t dim, int64_t by, at::ScalarType type, const Tensor &like) {
    const int64_t wide = (dim + by - 1) / by * by;
    if (wide == dim) return empty({rows, dim}, type, like);
    return empty({rows, wide}, type, like).narrow(1, 0, dim);
}

// A tensor of `size` and `strides` in the storage of `bytes`, from byte `at` (a multiple of an element).
Tensor within(const Tensor &bytes, int64_t at, c10::IntArrayRef size, c10::IntArrayRef strides, at::ScalarType type) {
    Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(bytes.storage()), bytes.key_set(),
                                                        c10::scalarTypeToTypeMeta(type));
    t.unsafeGetTensorImpl()->set_sizes_and_strides(size, strides, at / (int64_t)c10::elementSize(type));
    return t;
}

// Around a function's body: no C++ exception passes into Python.
#define BEGIN        \
    HANDLE_TH_ERRORS \
    try {
#define END                                  \
    }                                        \
    catch (const Mistake &m) {               \
        PyErr_SetString(m.kind, m.text);     \
        return nullptr;                      \
    }                                        \
    END_HANDLE_TH_ERRORS

#define ARGUMENTS(n)                                                                     \
    if (nargs != n) {                                                                    \
        PyErr_Format(PyExc_TypeError, "%s takes %d arguments, got %zd", __func__, n, nargs); \
        return nullptr;                                                                  \
    }

// (x, weight, eps, residual, residual_out) -> (q, scale, residual_out)
PyObject *add_rmsnorm_fp8(PyObject *, PyObject *const *o, Py_ssize_t nargs) {
    BEGIN
    ARGUMENTS(5)
    const Tensor &x = tensor(o[0], "x"), &w = tensor(o[1], "weight");
    const double eps = PyFloat_AsDouble(o[2]);
    if (eps == -1.0 && PyErr_Occurred()) return nullptr;
    const int dev = device_of(x, "x");
    need(x, "x", 2, dev);
    need(w, "weight", 1, dev);
    const int code = type_code(x.scalar_type());
    if (code < 0) throw TypeError("x must be bfloat16, float16 or float32");
    const int64_t rows = x.size(0), dim = x.size(1), groups = (dim + 127) / 128;
    if (w.size(0) != dim) throw ValueError("weight has %lld channels, x %lld", (long long)w.size(0), (long long)dim);
    if (w.scalar_type() != x.scalar_type()) throw TypeError("weight must have x's type");
    Tensor out;
    const Tensor *res = nullptr;
    if (o[3] != Py_None) {
        res = &tensor(o[3], "residual");
        need_like(*res, "residual", x, "x", dev);
        if (o[4] != Py_None) {
            out = tensor(o[4], "residual_out");
            need_like(out, "residual_out", x, "x", dev);
            need_apart(out, "residual_out");
        } else {
            out = padded_rows(rows, dim, 8, x.scalar_type(), x);
        }
    } else if (o[4] != Py_None) {
        throw ValueError("residual_out without a residual");
    }
    const c10::cuda::CUDAGuard guard((c10::DeviceIndex)dev);
    // q and its scales are used together, so they share a storage: an allocation less is 0.5 us
    // of a call of 6.
    const int64_t wide = (dim + 15) / 16 * 16, scale_at = (rows * wide + 255) / 256 * 256;
    const Tensor both = empty({scale_at + rows * groups * 4}, at::kByte, x);
    Tensor q = within(both, 0, {rows, dim}, {wide, 1}, at::kFloat8_e4m3fn);
    Tensor scale = within(both, scale_at, {rows, groups}, {1, rows}, at::kFloat);
    hv_norm_args a{};
    a.d_x = x.data_ptr(), a.d_weight = w.data_ptr(), a.d_q = q.data_ptr(), a.d_scale = scale.data_ptr<float>();
    a.rows = rows, a.x_stride = x.stride(0), a.q_stride = q.stride(0);
    if (res) {
        a.d_residual = res->data_ptr(), a.residual_stride = res->stride(0);
        a.d_residual_out = out.data_ptr(), a.residual_out_stride = out.stride(0);
    }
    a.scale_strides[0] = 1, a.scale_strides[1] = rows;
    a.dim = int_of(dim, "dim"), a.dtype = code, a.eps = (float)eps;
    if (const int rc = hv_add_rmsnorm_fp8(&a, stream_of(dev))) return PyLong_FromLong(rc);
    if (o[4] != Py_None) written(out);
    PyObject *r = PyTuple_New(3);
    if (!r) return nullptr;
    PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(std::move(q)));
    PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(std::move(scale)));
    PyTuple_SET_ITEM(r, 2, res ? THPVariable_Wrap(std::move(out)) : none());
    return r;
    END
}

// (a, a_scale, b, b_scale, out_dtype, out) -> out
PyObject *gemm_fp8(PyObject *, PyObject *const *o, Py_ssize_t nargs) {
    BEGIN
    ARGUMENTS(6)
    const Tensor &a = tensor(o[0], "a"), &as = tensor(o[1], "a_scale"), &b = tensor(o[2], "b"), &bs = tensor(o[3], "b_scale");
    const int dev = device_of(a, "a");
    need(a, "a", 2, dev);
    need(b, "b", 2, dev);
    if (a.scalar_type() != at::kFloat8_e4m3fn || b.scalar_type() != at::kFloat8_e4m3fn)
        throw TypeError("a and b must be float8_e4m3fn");
    const int64_t m = a.size(0), n = b.size(0), k = a.size(1), groups = (k + 127) / 128;
    if (b.size(1) != k) throw ValueError("K mismatch: a has %lld, b has %lld", (long long)k, (long long)b.size(1));
    if (k < 1) throw ValueError("k must be positive");
    const auto scale_of = [&](const Tensor &t, const char *name, int64_t rows) {
        on(t, name, dev);
        if (t.scalar_type() != at::kFloat) throw TypeError("%s must be float32", name);
        if (t.dim() != 2 || t.size(0) != rows || t.size(1) != groups)
            throw ValueError("%s must be [%lld, %lld]", name, (long long)rows, (long long)groups);
    };
    scale_of(as, "a_scale", m);
    scale_of(bs, "b_scale", (n + 127) / 128);
    at::ScalarType type = at::kBFloat16;
    if (o[4] != Py_None) {
        if (!THPDtype_Check(o[4])) throw TypeError("out_dtype must be a torch.dtype");
        type = ((THPDtype *)o[4])->scalar_type;
    }
    Tensor out;
    if (o[5] != Py_None) {
        out = tensor(o[5], "out");
        need(out, "out", 2, dev);
        need_apart(out, "out");
        if (out.size(0) != m || out.size(1) != n) throw ValueError("out must be [%lld, %lld]", (long long)m, (long long)n);
        if (o[4] != Py_None && out.scalar_type() != type) throw TypeError("out has another type than out_dtype");
        type = out.scalar_type();
    }
    const int code = type_code(type);
    if (code < 0) throw TypeError("out must be bfloat16, float16 or float32");
    const c10::cuda::CUDAGuard guard((c10::DeviceIndex)dev);
    if (!out.defined()) out = empty({m, n}, type, a);
    hv_gemm_fp8_args g{};
    g.d_a = a.data_ptr(), g.d_b = b.data_ptr(), g.d_a_scale = as.data_ptr<float>(), g.d_b_scale = bs.data_ptr<float>();
    g.d_out = out.data_ptr();
    g.m = m, g.n = n, g.k = k, g.a_stride = a.stride(0), g.b_stride = b.stride(0), g.out_stride = out.stride(0);
    for (int i = 0; i < 2; ++i) g.a_scale_strides[i] = as.stride(i), g.b_scale_strides[i] = bs.stride(i);
    g.out_dtype = code;
    if (const int rc = hv_gemm_fp8(&g, stream_of(dev))) return PyLong_FromLong(rc);
    if (o[5] != Py_None) written(out);
    return THPVariable_Wrap(std::move(out));
    END
}

void need_caches(const Tensor &kc, const Tensor &vc, int dev) {
    need(kc, "k_cache", 4, dev);
    need_like(vc, "v_cache", kc, "k_cache", dev);
}

// The weight of a norm of heads of `dim`, or null.
const void *head_weight(PyObject *o, const char *name, int64_t dim, at::ScalarType type, int dev) {
    if (o == Py_None) return nullptr;
    const Tensor &w = tensor(o, name);
    need(w, name, 1, dev);
    if (w.size(0) != dim) throw ValueError("%s has %lld channels, a head %lld", name, (long long)w.size(0), (long long)dim);
    if (w.scalar_type() != type) throw TypeError("%s must have k's type", name);
    return w.data_ptr();
}

// (k, v, k_cache, v_cache, page_table, positions, seq_ids, rope, q, interleaved, q_out) -> q_out; with the norms'
// (q_weight, k_weight, eps) behind them where `norm`
PyObject *append(PyObject *const *o, bool norm) {
    BEGIN
    const Tensor &k = tensor(o[0], "k"), &v = tensor(o[1], "v"), &kc = tensor(o[2], "k_cache"), &vc = tensor(o[3], "v_cache");
    const Tensor &table = tensor(o[4], "page_table"), &pos = tensor(o[5], "positions");
    const int dev = device_of(k, "k");
    need(k, "k", 3, dev);
    need_like(v, "v", k, "k", dev);
    need_caches(kc, vc, dev);
    need_apart(kc, "k_cache");
    need_apart(vc, "v_cache");
    need_ints(table, "page_table", 2, dev);
    need_ints(pos, "positions", 1, dev);
    const int code = type_code(k.scalar_type());
    if (code != HV_BF16 && code != HV_F16) throw TypeError("k must be bfloat16 or float16");
    if (kc.scalar_type() != k.scalar_type()) throw TypeError("k, v and the caches must have the same type");
    const int64_t tokens = k.size(0), kv_heads = k.size(1), dim = k.size(2);
    if (kc.size(2) != kv_heads || kc.size(3) != dim)
        throw ValueError("the caches hold other heads or another head dimension");
    if (pos.size(0) != tokens) throw ValueError("one position per token");
    hv_append_args a{};
    if (o[6] != Py_None) {
        const Tensor &ids = tensor(o[6], "seq_ids");
        need_ints(ids, "seq_ids", 1, dev);
        if (ids.size(0) != tokens) throw ValueError("one sequence id per token");
        a.d_seq_ids = ids.data_ptr<int32_t>();
    } else if (table.size(0) < tokens) {
        throw ValueError("without seq_ids the page table has one row per token");
    }
    if (o[7] != Py_None) {
        const Tensor &rope = tensor(o[7], "rope");
        need(rope, "rope", 2, dev);
        if (rope.scalar_type() != at::kFloat) throw TypeError("rope must be float32");
        a.d_rope = rope.data_ptr<float>(), a.rope_stride = rope.stride(0);
        a.rope_rows = int_of(rope.size(0), "rope"), a.rot = int_of(rope.size(1), "rope");
    }
    const int interleaved = PyObject_IsTrue(o[9]);
    if (interleaved < 0) return nullptr;
    const c10::cuda::CUDAGuard guard((c10::DeviceIndex)dev);
    Tensor out;
    if (o[8] != Py_None) {
        const Tensor &q = tensor(o[8], "q");
        need(q, "q", 3, dev);
        if (q.size(0) != tokens || q.size(2) != dim) throw ValueError("q must be [tokens, heads, dim]");
        if (q.scalar_type() != k.scalar_type()) throw TypeError("q must have k's type");
        if (o[10] != Py_None) {
            out = tensor(o[10], "q_out");
            need_like(out, "q_out", q, "q", dev);
            need_apart(out, "q_out");
        } else {
            out = empty(q.sizes(), q.scalar_type(), q);
        }
        a.d_q = q.data_ptr(), a.d_q_out = out.data_ptr(), a.heads = int_of(q.size(1), "heads");
        for (int i = 0; i < 2; ++i) a.q_strides[i] = q.stride(i), a.q_out_strides[i] = out.stride(i);
    } else if (o[10] != Py_None) {
        throw ValueError("q_out without q");
    }
    a.d_k = k.data_ptr(), a.d_v = v.data_ptr(), a.d_k_cache = kc.data_ptr(), a.d_v_cache = vc.data_ptr();
    a.d_page_table = table.data_ptr<int32_t>(), a.d_positions = pos.data_ptr<int32_t>();
    for (int i = 0; i < 2; ++i) a.k_strides[i] = k.stride(i), a.v_strides[i] = v.stride(i);
    for (int i = 0; i < 3; ++i) a.k_cache_strides[i] = kc.stride(i), a.v_cache_strides[i] = vc.stride(i);
    a.page_table_stride = table.stride(0);
    a.tokens = int_of(tokens, "tokens"), a.kv_heads = int_of(kv_heads, "kv_heads"), a.dim = int_of(dim, "dim");
    a.interleaved = interleaved, a.dtype = code;
    a.num_pages = int_of(kc.size(0), "pages"), a.page_size = int_of(kc.size(1), "page size");
    a.seqs = int_of(table.size(0), "page_table"), a.max_pages = int_of(table.size(1), "page_table");
    int rc;
    if (norm) {
        hv_norm_append_args n{a, nullptr, nullptr, 0.f};
        if (o[11] != Py_None && o[8] == Py_None) throw ValueError("q_weight without q");
        n.d_q_weight = head_weight(o[11], "q_weight", dim, k.scalar_type(), dev);
        n.d_k_weight = head_weight(o[12], "k_weight", dim, k.scalar_type(), dev);
        const double eps = PyFloat_AsDouble(o[13]);
        if (eps == -1.0 && PyErr_Occurred()) return nullptr;
        n.eps = (float)eps;
        rc = hv_norm_append_kv(&n, stream_of(dev));
    } else {
        rc = hv_append_kv(&a, stream_of(dev));
    }
    if (rc) return PyLong_FromLong(rc);
    written(kc);
    written(vc);
    if (o[10] != Py_None) written(out);
    return out.defined() ? THPVariable_Wrap(std::move(out)) : none();
    END
}
PyObject *append_kv(PyObject *, PyObject *const *o, Py_ssize_t nargs) {
    ARGUMENTS(11)
    return append(o, false);
}
PyObject *norm_append_kv(PyObject *, PyObject *const *o, Py_ssize_t nargs) {
    ARGUMENTS(14)
    return append(o, true);
}

int64_t workspace_bytes(bool chunks) {
    int64_t most = 0, need = 0;
    for (const int dim : {32, 64, 96, 128, 192, 256}) {
        TORCH_CHECK(hv_paged_attention_workspace(dim, &need) == HV_OK, hv_last_error());
        most = std::max(most, need);
        if (!chunks) continue;
        TORCH_CHECK(hv_paged_chunk_attention_workspace(dim, &need) == HV_OK, hv_last_error());
        most = std::max(most, need);
    }
    return most;
}

// Only the counters have to be zero: a fill of the whole 5 MB took 2.3 us of every captured call.
Tensor new_workspace(int dev, bool chunks) {
    const c10::cuda::CUDAGuard guard((c10::DeviceIndex)dev);
    Tensor t = at::detail::empty_cuda({workspace_bytes(chunks)}, at::kByte, at::Device(at::kCUDA, (c10::DeviceIndex)dev),
                                      std::nullopt);
    t.narrow(0, 0, HV_ATTENTION_COUNTER_BYTES).zero_();
    return t;
}

// (device index) -> a workspace tensor, its counters zeroed
PyObject *attention_workspace(PyObject *, PyObject *const *o, Py_ssize_t nargs) {
    BEGIN
    ARGUMENTS(1)
    const long dev = PyLong_AsLong(o[0]);
    if (dev == -1 && PyErr_Occurred()) return nullptr;
    return THPVariable_Wrap(new_workspace((int)dev, false));
    END
}
// (device index) -> one that paged_chunk_attention can use as well
PyObject *chunk_attention_workspace(PyObject *, PyObject *const *o, Py_ssize_t nargs) {
    BEGIN
    ARGUMENTS(1)
    const long dev = PyLong_AsLong(o[0]);
    if (dev == -1 && PyErr_Occurred()) return nullptr;
    return THPVariable_Wrap(new_workspace((int)dev, true));
    END
}

// The current stream's own workspace, made at its first call; a fresh one while the stream is
// being captured, since a graph may be replayed on any stream.
Tensor workspace_of(int dev, cudaStream_t stream, bool chunks) {
    // never destroyed: the CUDA context may be gone before a static would be
    static auto *held = new std::map<std::pair<int, cudaStream_t>, Tensor>[2];
    cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
    C10_CUDA_CHECK(cudaStreamIsCapturing(stream, &status));
    if (status != cudaStreamCaptureStatusNone) return new_workspace(dev, chunks);
    Tensor &t = held[chunks][{dev, stream}];
    if (!t.defined()) t = new_workspace(dev, chunks);
    return t;
}

// The caller's workspace, or the current stream's.
Tensor workspace(PyObject *o, int dev, c10::cuda::CUDAStream current, bool chunks) {
    if (o == Py_None) return workspace_of(dev, current.stream(), chunks);
    const Tensor &ws = tensor(o, "workspace");
    on(ws, "workspace", dev);
    if (ws.scalar_type() != at::kByte || !ws.is_contiguous()) throw TypeError("workspace must be contiguous bytes");
    // made on another stream perhaps: its memory is not handed on before this call is through
    c10::cuda::CUDACachingAllocator::recordStream(ws.storage().data_ptr(), current);
    return ws;
}

// An attention's softmax scale: dim^-0.5 for None; false with a Python error set.
bool scale_of(PyObject *o, int64_t dim, float *scale) {
    const double v = o == Py_None ? 1.0 / std::sqrt((double)dim) : PyFloat_AsDouble(o);
    *scale = (float)v;
    return !(v == -1.0 && PyErr_Occurred());
}

PyObject *with_or_without(Tensor out, Tensor more) {
    if (!more.defined()) return THPVariable_Wrap(std::move(out));
    PyObject *r = PyTuple_New(2);
    if (!r) return nullptr;
    PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(std::move(out)));
    PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(std::move(more)));
    return r;
}

// (q, k_cache, v_cache, page_table, lens, scale, workspace, out, return_lse) -> out or (out, lse)
PyObject *paged_attention(PyObject *, PyObject *const *o, Py_ssize_t nargs) {
    BEGIN
    ARGUMENTS(9)
    const Tensor &q = tensor(o[0], "q"), &kc = tensor(o[1], "k_cache"), &vc = tensor(o[2], "v_cache");
    const Tensor &table = tensor(o[3], "page_table"), &lens = tensor(o[4], "lens");
    const int dev = device_of(q, "q");
    need(q, "q", 3, dev);
    need_caches(kc, vc, dev);
    need_ints(table, "page_table", 2, dev);
    need_ints(lens, "lens", 1, dev);
    const int code = type_code(q.scalar_type());
    if (code != HV_BF16 && code != HV_F16) throw TypeError("q must be bfloat16 or float16");
    if (kc.scalar_type() != q.scalar_type()) throw TypeError("q and the caches must have the same type");
    const int64_t seqs = q.size(0), heads = q.size(1), dim = q.size(2), kv_heads = kc.size(2);
    if (kc.size(3) != dim) throw ValueError("the caches have another head dimension");
    if (kv_heads < 1 || heads < 1 || heads % kv_heads) throw ValueError("heads must be a positive multiple of kv_heads");
    if (table.size(0) != seqs || lens.size(0) != seqs) throw ValueError("page_table and lens have one row per sequence");
    float scale = 0;
    if (!scale_of(o[5], dim, &scale)) return nullptr;
    const int with_lse = PyObject_IsTrue(o[8]);
    if (with_lse < 0) return nullptr;
    const c10::cuda::CUDAGuard guard((c10::DeviceIndex)dev);
    const c10::cuda::CUDAStream current = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev);
    const cudaStream_t stream = current.stream();
    Tensor out;
    if (o[7] != Py_None) {
        out = tensor(o[7], "out");
        need_like(out, "out", q, "q", dev);
        need_apart(out, "out");
    } else {
        out = empty(q.sizes(), q.scalar_type(), q);
    }
    const Tensor ws = workspace(o[6], dev, current, false);
    Tensor lse;
    if (with_lse) lse = empty({seqs, heads}, at::kFloat, q);
    hv_attention_args a{};
    a.d_q = q.data_ptr(), a.d_out = out.data_ptr(), a.d_lse = with_lse ? lse.data_ptr<float>() : nullptr;
    a.d_k_cache = kc.data_ptr(), a.d_v_cache = vc.data_ptr();
    a.d_page_table = table.data_ptr<int32_t>(), a.d_lens = lens.data_ptr<int32_t>();
    a.d_workspace = ws.data_ptr(), a.workspace_bytes = ws.numel();
    for (int i = 0; i < 2; ++i) a.q_strides[i] = q.stride(i), a.out_strides[i] = out.stride(i);
    a.lse_strides[0] = heads, a.lse_strides[1] = 1;
    for (int i = 0; i < 3; ++i) a.k_cache_strides[i] = kc.stride(i), a.v_cache_strides[i] = vc.stride(i);
    a.page_table_stride = table.stride(0);
    a.seqs = int_of(seqs, "seqs"), a.heads = int_of(heads, "heads"), a.kv_heads = int_of(kv_heads, "kv_heads");
    a.dim = int_of(dim, "dim"), a.dtype = code;
    a.num_pages = int_of(kc.size(0), "pages"), a.page_size = int_of(kc.size(1), "page size");
    a.max_pages = int_of(table.size(1), "page_table"), a.scale = scale;
    if (const int rc = hv_paged_attention(&a, stream)) return PyLong_FromLong(rc);
    if (o[7] != Py_None) written(out);
    return with_or_without(std::move(out), std::move(lse));
    END
}

// (q, k_cache, v_cache, page_table, lens, starts, causal, scale, workspace, out, return_lse) -> out or (out, lse)
PyObject *paged_chunk_attention(PyObject *, PyObject *const *o, Py_ssize_t nargs) {
    BEGIN
    ARGUMENTS(11)
    const Tensor &q = tensor(o[0], "q"), &kc = tensor(o[1], "k_cache"), &vc = tensor(o[2], "v_cache");
    const Tensor &table = tensor(o[3], "page_table"), &lens = tensor(o[4], "lens"), &starts = tensor(o[5], "starts");
    const int dev = device_of(q, "q");
    need(q, "q", 3, dev);
    need_caches(kc, vc, dev);
    need_ints(table, "page_table", 2, dev);
    need_ints(lens, "lens", 1, dev);
    need_ints(starts, "starts", 1, dev);
    const int code = type_code(q.scalar_type());
    if (code != HV_BF16 && code != HV_F16) throw TypeError("q must be bfloat16 or float16");
    if (kc.scalar_type() != q.scalar_type()) throw TypeError("q and the caches must have the same type");
    const int64_t tokens = q.size(0), heads = q.size(1), dim = q.size(2), kv_heads = kc.size(2), seqs = lens.size(0);
    if (kc.size(3) != dim) throw ValueError("the caches have another head dimension");
    if (kv_heads < 1 || heads < 1 || heads % kv_heads) throw ValueError("heads must be a positive multiple of kv_heads");
    if (table.size(0) != seqs) throw ValueError("page_table and lens have one row per sequence");
    if (starts.size(0) != seqs + 1) throw ValueError("starts has one more entry than there are sequences");
    const int causal = PyObject_IsTrue(o[6]), with_lse = PyObject_IsTrue(o[10]);
    if (causal < 0 || with_lse < 0) return nullptr;
    float scale = 0;
    if (!scale_of(o[7], dim, &scale)) return nullptr;
    const c10::cuda::CUDAGuard guard((c10::DeviceIndex)dev);
    const c10::cuda::CUDAStream current = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev);
    Tensor out;
    if (o[9] != Py_None) {
        out = tensor(o[9], "out");
        need_like(out, "out", q, "q", dev);
        need_apart(out, "out");
    } else {
        out = empty(q.sizes(), q.scalar_type(), q);
    }
    const Tensor ws = workspace(o[8], dev, current, true);
    Tensor lse;
    if (with_lse) lse = empty({tokens, heads}, at::kFloat, q);
    hv_chunk_args a{};
    a.d_q = q.data_ptr(), a.d_out = out.data_ptr(), a.d_lse = with_lse ? lse.data_ptr<float>() : nullptr;
    a.d_k_cache = kc.data_ptr(), a.d_v_cache = vc.data_ptr();
    a.d_page_table = table.data_ptr<int32_t>(), a.d_lens = lens.data_ptr<int32_t>(), a.d_starts = starts.data_ptr<int32_t>();
    a.d_workspace = ws.data_ptr(), a.workspace_bytes = ws.numel();
    for (int i = 0; i < 2; ++i) a.q_strides[i] = q.stride(i), a.out_strides[i] = out.stride(i);
    a.lse_strides[0] = heads, a.lse_strides[1] = 1;
    for (int i = 0; i < 3; ++i) a.k_cache_strides[i] = kc.stride(i), a.v_cache_strides[i] = vc.stride(i);
    a.page_table_stride = table.stride(0);
    a.tokens = int_of(tokens, "tokens"), a.seqs = int_of(seqs, "seqs"), a.heads = int_of(heads, "heads");
    a.kv_heads = int_of(kv_heads, "kv_heads"), a.dim = int_of(dim, "dim"), a.dtype = code, a.causal = causal;
    a.num_pages = int_of(kc.size(0), "pages"), a.page_size = int_of(kc.size(1), "page size");
    a.max_pages = int_of(table.size(1), "page_table"), a.scale = scale;
    if (const int rc = hv_paged_chunk_attention(&a, current.stream())) return PyLong_FromLong(rc);
    if (o[9] != Py_None) written(out);
    return with_or_without(std::move(out), std::move(lse));
    END
}

// A setting of sample_tokens: None (`otherwise`), a number for all rows, or a tensor [rows] of `type`.  False with a
// Python error set.
template <typename N>
bool setting(PyObject *o, const char *name, at::ScalarType type, int64_t rows, int dev, N otherwise, N *number, const N **each) {
    *number = otherwise, *each = nullptr;
    if (o == Py_None) return true;
    if (THPVariable_Check(o)) {
        const Tensor &t = THPVariable_Unpack(o);
        if (t.scalar_type() != type) throw TypeError("%s must be %s", name, type == at::kInt ? "int32" : "float32");
        need(t, name, 1, dev);
        if (t.size(0) != rows) throw ValueError("%s must be a number or have one entry per row", name);
        *each = t.data_ptr<N>();
        return true;
    }
    if (type == at::kInt) {
        const long v = PyLong_AsLong(o);
        if (v == -1 && PyErr_Occurred()) return false;
        *number = (N)std::min(std::max(v, (long)INT32_MIN), (long)INT32_MAX);
    } else {
        const double v = PyFloat_AsDouble(o);
        if (v == -1.0 && PyErr_Occurred()) return false;
        *number = (N)v;
    }
    return true;
}

// (logits, uniform, temperature, top_k, top_p, min_p, out, return_logprob) -> tokens or (tokens, logprobs)
PyObject *sample_tokens(PyObject *, PyObject *const *o, Py_ssize_t nargs) {
    BEGIN
    ARGUMENTS(8)
    const Tensor &z = tensor(o[0], "logits"), &u = tensor(o[1], "uniform");
    const int dev = device_of(z, "logits");
    need(z, "logits", 2, dev);
    const int code = type_code(z.scalar_type());
    if (code < 0) throw TypeError("logits must be bfloat16, float16 or float32");
    const int64_t rows = z.size(0), vocab = z.size(1);
    if (u.scalar_type() != at::kFloat) throw TypeError("uniform must be float32");
    need(u, "uniform", 1, dev);
    if (u.size(0) != rows) throw ValueError("one uniform number per row");
    const int with_logprob = PyObject_IsTrue(o[7]);
    if (with_logprob < 0) return nullptr;
    hv_sample_args a{};
    if (!setting(o[2], "temperature", at::kFloat, rows, dev, 1.f, &a.temperature, &a.d_temperature) ||
        !setting(o[3], "top_k", at::kInt, rows, dev, 0, &a.top_k, &a.d_top_k) ||
        !setting(o[4], "top_p", at::kFloat, rows, dev, 1.f, &a.top_p, &a.d_top_p) ||
        !setting(o[5], "min_p", at::kFloat, rows, dev, 0.f, &a.min_p, &a.d_min_p))
        return nullptr;
    const c10::cuda::CUDAGuard guard((c10::DeviceIndex)dev);
    Tensor out, logprobs;
    if (o[6] != Py_None) {
        out = tensor(o[6], "out");
        if (out.scalar_type() != at::kLong) throw TypeError("out must be int64");
        need(out, "out", 1, dev);
        if (out.size(0) != rows) throw ValueError("out must have one entry per row");
    } else {
        out = empty({rows}, at::kLong, z);
    }
    if (with_logprob) logprobs = empty({rows}, at::kFloat, z);
    a.d_logits = z.data_ptr(), a.d_uniform = u.data_ptr<float>(), a.d_tokens = out.data_ptr<int64_t>();
    a.d_logprobs = with_logprob ? logprobs.data_ptr<float>() : nullptr;
    a.row_stride = z.stride(0), a.rows = int_of(rows, "rows"), a.vocab = int_of(vocab, "vocab"), a.dtype = code;
    if (const int rc = hv_sample_tokens(&a, stream_of(dev))) return PyLong_FromLong(rc);
    if (o[6] != Py_None) written(out);
    return with_or_without(std::move(out), std::move(logprobs));
    END
}

#define METHOD(f) {#f, (PyCFunction)(void (*)(void))f, METH_FASTCALL, nullptr}
PyMethodDef g_methods[] = {METHOD(add_rmsnorm_fp8), METHOD(gemm_fp8), METHOD(append_kv), METHOD(norm_append_kv),
                           METHOD(attention_workspace), METHOD(chunk_attention_workspace), METHOD(paged_attention),
                           METHOD(paged_chunk_attention), METHOD(sample_tokens), {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_decode_native", "Calls of heatvit_b200.decode.", -1, g_methods,
                        nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject *PyInit__decode_native() { return PyModule_Create(&g_module); }
