// hv_decode_chunk.cu — attention of a chunk of new tokens of each sequence over a paged cache.
//
//   out[t, h] = sum_j softmax_j(scale * q[t, h] . K[j, h / group]) V[j, h / group],  j < seen(t),
//   seen(t) = lens - n + i + 1 for the i-th of a sequence's n new tokens (causal), or lens;
//   a row that sees nothing gives zeros (and a log-sum-exp of -inf).
//
// A warp takes a row, its lanes the head's dimensions.
#include <math_constants.h>

#include "hv_decode.cuh"

namespace hv {
namespace {

using namespace dec;

constexpr float LOWEST = -3.402823466e38f;  // a running maximum before the first score

struct ChunkArgs {
    const void *q, *kc, *vc;
    void *out;
    float *lse;
    const int32_t *pages, *lens, *starts;
    long long q_tok, q_head, o_tok, o_head, lse_tok, lse_head;
    long long kc_page, kc_slot, kc_head, vc_page, vc_slot, vc_head, pages_stride;
    int tokens, seqs, heads, kv_heads, group, num_pages, page, max_pages, causal;
    float scale_log2;
    int *err;
};

// Start of sequence b (or its end: b + 1), brought into [0, tokens] and past none before it.
__device__ __forceinline__ int length_of(const ChunkArgs &a, int b) {
    const int n = max(a.lens[b], 0);
    const long long cap = min((long long)a.max_pages * a.page, (long long)HV_ATTENTION_MAX_LENGTH);
    if (n > cap) {
        atomicOr(a.err, HV_DECODE_BAD_LENGTH);
        return (int)cap;
    }
    return n;
}

template <typename T, int D>
__global__ void __launch_bounds__(256) chunk_simple_kernel(const __grid_constant__ ChunkArgs a) {
    griddep_wait();
    griddep_launch();
    constexpr int E = D / 32;
    const int lane = threadIdx.x & 31;
    const long long id = (long long)blockIdx.x * 8 + threadIdx.x / 32;
    const int b = blockIdx.y;
    const int s0 = min(max(a.starts[b], 0), a.tokens), s1 = min(max(a.starts[b + 1], 0), a.tokens);
    if (s1 < s0 || s0 != a.starts[b] || s1 != a.starts[b + 1]) atomicOr(a.err, HV_DECODE_BAD_START);
    const int n = max(s1 - s0, 0);
    const int len = length_of(a, b);
    for (long long w = id; w < (long long)n * a.heads; w += (long long)gridDim.x * 8) {
        const int i = (int)(w / a.heads), h = (int)(w - (long long)i * a.heads), kvh = h / a.group;
        const int seen = a.causal ? max(len - n + i + 1, 0) : len;
        const T *q = (const T *)a.q + (long long)(s0 + i) * a.q_tok + h * a.q_head + lane * E;
        float qv[E], o[E], m = LOWEST, l = 0.f;
        for (int e = 0; e < E; ++e) qv[e] = to_f32(q[e]) * a.scale_log2, o[e] = 0.f;
        for (int j = 0; j < seen; ++j) {
            const int pg = a.pages[b * a.pages_stride + j / a.page], slot = j % a.page;
            const bool ok = pg >= 0 && pg < a.num_pages;
            if (!ok && lane == 0) atomicOr(a.err, HV_DECODE_BAD_PAGE);
            const T *k = (const T *)a.kc + (ok ? pg * a.kc_page + slot * a.kc_slot + kvh * a.kc_head + lane * E : 0);
            const T *v = (const T *)a.vc + (ok ? pg * a.vc_page + slot * a.vc_slot + kvh * a.vc_head + lane * E : 0);
            float s = 0.f;
            if (ok)
                for (int e = 0; e < E; ++e) s += qv[e] * to_f32(k[e]);
            for (int x = 16; x; x /= 2) s += __shfl_xor_sync(~0u, s, x);
            const float mn = fmaxf(m, s), f = exp2f(m - mn), p = exp2f(s - mn);
            m = mn;
            l = l * f + p;
            for (int e = 0; e < E; ++e) o[e] = o[e] * f + (ok ? p * to_f32(v[e]) : 0.f);
        }
        T *out = (T *)a.out + (long long)(s0 + i) * a.o_tok + h * a.o_head + lane * E;
        for (int e = 0; e < E; ++e) out[e] = from_f32<T>(seen ? o[e] / l : 0.f);
        if (a.lse && lane == 0)
            a.lse[(long long)(s0 + i) * a.lse_tok + h * a.lse_head] =
                seen ? (m + log2f(l)) * 0.69314718055994531f : -CUDART_INF_F;
    }
}

template <typename T, int D>
cudaError_t launch(const ChunkArgs &a, cudaStream_t st) {
    return launch_pdl(chunk_simple_kernel<T, D>, dim3(1024, (unsigned)a.seqs), dim3(256), 0, st, a);
}

template <typename T>
cudaError_t by_dim(const ChunkArgs &a, int dim, cudaStream_t st) {
    switch (dim) {
        case 32: return launch<T, 32>(a, st);
        case 64: return launch<T, 64>(a, st);
        case 96: return launch<T, 96>(a, st);
        case 128: return launch<T, 128>(a, st);
        case 192: return launch<T, 192>(a, st);
        default: return launch<T, 256>(a, st);
    }
}

bool known_dim(int d) { return d == 32 || d == 64 || d == 96 || d == 128 || d == 192 || d == 256; }

}  // namespace
}  // namespace hv

using namespace hv;

extern "C" int hv_paged_chunk_attention_workspace(int dim, int64_t *bytes) {
    if (!bytes) return fail(HV_ERR_VALUE, "null argument");
    if (!known_dim(dim)) return fail(HV_ERR_VALUE, "dim must be 32, 64, 96, 128, 192 or 256");
    *bytes = HV_ATTENTION_COUNTER_BYTES;
    return HV_OK;
}

extern "C" int hv_paged_chunk_attention(const hv_chunk_args *p, void *stream) {
    if (!p) return fail(HV_ERR_VALUE, "null argument");
    if (p->dtype != HV_BF16 && p->dtype != HV_F16) return fail(HV_ERR_TYPE, "dtype must be HV_BF16 or HV_F16");
    if (p->tokens < 0 || p->seqs < 0 || p->heads < 1 || p->kv_heads < 1 || p->heads % p->kv_heads)
        return fail(HV_ERR_VALUE, "heads must be a positive multiple of kv_heads");
    if (!known_dim(p->dim)) return fail(HV_ERR_VALUE, "dim must be 32, 64, 96, 128, 192 or 256");
    if (p->page_size < 1 || p->num_pages < 0 || p->max_pages < 0) return fail(HV_ERR_VALUE, "bad cache geometry");
    if ((double)p->tokens * (p->heads / p->kv_heads) > HV_ATTENTION_MAX_LENGTH)
        return fail(HV_ERR_VALUE, "too many rows for one call");
    if (p->seqs == 0 || p->tokens == 0) return HV_OK;
    if (!p->d_q || !p->d_out || !p->d_lens || !p->d_starts || (p->max_pages && !p->d_page_table) ||
        (p->num_pages && (!p->d_k_cache || !p->d_v_cache)))
        return fail(HV_ERR_VALUE, "null buffer");
    int64_t need = 0;
    const int rc = hv_paged_chunk_attention_workspace(p->dim, &need);
    if (rc) return rc;
    if (!p->d_workspace || p->workspace_bytes < need)
        return fail(HV_ERR_VALUE, "the workspace has %lld bytes of %lld", (long long)p->workspace_bytes, (long long)need);
    if (!dec::aligned(p->d_workspace, 256)) return fail(HV_ERR_VALUE, "the workspace must be 256-byte aligned");
    bool ok = dec::aligned(p->d_k_cache, 16) && dec::aligned(p->d_v_cache, 16);
    for (int i = 0; i < 3; ++i) ok = ok && p->k_cache_strides[i] % 8 == 0 && p->v_cache_strides[i] % 8 == 0;
    if (!ok) return fail(HV_ERR_VALUE, "cache rows must start on 16 bytes");
    int *err = dec::error_word();
    if (!err) return fail(HV_ERR_CUDA, "cannot resolve the device error word");
    ChunkArgs a{};
    a.q = p->d_q, a.kc = p->d_k_cache, a.vc = p->d_v_cache, a.out = p->d_out, a.lse = p->d_lse;
    a.pages = p->d_page_table, a.lens = p->d_lens, a.starts = p->d_starts;
    a.q_tok = p->q_strides[0], a.q_head = p->q_strides[1], a.o_tok = p->out_strides[0], a.o_head = p->out_strides[1];
    a.lse_tok = p->lse_strides[0], a.lse_head = p->lse_strides[1];
    a.kc_page = p->k_cache_strides[0], a.kc_slot = p->k_cache_strides[1], a.kc_head = p->k_cache_strides[2];
    a.vc_page = p->v_cache_strides[0], a.vc_slot = p->v_cache_strides[1], a.vc_head = p->v_cache_strides[2];
    a.pages_stride = p->page_table_stride;
    a.tokens = p->tokens, a.seqs = p->seqs, a.heads = p->heads, a.kv_heads = p->kv_heads, a.group = p->heads / p->kv_heads;
    a.num_pages = p->num_pages, a.page = p->page_size, a.max_pages = p->max_pages, a.causal = p->causal;
    a.scale_log2 = p->scale * 1.4426950408889634f;
    a.err = err;
    const cudaError_t e = p->dtype == HV_BF16 ? by_dim<__nv_bfloat16>(a, p->dim, (cudaStream_t)stream)
                                              : by_dim<__half>(a, p->dim, (cudaStream_t)stream);
    if (e != cudaSuccess) return fail(HV_ERR_CUDA, "paged_chunk_attention: %s", cudaGetErrorString(e));
    return HV_OK;
}
