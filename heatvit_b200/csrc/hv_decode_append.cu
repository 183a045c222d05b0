// hv_decode_append.cu — keys and values into a paged cache, with the position rotation on the way.
//
// Token t of sequence s = seq_ids[t] (or t) at position p goes to page page_table[s][p / page],
// slot p % page.  The first `rot` elements of every q and k head are turned in pairs (u, w) by
// the angle of their pair at p: (u cos - w sin, u sin + w cos), the pair being elements (i,
// i + rot/2), or (2i, 2i + 1) when interleaved; cosines and sines come from a float32 table.
// One rounding of the 32-bit result; v and the elements past rot are copied.
//
// Bound by HBM (each element read once and written once), and for a decode step by the
// launch.  A thread moves two groups of eight elements: for the half-split form the groups
// that hold each other's partners.  Consecutive threads take consecutive groups of a head,
// then the heads of a token, q, k and v in one grid.
#include "hv_decode.cuh"

namespace hv {
namespace {

using namespace dec;

struct AppendArgs {
    const void *q, *k, *v;
    void *q_out, *kc, *vc;
    const float *table;       // [table_rows][rot]: cosines, then sines
    const int32_t *pages;     // [seqs][max_pages]
    const int32_t *seq_ids, *positions;
    long long q_tok, q_head, k_tok, k_head, v_tok, v_head, qo_tok, qo_head;
    long long kc_page, kc_slot, kc_head, vc_page, vc_slot, vc_head, table_stride;
    int tokens, heads, kv_heads, dim, rot, num_pages, page, seqs, max_pages, table_rows;
    long long pages_stride;
    int *err;
};

constexpr int THREADS = 256;

// PAIR: how many elements of each partner group a thread handles (8, or 1 where sizes or
// alignment do not allow 16-byte accesses).  Unit u of a head covers, for half-split, elements
// [u*PAIR, +PAIR) and their partners [rot/2 + u*PAIR, +PAIR) while u*PAIR < rot/2, then 2*PAIR
// consecutive elements past rot; interleaved and unrotated heads: 2*PAIR consecutive elements.
template <typename T, int PAIR, bool INTER>
__global__ void __launch_bounds__(THREADS) append_kernel(const AppendArgs a) {
    griddep_wait();
    griddep_launch();
    const int units = (a.dim + 2 * PAIR - 1) / (2 * PAIR);
    const int nh = a.heads + 2 * a.kv_heads;
    const unsigned per_token = (unsigned)nh * units;
    const long long total = (long long)a.tokens * per_token;
    const long long id = (long long)blockIdx.x * THREADS + threadIdx.x;
    if (id >= total) return;
    const int tok = (int)(id / per_token);
    const unsigned in = (unsigned)(id - (long long)tok * per_token);
    const int hh = in / units, u = in - hh * units;
    const bool is_q = hh < a.heads, is_k = !is_q && hh < a.heads + a.kv_heads;
    const int head = is_q ? hh : is_k ? hh - a.heads : hh - a.heads - a.kv_heads;
    const int pos = a.positions[tok];
    if (pos < 0 && !is_q) return;  // a padding token stores nothing
    if (a.rot && pos >= a.table_rows) {  // nor does one that the rotation table does not reach
        atomicOr(a.err, HV_DECODE_BAD_POSITION);
        return;
    }

    T *dst;
    const T *src;
    if (is_q) {
        src = (const T *)a.q + tok * a.q_tok + head * a.q_head;
        dst = (T *)a.q_out + tok * a.qo_tok + head * a.qo_head;
    } else {
        const int s = a.seq_ids ? a.seq_ids[tok] : tok;
        const int col = pos / a.page, slot = pos - col * a.page;
        if (s < 0 || s >= a.seqs || col >= a.max_pages) {
            atomicOr(a.err, HV_DECODE_BAD_POSITION);
            return;
        }
        const int pg = a.pages[s * a.pages_stride + col];
        if (pg < 0 || pg >= a.num_pages) {
            atomicOr(a.err, HV_DECODE_BAD_PAGE);
            return;
        }
        if (is_k) {
            src = (const T *)a.k + tok * a.k_tok + head * a.k_head;
            dst = (T *)a.kc + pg * a.kc_page + slot * a.kc_slot + head * a.kc_head;
        } else {
            src = (const T *)a.v + tok * a.v_tok + head * a.v_head;
            dst = (T *)a.vc + pg * a.vc_page + slot * a.vc_slot + head * a.vc_head;
        }
    }

    const int rot = is_q || is_k ? a.rot : 0;
    const int half = rot / 2;
    int c0 = u * 2 * PAIR, c1 = c0 + PAIR;  // the two groups' first elements
    if (!INTER && u * PAIR < half) {
        c0 = u * PAIR;
        c1 = half + c0;
    }
    const bool turned = c0 < rot;
    const float *tab = nullptr;
    if (turned) tab = a.table + (pos < 0 ? 0 : pos) * a.table_stride;
    float x0[PAIR], x1[PAIR];
    if constexpr (PAIR == 8) {
        load8(src + c0, a.dim - c0, true, x0);
        load8(src + c1, a.dim - c1, true, x1);
    } else {
        x0[0] = to_f32(src[c0]);
        x1[0] = c1 < a.dim ? to_f32(src[c1]) : 0.f;
    }
    if (turned) {
        if (!INTER) {
#pragma unroll
            for (int i = 0; i < PAIR; ++i) {
                const float c = tab[c0 + i], s = tab[half + c0 + i];
                const float p = x0[i], w = x1[i];
                x0[i] = p * c - w * s;
                x1[i] = p * s + w * c;
            }
        } else if constexpr (PAIR == 1) {
            const float c = tab[c0 >> 1], s = tab[half + (c0 >> 1)];
            const float p = x0[0], w = x1[0];
            x0[0] = p * c - w * s;
            x1[0] = p * s + w * c;
        } else {
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                float(&x)[PAIR] = g ? x1 : x0;
                const int b = g ? c1 : c0;
                if (b >= rot) continue;
#pragma unroll
                for (int i = 0; i < PAIR; i += 2) {
                    const float c = tab[(b + i) >> 1], s = tab[half + ((b + i) >> 1)];
                    const float p = x[i], w = x[i + 1];
                    x[i] = p * c - w * s;
                    x[i + 1] = p * s + w * c;
                }
            }
        }
    }
    if (is_q && pos < 0) {  // a padding token's q is defined: zeros
#pragma unroll
        for (int i = 0; i < PAIR; ++i) x0[i] = x1[i] = 0.f;
    }
    if constexpr (PAIR == 8) {
        store8(dst + c0, a.dim - c0, true, x0);
        store8(dst + c1, a.dim - c1, true, x1);
    } else {
        dst[c0] = from_f32<T>(x0[0]);
        if (c1 < a.dim) dst[c1] = from_f32<T>(x1[0]);
    }
}

template <typename T>
cudaError_t launch(const AppendArgs &a, bool wide, bool inter, cudaStream_t st) {
    const int per = wide ? 16 : 2;
    const long long total = (long long)a.tokens * (a.heads + 2 * a.kv_heads) * ((a.dim + per - 1) / per);
    const dim3 grid((unsigned)((total + THREADS - 1) / THREADS)), block(THREADS);
    if (wide)
        return inter ? launch_pdl(append_kernel<T, 8, true>, grid, block, 0, st, a)
                     : launch_pdl(append_kernel<T, 8, false>, grid, block, 0, st, a);
    return inter ? launch_pdl(append_kernel<T, 1, true>, grid, block, 0, st, a)
                 : launch_pdl(append_kernel<T, 1, false>, grid, block, 0, st, a);
}

}  // namespace
}  // namespace hv

using namespace hv;

extern "C" int hv_append_kv(const hv_append_args *p, void *stream) {
    if (!p) return fail(HV_ERR_VALUE, "null argument");
    if (p->dtype != HV_BF16 && p->dtype != HV_F16) return fail(HV_ERR_TYPE, "dtype must be HV_BF16 or HV_F16");
    if (p->tokens < 0 || p->heads < 0) return fail(HV_ERR_VALUE, "negative token or head count");
    if (p->kv_heads < 1 || p->dim < 1) return fail(HV_ERR_VALUE, "kv_heads and dim must be positive");
    if (p->rot < 0 || p->rot > p->dim || p->rot % 2) return fail(HV_ERR_VALUE, "rot must be even and in [0, dim]");
    if (p->page_size < 1 || p->num_pages < 0 || p->seqs < 0 || p->max_pages < 0)
        return fail(HV_ERR_VALUE, "bad cache geometry");
    if (p->tokens == 0) return HV_OK;
    if (!p->d_k || !p->d_v || !p->d_k_cache || !p->d_v_cache || !p->d_page_table || !p->d_positions)
        return fail(HV_ERR_VALUE, "null buffer");
    if (p->heads && (!p->d_q || !p->d_q_out)) return fail(HV_ERR_VALUE, "q heads without a q or q_out buffer");
    if (p->rot && (!p->d_rope || p->rope_rows < 1)) return fail(HV_ERR_VALUE, "rot without a table");
    int *err = dec::error_word();
    if (!err) return fail(HV_ERR_CUDA, "cannot resolve the device error word");
    AppendArgs a{};
    a.q = p->d_q, a.k = p->d_k, a.v = p->d_v, a.q_out = p->d_q_out, a.kc = p->d_k_cache, a.vc = p->d_v_cache;
    a.table = p->d_rope, a.pages = p->d_page_table, a.seq_ids = p->d_seq_ids, a.positions = p->d_positions;
    a.q_tok = p->q_strides[0], a.q_head = p->q_strides[1], a.k_tok = p->k_strides[0], a.k_head = p->k_strides[1];
    a.v_tok = p->v_strides[0], a.v_head = p->v_strides[1];
    a.qo_tok = p->q_out_strides[0], a.qo_head = p->q_out_strides[1];
    a.kc_page = p->k_cache_strides[0], a.kc_slot = p->k_cache_strides[1], a.kc_head = p->k_cache_strides[2];
    a.vc_page = p->v_cache_strides[0], a.vc_slot = p->v_cache_strides[1], a.vc_head = p->v_cache_strides[2];
    a.table_stride = p->rope_stride, a.pages_stride = p->page_table_stride;
    a.tokens = p->tokens, a.heads = p->heads, a.kv_heads = p->kv_heads, a.dim = p->dim, a.rot = p->rot;
    a.num_pages = p->num_pages, a.page = p->page_size, a.seqs = p->seqs, a.max_pages = p->max_pages;
    a.table_rows = p->rope_rows, a.err = err;
    // 16-byte accesses: every row that a thread reads or writes starts on 16 bytes, and a
    // group of eight elements is wholly rotated or not at all.
    bool wide = p->dim % 8 == 0 && p->rot % (p->interleaved ? 8 : 16) == 0;
    auto rows = [&](const void *b, const int64_t *s, int n) {
        wide = wide && dec::aligned(b, 16);
        for (int i = 0; i < n; ++i) wide = wide && s[i] % 8 == 0;
    };
    rows(a.k, p->k_strides, 2), rows(a.v, p->v_strides, 2);
    rows(a.kc, p->k_cache_strides, 3), rows(a.vc, p->v_cache_strides, 3);
    if (p->heads) rows(a.q, p->q_strides, 2), rows(a.q_out, p->q_out_strides, 2);
    const double units = (double)a.tokens * (a.heads + 2.0 * a.kv_heads) * ((a.dim + 1) / 2);
    if (units > 256.0 * INT32_MAX) return fail(HV_ERR_VALUE, "too many elements for one call");
    const cudaStream_t st = (cudaStream_t)stream;
    const cudaError_t e = p->dtype == HV_BF16 ? launch<__nv_bfloat16>(a, wide, p->interleaved != 0, st)
                                              : launch<__half>(a, wide, p->interleaved != 0, st);
    if (e != cudaSuccess) return fail(HV_ERR_CUDA, "append_kv: %s", cudaGetErrorString(e));
    return HV_OK;
}
