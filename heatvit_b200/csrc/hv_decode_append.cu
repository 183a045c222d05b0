// hv_decode_append.cu — keys and values into a paged cache, with the position rotation on the way.
//
// Token t of sequence s = seq_ids[t] (or t) at position p goes to page page_table[s][p / page],
// slot p % page.  The first `rot` elements of every q and k head are turned in pairs (u, w) by
// the angle of their pair at p: (u cos - w sin, u sin + w cos), the pair being elements (i,
// i + rot/2), or (2i, 2i + 1) when interleaved; cosines and sines come from a float32 table.
// One rounding of the 32-bit result; v and the elements past rot are copied.
//
// Bound by HBM (each element read once and written once), and for a decode step by the
// launch.  q, k and v have their own blocks.  A thread has one place in the head, and with it one
// set of angles, for one or two heads of a token; their elements are asked for before the
// position, and with it page and angles, are known, so that a thread waits for two memory
// latencies and not for four.
//
// Measured on one B200: 24 ragged prompts (36,900 tokens, 36 heads of 64) 59 us, 5.75 TB/s of
// what is read and written; 8 x 1024 tokens of 48 heads of 128 38 us (4.0 TB/s: pairs half a
// head apart double what a thread holds, and so halve its company); a decode step of 64
// sequences 2.3 us, the launch.  Sizes or strides off 16 bytes take a thread an element: 8 x 1024
// tokens of 48 heads of 124 124 us (1.2 TB/s).
#include <algorithm>

#include "hv_decode.cuh"

namespace hv {
namespace {

using namespace dec;

// n / d for n < 2^31 by a multiplication: the reciprocal rounded up, in 33 bits of which the first is
// an addition (Granlund and Montgomery, Division by Invariant Integers using Multiplication, 1994).
struct Divider {
    uint32_t mul, shift, d;
    __host__ Divider(uint32_t by = 1) : mul(0), shift(0), d(by) {
        while ((1ull << shift) < by) ++shift;
        mul = (uint32_t)(((1ull << 32) * ((1ull << shift) - by)) / by + 1);
    }
    __device__ __forceinline__ uint32_t operator()(uint32_t n) const { return (__umulhi(n, mul) + n) >> shift; }
};

// What is done with one of q, k, v: `heads` of it, whose first `rot` elements turn, to `to` or
// to the cache (page and slot strides).
struct Tensor {
    const void *from;
    void *to;
    long long tok, to_tok, page, slot;
    int head, to_head, heads, rot, cached;
    uint32_t strips, total;  // threads: tokens * strips * places
    Divider by_token, by_place;
};

struct AppendArgs {
    Tensor t[3];
    uint32_t first[3];     // block of each
    const float *table;    // [table_rows][rot]: cosines, then sines
    const int32_t *pages;  // [seqs][max_pages]
    const int32_t *seq_ids, *positions;
    long long table_stride, pages_stride;
    int num_pages, seqs, max_pages, table_rows, rot;
    Divider by_page;
    int *err;
};

constexpr int THREADS = 256;

// Elements as stored, in groups of W: 8, as one 16-byte access, or 1 where sizes or alignment
// do not allow that.
template <typename T, int W>
struct alignas(W * sizeof(T)) Elems {
    T e[W];
    __device__ __forceinline__ void load(const T *p) { *this = *(const Elems *)p; }
    __device__ __forceinline__ void store(T *p) const { *(Elems *)p = *this; }
};

// Places of a head, a thread's work each: half-split, rot / 2 / W pairs of groups that hold each
// other's partners, then the groups past rot; interleaved, pairs of neighbouring elements are in
// a group (W = 8) or are the two groups of a place (W = 1).
template <typename T, int W, bool INTER, int NH>
__global__ void __launch_bounds__(THREADS) append_kernel(const __grid_constant__ AppendArgs a) {
    griddep_wait();
    griddep_launch();
    const int which = (blockIdx.x >= a.first[1]) + (blockIdx.x >= a.first[2]);
    const Tensor &t = a.t[which];
    const unsigned id = (blockIdx.x - a.first[which]) * THREADS + threadIdx.x;
    if (id >= t.total) return;
    const unsigned tok = t.by_token(id), in = id - tok * t.by_token.d;
    const int strip = t.by_place(in), u = in - strip * t.by_place.d;  // heads strip, strip + strips, ...
    const int half = t.rot / 2;
    constexpr bool PAIRED = !INTER || W == 1;  // the two groups of a rotated place
    const int rotated = PAIRED ? half / W : t.rot / W;
    const bool turned = u < rotated, two = PAIRED && turned;
    const int c0 = !turned && PAIRED ? t.rot + (u - rotated) * W : INTER && PAIRED ? u * 2 : u * W;
    const int c1 = INTER ? 1 : half;  // from c0
    const int n = min((t.heads - strip + (int)t.strips - 1) / (int)t.strips, NH);

    const T *src = (const T *)t.from + (tok * t.tok + (long long)strip * t.head + c0);
    Elems<T, W> x[NH], y[NH];
#pragma unroll
    for (int j = 0; j < NH; ++j)
        if (j < n) {
            const T *p = src + (long long)(j * (int)t.strips) * t.head;
            x[j].load(p);
            if (two) y[j].load(p + c1);
        }

    const int pos = a.positions[tok];
    const bool live = pos >= 0;
    if (a.rot && pos >= a.table_rows) {  // a token that the rotation table does not reach: nothing
        atomicOr(a.err, HV_DECODE_BAD_POSITION);
        return;
    }
    constexpr int NA = INTER && W == 8 ? 4 : W;  // angles of a place
    alignas(16) float cs[NA], sn[NA];
    if (turned && live) {
        const float *tab = a.table + pos * a.table_stride + (INTER ? c0 / 2 : c0);
        if constexpr (W == 8) {
#pragma unroll
            for (int i = 0; i < NA; i += 4) {
                *(float4 *)(cs + i) = *(const float4 *)(tab + i);
                *(float4 *)(sn + i) = *(const float4 *)(tab + half + i);
            }
        } else {
            cs[0] = tab[0];
            sn[0] = tab[half];
        }
    }
    T *dst = (T *)t.to + ((long long)strip * t.to_head + c0);
    if (t.cached) {
        if (!live) return;  // a padding token stores nothing
        const int s = a.seq_ids ? a.seq_ids[tok] : (int)tok;
        const int col = a.by_page(pos), slot = pos - col * a.by_page.d;
        if (s < 0 || s >= a.seqs || col >= a.max_pages) {
            atomicOr(a.err, HV_DECODE_BAD_POSITION);
            return;
        }
        const int pg = a.pages[s * a.pages_stride + col];
        if (pg < 0 || pg >= a.num_pages) {
            atomicOr(a.err, HV_DECODE_BAD_PAGE);
            return;
        }
        dst += pg * t.page + slot * t.slot;
    } else {
        dst += tok * t.to_tok;
    }

#pragma unroll
    for (int j = 0; j < NH; ++j) {
        if (j >= n) break;
        if (!live) {  // a padding token's q is defined: zeros
#pragma unroll
            for (int i = 0; i < W; ++i) x[j].e[i] = y[j].e[i] = from_f32<T>(0.f);
        } else if (turned) {
#pragma unroll
            for (int i = 0; i < NA; ++i) {
                T &p = PAIRED ? x[j].e[i % W] : x[j].e[(2 * i) % W], &w = PAIRED ? y[j].e[i % W] : x[j].e[(2 * i + 1) % W];
                const float fp = to_f32(p), fw = to_f32(w);
                p = from_f32<T>(fp * cs[i] - fw * sn[i]);
                w = from_f32<T>(fp * sn[i] + fw * cs[i]);
            }
        }
        T *p = dst + (long long)(j * (int)t.strips) * t.to_head;
        x[j].store(p);
        if (two) y[j].store(p + c1);
    }
}

template <typename T, int W, bool INTER, int NH>
int launch(AppendArgs &a, int tokens, int dim, cudaStream_t st) {
    uint32_t blocks = 0;
    for (int i = 0; i < 3; ++i) {
        Tensor &t = a.t[i];
        const int rotated = !INTER || W == 1 ? t.rot / 2 / W : t.rot / W, places = rotated + (dim - t.rot) / W;
        t.strips = (t.heads + NH - 1) / NH;
        const double total = (double)tokens * t.strips * places;
        if (total > 2147483392.0) return fail(HV_ERR_VALUE, "too many elements for one call");
        t.total = (uint32_t)total;
        t.by_token = Divider(std::max(1u, t.strips * places));
        t.by_place = Divider(places);
        a.first[i] = blocks;
        blocks += (t.total + THREADS - 1) / THREADS;
    }
    const cudaError_t e = launch_pdl(append_kernel<T, W, INTER, NH>, dim3(blocks), dim3(THREADS), 0, st, a);
    if (e != cudaSuccess) return fail(HV_ERR_CUDA, "append_kv: %s", cudaGetErrorString(e));
    return HV_OK;
}

template <typename T>
int launch(AppendArgs &a, int tokens, int dim, bool wide, bool inter, int sms, cudaStream_t st) {
    if (!wide) return inter ? launch<T, 1, true, 1>(a, tokens, dim, st) : launch<T, 1, false, 1>(a, tokens, dim, st);
    // One head a thread until that fills the SMs' threads twice, then two: 24 ragged prompts of 36
    // heads of 64 (interleaved) took 70 us with one, 59 with two, 62 with four, 8 x 1024 tokens of
    // 48 heads of 128 (half-split) 42, 38 and 43.
    if ((double)tokens * dim / 8 * (a.t[0].heads + 2.0 * a.t[1].heads) <= 2.0 * 2048 * sms)
        return inter ? launch<T, 8, true, 1>(a, tokens, dim, st) : launch<T, 8, false, 1>(a, tokens, dim, st);
    return inter ? launch<T, 8, true, 2>(a, tokens, dim, st) : launch<T, 8, false, 2>(a, tokens, dim, st);
}

}  // namespace
}  // namespace hv

using namespace hv;

extern "C" int hv_append_kv(const hv_append_args *p, void *stream) {
    if (!p) return fail(HV_ERR_VALUE, "null argument");
    if (p->dtype != HV_BF16 && p->dtype != HV_F16) return fail(HV_ERR_TYPE, "dtype must be HV_BF16 or HV_F16");
    if (p->tokens < 0 || p->heads < 0) return fail(HV_ERR_VALUE, "negative token or head count");
    if (p->kv_heads < 1 || p->dim < 1) return fail(HV_ERR_VALUE, "kv_heads and dim must be positive");
    if ((double)p->tokens * (p->heads + 2.0 * p->kv_heads) * p->dim > 2147483392.0 * (p->dim % 8 ? 1 : 8))
        return fail(HV_ERR_VALUE, "too many elements for one call");
    if (p->rot < 0 || p->rot > p->dim || p->rot % 2) return fail(HV_ERR_VALUE, "rot must be even and in [0, dim]");
    if (p->page_size < 1 || p->num_pages < 0 || p->seqs < 0 || p->max_pages < 0)
        return fail(HV_ERR_VALUE, "bad cache geometry");
    if (p->tokens == 0) return HV_OK;
    if (!p->d_k || !p->d_v || !p->d_k_cache || !p->d_v_cache || !p->d_page_table || !p->d_positions)
        return fail(HV_ERR_VALUE, "null buffer");
    if (p->heads && (!p->d_q || !p->d_q_out)) return fail(HV_ERR_VALUE, "q heads without a q or q_out buffer");
    if (p->rot && (!p->d_rope || p->rope_rows < 1)) return fail(HV_ERR_VALUE, "rot without a table");
    int *err = dec::error_word();
    const int sms = dec::sm_count();
    if (!err || !sms) return fail(HV_ERR_CUDA, "cannot read the device's properties");
    AppendArgs a;
    a.t[0] = {p->d_q, p->d_q_out, p->q_strides[0], p->q_out_strides[0], 0, 0, (int)p->q_strides[1],
              (int)p->q_out_strides[1], p->heads, p->rot, 0};
    a.t[1] = {p->d_k, p->d_k_cache, p->k_strides[0], 0, p->k_cache_strides[0], p->k_cache_strides[1],
              (int)p->k_strides[1], (int)p->k_cache_strides[2], p->kv_heads, p->rot, 1};
    a.t[2] = {p->d_v, p->d_v_cache, p->v_strides[0], 0, p->v_cache_strides[0], p->v_cache_strides[1],
              (int)p->v_strides[1], (int)p->v_cache_strides[2], p->kv_heads, 0, 1};
    a.table = p->d_rope, a.pages = p->d_page_table, a.seq_ids = p->d_seq_ids, a.positions = p->d_positions;
    a.table_stride = p->rope_stride, a.pages_stride = p->page_table_stride;
    a.num_pages = p->num_pages, a.seqs = p->seqs, a.max_pages = p->max_pages;
    a.table_rows = p->rope_rows, a.rot = p->rot, a.by_page = Divider(p->page_size), a.err = err;
    for (const int64_t s : {p->q_strides[1], p->q_out_strides[1], p->k_strides[1], p->v_strides[1], p->k_cache_strides[2],
                            p->v_cache_strides[2]})
        if (s > INT32_MAX || s < -INT32_MAX) return fail(HV_ERR_VALUE, "head strides must be under 2^31");
    // 16-byte accesses: every row that a thread reads or writes starts on 16 bytes, and a
    // group of eight elements is wholly rotated or not at all.
    bool wide = p->dim % 8 == 0 && p->rot % (p->interleaved ? 8 : 16) == 0 &&
                (!p->rot || (dec::aligned(p->d_rope, 16) && p->rope_stride % 4 == 0));
    auto rows = [&](const void *b, const int64_t *s, int n) {
        wide = wide && dec::aligned(b, 16);
        for (int i = 0; i < n; ++i) wide = wide && s[i] % 8 == 0;
    };
    rows(p->d_k, p->k_strides, 2), rows(p->d_v, p->v_strides, 2);
    rows(p->d_k_cache, p->k_cache_strides, 3), rows(p->d_v_cache, p->v_cache_strides, 3);
    if (p->heads) rows(p->d_q, p->q_strides, 2), rows(p->d_q_out, p->q_out_strides, 2);
    const cudaStream_t st = (cudaStream_t)stream;
    return p->dtype == HV_BF16 ? launch<__nv_bfloat16>(a, p->tokens, p->dim, wide, p->interleaved != 0, sms, st)
                               : launch<__half>(a, p->tokens, p->dim, wide, p->interleaved != 0, sms, st);
}
