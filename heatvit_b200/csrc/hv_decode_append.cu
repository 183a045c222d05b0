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
    int lanes;  // of a head, where a norm adds up its squares
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
    const void *weight[3];  // of the norms ahead of the rotation; null: none
    float eps;
    int dim;
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

// Where a cached head of this token goes: its page and slot, -1 after a mistake, which is reported.
__device__ __forceinline__ long long cached_at(const AppendArgs &a, const Tensor &t, unsigned tok, int pos) {
    const int s = a.seq_ids ? a.seq_ids[tok] : (int)tok;
    const int col = a.by_page(pos), slot = pos - col * a.by_page.d;
    if (s < 0 || s >= a.seqs || col >= a.max_pages) {
        atomicOr(a.err, HV_DECODE_BAD_POSITION);
        return -1;
    }
    const int pg = a.pages[s * a.pages_stride + col];
    if (pg < 0 || pg >= a.num_pages) {
        atomicOr(a.err, HV_DECODE_BAD_PAGE);
        return -1;
    }
    return pg * t.page + slot * t.slot;
}

// Pairs of 32-bit numbers, as the packed multiply-adds take them: a word of T as two of them and back.
__device__ __forceinline__ uint64_t two(float lo, float hi) {
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};\n" : "=l"(v) : "f"(lo), "f"(hi));
    return v;
}
__device__ __forceinline__ void split2(uint64_t v, float &lo, float &hi) { asm("mov.b64 {%0, %1}, %2;\n" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;\n" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t wide2(uint32_t v, __nv_bfloat16) { return two(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u)); }
__device__ __forceinline__ uint64_t wide2(uint32_t v, __half) {
    const float2 f = __half22float2(*(const __half2 *)&v);
    return two(f.x, f.y);
}
__device__ __forceinline__ uint32_t narrow2(uint64_t v, __nv_bfloat16) {
    float lo, hi;
    split2(v, lo, hi);
    const __nv_bfloat162 r = __floats2bfloat162_rn(lo, hi);
    return *(const uint32_t *)&r;
}
__device__ __forceinline__ uint32_t narrow2(uint64_t v, __half) {
    float lo, hi;
    split2(v, lo, hi);
    const __half2 r = __floats2half2_rn(lo, hi);
    return *(const uint32_t *)&r;
}
__device__ __forceinline__ uint64_t swapped(uint64_t v) {
    float lo, hi;
    split2(v, lo, hi);
    return two(hi, lo);
}

// With a norm of each head ahead of the rotation: y = x * rsqrt(mean(x^2) + eps) * weight.  The
// lanes of a head, a power of two of them, add up their squares; places as in append_kernel, one to a lane.  What an
// element is multiplied by beside its head's root (weights, cosines, sines) is the same for all heads of a token, so a
// thread has it once for the NH heads that it takes.
//
// Measured on one B200: 8 ragged prompts (24,004 tokens, 40 + 2 x 8 heads of 96 in fp16, two thirds rotated in
// neighbouring pairs) 146 us, 3.6 TB/s of what is read and written (a quarter of its lanes have no place); 12,004 tokens of
// 48 heads of 128 69 us, 4.3 TB/s; a decode step of 64 sequences 2.6 us, the launch and three memory latencies.
template <typename T, bool INTER, int NH>
__global__ void __launch_bounds__(THREADS) norm_append_kernel(const __grid_constant__ AppendArgs a) {
    griddep_wait();
    griddep_launch();
    constexpr int W = 8;
    const int which = (blockIdx.x >= a.first[1]) + (blockIdx.x >= a.first[2]);
    const Tensor &t = a.t[which];
    const unsigned id = (blockIdx.x - a.first[which]) * THREADS + threadIdx.x;
    const bool exists = id < t.total;
    const unsigned tok = exists ? t.by_token(id) : 0, in = exists ? id - tok * t.by_token.d : 0;
    const int lanes = t.lanes, strip = in / lanes, u = in & (lanes - 1);
    const int half = t.rot / 2;
    constexpr bool PAIRED = !INTER;
    const int rotated = PAIRED ? half / W : t.rot / W;
    const bool works = exists && u < rotated + (a.dim - t.rot) / W;
    const bool turned = works && u < rotated, two_groups = PAIRED && turned;
    const int c0 = !works ? 0 : !turned && PAIRED ? t.rot + (u - rotated) * W : u * W;
    const int n = works ? min((t.heads - strip + (int)t.strips - 1) / (int)t.strips, NH) : 0;

    const T *src = (const T *)t.from + (tok * t.tok + (long long)strip * t.head + c0);
    uint4 x[NH], y[NH];
#pragma unroll
    for (int j = 0; j < NH; ++j) {
        x[j] = y[j] = make_uint4(0, 0, 0, 0);
        if (j < n) {
            const T *p = src + (long long)(j * (int)t.strips) * t.head;
            x[j] = *(const uint4 *)p;
            if (two_groups) y[j] = *(const uint4 *)(p + half);
        }
    }
    const T *weight = (const T *)a.weight[which];
    const int pos = works ? a.positions[tok] : -1;
    uint4 wx = make_uint4(0, 0, 0, 0), wy = wx;
    if (weight && works) {
        wx = *(const uint4 *)(weight + c0);
        if (two_groups) wy = *(const uint4 *)(weight + c0 + half);
    }
    float inv[NH];
#pragma unroll
    for (int j = 0; j < NH; ++j) {
        inv[j] = 1.f;
        if (!weight) continue;
        const uint32_t(&xw)[4] = *(const uint32_t(*)[4])&x[j], (&yw)[4] = *(const uint32_t(*)[4])&y[j];
        uint64_t s2 = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint64_t v = wide2(xw[i], T());
            s2 = fma2(v, v, s2);
            if (PAIRED) {
                const uint64_t z = wide2(yw[i], T());
                s2 = fma2(z, z, s2);
            }
        }
        float lo, hi;
        split2(s2, lo, hi);
        float s = lo + hi;
        for (int o = lanes / 2; o; o /= 2) s += __shfl_xor_sync(~0u, s, o);
        inv[j] = rsqrtf(s / (float)a.dim + a.eps);
    }
    if (!works) return;
    const bool live = pos >= 0;
    if (a.rot && pos >= a.table_rows) {
        atomicOr(a.err, HV_DECODE_BAD_POSITION);
        return;
    }
    T *dst = (T *)t.to + ((long long)strip * t.to_head + c0);
    if (t.cached) {
        if (!live) return;
        const long long at = cached_at(a, t, tok, pos);
        if (at == -1) return;
        dst += at;
    } else {
        dst += tok * t.to_tok;
    }
    // x' = (x A + y B) inv, y' = (y D + x C) inv; where pairs are neighbours, (p, w)' = ((p, w) A + (w, p) B) inv
    uint64_t A[4], B[4], C[4], D[4];
    if (live && (weight || turned)) {
        const uint32_t(&xw)[4] = *(const uint32_t(*)[4])&wx, (&yw)[4] = *(const uint32_t(*)[4])&wy;
        const float *tab = a.table + pos * a.table_stride + (INTER ? c0 / 2 : c0);
        const uint64_t one = two(1.f, 1.f), minus = two(-1.f, -1.f);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint64_t v = weight ? wide2(xw[i], T()) : one, z = weight ? wide2(yw[i], T()) : one;
            A[i] = v, B[i] = C[i] = 0, D[i] = z;
            if (!turned) continue;
            if (PAIRED) {
                const float2 c = *(const float2 *)(tab + 2 * i), s = *(const float2 *)(tab + half + 2 * i);
                const uint64_t cs = two(c.x, c.y), sn = two(s.x, s.y);
                A[i] = mul2(v, cs), B[i] = mul2(mul2(z, sn), minus), C[i] = mul2(v, sn), D[i] = mul2(z, cs);
            } else {
                const float c = tab[i], s = tab[half + i];
                A[i] = mul2(v, two(c, c)), B[i] = mul2(swapped(v), two(-s, s));
            }
        }
    }
#pragma unroll
    for (int j = 0; j < NH; ++j) {
        if (j >= n) break;
        uint32_t(&xw)[4] = *(uint32_t(*)[4])&x[j], (&yw)[4] = *(uint32_t(*)[4])&y[j];
        if (!live) {
            x[j] = y[j] = make_uint4(0, 0, 0, 0);
        } else if (weight || turned) {
            const uint64_t f = two(inv[j], inv[j]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint64_t v = wide2(xw[i], T());
                if (!turned) {
                    xw[i] = narrow2(mul2(mul2(v, A[i]), f), T());
                } else if (PAIRED) {
                    const uint64_t z = wide2(yw[i], T());
                    xw[i] = narrow2(mul2(fma2(z, B[i], mul2(v, A[i])), f), T());
                    yw[i] = narrow2(mul2(fma2(v, C[i], mul2(z, D[i])), f), T());
                } else {
                    xw[i] = narrow2(mul2(fma2(swapped(v), B[i], mul2(v, A[i])), f), T());
                }
            }
        }
        T *p = dst + (long long)(j * (int)t.strips) * t.to_head;
        *(uint4 *)p = x[j];
        if (two_groups) *(uint4 *)(p + half) = y[j];
    }
}

// The same for sizes and alignments that 16-byte accesses or 32 lanes of them do not cover: a
// warp a head, an element or a pair a lane, the head read again (from L1) for the result.  12,004 tokens of 48 heads in bf16, of
// 128 off 16 bytes 201 us (without norms 252), of 320 376 (194, which has 16-byte accesses there).
template <typename T>
__global__ void __launch_bounds__(THREADS) norm_append_any_kernel(const __grid_constant__ AppendArgs a, int inter) {
    griddep_wait();
    griddep_launch();
    const int which = (blockIdx.x >= a.first[1]) + (blockIdx.x >= a.first[2]);
    const Tensor &t = a.t[which];
    const unsigned id = ((blockIdx.x - a.first[which]) * THREADS + threadIdx.x) / 32, lane = threadIdx.x % 32;
    if (id >= t.total) return;  // of warps
    const unsigned tok = t.by_token(id);
    const int head = id - tok * t.by_token.d, half = t.rot / 2;
    const T *src = (const T *)t.from + (tok * t.tok + (long long)head * t.head);
    const T *weight = (const T *)a.weight[which];
    float inv = 1.f;
    if (weight) {
        float s = 0.f;
        for (int i = lane; i < a.dim; i += 32) s += to_f32(src[i]) * to_f32(src[i]);
        for (int o = 16; o; o /= 2) s += __shfl_xor_sync(~0u, s, o);
        inv = rsqrtf(s / (float)a.dim + a.eps);
    }
    const int pos = a.positions[tok];
    const bool live = pos >= 0;
    if (a.rot && pos >= a.table_rows) {
        if (lane == 0) atomicOr(a.err, HV_DECODE_BAD_POSITION);
        return;
    }
    T *dst = (T *)t.to + (long long)head * t.to_head;
    if (t.cached) {
        if (!live) return;
        const long long at = cached_at(a, t, tok, pos);
        if (at == -1) return;
        dst += at;
    } else {
        dst += tok * t.to_tok;
    }
    const float *tab = a.table + (live ? pos : 0) * a.table_stride;
    auto normed = [&](int i) {
        const float v = to_f32(src[i]);
        return weight ? v * inv * to_f32(weight[i]) : v;
    };
    for (int i = lane; i < half; i += 32) {
        const int c0 = inter ? 2 * i : i, c1 = inter ? 2 * i + 1 : i + half;
        float p = 0.f, w = 0.f;
        if (live) {
            const float fp = normed(c0), fw = normed(c1), cs = tab[i], sn = tab[half + i];
            p = fp * cs - fw * sn;
            w = fp * sn + fw * cs;
        }
        dst[c0] = from_f32<T>(p);
        dst[c1] = from_f32<T>(w);
    }
    for (int i = t.rot + lane; i < a.dim; i += 32) dst[i] = !live ? from_f32<T>(0.f) : weight ? from_f32<T>(normed(i)) : src[i];
}

template <typename T, bool INTER, int NH>
int launch_norm(AppendArgs &a, int tokens, cudaStream_t st) {
    uint32_t blocks = 0;
    for (int i = 0; i < 3; ++i) {
        Tensor &t = a.t[i];
        const int places = (INTER ? t.rot : t.rot / 2) / 8 + (a.dim - t.rot) / 8;
        for (t.lanes = 1; t.lanes < places;) t.lanes *= 2;
        t.strips = (t.heads + NH - 1) / NH;
        const double total = (double)tokens * t.strips * t.lanes;
        if (total > 2147483392.0) return fail(HV_ERR_VALUE, "too many elements for one call");
        t.total = (uint32_t)total;
        t.by_token = Divider(std::max(1u, t.strips * t.lanes));
        a.first[i] = blocks;
        blocks += (t.total + THREADS - 1) / THREADS;
    }
    const cudaError_t e = launch_pdl(norm_append_kernel<T, INTER, NH>, dim3(blocks), dim3(THREADS), 0, st, a);
    if (e != cudaSuccess) return fail(HV_ERR_CUDA, "append_kv: %s", cudaGetErrorString(e));
    return HV_OK;
}

template <typename T>
int launch_norm_any(AppendArgs &a, int tokens, bool inter, cudaStream_t st) {
    uint32_t blocks = 0;
    for (int i = 0; i < 3; ++i) {
        Tensor &t = a.t[i];
        const double total = (double)tokens * t.heads;
        if (total * 32 > 2147483392.0) return fail(HV_ERR_VALUE, "too many elements for one call");
        t.total = (uint32_t)total;
        t.by_token = Divider(std::max(1, t.heads));
        a.first[i] = blocks;
        blocks += (t.total * 32 + THREADS - 1) / THREADS;
    }
    const cudaError_t e = launch_pdl(norm_append_any_kernel<T>, dim3(blocks), dim3(THREADS), 0, st, a, (int)inter);
    if (e != cudaSuccess) return fail(HV_ERR_CUDA, "append_kv: %s", cudaGetErrorString(e));
    return HV_OK;
}

template <typename T>
int launch_norm(AppendArgs &a, int tokens, bool wide, bool inter, int sms, cudaStream_t st) {
    // 32 lanes hold 256 elements of a head that is not rotated, or in neighbouring pairs; all three share a layout
    if (!wide || a.dim > 256) return launch_norm_any<T>(a, tokens, inter, st);
    // One head a thread until that fills the SMs' threads once, two until four times, then four.  us with one, two and
    // four: the 8 prompts above 270, 183, 146; 48 heads of 128, 12,004 tokens 91.5, 72.4, 69.1; 2048 15.1, 11.7, 11.4; 1024
    // 8.5, 6.8, 7.7; 512 5.3, 4.3, 5.1; 256 3.9, 3.8, 4.1; 128 3.1, 3.2, 4.1; the decode step 2.6, 3.2, 3.9.
    const double threads = (double)tokens * a.dim / 8 * (a.t[0].heads + 2.0 * a.t[1].heads), room = 2048.0 * sms;
    if (threads <= room) return inter ? launch_norm<T, true, 1>(a, tokens, st) : launch_norm<T, false, 1>(a, tokens, st);
    if (threads <= 4 * room) return inter ? launch_norm<T, true, 2>(a, tokens, st) : launch_norm<T, false, 2>(a, tokens, st);
    return inter ? launch_norm<T, true, 4>(a, tokens, st) : launch_norm<T, false, 4>(a, tokens, st);
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

static int append(const hv_append_args *p, const void *q_weight, const void *k_weight, float eps, void *stream) {
    const bool norm = q_weight || k_weight;
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
    a.weight[0] = q_weight, a.weight[1] = k_weight, a.weight[2] = nullptr, a.eps = eps, a.dim = p->dim;
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
    if (norm) {
        wide = wide && dec::aligned(q_weight, 16) && dec::aligned(k_weight, 16);
        return p->dtype == HV_BF16 ? launch_norm<__nv_bfloat16>(a, p->tokens, wide, p->interleaved != 0, sms, st)
                                   : launch_norm<__half>(a, p->tokens, wide, p->interleaved != 0, sms, st);
    }
    return p->dtype == HV_BF16 ? launch<__nv_bfloat16>(a, p->tokens, p->dim, wide, p->interleaved != 0, sms, st)
                               : launch<__half>(a, p->tokens, p->dim, wide, p->interleaved != 0, sms, st);
}

extern "C" int hv_append_kv(const hv_append_args *p, void *stream) {
    if (!p) return fail(HV_ERR_VALUE, "null argument");
    return append(p, nullptr, nullptr, 0.f, stream);
}

extern "C" int hv_norm_append_kv(const hv_norm_append_args *p, void *stream) {
    if (!p) return fail(HV_ERR_VALUE, "null argument");
    if (!(p->eps >= 0.f)) return fail(HV_ERR_VALUE, "eps must not be negative");
    if (p->d_q_weight && !p->append.heads) return fail(HV_ERR_VALUE, "a weight for q without q heads");
    return append(&p->append, p->d_q_weight, p->d_k_weight, p->eps, stream);
}
