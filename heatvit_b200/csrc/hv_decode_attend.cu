// hv_decode_attend.cu — attention of one new token per sequence over a paged cache.
//
//   out[b, h] = sum_t softmax_t(scale * q[b, h] . K[t, h / group]) V[t, h / group],
//   t < lens[b];  a sequence of no tokens gives zeros (and a log-sum-exp of -inf).
//
// Bound by HBM: each live key and value is read once, for up to 16 query heads that share
// it.  Those heads are the 16 rows of an m16n8k16 matrix product: at 23 bytes of cache an
// SM clock, 16 multiply-adds an element leave the warp-level tensor path under a fifth
// busy, and it needs none of the 128 rows that a tcgen05 tile would pad to.  (More heads read
// the cache again for every 16: 32 x 4000 tokens, 16 heads over one 23 us, 32 over one 35.)
//
// Work: the (sequence, head tile) items are cut into tiles of 64 tokens (128 for heads of up
// to 64 dimensions), the tiles of all items are laid end to end, and the CTAs of one resident
// wave take equal shares of that line.  So a ragged batch is even, and a single long sequence
// uses every SM; every CTA works the cuts out for itself from the lengths, which stay on the
// device.  A warp owns its tokens of a tile and its own cp.async ring, so that warps do not
// wait for one another inside an item; the ring runs ahead across item borders.
//
// An item inside one share is written straight out.  One that is cut leaves a part (the
// unnormalised sum, the running maximum and the sum of weights, in 32 bits) per CTA in the
// workspace, and the CTA that finishes last joins the parts in the order of the shares: the
// result does not depend on which that is.
//
// Measured on one B200, bf16, in bursts: 64 sequences of 0 to 8192 tokens (32 heads of 128 over 8)
// 182 us, 5.9 TB/s of the cache (201 when calls follow one another for long); two of 131071 (64 over
// 8) 187 us, 5.7 TB/s.  CTAs stream for 150 to 170 us of that; the rest is what the latest of them
// join.  One sequence of 197 tokens, 5.7 us: length, page, key, join, each a memory latency after the
// other.  (A workspace made outside the graph; a captured call that makes its own takes 1 us more.)
#include <math_constants.h>

#include "hv_decode.cuh"
#include "hv_tc05.cuh"

namespace hv {
namespace {

using namespace dec;

constexpr int ROWS = 16, BLOCK = 16, SLICES = 4;
// A running maximum before the first score.  Finite, so that a score of -inf (a product out of
// range) weighs exp2(-inf) = 0 and not NaN; a NaN passes every maximum and shows in the sums.
constexpr float LOWEST = -3.402823466e38f;
// Tiles: a part costs more than the loads of fewer.  One sequence of 1000 tokens, heads of 128: 10.3
// us with one, 10.7 with two, 13.0 with four; one of 197, heads of 64: 9.1, 8.2, 11.8.
constexpr int MIN_SHARE = 2;
// Tiles that a share may grow by so that items of one length end where shares do and none is cut.
// Sequences of one length, 32 heads of 128 over 8, without and with it: 32 of 512 tokens (shares of 7,
// items of 8) 22.1 and 18.0 us, 64 of 512 (14, 16) 35.6 and 31.8, 24 of 384 (4, 6) 17.1 and 14.3, 22 of
// 320 (3, 5) 15.4 and 12.3.  By four, 16 of 512 (4, 8) took 18.9 instead of 16.0.
constexpr int SLACK = 2;
// A row's weights are taken beside a reference that makes its largest 2^TOP when it is set, and that moves
// when one passes it by more than 2^SOFT.  fp16 has normal numbers from 2^-14 to 2^15 and none under 2^-24: its
// weights begin at 2^9, so that those of a long tail, each 2^-23 of one large weight, keep their bits, and those
// under 2^-34 of it are lost (with TOP = 0, weights 16 nats under one had a single bit left).  bf16 has the
// range of the 32-bit weights.
template <typename T>
constexpr float TOP = 0.f;
template <>
constexpr float TOP<__half> = 9.f;
constexpr float SOFT = 6.f;
constexpr int FAN = 16;       // parts whose loads a joining CTA has in flight together
// A further FAN parts cost a joining CTA about 1.5 us, a second level about 7.
constexpr int ONE_LEVEL = 4 * FAN, GROUP = FAN;
constexpr int MAX_GRID = 1024;

struct AttendArgs {
    const void *q, *kc, *vc;
    void *out;
    float *lse;
    const int32_t *pages, *lens;
    long long q_seq, q_head, o_seq, o_head, lse_seq, lse_head;
    long long kc_page, kc_slot, kc_head, vc_page, vc_slot, vc_head, pages_stride;
    int seqs, heads, kv_heads, group, head_tiles, num_pages, page, max_pages, q_pairs, o_vec;
    int page16, page_shift;  // the page is a multiple of 16 tokens; log2 of a page that is a power of two, or -1
    float scale_log2;
    float *parts;      // [grid][2][ROWS][D], then [grid][2][ROWS][2]
    uint32_t *counts;  // [3][MAX_GRID], see the end of an item; zero between calls
    int *err;
};

// A head of over 128 dimensions is split between two warps (HALVES), which add their halves of
// the scores through shared memory: one warp's sums and q would take all of its registers.
template <int D>
struct Lay {
    static constexpr int HALVES = D > 128 ? 2 : 1, DH = D / HALVES;
    static constexpr int WARPS = SLICES * HALVES, THREADS = WARPS * 32;
    // 16-token blocks of a warp's step: a step costs about the same for 32 tokens of 64
    // dimensions (16 heads of 64 over 64 x 4000 tokens: 245 us with 16, 223 with 32) as for 16 of 128
    static constexpr int BLOCKS = D <= 64 ? 2 : 1, WTOK = BLOCKS * BLOCK, TILE = SLICES * WTOK;
    static constexpr int ROW = DH * 2 + 16;  // bytes: rows 16 bytes apart modulo 128 (ldmatrix without conflicts)
    // Three CTAs an SM of two stages where registers allow, else two of three: 16 heads of 64 took
    // 223 us as two of three, 186 as three of two; heads of 128 spill at 168 registers (187, 381).
    // (So do 64 bytes of heads of 64 in groups of over eight.)
    static constexpr int PER_SM = D <= 64 ? 3 : D <= 128 ? 2 : 1, STAGES = D <= 64 ? 2 : 3;
    static constexpr int STAGE = 2 * WTOK * ROW;
    static constexpr int PART_ROW = DH + 4;  // a warp's sums at an item's end, where its last stage was
    static constexpr int SUM = WARPS * STAGES * STAGE;  // weights of parts, or halves of scores before that
    static constexpr int EXCHANGE = HALVES == 1 ? 0 : 2 * WARPS * 32 * 8 * 4, JOIN = 2 * FAN * ROWS * 4;
    static constexpr int STAT = SUM + (JOIN > EXCHANGE ? JOIN : EXCHANGE);  // [SLICES + 1][ROWS][2] float
    static constexpr int MISC = STAT + (SLICES + 1) * ROWS * 2 * 4;
    static_assert(ROWS * PART_ROW * 4 <= STAGE, "a warp's sums fit in a stage");
    static constexpr int BYTES = MISC + 32;
    static_assert(PER_SM * (BYTES + 1024) <= 228 * 1024, "the CTAs of a wave are resident together");
};

__device__ __forceinline__ void cp16(uint32_t dst, const void *src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ float exp2_(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void ldsm4(uint32_t a, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(a)
                 : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t a, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(a)
                 : "memory");
}
template <typename T>
__device__ __forceinline__ uint32_t load_pair(const T *p, bool pairs) {
    if (pairs) return *(const uint32_t *)p;
    return *(const uint16_t *)p | (uint32_t) * (const uint16_t *)(p + 1) << 16;
}
template <typename T>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack(float lo, float hi, __nv_bfloat16) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *(uint32_t *)&v;
}
__device__ __forceinline__ uint32_t pack(float lo, float hi, __half) {
    __half2 v = __floats2half2_rn(lo, hi);
    return *(uint32_t *)&v;
}

// What a number of T that stands for a weight leaves of it, rounded in turn, for a pair: the two
// together are within 2^-16 of a weight (bf16; fp16 2^-22, and 2^-25).
__device__ __forceinline__ uint32_t pack_rest(float lo, float hi, uint32_t p, __nv_bfloat16 t) {
    return pack(lo - __uint_as_float(p << 16), hi - __uint_as_float(p & 0xffff0000u), t);
}
__device__ __forceinline__ uint32_t pack_rest(float lo, float hi, uint32_t p, __half t) {
    const float2 v = __half22float2(*(const __half2 *)&p);
    return pack(lo - v.x, hi - v.y, t);
}
// A number of T a little under a weight, for a pair, so that what it leaves is above zero and not
// rounded to it: both times infinity are then that infinity, and not 0 * inf or inf - inf.  (fp16
// weights under 2^-24 are zeros either way.)
__device__ __forceinline__ uint32_t pack_under(float lo, float hi, __nv_bfloat16) {
    constexpr float F = 1.f - 0x1p-20f;
    uint32_t p;
    asm("cvt.rz.bf16x2.f32 %0, %1, %2;\n" : "=r"(p) : "f"(hi * F), "f"(lo * F));
    return p;
}
__device__ __forceinline__ uint32_t pack_under(float lo, float hi, __half) {
    constexpr float F = 1.f - 0x1p-22f, D = 0x1.01p-25f;
    uint32_t p;
    asm("cvt.rz.f16x2.f32 %0, %1, %2;\n" : "=r"(p) : "f"(fmaf(hi, F, -D)), "f"(fmaf(lo, F, -D)));
    return p;
}

// Live tokens of sequence b: never beyond what its page table row can name, and so few that
// the end of their last tile is an int as well.
__device__ __forceinline__ int length_of(const AttendArgs &a, int b) {
    const int n = max(a.lens[b], 0);
    const long long cap = min((long long)a.max_pages * a.page, (long long)HV_ATTENTION_MAX_LENGTH);
    if (n > cap) {
        atomicOr(a.err, HV_DECODE_BAD_LENGTH);
        return (int)cap;
    }
    return n;
}

// A place on the line of tiles: tile `tile` of item (sequence b, head tile h).
template <int TILE>
struct Place {
    int b, h, tile, len, tiles;
    __device__ __forceinline__ void set(const AttendArgs &a, int seq) {
        b = seq;
        len = length_of(a, b);
        tiles = (len + TILE - 1) / TILE;
    }
    __device__ __forceinline__ void next(const AttendArgs &a, int heads) {
        if (++tile < tiles) return;
        tile = 0;
        if (++h < heads) return;
        h = 0;
        do set(a, b + 1);  // only called where a further tile exists
        while (tiles == 0);
    }
};

template <typename T>
__device__ __forceinline__ void store4(T *p, bool vec, float4 v, float f) {
    T e[4] = {from_f32<T>(v.x * f), from_f32<T>(v.y * f), from_f32<T>(v.z * f), from_f32<T>(v.w * f)};
    if (vec) {
        *(uint2 *)p = *(const uint2 *)e;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = e[i];
    }
}

// Joins n parts of one item, by the whole CTA: FAN parts at a time, the loads of a round
// issued together (the parts come from L2, and its latency under load, once a part, would be
// the time).  Part k is in slot(k).  The order of every sum is that of the parts.  Goes to the
// output if `out`, else back to slot(0).  `sum` has room for 2 * FAN * ROWS, `stat` for
// 3 * ROWS numbers.
template <typename T, int D, typename Slot>
__device__ __forceinline__ void join_parts(float *parts, float *sum, float *stat, Slot slot, int n, int nrows, T *out,
                                           long long o_head, bool o_vec, float *lse, long long lse_head) {
    constexpr int THREADS = Lay<D>::THREADS, PER = FAN * ROWS / THREADS;  // (part, row) pairs of a thread
    constexpr int NV = ROWS * D / 4 / THREADS;
    const int tid = threadIdx.x;
    float4 *po = (float4 *)parts;
    float2 *pst = (float2 *)(parts + 2ll * gridDim.x * (ROWS * D));
    const int nvec = nrows * (D / 4);
    float *factor = stat + 2 * ROWS;
    float4 acc[NV] = {};
    for (int k0 = 0; k0 < n; k0 += FAN) {
        const int m = min(FAN, n - k0);
        float2 v[PER];
#pragma unroll
        for (int e = 0; e < PER; ++e) {
            const int k = (tid + e * THREADS) / ROWS, r = tid % ROWS;
            v[e] = k < m && r < nrows ? __ldcg(pst + slot(k0 + k) * ROWS + r) : make_float2(LOWEST, 0.f);
        }
        float4 x[FAN];
        auto fetch = [&](int t) {
#pragma unroll
            for (int k = 0; k < FAN; ++k)
                x[k] = k < m && t < nvec ? __ldcg(po + slot(k0 + k) * (ROWS * D / 4) + t) : make_float4(0.f, 0.f, 0.f, 0.f);
        };
        fetch(tid);
        __syncthreads();
#pragma unroll
        for (int e = 0; e < PER; ++e) {
            sum[tid + e * THREADS] = v[e].x;
            sum[FAN * ROWS + tid + e * THREADS] = v[e].y;
        }
        __syncthreads();
        if (tid < ROWS) {  // weights of the parts of row `tid`
            const float was = k0 ? stat[2 * tid] : LOWEST;
            float M = was;
            for (int k = 0; k < m; ++k) M = fmaxf(M, sum[k * ROWS + tid]);
            const float f = k0 ? exp2_(was - M) : 0.f;
            float S = k0 ? stat[2 * tid + 1] * f : 0.f;
            for (int k = 0; k < m; ++k) {
                const float w = exp2_(sum[k * ROWS + tid] - M);
                S += w * sum[(FAN + k) * ROWS + tid];
                sum[k * ROWS + tid] = w;
            }
            stat[2 * tid] = M;
            stat[2 * tid + 1] = S;
            factor[tid] = f;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int t = tid + i * THREADS;
            if (t >= nvec) break;
            if (i) fetch(t);
            const int row = t / (D / 4);
            const float f = factor[row];
            acc[i] = make_float4(acc[i].x * f, acc[i].y * f, acc[i].z * f, acc[i].w * f);
#pragma unroll
            for (int k = 0; k < FAN; ++k) {
                if (k >= m) break;
                const float w = sum[k * ROWS + row];
                acc[i].x += w * x[k].x;
                acc[i].y += w * x[k].y;
                acc[i].z += w * x[k].z;
                acc[i].w += w * x[k].w;
            }
        }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int t = tid + i * THREADS, row = t / (D / 4);
        if (t >= nvec) break;
        if (out) store4(out + row * o_head + (t - row * (D / 4)) * 4, o_vec, acc[i], 1.f / stat[2 * row + 1]);
        else __stcg(po + slot(0) * (ROWS * D / 4) + t, acc[i]);
    }
    if (tid < nrows) {
        if (!out) __stcg(pst + slot(0) * ROWS + tid, make_float2(stat[2 * tid], stat[2 * tid + 1]));
        else if (lse) lse[tid * lse_head] = (stat[2 * tid] + log2f(stat[2 * tid + 1])) * 0.69314718055994531f;
    }
}

// Counts this CTA in; true in the one that comes last, for which the counter is zero again
// and the others' stores are visible.
__device__ __forceinline__ bool comes_last(uint32_t *counter, uint32_t of, long long *flag) {
    __syncthreads();
    if (threadIdx.x == 0) {
        __threadfence();  // the CTA's stores, which the barrier put before this
        const bool last = atomicAdd(counter, 1u) == of - 1;
        if (last) *counter = 0;
        __threadfence();  // and the others', before what follows the next barrier
        *flag = last;
    }
    __syncthreads();
    const bool last = *flag;
    __syncthreads();
    return last;
}

// HALF: items of up to eight heads.  Their weights take eight rows of the second product, and
// the other eight take what rounding left of those (see there).
template <typename T, int D, bool HALF>
__global__ void __launch_bounds__(Lay<D>::THREADS, Lay<D>::PER_SM)
    attend_kernel(const __grid_constant__ AttendArgs a) {
    griddep_wait();
    griddep_launch();
    using L = Lay<D>;
    constexpr int NR = HALF ? 1 : 2;  // rows of a thread: lane / 4 + 8 i
    constexpr int DH = L::DH, THREADS = L::THREADS, BLOCKS = L::BLOCKS, WTOK = L::WTOK, TILE = L::TILE;
    using Place = Place<L::TILE>;
    extern __shared__ __align__(128) uint8_t smem[];
    float *sum = (float *)(smem + L::SUM);
    float *stat = (float *)(smem + L::STAT);
    long long *misc = (long long *)(smem + L::MISC);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int slice = warp % SLICES, half = warp / SLICES;  // tokens and dimensions of this warp
    const int items = a.kv_heads * a.head_tiles;            // of a sequence

    // Sequences of no tokens: nobody's share holds them.
    for (int b = blockIdx.x; b < a.seqs; b += gridDim.x)
        if (a.lens[b] <= 0 || a.max_pages == 0) {
            for (int i = tid; i < a.heads * D; i += THREADS)
                ((T *)a.out)[b * a.o_seq + (i / D) * a.o_head + i % D] = from_f32<T>(0.f);
            if (a.lse)
                for (int i = tid; i < a.heads; i += THREADS) a.lse[b * a.lse_seq + i * a.lse_head] = -CUDART_INF_F;
        }

    // The line's length, this CTA's share of it, and the share's first place.
    if (warp == 0) {
        long long total = 0;
        int held = 0;  // this lane's sequence of the last 32
        int most = 0, live = 0;  // the longest of this lane's sequences, and how many have tokens
        for (int b0 = 0; b0 < a.seqs; b0 += 32) {
            const int b = b0 + lane;
            held = b < a.seqs ? (length_of(a, b) + TILE - 1) / TILE : 0;
            total += __reduce_add_sync(~0u, held);
            most = max(most, held);
            live += held > 0;
        }
        const long long tiles = total;
        total *= items;
        long long share = (total + gridDim.x - 1) / gridDim.x;
        if (share <= MIN_SHARE) {
            share = MIN_SHARE;
        } else {
            most = __reduce_max_sync(~0u, most);
            if (tiles == (long long)most * __reduce_add_sync(~0u, live)) {
                const long long whole = share <= most ? most : (share + most - 1) / most * most;
                if (whole - share <= SLACK) share = whole;
            }
        }
        const long long first = share * blockIdx.x;
        long long before = 0;  // tiles of the sequences ahead of b0
        int found = -1;
        for (int b0 = 0; b0 < a.seqs && found < 0 && first < total; b0 += 32) {
            const int b = b0 + lane;
            const int n = a.seqs <= 32 ? held : b < a.seqs ? (length_of(a, b) + TILE - 1) / TILE : 0;
            int incl = n;
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(~0u, incl, o);
                if (lane >= o) incl += v;
            }
            const bool here = (before + incl) * items > first;
            const unsigned m = __ballot_sync(~0u, here);
            if (m) {
                const int l = __ffs(m) - 1;
                found = b0 + l;
                before += __shfl_sync(~0u, incl - n, l);
            } else {
                before += __shfl_sync(~0u, incl, 31);
            }
        }
        if (lane == 0) {
            misc[0] = total;
            misc[1] = share;
            misc[2] = before * items;
            misc[3] = found;
        }
    }
    __syncthreads();
    const long long total = misc[0], share = misc[1], first = share * blockIdx.x;
    if (first >= total) return;
    const int count = (int)min(share, total - first);
    Place ld, cur;
    cur.set(a, (int)misc[3]);
    {
        const long long in = first - misc[2];
        cur.h = (int)(in / cur.tiles);
        cur.tile = (int)(in - (long long)cur.h * cur.tiles);
    }
    ld = cur;
    long long item_first = first - cur.tile;  // the line's index of the current item's first tile

    uint8_t *ring = smem + warp * L::STAGES * L::STAGE;
    const T *kc = (const T *)a.kc, *vc = (const T *)a.vc;

    // The page of a block of 16 tokens (page16: they share one), or of this lane's token of it
    // (lane & 15), at place p; -1 past the length.
    struct Pages {
        int of[BLOCKS];
    };
    auto pages_of = [&](const Place &p) {
        Pages r;
#pragma unroll
        for (int k = 0; k < BLOCKS; ++k) {
            const int t = p.tile * TILE + slice * WTOK + k * BLOCK + (a.page16 ? 0 : lane & 15);
            r.of[k] = t < p.len ? a.pages[p.b * a.pages_stride + (a.page_shift >= 0 ? t >> a.page_shift : t / a.page)] : -1;
        }
        return r;
    };
    auto load = [&](int stage, const Place &p, const Pages &pgs) {
        const int t0 = p.tile * TILE + slice * WTOK;
        if (t0 >= p.len) return;  // not read either
        const int head = p.h / a.head_tiles;
        constexpr int CH = DH / 8;  // 16-byte pieces of a row
        constexpr int N = BLOCK * CH / 32;
#pragma unroll
        for (int b = 0; b < BLOCKS; ++b) {
            const uint32_t dst = tc05::smem_u32(ring + stage * L::STAGE) + b * BLOCK * L::ROW;
            const int t1 = t0 + b * BLOCK;
            if (a.page16) {
                int pg = pgs.of[b], live = p.len - t1;  // rows of the 16 that exist
                if (pg < 0 || pg >= a.num_pages) {
                    if (live > 0) atomicOr(a.err, HV_DECODE_BAD_PAGE);
                    pg = live = 0;
                }
                const int slot = a.page_shift >= 0 ? t1 & (a.page - 1) : t1 % a.page;
                const T *k = kc + (pg * a.kc_page + slot * a.kc_slot + head * a.kc_head + half * DH);
                const T *v = vc + (pg * a.vc_page + slot * a.vc_slot + head * a.vc_head + half * DH);
                if constexpr (32 % CH == 0) {
                    const int row0 = lane / CH, col = lane % CH;
                    k += row0 * a.kc_slot + col * 8;
                    v += row0 * a.vc_slot + col * 8;
                    const uint32_t to = dst + row0 * L::ROW + col * 16;
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        const int n = row0 + i * (32 / CH) < live ? 16 : 0;
                        cp16(to + i * (32 / CH) * L::ROW, k, n);
                        cp16(to + (WTOK + i * (32 / CH)) * L::ROW, v, n);
                        k += (32 / CH) * a.kc_slot;
                        v += (32 / CH) * a.vc_slot;
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        const int c = i * 32 + lane, row = c / CH, col = c % CH, n = row < live ? 16 : 0;
                        cp16(dst + row * L::ROW + col * 16, k + row * a.kc_slot + col * 8, n);
                        cp16(dst + (WTOK + row) * L::ROW + col * 16, v + row * a.vc_slot + col * 8, n);
                    }
                }
                continue;
            }
            const int t = t1 + (lane & 15), pg = pgs.of[b];
            bool ok = t < p.len;
            if (ok && (pg < 0 || pg >= a.num_pages)) {
                atomicOr(a.err, HV_DECODE_BAD_PAGE);
                ok = false;
            }
            const int slot = a.page_shift >= 0 ? t & (a.page - 1) : t % a.page;
            const long long ko = ok ? pg * a.kc_page + slot * a.kc_slot + head * a.kc_head + half * DH : -1;
            const long long vo = ok ? pg * a.vc_page + slot * a.vc_slot + head * a.vc_head + half * DH : -1;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int c = i * 32 + lane, row = c / CH, col = c % CH;
                const long long k = __shfl_sync(~0u, ko, row), v = __shfl_sync(~0u, vo, row);
                cp16(dst + row * L::ROW + col * 16, kc + (k < 0 ? 0 : k + col * 8), k < 0 ? 0 : 16);
                cp16(dst + (WTOK + row) * L::ROW + col * 16, vc + (v < 0 ? 0 : v + col * 8), v < 0 ? 0 : 16);
            }
        }
    };

    Pages pg = pages_of(ld);
    int loaded = 0;
    auto load_next = [&]() {
        if (loaded < count) {
            load(loaded % L::STAGES, ld, pg);
            if (++loaded < count) {
                ld.next(a, items);
                pg = pages_of(ld);
            }
        }
        asm volatile("cp.async.commit_group;\n" ::: "memory");
    };
    for (int s = 0; s < L::STAGES - 1; ++s) load_next();

    uint32_t qf[DH / 16][4];
    float o[DH / 8][4];
    float m[NR], l[NR];
    bool fresh = true;
    for (int u = 0; u < count; ++u) {
        const int head = cur.h / a.head_tiles, ht = cur.h - head * a.head_tiles;
        const int nrows = min(ROWS, a.group - ht * ROWS);
        const int h0 = head * a.group + ht * ROWS;
        if (fresh) {
            const T *q = (const T *)a.q + cur.b * a.q_seq + h0 * a.q_head;
#pragma unroll
            for (int j = 0; j < DH / 16; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int r = (lane >> 2) + (i & 1) * 8, c = half * DH + j * 16 + (lane & 3) * 2 + (i >> 1) * 8;
                    qf[j][i] = (i & 1) < NR && r < nrows ? load_pair(q + r * a.q_head + c, a.q_pairs) : 0;
                }
#pragma unroll
            for (int j = 0; j < DH / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
#pragma unroll
            for (int i = 0; i < NR; ++i) m[i] = LOWEST, l[i] = 0.f;
            fresh = false;
        }
        asm volatile("cp.async.wait_group %0;\n" ::"n"(L::STAGES - 2) : "memory");
        __syncwarp();
        const int t0 = cur.tile * TILE + slice * WTOK;
        if (t0 < cur.len) {
            const uint32_t kb = tc05::smem_u32(ring + (u % L::STAGES) * L::STAGE), vb = kb + WTOK * L::ROW;
            float s[2 * BLOCKS][4] = {};
            const uint32_t ka = kb + ((lane >> 4) * 8 + (lane & 7)) * L::ROW + ((lane >> 3) & 1) * 16;
#pragma unroll
            for (int j = 0; j < DH / 16; ++j)
#pragma unroll
                for (int b = 0; b < BLOCKS; ++b) {
                    uint32_t r[4];
                    ldsm4(ka + b * BLOCK * L::ROW + j * 32, r);
                    mma<T>(s[2 * b], qf[j], r[0], r[1]);
                    mma<T>(s[2 * b + 1], qf[j], r[2], r[3]);
                }
            if constexpr (L::HALVES == 2) {
                // two buffers in turn: the partner has read a buffer before the step's barrier
                // after the one that filled it
                float4 *mine = (float4 *)sum + ((u & 1) * L::WARPS + warp) * 64 + lane;
                const float4 *its = (float4 *)sum + ((u & 1) * L::WARPS + (warp ^ SLICES)) * 64 + lane;
                mine[0] = make_float4(s[0][0], s[0][1], s[0][2], s[0][3]);
                mine[32] = make_float4(s[1][0], s[1][1], s[1][2], s[1][3]);
                asm volatile("bar.sync %0, 64;\n" ::"r"(1 + slice) : "memory");
                const float4 x = its[0], y = its[32];
                s[0][0] += x.x, s[0][1] += x.y, s[0][2] += x.z, s[0][3] += x.w;
                s[1][0] += y.x, s[1][1] += y.y, s[1][2] += y.z, s[1][3] += y.w;
            }
            // s[n][2 * i + e]: row lane / 4 + 8 i, token t0 + 8 n + 2 (lane % 4) + e
#pragma unroll
            for (int n = 0; n < 2 * BLOCKS; ++n)
#pragma unroll
                for (int e = 0; e < 2 * NR; ++e) s[n][e] *= a.scale_log2;
            if (t0 + WTOK > cur.len)
#pragma unroll
                for (int n = 0; n < 2 * BLOCKS; ++n)
#pragma unroll
                    for (int e = 0; e < 2 * NR; ++e)
                        if (t0 + n * 8 + (lane & 3) * 2 + (e & 1) >= cur.len) s[n][e] = -CUDART_INF_F;
            float x[NR];
            bool moves = false;
#pragma unroll
            for (int i = 0; i < NR; ++i) {
                x[i] = fmaxf(s[0][2 * i], s[0][2 * i + 1]);
#pragma unroll
                for (int n = 1; n < 2 * BLOCKS; ++n) x[i] = fmaxf(x[i], fmaxf(s[n][2 * i], s[n][2 * i + 1]));
                x[i] = fmaxf(x[i], __shfl_xor_sync(~0u, x[i], 1));
                x[i] = fmaxf(x[i], __shfl_xor_sync(~0u, x[i], 2));
                moves |= x[i] > m[i] + (TOP<T> + SOFT);
            }
            if (__any_sync(~0u, moves)) {
                float f[NR];
#pragma unroll
                for (int i = 0; i < NR; ++i) {
                    x[i] = fmaxf(x[i] - TOP<T>, m[i]);
                    f[i] = exp2_(m[i] - x[i]);
                    m[i] = x[i];
                    l[i] *= f[i];
                }
#pragma unroll
                for (int j = 0; j < DH / 8; ++j) {
                    o[j][0] *= f[0];
                    o[j][1] *= f[0];
                    o[j][2] *= f[NR - 1];
                    o[j][3] *= f[NR - 1];
                }
            }
#pragma unroll
            for (int n = 0; n < 2 * BLOCKS; ++n)
#pragma unroll
                for (int e = 0; e < 2 * NR; ++e) {
                    s[n][e] = exp2_(s[n][e] - m[e >> 1]);
                    l[e >> 1] += s[n][e];
                }
            // A weight goes into the product as two numbers of type T, the rounded one and what that
            // leaves: rounded alone, weights that are alike would all be off the same way, by up to 2^-8
            // (bf16), against a sum that is not.  With up to eight heads the second ones take the rows
            // that no head has, with more a product of their own (64 heads over 4, 64 x 4000 tokens: 99 us
            // without it, 103 with).
#pragma unroll
            for (int b = 0; b < BLOCKS; ++b) {
                const float(&x)[4] = s[2 * b], (&y)[4] = s[2 * b + 1];
                const uint32_t x0 = HALF ? pack(x[0], x[1], T()) : pack_under(x[0], x[1], T());
                const uint32_t y0 = HALF ? pack(y[0], y[1], T()) : pack_under(y[0], y[1], T());
                const uint32_t x0r = pack_rest(x[0], x[1], x0, T()), y0r = pack_rest(y[0], y[1], y0, T());
                const uint32_t x1 = HALF ? x0r : pack_under(x[2], x[3], T());
                const uint32_t y1 = HALF ? y0r : pack_under(y[2], y[3], T());
                const uint32_t p[4] = {x0, x1, y0, y1};
                const uint32_t va = vb + (b * BLOCK + (lane & 15)) * L::ROW + (lane >> 4) * 16;
#pragma unroll
                for (int j = 0; j < DH / 16; ++j) {
                    uint32_t r[4];
                    ldsm4t(va + j * 32, r);
                    mma<T>(o[2 * j], p, r[0], r[1]);
                    mma<T>(o[2 * j + 1], p, r[2], r[3]);
                    if constexpr (!HALF) {
                        const uint32_t d[4] = {x0r, pack_rest(x[2], x[3], x1, T()), y0r, pack_rest(y[2], y[3], y1, T())};
                        mma<T>(o[2 * j], d, r[0], r[1]);
                        mma<T>(o[2 * j + 1], d, r[2], r[3]);
                    }
                }
            }
        }
        __syncwarp();  // the stage that is refilled next was read in the step before
        load_next();

        const bool item_ends = cur.tile + 1 == cur.tiles;
        if (item_ends || u + 1 == count) {
            // Join the slices of tokens: rows' maxima, then the sums in the order of the slices.
            if (L::HALVES == 2) __syncthreads();  // the scores that were exchanged last have been read
#pragma unroll
            for (int i = 0; i < NR; ++i) {
                l[i] += __shfl_xor_sync(~0u, l[i], 1);
                l[i] += __shfl_xor_sync(~0u, l[i], 2);
                if ((lane & 3) == 0 && half == 0) {
                    float *st = stat + (slice * ROWS + (lane >> 2) + 8 * i) * 2;
                    st[0] = m[i];
                    st[1] = l[i];
                }
            }
            __syncthreads();
            float f[NR];
#pragma unroll
            for (int i = 0; i < NR; ++i) {
                float top = LOWEST;
                for (int w = 0; w < SLICES; ++w) top = fmaxf(top, stat[(w * ROWS + (lane >> 2) + 8 * i) * 2]);
                f[i] = exp2_(m[i] - top);
            }
            float *mine = (float *)(ring + (u % L::STAGES) * L::STAGE);  // read, and not yet refilled
#pragma unroll
            for (int j = 0; j < DH / 8; ++j) {
                if (HALF) {  // an infinity stays: the rest may have had a zero or another sign for it
                    if (!isinf(o[j][0])) o[j][0] += o[j][2];
                    if (!isinf(o[j][1])) o[j][1] += o[j][3];
                }
#pragma unroll
                for (int i = 0; i < NR; ++i)
                    *(float2 *)(mine + ((lane >> 2) + 8 * i) * L::PART_ROW + j * 8 + (lane & 3) * 2) =
                        make_float2(o[j][2 * i] * f[i], o[j][2 * i + 1] * f[i]);
            }
            float M = LOWEST, S = 0.f;
            float *of_row = stat + SLICES * ROWS * 2;
            if (tid < 8 * NR) {  // a row's maximum and sum
                for (int w = 0; w < SLICES; ++w) M = fmaxf(M, stat[(w * ROWS + tid) * 2]);
                for (int w = 0; w < SLICES; ++w)
                    S += stat[(w * ROWS + tid) * 2 + 1] * exp2_(stat[(w * ROWS + tid) * 2] - M);
                of_row[tid * 2 + 1] = S;
            }
            __syncthreads();
            // four columns of the item's sums
            auto four = [&](int r, int c) {
                const float *p = (const float *)(smem + (c / DH * SLICES * L::STAGES + u % L::STAGES) * L::STAGE) +
                                 r * L::PART_ROW + c % DH;
                float4 v = *(const float4 *)p;
#pragma unroll
                for (int w = 1; w < SLICES; ++w) {
                    const float4 x = *(const float4 *)(p + w * (L::STAGES * L::STAGE / 4));
                    v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
                }
                return v;
            };
            const int nvec = nrows * (D / 4);
            T *out = (T *)a.out + cur.b * a.o_seq + h0 * a.o_head;
            float *lse = a.lse ? a.lse + cur.b * a.lse_seq + h0 * a.lse_head : nullptr;
            const int c_first = (int)(item_first / share), c_last = (int)((item_first + cur.tiles - 1) / share);
            if (c_first == c_last) {
                for (int i = tid; i < nvec; i += THREADS) {
                    const int r = i / (D / 4), c = (i - r * (D / 4)) * 4;
                    store4(out + r * a.o_head + c, a.o_vec, four(r, c), 1.f / of_row[r * 2 + 1]);
                }
                if (lse && tid < nrows) lse[tid * a.lse_head] = (M + log2f(S)) * 0.69314718055994531f;
            } else {
                // A part.  The last CTA of up to ONE_LEVEL to come joins them all; of more, the last of
                // every GROUP neighbouring shares joins theirs, and the last of those the rest.  A
                // share leaves its second slot to the item that starts in it, its first to one that
                // started before; likewise at most one item enters a group of shares from before.
                auto slot = [&](int c) { return 2ll * c + (c == c_first); };
                const long long mine = slot(blockIdx.x);
                float4 *po = (float4 *)(a.parts + mine * (ROWS * D));
                float2 *pst = (float2 *)(a.parts + 2ll * gridDim.x * (ROWS * D)) + mine * ROWS;
                for (int i = tid; i < nvec; i += THREADS)
                    __stcg(po + i, four(i / (D / 4), i % (D / 4) * 4));
                if (tid < nrows) __stcg(pst + tid, make_float2(M, S));
                const int n = c_last - c_first + 1;
                if (n <= ONE_LEVEL) {
                    if (comes_last(a.counts + c_first, n, misc))
                        join_parts<T, D>(a.parts, sum, stat, [&](int k) { return slot(c_first + k); }, n, nrows, out,
                                         a.o_head, a.o_vec, lse, a.lse_head);
                } else {
                    const int g = blockIdx.x / GROUP, g_first = c_first / GROUP, groups = c_last / GROUP - g_first + 1;
                    const int lo = max(c_first, g * GROUP), ng = min(c_last, g * GROUP + GROUP - 1) - lo + 1;
                    if (comes_last(lo == c_first ? a.counts + c_first : a.counts + MAX_GRID + g, ng, misc)) {
                        if (ng > 1)
                            join_parts<T, D>(a.parts, sum, stat, [&](int k) { return slot(lo + k); }, ng, nrows,
                                             (T *)nullptr, 0, false, nullptr, 0);
                        if (comes_last(a.counts + 2 * MAX_GRID + c_first, groups, misc))
                            join_parts<T, D>(a.parts, sum, stat,
                                             [&](int k) { return slot(k ? (g_first + k) * GROUP : c_first); }, groups,
                                             nrows, out, a.o_head, a.o_vec, lse, a.lse_head);
                    }
                }
            }
            __syncthreads();  // sum, stat and misc are free again
            fresh = true;
            item_first += cur.tiles;
        }
        if (u + 1 < count) cur.next(a, items);
    }
    asm volatile("cp.async.wait_all;\n" ::: "memory");
}

// The counters come first and take the same room for every call, so that calls of other
// sizes with the same workspace never find a part where a zero belongs.
constexpr int COUNT_BYTES = 3 * MAX_GRID * 4;
static_assert(HV_ATTENTION_MAX_LENGTH + (long long)Lay<64>::TILE + ROWS <= INT32_MAX && Lay<64>::TILE >= Lay<128>::TILE,
              "token numbers of a last tile are ints");
static_assert(COUNT_BYTES == HV_ATTENTION_COUNTER_BYTES, "what the caller zeroes");

// CTAs of one resident wave on the current device.
int wave(int d) {
    const int sms = sm_count();
    const int grid = sms * (d <= 64 ? Lay<64>::PER_SM : d <= 128 ? Lay<128>::PER_SM : Lay<256>::PER_SM);
    return grid < MAX_GRID ? grid : MAX_GRID;
}

template <typename T, int D, bool HALF>
cudaError_t launch(const AttendArgs &a, int grid, cudaStream_t st) {
    static std::atomic<uint64_t> ready;
    const cudaError_t e = allow_shared(attend_kernel<T, D, HALF>, ready);
    if (e != cudaSuccess) return e;
    return launch_pdl(attend_kernel<T, D, HALF>, dim3((unsigned)grid), dim3(Lay<D>::THREADS), Lay<D>::BYTES, st, a);
}
template <typename T, int D>
cudaError_t by_group(const AttendArgs &a, int grid, cudaStream_t st) {
    return a.group <= ROWS / 2 ? launch<T, D, true>(a, grid, st) : launch<T, D, false>(a, grid, st);
}

template <typename T>
cudaError_t by_dim(const AttendArgs &a, int dim, int grid, cudaStream_t st) {
    switch (dim) {
        case 32: return by_group<T, 32>(a, grid, st);
        case 64: return by_group<T, 64>(a, grid, st);
        case 96: return by_group<T, 96>(a, grid, st);
        case 128: return by_group<T, 128>(a, grid, st);
        case 192: return by_group<T, 192>(a, grid, st);
        default: return by_group<T, 256>(a, grid, st);
    }
}

bool known_dim(int d) { return d == 32 || d == 64 || d == 96 || d == 128 || d == 192 || d == 256; }

}  // namespace
}  // namespace hv

using namespace hv;

extern "C" int hv_paged_attention_workspace(int dim, int64_t *bytes) {
    if (!bytes) return fail(HV_ERR_VALUE, "null argument");
    if (!known_dim(dim)) return fail(HV_ERR_VALUE, "dim must be 32, 64, 96, 128, 192 or 256");
    const int grid = wave(dim);
    if (!grid) return fail(HV_ERR_CUDA, "cannot read the device's SM count");
    *bytes = COUNT_BYTES + 2ll * grid * ROWS * (dim + 2) * 4;
    return HV_OK;
}

extern "C" int hv_paged_attention(const hv_attention_args *p, void *stream) {
    if (!p) return fail(HV_ERR_VALUE, "null argument");
    if (p->dtype != HV_BF16 && p->dtype != HV_F16) return fail(HV_ERR_TYPE, "dtype must be HV_BF16 or HV_F16");
    if (p->seqs < 0 || p->heads < 1 || p->kv_heads < 1 || p->heads % p->kv_heads)
        return fail(HV_ERR_VALUE, "heads must be a positive multiple of kv_heads");
    if (!known_dim(p->dim)) return fail(HV_ERR_VALUE, "dim must be 32, 64, 96, 128, 192 or 256");
    if (p->page_size < 1 || p->num_pages < 0 || p->max_pages < 0) return fail(HV_ERR_VALUE, "bad cache geometry");
    if (p->seqs == 0) return HV_OK;
    if (!p->d_q || !p->d_out || !p->d_lens || (p->max_pages && !p->d_page_table) ||
        (p->num_pages && (!p->d_k_cache || !p->d_v_cache)))
        return fail(HV_ERR_VALUE, "null buffer");
    int64_t need = 0;
    const int rc = hv_paged_attention_workspace(p->dim, &need);
    if (rc) return rc;
    if (!p->d_workspace || p->workspace_bytes < need)
        return fail(HV_ERR_VALUE, "the workspace has %lld bytes of %lld", (long long)p->workspace_bytes, (long long)need);
    if (!dec::aligned(p->d_workspace, 256)) return fail(HV_ERR_VALUE, "the workspace must be 256-byte aligned");
    bool ok = dec::aligned(p->d_k_cache, 16) && dec::aligned(p->d_v_cache, 16);
    for (int i = 0; i < 3; ++i) ok = ok && p->k_cache_strides[i] % 8 == 0 && p->v_cache_strides[i] % 8 == 0;
    if (!ok) return fail(HV_ERR_VALUE, "cache rows must start on 16 bytes");
    int *err = dec::error_word();
    if (!err) return fail(HV_ERR_CUDA, "cannot resolve the device error word");
    const int group = p->heads / p->kv_heads;
    AttendArgs a{};
    a.q = p->d_q, a.kc = p->d_k_cache, a.vc = p->d_v_cache, a.out = p->d_out, a.lse = p->d_lse;
    a.pages = p->d_page_table, a.lens = p->d_lens;
    a.q_seq = p->q_strides[0], a.q_head = p->q_strides[1], a.o_seq = p->out_strides[0], a.o_head = p->out_strides[1];
    a.lse_seq = p->lse_strides[0], a.lse_head = p->lse_strides[1];
    a.kc_page = p->k_cache_strides[0], a.kc_slot = p->k_cache_strides[1], a.kc_head = p->k_cache_strides[2];
    a.vc_page = p->v_cache_strides[0], a.vc_slot = p->v_cache_strides[1], a.vc_head = p->v_cache_strides[2];
    a.pages_stride = p->page_table_stride;
    a.seqs = p->seqs, a.heads = p->heads, a.kv_heads = p->kv_heads, a.group = group;
    a.head_tiles = (group + ROWS - 1) / ROWS;
    a.num_pages = p->num_pages, a.page = p->page_size, a.max_pages = p->max_pages;
    a.q_pairs = dec::aligned(a.q, 4) && a.q_seq % 2 == 0 && a.q_head % 2 == 0;
    a.o_vec = dec::aligned(a.out, 8) && a.o_seq % 4 == 0 && a.o_head % 4 == 0;
    a.page16 = a.page % BLOCK == 0;
    a.page_shift = (a.page & (a.page - 1)) == 0 ? __builtin_ctz(a.page) : -1;
    a.scale_log2 = p->scale * 1.4426950408889634f;
    a.counts = (uint32_t *)p->d_workspace;
    a.parts = (float *)((char *)p->d_workspace + COUNT_BYTES);
    a.err = err;
    const int grid = wave(p->dim);
    const cudaError_t e = p->dtype == HV_BF16 ? by_dim<__nv_bfloat16>(a, p->dim, grid, (cudaStream_t)stream)
                                              : by_dim<__half>(a, p->dim, grid, (cudaStream_t)stream);
    if (e != cudaSuccess) return fail(HV_ERR_CUDA, "paged_attention: %s", cudaGetErrorString(e));
    return HV_OK;
}
