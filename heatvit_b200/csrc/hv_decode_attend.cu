// hv_decode_attend.cu — attention of one new token per sequence over a paged cache.
//
//   out[b, h] = sum_t softmax_t(scale * q[b, h] . K[t, h / group]) V[t, h / group],
//   t < lens[b];  a sequence of no tokens gives zeros (and a log-sum-exp of -inf).
//
// Bound by HBM: each live key and value is read once, for up to 16 query heads that share
// it.  Those heads are the 16 rows of an m16n8k16 matrix product: at 23 bytes of cache an
// SM clock, 16 multiply-adds an element leave the warp-level tensor path under a fifth
// busy, and it needs none of the 128 rows that a tcgen05 tile would pad to.
//
// Work: the (sequence, head tile) items are cut into tiles of 64 tokens, the tiles of all
// items are laid end to end, and the CTAs of one resident wave take equal shares of that
// line.  So a ragged batch is even, and a single long sequence uses every SM; every CTA
// works the cuts out for itself from the lengths, which stay on the device.  A warp owns 16
// tokens of a tile and its own cp.async ring, so that warps do not wait for one another
// inside an item; the ring runs ahead across item borders.
//
// An item inside one share is written straight out.  One that is cut leaves a part (the
// unnormalised sum, the running maximum and the sum of weights, in 32 bits) per CTA in the
// workspace, and the CTA that finishes last joins the parts in the order of the shares: the
// result does not depend on which that is.
#include <math_constants.h>

#include "hv_decode.cuh"
#include "hv_tc05.cuh"

namespace hv {
namespace {

using namespace dec;

constexpr int WARPS = 4, THREADS = WARPS * 32, ROWS = 16, WTOK = 16, TILE = WARPS * WTOK;
constexpr int MIN_SHARE = 4;  // tiles: a part costs more than the loads of fewer

struct AttendArgs {
    const void *q, *kc, *vc;
    void *out;
    float *lse;
    const int32_t *pages, *lens;
    long long q_seq, q_head, o_seq, o_head, lse_seq, lse_head;
    long long kc_page, kc_slot, kc_head, vc_page, vc_slot, vc_head, pages_stride;
    int seqs, heads, kv_heads, group, head_tiles, num_pages, page, max_pages, q_pairs;
    float scale_log2;
    float *parts;      // [grid][2][ROWS][D], then [grid][2][ROWS][2]
    uint32_t *counts;  // [grid], by the share that a cut item starts in; zero between calls
    int *err;
};

template <int D>
struct Lay {
    static constexpr int ROW = D * 2 + 16;  // bytes: rows 16 bytes apart modulo 128 (ldmatrix without conflicts)
    static constexpr int STAGES = D <= 64 ? 4 : 3;
    static constexpr int STAGE = 2 * WTOK * ROW;
    static constexpr int SUM = WARPS * STAGES * STAGE;  // [ROWS][D + 4] float
    static constexpr int STAT = SUM + ROWS * (D + 4) * 4;  // [WARPS][ROWS][2] float
    static constexpr int MISC = STAT + WARPS * ROWS * 2 * 4;
    static constexpr int BYTES = MISC + 32;
    // registers cap it at two or three, shared memory at one for D = 256
    static constexpr int PER_SM = D <= 64 ? 3 : D <= 128 ? 2 : 1;
};

__device__ __forceinline__ void cp16(uint32_t dst, const void *src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
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

// Live tokens of sequence b: never beyond what its page table row can name.
__device__ __forceinline__ int length_of(const AttendArgs &a, int b) {
    const int n = max(a.lens[b], 0);
    const long long cap = (long long)a.max_pages * a.page;
    if (n > cap) {
        atomicOr(a.err, HV_DECODE_BAD_LENGTH);
        return (int)cap;
    }
    return n;
}

// A place on the line of tiles: tile `tile` of item (sequence b, head tile h).
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

template <typename T, int D>
__global__ void __launch_bounds__(THREADS, Lay<D>::PER_SM) attend_kernel(const AttendArgs a) {
    griddep_wait();
    griddep_launch();
    using L = Lay<D>;
    extern __shared__ __align__(128) uint8_t smem[];
    float *sum = (float *)(smem + L::SUM);
    float *stat = (float *)(smem + L::STAT);
    long long *misc = (long long *)(smem + L::MISC);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int items = a.kv_heads * a.head_tiles;  // of a sequence

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
        for (int b0 = 0; b0 < a.seqs; b0 += 32) {
            const int b = b0 + lane;
            int n = b < a.seqs ? (length_of(a, b) + TILE - 1) / TILE : 0;
            for (int o = 16; o; o >>= 1) n += __shfl_xor_sync(~0u, n, o);
            total += n;
        }
        total *= items;
        long long share = (total + gridDim.x - 1) / gridDim.x;
        if (share < MIN_SHARE) share = MIN_SHARE;
        const long long first = share * blockIdx.x;
        long long before = 0;  // tiles of the sequences ahead of b0
        int found = -1;
        for (int b0 = 0; b0 < a.seqs && found < 0 && first < total; b0 += 32) {
            const int b = b0 + lane;
            const int n = b < a.seqs ? (length_of(a, b) + TILE - 1) / TILE : 0;
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

    // The page of this lane's token (lane & 15) at place p; -1 past the length.
    auto page_of = [&](const Place &p) {
        const int t = p.tile * TILE + warp * WTOK + (lane & 15);
        return t < p.len ? a.pages[p.b * a.pages_stride + t / a.page] : -1;
    };
    auto load = [&](int stage, const Place &p, int pg) {
        const int t = p.tile * TILE + warp * WTOK + (lane & 15);
        const int head = p.h / a.head_tiles;
        bool ok = t < p.len;
        if (ok && (pg < 0 || pg >= a.num_pages)) {
            atomicOr(a.err, HV_DECODE_BAD_PAGE);
            ok = false;
        }
        const int slot = t % a.page;
        const long long ko = ok ? pg * a.kc_page + slot * a.kc_slot + head * a.kc_head : -1;
        const long long vo = ok ? pg * a.vc_page + slot * a.vc_slot + head * a.vc_head : -1;
        const uint32_t dst = tc05::smem_u32(ring + stage * L::STAGE);
        constexpr int CH = D / 8;  // 16-byte pieces of a row
        constexpr int N = WTOK * CH / 32;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int c = i * 32 + lane, row = c / CH, col = c % CH;
            const long long k = __shfl_sync(~0u, ko, row), v = __shfl_sync(~0u, vo, row);
            cp16(dst + row * L::ROW + col * 16, kc + (k < 0 ? 0 : k + col * 8), k < 0 ? 0 : 16);
            cp16(dst + (WTOK + row) * L::ROW + col * 16, vc + (v < 0 ? 0 : v + col * 8), v < 0 ? 0 : 16);
        }
    };

    int pg = page_of(ld);
    int loaded = 0;
    auto load_next = [&]() {
        if (loaded < count) {
            load(loaded % L::STAGES, ld, pg);
            if (++loaded < count) {
                ld.next(a, items);
                pg = page_of(ld);
            }
        }
        asm volatile("cp.async.commit_group;\n" ::: "memory");
    };
    for (int s = 0; s < L::STAGES - 1; ++s) load_next();

    uint32_t qf[D / 16][4];
    float o[D / 8][4];
    float m[2], l[2];
    bool fresh = true;
    for (int u = 0; u < count; ++u) {
        const int head = cur.h / a.head_tiles, ht = cur.h - head * a.head_tiles;
        const int nrows = min(ROWS, a.group - ht * ROWS);
        const int h0 = head * a.group + ht * ROWS;
        if (fresh) {
            const T *q = (const T *)a.q + cur.b * a.q_seq;
#pragma unroll
            for (int j = 0; j < D / 16; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int r = (lane >> 2) + (i & 1) * 8, c = j * 16 + (lane & 3) * 2 + (i >> 1) * 8;
                    uint32_t w = 0;
                    if (r < nrows) {
                        const T *p = q + (h0 + r) * a.q_head + c;
                        if (a.q_pairs) w = *(const uint32_t *)p;
                        else w = *(const uint16_t *)p | (uint32_t) * (const uint16_t *)(p + 1) << 16;
                    }
                    qf[j][i] = w;
                }
#pragma unroll
            for (int j = 0; j < D / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
            m[0] = m[1] = -CUDART_INF_F;
            l[0] = l[1] = 0.f;
            fresh = false;
        }
        asm volatile("cp.async.wait_group %0;\n" ::"n"(L::STAGES - 2) : "memory");
        __syncwarp();
        const int t0 = cur.tile * TILE + warp * WTOK;
        if (t0 < cur.len) {
            const uint32_t kb = tc05::smem_u32(ring + (u % L::STAGES) * L::STAGE), vb = kb + WTOK * L::ROW;
            float s[2][4] = {};
            const uint32_t ka = kb + ((lane >> 4) * 8 + (lane & 7)) * L::ROW + ((lane >> 3) & 1) * 16;
#pragma unroll
            for (int j = 0; j < D / 16; ++j) {
                uint32_t r[4];
                ldsm4(ka + j * 32, r);
                mma<T>(s[0], qf[j], r[0], r[1]);
                mma<T>(s[1], qf[j], r[2], r[3]);
            }
            // s[n][2 * i + e]: row lane / 4 + 8 i, token t0 + 8 n + 2 (lane % 4) + e
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    s[n][e] = t0 + n * 8 + (lane & 3) * 2 + (e & 1) < cur.len ? s[n][e] * a.scale_log2 : -CUDART_INF_F;
            float f[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float x = fmaxf(fmaxf(s[0][2 * i], s[0][2 * i + 1]), fmaxf(s[1][2 * i], s[1][2 * i + 1]));
                x = fmaxf(x, __shfl_xor_sync(~0u, x, 1));
                x = fmaxf(x, __shfl_xor_sync(~0u, x, 2));
                x = fmaxf(x, m[i]);
                f[i] = exp2f(m[i] - x);
                m[i] = x;
                float p = 0.f;
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        s[n][2 * i + e] = exp2f(s[n][2 * i + e] - x);
                        p += s[n][2 * i + e];
                    }
                l[i] = l[i] * f[i] + p;
            }
            if (__any_sync(~0u, f[0] != 1.f || f[1] != 1.f)) {
#pragma unroll
                for (int j = 0; j < D / 8; ++j) {
                    o[j][0] *= f[0];
                    o[j][1] *= f[0];
                    o[j][2] *= f[1];
                    o[j][3] *= f[1];
                }
            }
            // weights in T for the product: each is within 2^-9 (bf16) of its 32-bit value,
            // as the values that it multiplies are of theirs; the sums stay in 32 bits
            uint32_t p[4] = {pack(s[0][0], s[0][1], T()), pack(s[0][2], s[0][3], T()), pack(s[1][0], s[1][1], T()),
                             pack(s[1][2], s[1][3], T())};
            const uint32_t va = vb + (lane & 15) * L::ROW + (lane >> 4) * 16;
#pragma unroll
            for (int j = 0; j < D / 16; ++j) {
                uint32_t r[4];
                ldsm4t(va + j * 32, r);
                mma<T>(o[2 * j], p, r[0], r[1]);
                mma<T>(o[2 * j + 1], p, r[2], r[3]);
            }
        }
        __syncwarp();  // the stage that is refilled next was read in the step before
        load_next();

        const bool item_ends = cur.tile + 1 == cur.tiles;
        if (item_ends || u + 1 == count) {
            // Join the four warps: rows' maxima, then the sums in the order of the warps.
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                l[i] += __shfl_xor_sync(~0u, l[i], 1);
                l[i] += __shfl_xor_sync(~0u, l[i], 2);
                if ((lane & 3) == 0) {
                    float *st = stat + (warp * ROWS + (lane >> 2) + 8 * i) * 2;
                    st[0] = m[i];
                    st[1] = l[i];
                }
            }
            __syncthreads();
            float top[2], f[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                top[i] = -CUDART_INF_F;
                for (int w = 0; w < WARPS; ++w) top[i] = fmaxf(top[i], stat[(w * ROWS + (lane >> 2) + 8 * i) * 2]);
                f[i] = m[i] == -CUDART_INF_F ? 0.f : exp2f(m[i] - top[i]);
            }
            for (int w = 0; w < WARPS; ++w) {
                if (warp == w) {
#pragma unroll
                    for (int j = 0; j < D / 8; ++j)
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            float2 *d = (float2 *)(sum + ((lane >> 2) + 8 * i) * (D + 4) + j * 8 + (lane & 3) * 2);
                            float2 v = make_float2(o[j][2 * i] * f[i], o[j][2 * i + 1] * f[i]);
                            if (w) {
                                const float2 x = *d;
                                v.x += x.x;
                                v.y += x.y;
                            }
                            *d = v;
                        }
                }
                __syncthreads();
            }
            auto row_stat = [&](int r, float &M, float &S) {
                M = -CUDART_INF_F;
                S = 0.f;
                for (int w = 0; w < WARPS; ++w) M = fmaxf(M, stat[(w * ROWS + r) * 2]);
                for (int w = 0; w < WARPS; ++w) {
                    const float mw = stat[(w * ROWS + r) * 2];
                    if (mw != -CUDART_INF_F) S += stat[(w * ROWS + r) * 2 + 1] * exp2f(mw - M);
                }
            };
            T *out = (T *)a.out + cur.b * a.o_seq + h0 * a.o_head;
            float *lse = a.lse ? a.lse + cur.b * a.lse_seq + h0 * a.lse_head : nullptr;
            const long long c_first = item_first / share, c_last = (item_first + cur.tiles - 1) / share;
            if (c_first == c_last) {
                for (int i = tid; i < nrows * D; i += THREADS) {
                    const int r = i / D, c = i - r * D;
                    float M, S;
                    row_stat(r, M, S);
                    out[r * a.o_head + c] = from_f32<T>(sum[r * (D + 4) + c] / S);
                    if (lse && c == 0) lse[r * a.lse_head] = (M + log2f(S)) * 0.69314718055994531f;
                }
            } else {
                const long long slot = 2ll * blockIdx.x + (blockIdx.x == c_first ? 1 : 0);
                float *po = a.parts + slot * (ROWS * D);
                float *pst = a.parts + 2ll * gridDim.x * (ROWS * D);
                for (int i = tid; i < nrows * D; i += THREADS) __stcg(po + i, sum[(i / D) * (D + 4) + i % D]);
                if (tid < nrows) {
                    float M, S;
                    row_stat(tid, M, S);
                    __stcg(pst + (slot * ROWS + tid) * 2, M);
                    __stcg(pst + (slot * ROWS + tid) * 2 + 1, S);
                }
                __threadfence();
                __syncthreads();
                uint32_t *cnt = a.counts + c_first;  // one cut item at most starts in a share
                if (tid == 0) misc[0] = atomicAdd(cnt, 1u) == (uint32_t)(c_last - c_first);
                __syncthreads();
                if (misc[0]) {
                    __threadfence();
                    for (int i = tid; i < nrows * D; i += THREADS) {
                        const int r = i / D, c = i - r * D;
                        float M = -CUDART_INF_F, S = 0.f, acc = 0.f;
                        for (long long k = c_first; k <= c_last; ++k)
                            M = fmaxf(M, __ldcg(pst + ((2 * k + (k == c_first)) * ROWS + r) * 2));
                        for (long long k = c_first; k <= c_last; ++k) {
                            const long long sl = 2 * k + (k == c_first);
                            const float w = exp2f(__ldcg(pst + (sl * ROWS + r) * 2) - M);
                            S += w * __ldcg(pst + (sl * ROWS + r) * 2 + 1);
                            acc += w * __ldcg(a.parts + sl * (ROWS * D) + r * D + c);
                        }
                        out[r * a.o_head + c] = from_f32<T>(acc / S);
                        if (lse && c == 0) lse[r * a.lse_head] = (M + log2f(S)) * 0.69314718055994531f;
                    }
                    if (tid == 0) *cnt = 0;
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
constexpr int MAX_GRID = 1024, COUNT_BYTES = MAX_GRID * 4;

// CTAs of one resident wave on the current device.
int wave(int d) {
    int dev = 0, sms = 0;
    if (cudaGetDevice(&dev) != cudaSuccess ||
        cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
        return 0;
    const int grid = sms * (d <= 64 ? Lay<64>::PER_SM : d <= 128 ? Lay<128>::PER_SM : Lay<256>::PER_SM);
    return grid < MAX_GRID ? grid : MAX_GRID;
}

template <typename T, int D>
cudaError_t launch(const AttendArgs &a, int grid, cudaStream_t st) {
    const cudaError_t e =
        cudaFuncSetAttribute(attend_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, Lay<D>::BYTES);
    if (e != cudaSuccess) return e;
    return launch_pdl(attend_kernel<T, D>, dim3((unsigned)grid), dim3(THREADS), Lay<D>::BYTES, st, a);
}

template <typename T>
cudaError_t by_dim(const AttendArgs &a, int dim, int grid, cudaStream_t st) {
    switch (dim) {
        case 32: return launch<T, 32>(a, grid, st);
        case 64: return launch<T, 64>(a, grid, st);
        case 96: return launch<T, 96>(a, grid, st);
        case 128: return launch<T, 128>(a, grid, st);
        case 192: return launch<T, 192>(a, grid, st);
        default: return launch<T, 256>(a, grid, st);
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
