// hv_decode_norm.cu — residual addition, root-mean-square norm and e4m3 output in one pass.
//
//   h = x + residual                         (32 bits; its rounding to T is residual_out)
//   y = h * rsqrt(mean(h^2) + eps) * weight
//   scale = max(amax |y|, 2^-100) / 448 over each 128 channels, q = e4m3(y / scale)
//
// The norm is taken of the unrounded sum: residual_out is one rounding of h, q one
// rounding of y.  The floor keeps the scale of an all-zero block a normal number.
//
// Bound by HBM: x, residual, residual_out and q cross it once each (7 bytes an element in
// bf16), so a row stays in registers between its sum of squares and its scales.  A thread has
// NV groups of eight consecutive channels, a row's threads apart: 16-byte accesses, and a
// block of 128 channels is 16 neighbouring lanes, whose amax is four shuffles.  Rows of up to
// 1024 channels take a warp each, longer ones a CTA; many long ones go through a ring of bulk
// copies (see norm_ring_kernel).
//
// Measured on one B200, in bursts: 16384 x 8192 bf16 with residual 146 us, 6.48 TB/s, the rate of a
// plain copy (164 us, 5.7 TB/s, when calls follow one another for long and the memory slows down);
// 1999 x 5000 fp32 26.6 us (4.9 TB/s: 13 or 14 rows a CTA, and filling and emptying the ring);
// 8192 x 8192 fp16 without residual 49 us, where half of the issue slots convert; 4096 x 32768 bf16
// 207 us (4.5 TB/s: rows over 16384 channels take 1024 threads of 64 registers, which spill 112 to
// 756 bytes); 8 x 4096 1.8 us, the launch.
#include <cuda_fp8.h>

#include <algorithm>

#include "hv_decode.cuh"
#include "hv_tc05.cuh"

namespace hv {
namespace {

using namespace dec;

struct NormArgs {
    const void *x, *res, *w;
    void *res_out;
    uint8_t *q;
    float *scale;
    long long x_stride, res_stride, res_out_stride, q_stride;  // elements
    long long scale_row, scale_group;
    int rows, dim, full;
    float eps;
};

__device__ __forceinline__ void mbar_expect(uint64_t *mbar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(tc05::smem_u32(mbar)), "r"(bytes)
                 : "memory");
}
// `bytes` (a multiple of 16, both addresses 16-byte aligned) into shared memory, completing on `mbar`.
__device__ __forceinline__ void bulk_copy(uint32_t dst, const void *src, uint32_t bytes, uint64_t *mbar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n" ::"r"(dst),
                 "l"(src), "r"(bytes), "r"(tc05::smem_u32(mbar))
                 : "memory");
}

constexpr float kE4m3Max = 448.f;
constexpr float kAmaxFloor = 7.888609052210118e-31f;  // 2^-100
constexpr float kSafeLow = 1e-30f, kSafeHigh = 1e30f;

// A row is worked on in groups of eight channels, of which the group at channel c has
// a.dim - c.  FULL: every group has eight or none, and starts on 16 bytes (8 in q).
template <typename T, bool FULL>
struct alignas(16) Group {
    T e[8];  // as stored, so that a load can be under way while others are used
    __device__ __forceinline__ void load(const T *p, int n) {
        if (FULL) {
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; ++i)
                ((uint4 *)e)[i] = n > 0 ? ((const uint4 *)p)[i] : make_uint4(0, 0, 0, 0);
        } else if (n < 8) {
#pragma unroll
            for (int i = 0; i < 8; ++i) e[i] = i < n ? p[i] : from_f32<T>(0.f);
        } else if ((uintptr_t)p % 16 == 0) {
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; ++i) ((uint4 *)e)[i] = ((const uint4 *)p)[i];
        } else if ((uintptr_t)p % 4 == 0) {
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) * 2; ++i) ((uint32_t *)e)[i] = ((const uint32_t *)p)[i];
        } else {  // 16 bits and odd: whole words between the first element and the last
            const uint32_t *m = (const uint32_t *)(p + 1);
            uint32_t v[5] = {(uint32_t) * (const uint16_t *)p << 16, m[0], m[1], m[2], *(const uint16_t *)(p + 7)};
#pragma unroll
            for (int i = 0; i < 4; ++i) ((uint32_t *)e)[i] = __funnelshift_r(v[i], v[i + 1], 16);
        }
    }
    __device__ __forceinline__ void store(T *p, int n) const {
        if (FULL) {
            if (n > 0)
#pragma unroll
                for (int i = 0; i < (int)sizeof(T) / 2; ++i) ((uint4 *)p)[i] = ((const uint4 *)e)[i];
        } else if (n < 8) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < n) p[i] = e[i];
        } else if ((uintptr_t)p % 16 == 0) {
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; ++i) ((uint4 *)p)[i] = ((const uint4 *)e)[i];
        } else if ((uintptr_t)p % 4 == 0) {
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) * 2; ++i) ((uint32_t *)p)[i] = ((const uint32_t *)e)[i];
        } else {
            const uint32_t *v = (const uint32_t *)e;
            uint32_t *m = (uint32_t *)(p + 1);
            p[0] = e[0];
#pragma unroll
            for (int i = 0; i < 3; ++i) m[i] = __funnelshift_r(v[i], v[i + 1], 16);
            p[7] = e[7];
        }
    }
};

// An approximate reciprocal and one Newton step: a block's 128 quotients share its error.
__device__ __forceinline__ float reciprocal(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return fmaf(y, fmaf(-x, y, 1.f), y);
}

// e4m3(y * f) of a group.
template <bool FULL>
__device__ __forceinline__ void put_q(const NormArgs &a, long long row, int c, int n, const float (&y)[8], float f) {
    uint32_t b[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(y[4 * j] * f, y[4 * j + 1] * f), __NV_SATFINITE,
                                                     __NV_E4M3);
        const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(y[4 * j + 2] * f, y[4 * j + 3] * f),
                                                     __NV_SATFINITE, __NV_E4M3);
        b[j] = lo | hi << 16;
    }
    uint8_t *q = a.q + row * a.q_stride + c;
    if (FULL) {
        if (n > 0) *(uint2 *)q = make_uint2(b[0], b[1]);
    } else if (n >= 8 && (uintptr_t)q % 8 == 0) {
        *(uint2 *)q = make_uint2(b[0], b[1]);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < n) q[j] = (uint8_t)(b[j >> 2] >> (8 * (j & 3)));
    }
}
// The larger, or a NaN where either is one (fmaxf would drop it): the NaN then reaches the scale.
__device__ __forceinline__ float max_or_nan(float a, float b) {
    float m;
    asm("max.NaN.f32 %0, %1, %2;\n" : "=f"(m) : "f"(a), "f"(b));
    return m;
}
// A block's amax: 16 neighbouring lanes hold its 128 channels, and every lane of the warp
// takes part.
__device__ __forceinline__ float block_amax(const float (&y)[8]) {
    float m = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max_or_nan(m, fabsf(y[j]));
#pragma unroll
    for (int o = 8; o; o >>= 1) m = max_or_nan(m, __shfl_xor_sync(~0u, m, o));
    return m;
}
// A row's 1 / rms cancels in y / scale, so q goes out before the row's sum is known:
// q = e4m3(h w 448 / amax|h w|).  Returns amax|h w|, from which put_scales makes the scale.
template <typename T, bool FULL>
__device__ __forceinline__ float put_group(const NormArgs &a, long long row, int c, const float (&h)[8],
                                           const Group<T, FULL> &w) {
    float y[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = h[j] * to_f32(w.e[j]);
    const float amax = block_amax(y);
    put_q<FULL>(a, row, c, a.dim - c, y, kE4m3Max * reciprocal(amax));
    return amax;
}
template <typename T, int TPR, int NV, bool FULL>
__device__ __forceinline__ void put_scales(const NormArgs &a, long long row, int t, const float (&h)[NV][8],
                                           const Group<T, FULL> (&w)[NV], const float (&amax)[NV], float rstd) {
    // A block under the floor, or whose products or quotients may have left the range, is done
    // again in the order of the formula.
    bool redo = false;
#pragma unroll
    for (int i = 0; i < NV; ++i)
        redo |= (t + i * TPR) * 8 < a.dim && !(amax[i] * rstd >= kAmaxFloor && amax[i] > kSafeLow && amax[i] < kSafeHigh);
    if (!__any_sync(~0u, redo)) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (t + i * TPR) * 8;
            if ((t & 15) == 0 && c < a.dim)
                a.scale[row * a.scale_row + (c >> 7) * a.scale_group] = amax[i] * rstd * (1.f / kE4m3Max);
        }
        return;
    }
#pragma unroll 1
    for (int i = 0; i < NV; ++i) {
        const int c = (t + i * TPR) * 8;
        float y[8];
#pragma unroll
        for (int k = 0; k < NV; ++k)
            if (k == i)
#pragma unroll
                for (int j = 0; j < 8; ++j) y[j] = h[k][j] * rstd * to_f32(w[k].e[j]);
        const float top = max_or_nan(block_amax(y), kAmaxFloor);
        put_q<FULL>(a, row, c, a.dim - c, y, kE4m3Max / top);
        if ((t & 15) == 0 && c < a.dim) a.scale[row * a.scale_row + (c >> 7) * a.scale_group] = top * (1.f / kE4m3Max);
    }
}

// One row for each group of TPR threads: a CTA of it, or (TPR = 32) warps that take a row
// after another and load the next while they work on one.
template <typename T, int TPR, int NV, bool RES, bool FULL>
__global__ void __launch_bounds__(TPR == 32 ? 256 : TPR) norm_kernel(const __grid_constant__ NormArgs a) {
    griddep_wait();
    griddep_launch();
    const int t = TPR == 32 ? threadIdx.x & 31 : threadIdx.x;
    const long long step = TPR == 32 ? gridDim.x * 8ll : gridDim.x;
    long long row = TPR == 32 ? blockIdx.x * 8ll + (threadIdx.x >> 5) : blockIdx.x;
    Group<T, FULL> x[NV], r[RES ? NV : 1], w[NV];
    auto fetch = [&](long long k) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (t + i * TPR) * 8;
            x[i].load((const T *)a.x + k * a.x_stride + c, a.dim - c);
            if (RES) r[i].load((const T *)a.res + k * a.res_stride + c, a.dim - c);
        }
    };
    if (row < a.rows) fetch(row);
#pragma unroll
    for (int i = 0; i < NV; ++i) w[i].load((const T *)a.w + (t + i * TPR) * 8, a.dim - (t + i * TPR) * 8);
    for (; row < a.rows; row += step) {  // once, where TPR > 32
        float h[NV][8], amax[NV], ss = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                h[i][j] = to_f32(x[i].e[j]);
                if (RES) h[i][j] += to_f32(r[i].e[j]);
            }
        if (TPR == 32 && row + step < a.rows) fetch(row + step);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (t + i * TPR) * 8;
            if (RES) {
                Group<T, FULL> o;
#pragma unroll
                for (int j = 0; j < 8; ++j) o.e[j] = from_f32<T>(h[i][j]);
                o.store((T *)a.res_out + row * a.res_out_stride + c, a.dim - c);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) ss += h[i][j] * h[i][j];
            amax[i] = put_group(a, row, c, h[i], w[i]);
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(~0u, ss, o);
        if (TPR > 32) {
            __shared__ float part[32];
            if ((t & 31) == 0) part[t >> 5] = ss;
            __syncthreads();
            ss = 0.f;
#pragma unroll
            for (int i = 0; i < TPR / 32; ++i) ss += part[i];
        }
        put_scales<T, TPR, NV, FULL>(a, row, t, h, w, amax, rsqrtf(ss / (float)a.dim + a.eps));
        if (TPR > 32) break;
    }
}

// Many long rows: CTAs that stay, rows copied ahead into a ring in shared memory by the bulk
// copy engine, so that loads are on the way while a row is reduced and written (one CTA a row
// leaves the memory idle between its phases: 16384 x 8192 bf16 took 194 us that way, 222 with
// 256 threads).  Everyone has read a stage by the barrier of its row's reduction, after which
// one thread refills it.
constexpr int MAX_STAGES = 8;

template <typename T, int THREADS, int NV, bool RES>
__global__ void __launch_bounds__(THREADS) norm_ring_kernel(const __grid_constant__ NormArgs a, int stages,
                                                            int stage_bytes, int row_bytes, uint32_t expect,
                                                            int *err) {
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint64_t full[MAX_STAGES];
    __shared__ float part[2][THREADS / 32];
    __shared__ volatile int stop;
    const int t = threadIdx.x;
    if (t == 0) {
        stop = 0;
        for (int i = 0; i < stages; ++i) tc05::mbar_init(&full[i], 1);
        tc05::fence_mbar_init();
    }
    __syncthreads();
    griddep_wait();
    griddep_launch();
    const int mine = (a.rows - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x;  // rows of this CTA
    auto fetch = [&](int i, int s) {
        const long long row = blockIdx.x + (long long)i * gridDim.x;
        const uint32_t dst = tc05::smem_u32(smem + s * stage_bytes);
        mbar_expect(&full[s], expect);  // what is copied here
        bulk_copy(dst, (const T *)a.x + row * a.x_stride, row_bytes, &full[s]);
        if (RES) bulk_copy(dst + stage_bytes / 2, (const T *)a.res + row * a.res_stride, row_bytes, &full[s]);
    };
    if (t == 0)
        for (int i = 0; i < min(stages, mine); ++i) fetch(i, i);
    Group<T, true> w[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) w[i].load((const T *)a.w + (t + i * THREADS) * 8, a.dim - (t + i * THREADS) * 8);

    int s = 0, phase = 0;
    for (int k = 0; k < mine; ++k) {
        const long long row = blockIdx.x + (long long)k * gridDim.x;
        const T *x = (const T *)(smem + s * stage_bytes), *res = (const T *)(smem + s * stage_bytes + stage_bytes / 2);
        if (!tc05::mbar_wait(&full[s], phase, WAIT_ITERS)) stop = 1;
        float h[NV][8], amax[NV], ss = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (t + i * THREADS) * 8, n = a.dim - c;
            Group<T, true> g;
            g.load(x + c, n);
#pragma unroll
            for (int j = 0; j < 8; ++j) h[i][j] = to_f32(g.e[j]);
            if (RES) {
                g.load(res + c, n);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    h[i][j] += to_f32(g.e[j]);
                    g.e[j] = from_f32<T>(h[i][j]);
                }
                g.store((T *)a.res_out + row * a.res_out_stride + c, n);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) ss += h[i][j] * h[i][j];
            amax[i] = put_group(a, row, c, h[i], w[i]);
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(~0u, ss, o);
        if ((t & 31) == 0) part[k & 1][t >> 5] = ss;
        __syncthreads();
        if (stop) {  // a copy that does not come: report it, and leave when the others are in
            if (t == 0) {
                atomicOr(err, HV_DECODE_STALLED);
                for (int i = k; i < min(k + stages, mine); ++i) tc05::mbar_wait(&full[i % stages], (i / stages) & 1, DRAIN_ITERS);
            }
            break;
        }
        if (t == 0 && k + stages < mine) fetch(k + stages, s);
        if (++s == stages) {
            s = 0;
            phase ^= 1;
        }
        ss = 0.f;
#pragma unroll
        for (int i = 0; i < THREADS / 32; ++i) ss += part[k & 1][i];
        put_scales<T, THREADS, NV, true>(a, row, t, h, w, amax, rsqrtf(ss / (float)a.dim + a.eps));
    }
}

template <typename T, int TPR, int NV>
cudaError_t launch(const NormArgs &a, int sms, cudaStream_t st) {
    const int warps_grid = (int)std::min<long long>((a.rows + 7ll) / 8, (long long)sms * (NV == 1 ? 5 : NV == 2 ? 4 : 2));
    const dim3 grid((unsigned)(TPR == 32 ? warps_grid : a.rows)), block(TPR == 32 ? 256 : TPR);
    if (a.full)
        return a.res ? launch_pdl(norm_kernel<T, TPR, NV, true, true>, grid, block, 0, st, a)
                     : launch_pdl(norm_kernel<T, TPR, NV, false, true>, grid, block, 0, st, a);
    return a.res ? launch_pdl(norm_kernel<T, TPR, NV, true, false>, grid, block, 0, st, a)
                 : launch_pdl(norm_kernel<T, TPR, NV, false, false>, grid, block, 0, st, a);
}

// CTAs of an SM and stages of a ring: enough threads to keep up (16-bit rows with a residual
// 512 an SM, without one twice as many, float32 half of those, but one CTA at least: float32 rows of
// over 4096 channels have 512), and 64 KB ahead an SM (128 where one CTA has it): 32768 x 2048 bf16 took 72 us with 64 KB, 83 with 96 and 94 with 128.
template <typename T, int THREADS, int NV>
cudaError_t launch_ring(const NormArgs &a, int sms, int row_bytes, int *err, cudaStream_t st) {
    const auto kernel = a.res ? norm_ring_kernel<T, THREADS, NV, true> : norm_ring_kernel<T, THREADS, NV, false>;
    const int stage = (row_bytes + 127) / 128 * 128 * (a.res ? 2 : 1);
    const int per_sm = std::max(1, (a.res ? 512 : 1024) * 2 / (int)sizeof(T) / THREADS);
    const int ahead = (per_sm > 1 ? 64 : 128) * 1024 / (per_sm * stage);
    const int stages = std::max(2, std::min(MAX_STAGES, ahead)), smem = stages * stage;
    // with hv_test_decode_stall 16 bytes more, which do not come (a test in the kernel for a row to leave
    // out took 1.5% of 16384 x 8192)
    const uint32_t expect = row_bytes * (a.res ? 2 : 1) + (skipped_copy() == NO_COPY ? 0 : 16);
    static std::atomic<uint64_t> ready[2];
    const cudaError_t e = allow_shared(kernel, ready[a.res != nullptr]);
    if (e != cudaSuccess) return e;
    return launch_pdl(kernel, dim3((unsigned)std::min(a.rows, sms * per_sm)), dim3(THREADS), smem, st, a, stages, stage,
                      row_bytes, expect, err);
}

template <typename T>
cudaError_t by_dim(const NormArgs &a, int sms, int *err, cudaStream_t st) {
    const int d = a.dim;
    if (d <= 256) return launch<T, 32, 1>(a, sms, st);
    if (d <= 512) return launch<T, 32, 2>(a, sms, st);
    if (d <= 1024) return launch<T, 32, 4>(a, sms, st);
    // The ring wants whole 16-byte pieces, room for two stages, and some rows for each CTA.
    const int bytes = d * (int)sizeof(T);
    if (a.full && bytes % 16 == 0 && d <= 16384 && a.rows >= 4 * sms && 2 * (a.res ? 2 : 1) * (bytes + 127) <= 222 * 1024) {
        if (d <= 2048) return launch_ring<T, 128, 2>(a, sms, bytes, err, st);
        if (d <= 4096) return launch_ring<T, 256, 2>(a, sms, bytes, err, st);
        if (d <= 8192) return launch_ring<T, 512, 2>(a, sms, bytes, err, st);
        return launch_ring<T, 512, 4>(a, sms, bytes, err, st);
    }
    if (d <= 2048) return launch<T, 128, 2>(a, sms, st);
    if (d <= 4096) return launch<T, 256, 2>(a, sms, st);
    if (d <= 8192) return launch<T, 512, 2>(a, sms, st);
    if (d <= 16384) return launch<T, 512, 4>(a, sms, st);
    return launch<T, 1024, 4>(a, sms, st);
}

}  // namespace
}  // namespace hv

using namespace hv;

extern "C" int hv_add_rmsnorm_fp8(const hv_norm_args *p, void *stream) {
    if (!p) return fail(HV_ERR_VALUE, "null argument");
    if (!dec::known_dtype(p->dtype)) return fail(HV_ERR_TYPE, "dtype must be HV_BF16, HV_F16 or HV_F32");
    if (p->rows < 0 || p->rows > INT32_MAX) return fail(HV_ERR_VALUE, "rows outside [0, 2^31)");
    if (p->dim < 1 || p->dim > 32768) return fail(HV_ERR_VALUE, "dim outside [1, 32768]");
    if (!(p->eps >= 0.f)) return fail(HV_ERR_VALUE, "eps must not be negative");
    if (!p->d_residual != !p->d_residual_out)
        return fail(HV_ERR_VALUE, "residual and residual_out are given together or not at all");
    if (p->rows == 0) return HV_OK;
    if (!p->d_x || !p->d_weight || !p->d_q || !p->d_scale) return fail(HV_ERR_VALUE, "null buffer");
    NormArgs a{p->d_x, p->d_residual, p->d_weight, p->d_residual_out, (uint8_t *)p->d_q, p->d_scale, p->x_stride,
               p->residual_stride, p->residual_out_stride, p->q_stride, p->scale_strides[0], p->scale_strides[1],
               (int)p->rows, p->dim, 0, p->eps};
    const int es = dec::elem_size(p->dtype);
    auto wide = [&](const void *b, int64_t stride) {
        return dec::aligned(b, 16) && (p->rows == 1 || stride * es % 16 == 0);
    };
    a.full = p->dim % 8 == 0 && wide(a.x, a.x_stride) && dec::aligned(a.w, 16) &&
             (!a.res || (wide(a.res, a.res_stride) && wide(a.res_out, a.res_out_stride))) && dec::aligned(a.q, 8) &&
             (p->rows == 1 || a.q_stride % 8 == 0);
    int *err = dec::error_word();
    const int sms = dec::sm_count();
    if (!err || !sms) return fail(HV_ERR_CUDA, "cannot read the device's properties");
    const cudaStream_t st = (cudaStream_t)stream;
    const cudaError_t e = p->dtype == HV_BF16  ? by_dim<__nv_bfloat16>(a, sms, err, st)
                          : p->dtype == HV_F16 ? by_dim<__half>(a, sms, err, st)
                                               : by_dim<float>(a, sms, err, st);
    if (e != cudaSuccess) return fail(HV_ERR_CUDA, "add_rmsnorm_fp8: %s", cudaGetErrorString(e));
    return HV_OK;
}
