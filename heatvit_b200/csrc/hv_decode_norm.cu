// hv_decode_norm.cu — residual addition, root-mean-square norm and e4m3 output in one pass.
//
//   h = x + residual                         (32 bits; its rounding to T is residual_out)
//   y = h * rsqrt(mean(h^2) + eps) * weight
//   scale = max(amax |y|, 2^-100) / 448 over each 128 channels, q = e4m3(y / scale)
//
// The norm is taken of the unrounded sum: residual_out is one rounding of h, q one
// rounding of y.  The floor keeps the scale of an all-zero block a normal number.
//
// Bound by HBM: x, residual, residual_out and q cross it once each (7 bytes an element
// in bf16), so a row stays in registers between the sum of squares and the output.  A
// thread holds NV groups of eight consecutive channels, TPR threads apart: 16-byte
// accesses, and a block of 128 channels is 16 neighbouring lanes, whose amax is four
// shuffles.  Rows of up to 1024 channels take a warp each, longer ones a CTA.
#include <cuda_fp8.h>

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
    int rows, dim, vec, q8;
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

// Group `c / 8` of a row's output: eight channels of a thread, `n` of which exist; 16
// neighbouring lanes hold a block of 128.  Every lane of the warp takes part.
__device__ __forceinline__ void put_group(const NormArgs &a, long long row, int c, int n, const float (&h)[8],
                                          const float (&w)[8], float rstd) {
    float y[8], amax = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        y[j] = h[j] * rstd * w[j];
        amax = fmaxf(amax, fabsf(y[j]));
    }
#pragma unroll
    for (int o = 8; o; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(~0u, amax, o));
    amax = fmaxf(amax, kAmaxFloor);
    if (n <= 0) return;
    if ((c & 127) == 0) a.scale[row * a.scale_row + (long long)(c >> 7) * a.scale_group] = amax / kE4m3Max;
    const float inv = kE4m3Max / amax;
    uint32_t b[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(y[4 * j] * inv, y[4 * j + 1] * inv), __NV_SATFINITE,
                                                     __NV_E4M3);
        const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(y[4 * j + 2] * inv, y[4 * j + 3] * inv),
                                                     __NV_SATFINITE, __NV_E4M3);
        b[j] = lo | hi << 16;
    }
    uint8_t *q = a.q + row * a.q_stride + c;
    if (a.q8 && n >= 8) {
        *(uint2 *)q = make_uint2(b[0], b[1]);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < n) q[j] = (uint8_t)(b[j >> 2] >> (8 * (j & 3)));
    }
}

// One CTA a row, or (TPR = 32) one warp for RPW rows, whose loads are issued together.
template <typename T, int TPR, int NV, int RPW, bool RES>
__global__ void __launch_bounds__(TPR == 32 ? 256 : TPR) norm_kernel(const NormArgs a) {
    griddep_wait();
    griddep_launch();
    static_assert(TPR == 32 || RPW == 1, "a CTA's barrier is for one row");
    const int t = TPR == 32 ? threadIdx.x & 31 : threadIdx.x;
    const long long row0 = TPR == 32 ? ((long long)blockIdx.x * 8 + (threadIdx.x >> 5)) * RPW : blockIdx.x;
    if (row0 >= a.rows) return;  // whole warps, or none of a one-row CTA
    float h[RPW][NV][8], ss[RPW];
#pragma unroll
    for (int k = 0; k < RPW; ++k) {
        const long long row = min(row0 + k, (long long)a.rows - 1);
        const T *x = (const T *)a.x + row * a.x_stride;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (t + i * TPR) * 8;
            load8(x + c, a.dim - c, a.vec, h[k][i]);
        }
    }
    if (RES) {
#pragma unroll
        for (int k = 0; k < RPW; ++k) {
            const long long row = min(row0 + k, (long long)a.rows - 1);
            const T *res = (const T *)a.res + row * a.res_stride;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = (t + i * TPR) * 8;
                float r[8];
                load8(res + c, a.dim - c, a.vec, r);
#pragma unroll
                for (int j = 0; j < 8; ++j) h[k][i][j] += r[j];
            }
        }
    }
#pragma unroll
    for (int k = 0; k < RPW; ++k) {
        ss[k] = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (t + i * TPR) * 8;
            if (RES && row0 + k < a.rows)
                store8((T *)a.res_out + (row0 + k) * a.res_out_stride + c, a.dim - c, a.vec, h[k][i]);
#pragma unroll
            for (int j = 0; j < 8; ++j) ss[k] += h[k][i][j] * h[k][i][j];
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) ss[k] += __shfl_xor_sync(~0u, ss[k], o);
    }
    if (TPR > 32) {
        __shared__ float part[32];
        if ((t & 31) == 0) part[t >> 5] = ss[0];
        __syncthreads();
        ss[0] = 0.f;
#pragma unroll
        for (int i = 0; i < TPR / 32; ++i) ss[0] += part[i];
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (t + i * TPR) * 8;
        float w[8];
        load8((const T *)a.w + c, a.dim - c, a.vec, w);
#pragma unroll
        for (int k = 0; k < RPW; ++k)
            put_group(a, row0 + k, c, row0 + k < a.rows ? a.dim - c : 0, h[k][i], w,
                      rsqrtf(ss[k] / (float)a.dim + a.eps));
    }
}

// Many long rows: CTAs that stay, rows copied ahead into a ring in shared memory by the bulk
// copy engine, so that loads are on the way while a row is reduced and written (one CTA a row
// leaves the memory idle between its phases).  Everyone has read a stage by the barrier of its
// row's reduction, after which one thread refills it.
constexpr int RING_THREADS = 256, MAX_STAGES = 4;
constexpr uint32_t RING_WAIT = 1u << 22;

template <typename T, int NV, bool RES>
__global__ void __launch_bounds__(RING_THREADS) norm_ring_kernel(const NormArgs a, int stages, int stage_bytes,
                                                                 int row_bytes, int *err) {
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint64_t full[MAX_STAGES];
    __shared__ float part[2][RING_THREADS / 32];
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
    auto fetch = [&](int i) {
        const long long row = blockIdx.x + (long long)i * gridDim.x;
        const uint32_t dst = tc05::smem_u32(smem + (i % stages) * stage_bytes);
        uint64_t *bar = &full[i % stages];
        mbar_expect(bar, RES ? 2 * row_bytes : row_bytes);
        bulk_copy(dst, (const T *)a.x + row * a.x_stride, row_bytes, bar);
        if (RES) bulk_copy(dst + stage_bytes / 2, (const T *)a.res + row * a.res_stride, row_bytes, bar);
    };
    if (t == 0)
        for (int i = 0; i < min(stages, mine); ++i) fetch(i);
    float w[NV][8];
#pragma unroll
    for (int i = 0; i < NV; ++i) load8((const T *)a.w + (t + i * RING_THREADS) * 8, a.dim - (t + i * RING_THREADS) * 8, true, w[i]);

    for (int k = 0; k < mine; ++k) {
        const long long row = blockIdx.x + (long long)k * gridDim.x;
        const T *x = (const T *)(smem + (k % stages) * stage_bytes);
        const T *res = (const T *)(smem + (k % stages) * stage_bytes + stage_bytes / 2);
        if (!tc05::mbar_wait(&full[k % stages], (k / stages) & 1, RING_WAIT)) stop = 1;
        float h[NV][8], ss = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (t + i * RING_THREADS) * 8, n = a.dim - c;
            load8(x + c, n, true, h[i]);
            if (RES) {
                float r[8];
                load8(res + c, n, true, r);
#pragma unroll
                for (int j = 0; j < 8; ++j) h[i][j] += r[j];
                store8((T *)a.res_out + row * a.res_out_stride + c, n, true, h[i]);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) ss += h[i][j] * h[i][j];
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(~0u, ss, o);
        if ((t & 31) == 0) part[k & 1][t >> 5] = ss;
        __syncthreads();
        if (stop) {  // a copy that does not come: report it, and leave when the others are in
            if (t == 0) {
                atomicOr(err, HV_DECODE_STALLED);
                for (int i = k; i < min(k + stages, mine); ++i) tc05::mbar_wait(&full[i % stages], (i / stages) & 1, RING_WAIT);
            }
            break;
        }
        if (t == 0 && k + stages < mine) fetch(k + stages);
        ss = 0.f;
#pragma unroll
        for (int i = 0; i < RING_THREADS / 32; ++i) ss += part[k & 1][i];
        const float rstd = rsqrtf(ss / (float)a.dim + a.eps);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (t + i * RING_THREADS) * 8;
            put_group(a, row, c, a.dim - c, h[i], w[i], rstd);
        }
    }
}

template <typename T, int TPR, int NV, int RPW = 1>
cudaError_t launch(const NormArgs &a, cudaStream_t st) {
    const dim3 grid((unsigned)(TPR == 32 ? (a.rows + 8ll * RPW - 1) / (8 * RPW) : a.rows)), block(TPR == 32 ? 256 : TPR);
    return a.res ? launch_pdl(norm_kernel<T, TPR, NV, RPW, true>, grid, block, 0, st, a)
                 : launch_pdl(norm_kernel<T, TPR, NV, RPW, false>, grid, block, 0, st, a);
}

template <typename T, int NV>
cudaError_t launch_ring(const NormArgs &a, int sms, int per_sm, int stages, int stage_bytes, int *err, cudaStream_t st) {
    const auto kernel = a.res ? norm_ring_kernel<T, NV, true> : norm_ring_kernel<T, NV, false>;
    const int smem = stages * stage_bytes;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    const int grid = min(a.rows, sms * per_sm);
    return launch_pdl(kernel, dim3((unsigned)grid), dim3(RING_THREADS), smem, st, a, stages, stage_bytes,
                      a.dim * (int)sizeof(T), err);
}

template <typename T>
cudaError_t by_dim(const NormArgs &a, int sms, int *err, cudaStream_t st) {
    const int d = a.dim;
    if (d <= 256) return launch<T, 32, 1, 4>(a, st);
    if (d <= 512) return launch<T, 32, 2, 2>(a, st);
    if (d <= 1024) return launch<T, 32, 4>(a, st);
    // The ring wants whole 16-byte pieces, at least two stages, and some rows for each CTA.
    const int bytes = (d * (int)sizeof(T) + 127) / 128 * 128 * (a.res ? 2 : 1);
    if (a.vec && d * sizeof(T) % 16 == 0 && d <= 16384 && a.rows >= 4 * sms && 2 * bytes <= 220 * 1024) {
        const int per_sm = 2 * bytes <= 110 * 1024 ? 2 : 1;
        const int stages = min(MAX_STAGES, (per_sm == 2 ? 110 : 220) * 1024 / bytes);
        if (d <= 2048) return launch_ring<T, 1>(a, sms, per_sm, stages, bytes, err, st);
        if (d <= 4096) return launch_ring<T, 2>(a, sms, per_sm, stages, bytes, err, st);
        if (d <= 8192) return launch_ring<T, 4>(a, sms, per_sm, stages, bytes, err, st);
        return launch_ring<T, 8>(a, sms, per_sm, stages, bytes, err, st);
    }
    if (d <= 2048) return launch<T, 128, 2>(a, st);
    if (d <= 4096) return launch<T, 256, 2>(a, st);
    if (d <= 8192) return launch<T, 512, 2>(a, st);
    if (d <= 16384) return launch<T, 512, 4>(a, st);
    return launch<T, 1024, 4>(a, st);
}

}  // namespace
}  // namespace hv

using namespace hv;

extern "C" int hv_add_rmsnorm_fp8(const void *d_x, int64_t x_stride, const void *d_residual, int64_t residual_stride,
                                  const void *d_weight, int64_t rows, int dim, int dtype, float eps,
                                  void *d_residual_out, int64_t residual_out_stride, void *d_q, int64_t q_stride,
                                  float *d_scale, int64_t scale_row_stride, int64_t scale_group_stride,
                                  void *stream) {
    if (!dec::known_dtype(dtype)) return fail(HV_ERR_TYPE, "dtype must be HV_BF16, HV_F16 or HV_F32");
    if (rows < 0 || rows > INT32_MAX) return fail(HV_ERR_VALUE, "rows outside [0, 2^31)");
    if (dim < 1 || dim > 32768) return fail(HV_ERR_VALUE, "dim outside [1, 32768]");
    if (rows == 0) return HV_OK;
    if (!d_x || !d_weight || !d_q || !d_scale) return fail(HV_ERR_VALUE, "null buffer");
    if (!d_residual != !d_residual_out)
        return fail(HV_ERR_VALUE, "residual and residual_out are given together or not at all");
    if (!(eps >= 0.f)) return fail(HV_ERR_VALUE, "eps must not be negative");
    NormArgs a{d_x, d_residual, d_weight, d_residual_out, (uint8_t *)d_q, d_scale, x_stride, residual_stride,
               residual_out_stride, q_stride, scale_row_stride, scale_group_stride, (int)rows, dim, 1, 0, eps};
    const int es = dec::elem_size(dtype);
    auto wide = [&](const void *p, int64_t stride) {
        return dec::aligned(p, 16) && (rows == 1 || stride * es % 16 == 0);
    };
    a.vec = wide(d_x, x_stride) && dec::aligned(d_weight, 16) &&
            (!d_residual || (wide(d_residual, residual_stride) && wide(d_residual_out, residual_out_stride)));
    a.q8 = dec::aligned(d_q, 8) && (rows == 1 || q_stride % 8 == 0);
    int *err = dec::error_word();
    const int sms = dec::sm_count();
    if (!err || !sms) return fail(HV_ERR_CUDA, "cannot read the device's properties");
    const cudaStream_t st = (cudaStream_t)stream;
    const cudaError_t e = dtype == HV_BF16  ? by_dim<__nv_bfloat16>(a, sms, err, st)
                          : dtype == HV_F16 ? by_dim<__half>(a, sms, err, st)
                                            : by_dim<float>(a, sms, err, st);
    if (e != cudaSuccess) return fail(HV_ERR_CUDA, "add_rmsnorm_fp8: %s", cudaGetErrorString(e));
    return HV_OK;
}
