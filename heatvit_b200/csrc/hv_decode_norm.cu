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

constexpr float kE4m3Max = 448.f;
constexpr float kAmaxFloor = 7.888609052210118e-31f;  // 2^-100

template <typename T, int TPR, int NV, bool RES>
__global__ void __launch_bounds__(TPR == 32 ? 256 : TPR) norm_kernel(const NormArgs a) {
    griddep_wait();
    griddep_launch();
    constexpr int RPC = TPR == 32 ? 8 : 1;  // rows of a CTA
    const int t = TPR == 32 ? threadIdx.x & 31 : threadIdx.x;
    const int row = blockIdx.x * RPC + (TPR == 32 ? threadIdx.x >> 5 : 0);
    if (row >= a.rows) return;  // whole warps, or none of a one-row CTA
    const T *x = (const T *)a.x + (long long)row * a.x_stride;
    const T *res = RES ? (const T *)a.res + (long long)row * a.res_stride : nullptr;
    T *ro = RES ? (T *)a.res_out + (long long)row * a.res_out_stride : nullptr;

    float h[NV][8];
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (t + i * TPR) * 8, n = a.dim - c;
        load8(x + c, n, a.vec, h[i]);
        if (RES) {
            float r[8];
            load8(res + c, n, a.vec, r);
#pragma unroll
            for (int j = 0; j < 8; ++j) h[i][j] += r[j];
        }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (t + i * TPR) * 8;
        if (RES) store8(ro + c, a.dim - c, a.vec, h[i]);
#pragma unroll
        for (int j = 0; j < 8; ++j) ss += h[i][j] * h[i][j];
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
    const float rstd = rsqrtf(ss / (float)a.dim + a.eps);

#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (t + i * TPR) * 8, n = a.dim - c;
        float w[8], y[8], amax = 0.f;
        load8((const T *)a.w + c, n, a.vec, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            y[j] = h[i][j] * rstd * w[j];
            amax = fmaxf(amax, fabsf(y[j]));
        }
#pragma unroll
        for (int o = 8; o; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(~0u, amax, o));
        amax = fmaxf(amax, kAmaxFloor);
        if (n <= 0) continue;
        if ((t & 15) == 0)
            a.scale[(long long)row * a.scale_row + (long long)(c >> 7) * a.scale_group] = amax / kE4m3Max;
        const float inv = kE4m3Max / amax;
        uint32_t b[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(y[4 * j] * inv, y[4 * j + 1] * inv),
                                                         __NV_SATFINITE, __NV_E4M3);
            const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(y[4 * j + 2] * inv, y[4 * j + 3] * inv),
                                                         __NV_SATFINITE, __NV_E4M3);
            b[j] = lo | hi << 16;
        }
        uint8_t *q = a.q + (long long)row * a.q_stride + c;
        if (a.q8 && n >= 8) {
            *(uint2 *)q = make_uint2(b[0], b[1]);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (j < n) q[j] = (uint8_t)(b[j >> 2] >> (8 * (j & 3)));
        }
    }
}

template <typename T, int TPR, int NV>
cudaError_t launch(const NormArgs &a, cudaStream_t st) {
    const dim3 grid((unsigned)(TPR == 32 ? (a.rows + 7) / 8 : a.rows)), block(TPR == 32 ? 256 : TPR);
    return a.res ? launch_pdl(norm_kernel<T, TPR, NV, true>, grid, block, 0, st, a)
                 : launch_pdl(norm_kernel<T, TPR, NV, false>, grid, block, 0, st, a);
}

template <typename T>
cudaError_t by_dim(const NormArgs &a, cudaStream_t st) {
    const int d = a.dim;
    if (d <= 256) return launch<T, 32, 1>(a, st);
    if (d <= 512) return launch<T, 32, 2>(a, st);
    if (d <= 1024) return launch<T, 32, 4>(a, st);
    if (d <= 2048) return launch<T, 128, 2>(a, st);
    if (d <= 4096) return launch<T, 256, 2>(a, st);
    if (d <= 8192) return launch<T, 256, 4>(a, st);
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
    cudaError_t e;
    if (dtype == HV_BF16) e = by_dim<__nv_bfloat16>(a, (cudaStream_t)stream);
    else if (dtype == HV_F16) e = by_dim<__half>(a, (cudaStream_t)stream);
    else e = by_dim<float>(a, (cudaStream_t)stream);
    if (e != cudaSuccess) return fail(HV_ERR_CUDA, "add_rmsnorm_fp8: %s", cudaGetErrorString(e));
    return HV_OK;
}
