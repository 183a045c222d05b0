// hv_decode.cuh — what the decode operators (norm, e4m3 GEMM, cache append, paged
// attention) share: element types, their 32-bit conversions, and the device error word.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "hv_internal.cuh"
#include "hv_launch.cuh"

namespace hv {
namespace dec {

// Device word that the decode kernels OR HV_DECODE_* bits into (hv_decode_error reads
// and clears it); null when its address cannot be resolved.
int *error_word();
// SMs of the current device; 0 when that cannot be read.
int sm_count();

// Polls of an mbarrier before a wait gives up: a poll takes 4 us where bytes of a copy are missing and 24 ns
// where nobody has arrived, so 1 s and 6 ms (2^22 polls held the GPU for 17 s).  Then, before memory goes,
// for what is under way, which has had that long already.
constexpr uint32_t WAIT_ITERS = 1u << 18, DRAIN_ITERS = 1u << 14;
// The copy that each CTA leaves out: NO_COPY unless hv_test_decode_stall asked for one.
constexpr uint32_t NO_COPY = UINT32_MAX;
uint32_t skipped_copy();

// Lets `kernel` have all of an SM's shared memory, once a device: `ready` has a bit for each.
template <typename K>
cudaError_t allow_shared(K kernel, std::atomic<uint64_t> &ready) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess || (dev < 64 && ready.load(std::memory_order_relaxed) >> dev & 1)) return e;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024 - 512);
    if (e == cudaSuccess && dev < 64) ready.fetch_or(1ull << dev, std::memory_order_relaxed);
    return e;
}

inline int elem_size(int dtype) { return dtype == HV_F32 ? 4 : 2; }
inline bool known_dtype(int dtype) { return dtype == HV_BF16 || dtype == HV_F16 || dtype == HV_F32; }
inline bool aligned(const void *p, size_t n) { return (uintptr_t)p % n == 0; }

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

}  // namespace dec
}  // namespace hv
