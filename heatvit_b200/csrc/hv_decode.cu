// hv_decode.cu — the decode operators' device error word and device properties.
#include <atomic>

#include "hv_decode.cuh"

namespace hv {
namespace {

__device__ int g_decode_error;

constexpr int MAX_DEVICES = 64;
std::atomic<int *> g_address[MAX_DEVICES];
std::atomic<int> g_sms[MAX_DEVICES];
std::atomic<uint32_t> g_skip{dec::NO_COPY};

}  // namespace

namespace dec {

int *error_word() {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= MAX_DEVICES) return nullptr;
    int *p = g_address[dev].load(std::memory_order_acquire);
    if (!p) {
        void *v = nullptr;
        if (cudaGetSymbolAddress(&v, g_decode_error) != cudaSuccess) return nullptr;
        p = (int *)v;
        g_address[dev].store(p, std::memory_order_release);
    }
    return p;
}

int sm_count() {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= MAX_DEVICES) return 0;
    int n = g_sms[dev].load(std::memory_order_relaxed);
    if (!n) {
        if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
        g_sms[dev].store(n, std::memory_order_relaxed);
    }
    return n;
}

uint32_t skipped_copy() { return g_skip.load(std::memory_order_relaxed); }

}  // namespace dec
}  // namespace hv

extern "C" int hv_test_decode_stall(int skip_copy) {
    using namespace hv;
    if (skip_copy < -1) return fail(HV_ERR_VALUE, "skip_copy must be -1 (none) or a copy's number");
    g_skip.store(skip_copy < 0 ? dec::NO_COPY : (uint32_t)skip_copy, std::memory_order_relaxed);
    return HV_OK;
}

extern "C" int hv_decode_error(int *bits) {
    using namespace hv;
    if (!bits) return fail(HV_ERR_VALUE, "null argument");
    int *p = dec::error_word();
    if (!p) return fail(HV_ERR_CUDA, "cannot resolve the device error word");
    const int zero = 0;
    cudaError_t e = cudaDeviceSynchronize();
    if (e == cudaSuccess) e = cudaMemcpy(bits, p, sizeof(int), cudaMemcpyDeviceToHost);
    if (e == cudaSuccess && *bits) e = cudaMemcpy(p, &zero, sizeof(int), cudaMemcpyHostToDevice);
    if (e != cudaSuccess) return fail(HV_ERR_CUDA, "decode error word: %s", cudaGetErrorString(e));
    return HV_OK;
}
