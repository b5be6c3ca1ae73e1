// Host-side helpers shared by the library's translation units.
#pragma once

#include <cuda_runtime.h>

#include <atomic>
#include <cstddef>
#include <cstdint>

#include "swiglu_b200.h"

namespace swb {

// Shared-memory capacities of sm_100: 228 KB per SM, 227 KB opt-in per CTA,
// 1 KB reserved per resident CTA.
constexpr size_t kSmemPerSm = 233472;
constexpr size_t kSmemPerCtaMax = 232448;

// Records `status`'s message (and `detail`) for swb_last_error and returns it.
int fail(int status, const char* detail = nullptr);
// SWB_OK, or the pending CUDA error as SWB_E_CUDA.
int check_launch();
// SMs of the current device, -1 on a CUDA error.
int sm_count();
// Whether every address is a multiple of `bytes` (null is).
template <typename... P>
bool aligned(size_t bytes, P... p) {
    return ((reinterpret_cast<uintptr_t>(p) | ... | uintptr_t(0)) & (bytes - 1)) == 0;
}
bool overlaps(const void* a, size_t abytes, const void* b, size_t bbytes);

// Device error words of the other translation units (each holds its own).
int moe_device_error(int clear, int* out);
int mx4_matmul_device_error(int clear, int* out);
int mx4_wide_device_error(int clear, int* out);
int moe_wide_device_error(int clear, int* out);
int mx4_deep_device_error(int clear, int* out);

// Launches an attribute-carrying kernel; the returned error is the launch's own.
template <typename... Args>
int launch_ex(void (*kernel)(Args...), unsigned grid, unsigned block, size_t smem, cudaStream_t stream,
              bool cooperative, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeCooperative;
    attr[0].val.cooperative = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cooperative ? 1 : 0;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
    if (e != cudaSuccess) {
        (void)cudaGetLastError();
        return fail(SWB_E_CUDA, cudaGetErrorString(e));
    }
    return SWB_OK;
}

// Raises a kernel's dynamic shared-memory limit to `bytes` once per device (`done_mask`).
template <typename Kernel>
int allow_smem(Kernel kernel, std::atomic<uint64_t>& done_mask, size_t bytes) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return check_launch();
    const uint64_t bit = dev < 64 ? (uint64_t(1) << dev) : 0;
    if (bit && (done_mask.load(std::memory_order_acquire) & bit)) return SWB_OK;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(bytes));
    if (e != cudaSuccess) {
        (void)cudaGetLastError();
        return fail(SWB_E_CUDA, cudaGetErrorString(e));
    }
    if (bit) done_mask.fetch_or(bit, std::memory_order_acq_rel);
    return SWB_OK;
}

}  // namespace swb
