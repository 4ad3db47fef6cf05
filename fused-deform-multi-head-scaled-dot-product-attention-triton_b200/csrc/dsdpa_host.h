// What the library's C-ABI translation units share on the host side.
#pragma once

#include <cuda_runtime.h>
#include <float.h>
#include <math.h>
#include <stdint.h>
#include <atomic>

#include "../../include/dsdpa.h"

namespace dsdpa {

// dsdpa_api.cu: record a failed CUDA call (what dsdpa_last_cuda_error() returns); returns DSDPA_ERR_CUDA
int report_cuda_failure(int cuda_error);
// dsdpa_api.cu: the device's error word (what dsdpa_device_error() reads), `device` being current
cudaError_t device_error_word(int device, int** out);
// dsdpa_api.cu: kernels launched, for dsdpa_kernel_launches()
void count_launches(int n);

inline bool misaligned(const void* p) { return ((uintptr_t)p & 15u) != 0; }

// Strides of dimensions that have one element do not matter.
inline bool bad_stride(const long long (&st)[3], int dtype, int B, int H, int L) {
    const int n[3] = { B, H, L };
    for (int i = 0; i < 3; ++i)
        if (n[i] > 1 && (st[i] <= 0 || (st[i] * (dtype == DSDPA_F32 ? 4 : 2)) % 16)) return true;
    return false;
}

// A scale or a cap that the kernels' fp32 cannot carry: they work with 2 |sm_scale| / softcap and softcap log2(e).
inline bool bad_score(float sm_scale, float softcap) {
    if (!isfinite(sm_scale) || !isfinite(softcap)) return true;
    if (softcap <= 0.0f) return false;
    const double in = 2.0 * fabs((double)sm_scale) / softcap;
    return softcap < FLT_MIN || softcap > FLT_MAX / 2 || in > FLT_MAX || (sm_scale != 0.0f && in < FLT_MIN);
}

struct DeviceGuard {
    int prev = -1;
    cudaError_t err = cudaSuccess;
    explicit DeviceGuard(int device) {
        err = cudaGetDevice(&prev);
        if (err == cudaSuccess && prev != device) err = cudaSetDevice(device);
    }
    ~DeviceGuard() {
        int cur = -1;
        if (prev >= 0 && cudaGetDevice(&cur) == cudaSuccess && cur != prev) (void)cudaSetDevice(prev);
    }
};

// Lets a kernel have `bytes` of dynamic shared memory, once per device; `done` is the calling instantiation's own.
struct SmemOnce {
    std::atomic<bool> done[64] = {};
};
template <typename K>
inline cudaError_t allow_smem(K kern, int bytes, SmemOnce& once) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64 && once.done[dev].load(std::memory_order_relaxed)) return cudaSuccess;
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess && dev >= 0 && dev < 64) once.done[dev].store(true, std::memory_order_relaxed);
    return e;
}

}  // namespace dsdpa
