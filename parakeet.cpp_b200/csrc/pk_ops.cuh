// pk_ops.cuh -- what the entry points that take a caller's device pointers and stream
// (pk_mx4.cu, pk_sample.cu) share: the current device kept as the caller left it, the
// device check, error texts, and loads of the three element types.
#pragma once

#include "pk_internal.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdio>
#include <utility>

namespace pk {
namespace {

// Makes `device` current for a scope; the caller's device is current again after it.
struct DeviceScope {
    int before = -1, now = -1;
    cudaError_t err;
    explicit DeviceScope(int device) {
        err = cudaGetDevice(&before);
        now = before;
        if (err == cudaSuccess && before != device) {
            err = cudaSetDevice(device);
            if (err == cudaSuccess) now = device;
        }
    }
    ~DeviceScope() {
        if (before >= 0 && now != before) cudaSetDevice(before);
    }
    DeviceScope(const DeviceScope &) = delete;
    DeviceScope & operator=(const DeviceScope &) = delete;
};

inline pk_status op_fail(pk_status s, const char * fn, const char * what) {
    char msg[256];
    std::snprintf(msg, sizeof(msg), "%s: %s", fn, what);
    return set_error(s, msg);
}

// The runtime keeps an error until somebody asks for the last one: it is this call's, and no later launch's.
inline pk_status op_cuda_fail(cudaError_t e, const char * fn) {
    cudaGetLastError();
    return op_fail(e == cudaErrorMemoryAllocation ? PK_ERR_OOM : PK_ERR_CUDA, fn, cudaGetErrorString(e));
}

// A launch whose status is its own, not an earlier call's that nobody has asked for.
template <class... P, class... A>
inline cudaError_t launch_on(void (*kernel)(P...), dim3 grid, unsigned threads, size_t smem, cudaStream_t s, A &&... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    return cudaLaunchKernelEx(&cfg, kernel, std::forward<A>(args)...);
}

// Whether `device` exists and is sm_100 (asked of the runtime once per device).
inline bool device_ok(int device) {
    constexpr int kMax = 64;
    static int known[kMax];   // 0 not asked, 1 yes, 2 no; a race writes the same answer twice
    if (device < 0 || device >= kMax) return false;
    int k = __atomic_load_n(&known[device], __ATOMIC_RELAXED);
    if (k == 0) {
        int n = 0, major = 0;
        if (cudaGetDeviceCount(&n) != cudaSuccess || device >= n) {
            cudaGetLastError();
            return false;
        }
        if (cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, device) != cudaSuccess) {
            cudaGetLastError();
            return false;
        }
        k = major == 10 ? 1 : 2;
        __atomic_store_n(&known[device], k, __ATOMIC_RELAXED);
    }
    return k == 1;
}

inline int elem_size(int type) { return type == PK_GGML_F32 ? 4 : (type == PK_GGML_F16 || type == PK_GGML_BF16) ? 2 : 0; }

inline bool aligned_to(const void * p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }

template <class T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

}  // namespace
}  // namespace pk
