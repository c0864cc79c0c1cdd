// What the launchers of the generation-step kernels (df11_kv.cu, df11_sample.cu) share.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "../../include/df11.h"
#include "df11_error.h"

// Makes `device` current for the calling thread and puts the previous one back.
struct Df11DeviceScope {
    int prev = -1;
    bool ok = true;
    explicit Df11DeviceScope(int device)
    {
        if (cudaGetDevice(&prev) != cudaSuccess) prev = -1;
        if (prev == device) prev = -1;
        else ok = cudaSetDevice(device) == cudaSuccess;
    }
    ~Df11DeviceScope()
    {
        if (prev >= 0) cudaSetDevice(prev);
    }
    Df11DeviceScope(const Df11DeviceScope &) = delete;
    Df11DeviceScope &operator=(const Df11DeviceScope &) = delete;
};

// Lets `kernel` use `bytes` of shared memory on the current device, which is `device`.  The runtime is asked once per
// kernel and device: the answer stays, and asking costs as much as a launch's other bookkeeping together.
inline cudaError_t df11_allow_shared(const void *kernel, size_t bytes, int device)
{
    constexpr int kPlaces = 256;
    static std::atomic<const void *> known[kPlaces];
    const size_t at = ((reinterpret_cast<uintptr_t>(kernel) >> 3) + (size_t)device * 61) % kPlaces;
    const void *const tag = reinterpret_cast<const char *>(kernel) + (device & 7);
    if (device < 8 && known[at].load(std::memory_order_relaxed) == tag) return cudaSuccess;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e == cudaSuccess && device < 8) known[at].store(tag, std::memory_order_relaxed);
    return e;
}

template <typename T> __device__ __forceinline__ float df11_to_float(T x);
template <> __device__ __forceinline__ float df11_to_float<float>(float x) { return x; }
template <> __device__ __forceinline__ float df11_to_float<__half>(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float df11_to_float<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }

template <typename T> __device__ __forceinline__ T df11_from_float(float x);
template <> __device__ __forceinline__ __half df11_from_float<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 df11_from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
