// What the launchers of the generation-step kernels (df11_kv.cu, df11_sample.cu) share.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

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

template <typename T> __device__ __forceinline__ float df11_to_float(T x);
template <> __device__ __forceinline__ float df11_to_float<float>(float x) { return x; }
template <> __device__ __forceinline__ float df11_to_float<__half>(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float df11_to_float<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }

template <typename T> __device__ __forceinline__ T df11_from_float(float x);
template <> __device__ __forceinline__ __half df11_from_float<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 df11_from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
