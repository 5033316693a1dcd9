// layers.h -- what the network's layers (rotary.cu, groupnorm.cu, gated.cu) share: element
// types, aligned vectors, activations, and the checks of their entry points.
#pragma once
#include "engine.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace stg {

// The engine's device for one call; the caller's current device again afterwards.
struct DeviceScope {
    int before = -1, device;
    explicit DeviceScope(const stg_engine* e) : device(e->device) {
        cuda_check(cudaGetDevice(&before), "cudaGetDevice");
        if (before != device) cuda_check(cudaSetDevice(device), "cudaSetDevice");
    }
    ~DeviceScope() { if (before != device) cudaSetDevice(before); }
    DeviceScope(const DeviceScope&) = delete;
    DeviceScope& operator=(const DeviceScope&) = delete;
};

template <class Cfg> void check_sized(const Cfg* c, const char* op) {
    if (!c || c->size < sizeof(Cfg)) fail(STG_INVALID_ARGUMENT, std::string(op) + ": config is NULL or config.size is too small");
}
inline void check(bool ok, const char* what) { if (!ok) fail(STG_INVALID_ARGUMENT, what); }
inline size_t elem_size(int dtype) { return dtype == STG_F32 ? 4 : 2; }
inline bool valid_dtype(int dtype) { return dtype == STG_F32 || dtype == STG_F16 || dtype == STG_BF16; }
inline bool valid_activation(int a) { return a >= STG_ACT_NONE && a <= STG_ACT_SIGMOID; }
inline bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// Unsigned division by a constant of the launch: n / d for n < 2^31, d < 2^31, as the high
// half of one multiplication (Granlund and Montgomery 1994: with l = ceil(log2 d) and
// m = floor(2^32 (2^l - d) / d) + 1, n / d = (mulhi(m, n) + n) >> l).
struct FastDiv {
    uint32_t d = 1, m = 1, l = 0;
    FastDiv() = default;
    explicit FastDiv(uint32_t div) : d(div) {
        while ((1ull << l) < d) l++;
        m = (uint32_t)(((1ull << 32) * ((1ull << l) - d)) / d + 1);
    }
    __device__ __forceinline__ uint32_t div(uint32_t n) const { return (__umulhi(n, m) + n) >> l; }
};

template <class T, int N> struct alignas(sizeof(T) * N) Pack { T v[N]; };

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
template <class T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ float from_float<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// Calls fn with a null pointer of the element type as its tag.
template <class Fn> void with_dtype(int dtype, Fn&& fn) {
    if (dtype == STG_F32) fn((float*)nullptr);
    else if (dtype == STG_F16) fn((__half*)nullptr);
    else fn((__nv_bfloat16*)nullptr);
}

// 1 / (1 + e^-z). For z below about -88 e^-z is infinite and the result 0, its limit.
__device__ __forceinline__ float sigmoidf(float z) { return __fdividef(1.0f, 1.0f + __expf(-z)); }

} // namespace stg
