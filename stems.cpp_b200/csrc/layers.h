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

// ---- activations --------------------------------------------------------------------------------
// Float results (kFast false) use CUDA's expf, erfcf and division. Results that are rounded to 16
// bits use the approximate exponential and reciprocal (2^-22 relative each): a function then
// costs two special-function instructions and a few multiplications, where the
// accurate ones made group norm with GELU compute-bound (213 us where the memory takes 40).
__device__ __forceinline__ float ex2(float x) { float r; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x)); return r; }
__device__ __forceinline__ float rcp(float x) { float r; asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x)); return r; }
// 1 / (1 + 2^(-z log2 e)); 0 where the power is infinite.
template <bool kFast> __device__ __forceinline__ float sigmoid(float z) {
    return kFast ? rcp(1.0f + ex2(-1.4426950408889634f * z)) : 1.0f / (1.0f + expf(-z));
}
// Phi(z), the normal distribution function, and e = exp(-z^2 / 2). Phi(-|z|) = e R(|z|) with R(x) =
// erfcx(x / sqrt 2) / 2, which falls smoothly from 1/2 to 1 / (x sqrt(2 pi)) and is fitted here by
// t P(t), t = 1 / (1 + 0.36 x), P of degree 6: minimax on [0, 14] (iteratively reweighted least
// squares in double), 1.2e-6 relative in float. Past 13 e is zero in float.
__device__ __forceinline__ float gauss(float z, float& e) {
    const float t = rcp(fmaf(0.36f, fabsf(z), 1.0f));
    e = ex2(-0.72134752044448170f * z * z);
    float p = fmaf(t, 0.047056273f, -0.17976463f);
    p = fmaf(t, p, 0.18095392f);
    p = fmaf(t, p, 0.026549397f);
    p = fmaf(t, p, 0.13971923f);
    p = fmaf(t, p, 0.14177246f);
    p = fmaf(t, p, 0.14371304f);
    const float tail = p * t * e;
    return z < 0.0f ? tail : 1.0f - tail;   // a NaN in z is one in tail
}
// act(z) and its derivative.
template <int ACT, bool kFast> __device__ __forceinline__ void act_both(float z, float& a, float& d) {
    if (ACT == STG_ACT_RELU) {
        a = z < 0.0f ? 0.0f : z;                             // keeps NaN
        d = z > 0.0f ? 1.0f : (z <= 0.0f ? 0.0f : z);
    } else if (ACT == STG_ACT_SILU) {
        const float s = sigmoid<kFast>(z);
        a = z * s;
        d = fmaf(a, 1.0f - s, s);
    } else if (ACT == STG_ACT_GELU) {
        float e, phi;
        if (kFast) phi = gauss(z, e);
        else {
            phi = 0.5f * erfcf(-z * 0.70710678118654752f);
            e = expf(-0.5f * z * z);
        }
        a = z * phi;
        d = fmaf(0.3989422804014327f * z, e, phi);
    } else if (ACT == STG_ACT_SIGMOID) {
        a = sigmoid<kFast>(z);
        d = a * (1.0f - a);
    } else {
        a = z;
        d = 1.0f;
    }
}
template <int ACT, bool kFast> __device__ __forceinline__ float act(float z) {
    float a, d;
    act_both<ACT, kFast>(z, a, d);
    return a;
}
template <int ACT, bool kFast> __device__ __forceinline__ float act_grad(float z) {
    float a, d;
    act_both<ACT, kFast>(z, a, d);
    return d;
}

// Calls fn with the activation as an integral_constant.
template <class Fn> void with_activation(int a, Fn&& fn) {
    switch (a) {
        case STG_ACT_RELU: return fn(std::integral_constant<int, STG_ACT_RELU>{});
        case STG_ACT_SILU: return fn(std::integral_constant<int, STG_ACT_SILU>{});
        case STG_ACT_GELU: return fn(std::integral_constant<int, STG_ACT_GELU>{});
        case STG_ACT_SIGMOID: return fn(std::integral_constant<int, STG_ACT_SIGMOID>{});
        default: return fn(std::integral_constant<int, STG_ACT_NONE>{});
    }
}

} // namespace stg
