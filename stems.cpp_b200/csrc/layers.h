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

// ---- pairs: two floats to an instruction --------------------------------------------------------
struct f2 { uint64_t v; };
__device__ __forceinline__ f2 make_f2(float x, float y) { f2 r; asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(x), "f"(y)); return r; }
__device__ __forceinline__ f2 make_f2(float x) { return make_f2(x, x); }
__device__ __forceinline__ float2 split(f2 a) { float2 r; asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v)); return r; }
__device__ __forceinline__ f2 operator+(f2 a, f2 b) { f2 r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v)); return r; }
__device__ __forceinline__ f2 operator*(f2 a, f2 b) { f2 r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v)); return r; }
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) { f2 r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v)); return r; }
template <class Fn> __device__ __forceinline__ f2 each(f2 a, Fn&& fn) { const float2 v = split(a); return make_f2(fn(v.x), fn(v.y)); }

__device__ __forceinline__ f2 load2(const float* p) { return make_f2(p[0], p[1]); }
__device__ __forceinline__ f2 load2(const __half* p) { const float2 v = __half22float2(*reinterpret_cast<const __half2*>(p)); return make_f2(v.x, v.y); }
__device__ __forceinline__ f2 load2(const __nv_bfloat16* p) {   // a bf16 is the upper half of a float
    const uint32_t u = *reinterpret_cast<const uint32_t*>(p);
    return make_f2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}
__device__ __forceinline__ void store2(float* p, f2 a) { const float2 v = split(a); p[0] = v.x; p[1] = v.y; }
__device__ __forceinline__ void store2(__half* p, f2 a) { const float2 v = split(a); *reinterpret_cast<__half2*>(p) = __floats2half2_rn(v.x, v.y); }
__device__ __forceinline__ void store2(__nv_bfloat16* p, f2 a) {
    const float2 v = split(a);
    *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(v.x, v.y);
}

// exp(-z) for float results: 2^t, t = -z log2 e rounded, times 1 + ln 2 (what t lost), so that what
// is left is the approximate power's own 2^-22. Infinite powers are kept finite for that product.
__device__ __forceinline__ f2 exp_neg(f2 z) {
    const f2 c = make_f2(-1.4426950216293335f), t = z * c;
    const f2 lost = each(fma2(z, make_f2(-1.9259629911266175e-8f), fma2(z, c, t * make_f2(-1.0f))),
                         [](float x) { return fabsf(x) < 1.0f ? x : 0.0f; });   // (infinite z lose nothing)
    const f2 e = each(t, [](float x) { return fminf(ex2(x), 3.0e38f); });
    return fma2(e, lost * make_f2(0.6931471805599453f), e);
}
template <bool kFast> __device__ __forceinline__ f2 sigmoid2(f2 z) {
    const f2 e = kFast ? each(z * make_f2(-1.4426950408889634f), [](float x) { return ex2(x); }) : exp_neg(z);
    return each(e + make_f2(1.0f), [](float x) { return rcp(x); });
}
constexpr float kGaussStep = 0.27f;
__device__ constexpr float kGauss[9] = {0.107720181f, 0.107550503f, 0.10175919f, 0.0722401889f, 0.107399681f, -0.068621354f, 0.169291745f, -0.126255433f, 0.0289153096f};
// |z| and Phi(-|z|), exp(-z^2 / 2): see gauss(). For float results P has degree 8 on t = 1 / (1 + 0.27 x)
// (3e-8) and the power makes up for the rounding of z^2.
template <bool kFast> __device__ __forceinline__ f2 gauss2(f2 z, f2& size, f2& e) {
    size = each(z, [](float x) { return fminf(fabsf(x), 100.0f); });
    const f2 t = each(fma2(make_f2(kFast ? 0.36f : kGaussStep), size, make_f2(1.0f)), [](float x) { return rcp(x); });
    f2 p;
    if (kFast) {
        e = each(z * z * make_f2(-0.72134752044448170f), [](float x) { return ex2(x); });
        p = fma2(t, make_f2(0.047056273f), make_f2(-0.17976463f));
        p = fma2(t, p, make_f2(0.18095392f));
        p = fma2(t, p, make_f2(0.026549397f));
        p = fma2(t, p, make_f2(0.13971923f));
        p = fma2(t, p, make_f2(0.14177246f));
        p = fma2(t, p, make_f2(0.14371304f));
    } else {
        const f2 zz = each(z * z, [](float x) { return fminf(x, 400.0f); });   // past 14 both factors vanish
        const f2 lost = fma2(z, z, z * z * make_f2(-1.0f));
        e = exp_neg(zz * make_f2(0.5f));
        e = fma2(e, each(lost, [](float x) { return fabsf(x) < 1.0f ? -0.5f * x : 0.0f; }), e);
        p = make_f2(kGauss[8]);
#pragma unroll
        for (int i = 7; i >= 0; i--) p = fma2(t, p, make_f2(kGauss[i]));
    }
    return p * t * e;
}
// act(z), and act(z) and its derivative, of pairs.
template <int ACT, bool kFast> __device__ __forceinline__ f2 act2(f2 z) {
    if (ACT == STG_ACT_RELU) return each(z, [](float x) { return x < 0.0f ? 0.0f : x; });
    if (ACT == STG_ACT_SILU) return z * sigmoid2<kFast>(z);
    if (ACT == STG_ACT_GELU) {   // max(z, 0) - |z| Phi(-|z|)
        f2 size, e;
        const f2 tail = gauss2<kFast>(z, size, e);
        return fma2(size * make_f2(-1.0f), tail, each(z, [](float x) { return x < 0.0f ? 0.0f : x; }));
    }
    if (ACT == STG_ACT_SIGMOID) return sigmoid2<kFast>(z);
    return z;
}
template <int ACT, bool kFast> __device__ __forceinline__ f2 act_grad2(f2 z) {
    if (ACT == STG_ACT_RELU) return each(z, [](float x) { return x > 0.0f ? 1.0f : (x <= 0.0f ? 0.0f : x); });
    if (ACT == STG_ACT_SILU || ACT == STG_ACT_SIGMOID) {
        const f2 s = sigmoid2<kFast>(z), rest = fma2(s, make_f2(-1.0f), make_f2(1.0f));
        return ACT == STG_ACT_SIGMOID ? s * rest : fma2(z * s, rest, s);
    }
    if (ACT == STG_ACT_GELU) {
        f2 size, e;
        const float2 tail = split(gauss2<kFast>(z, size, e)), x = split(z);
        const f2 phi = make_f2(x.x < 0.0f ? tail.x : 1.0f - tail.x, x.y < 0.0f ? tail.y : 1.0f - tail.y);
        return fma2(z * make_f2(0.3989422804014327f), e, phi);
    }
    return make_f2(1.0f);
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
