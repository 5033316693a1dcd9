// layers.h -- what the network's layers (rotary.cu, groupnorm.cu, gated.cu) share: element
// types, aligned vectors, activations, and the checks of their entry points.
#pragma once
#include "engine.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

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

struct Nothing { __device__ __forceinline__ void operator()() const {} };
// load() then use() n times, in that order each, with the loads U to 2U ahead; batch() after every U uses that are not the last. (Group norm's moments of
// 132 MB: 30 us; with twice the warps 34, and 39 with four plain loads at a time in place of this.)
template <class P, int U, class Load, class Use, class Batch = Nothing>
__device__ __forceinline__ void stream(int n, Load&& load, Use&& use, Batch&& batch = Batch{}) {
    P now[U], next[U];
    if (n >= U) {
#pragma unroll
        for (int u = 0; u < U; u++) load(now[u]);
#pragma unroll 2
        for (; n >= 2 * U; n -= U) {
#pragma unroll
            for (int u = 0; u < U; u++) load(next[u]);
#pragma unroll
            for (int u = 0; u < U; u++) use(now[u]);
            batch();
#pragma unroll
            for (int u = 0; u < U; u++) now[u] = next[u];
        }
        n -= U;
        // the rest is on its way while the last whole batch is used
#pragma unroll
        for (int u = 0; u < U; u++)
            if (u < n) load(next[u]);
#pragma unroll
        for (int u = 0; u < U; u++) use(now[u]);
        if (n > 0) batch();
    } else {
#pragma unroll
        for (int u = 0; u < U; u++)
            if (u < n) load(next[u]);
    }
#pragma unroll
    for (int u = 0; u < U; u++)
        if (u < n) use(next[u]);
}
// A vector's last read, and a result that is not read here: both leave L2 first.
template <class P, class T> __device__ __forceinline__ P load_stream(const T* p) {
    P v;
    if constexpr (sizeof(P) == 16) {
        const uint4 u = __ldcs(reinterpret_cast<const uint4*>(p));
        v = *reinterpret_cast<const P*>(&u);
    } else v = *reinterpret_cast<const P*>(p);
    return v;
}
template <class T, class P> __device__ __forceinline__ void store_stream(T* p, const P& v) {
    if constexpr (sizeof(P) == 16) __stcs(reinterpret_cast<uint4*>(p), *reinterpret_cast<const uint4*>(&v));
    else *reinterpret_cast<P*>(p) = v;
}

// ---- activations --------------------------------------------------------------------------------
// Built on the approximate power of two and reciprocal (2^-22 relative each). For results that are
// rounded to 16 bits (kFast) those do as they are; float results make up for the roundings of
// the exponent, which is what is left of an exponential's error otherwise. CUDA's accurate erfcf,
// expf and division made group norm with GELU compute-bound (213 us where the memory takes 40).
__device__ __forceinline__ float ex2(float x) { float r; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x)); return r; }
__device__ __forceinline__ float rcp(float x) { float r; asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x)); return r; }
__device__ __forceinline__ float relu(float x) { float r; asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(r) : "f"(x)); return r; }   // keeps NaN
// exp(-z) for float results: 2^t, t = -z log2 e rounded, times 1 + ln 2 (what t lost), so that what
// is left is the approximate power's own 2^-22. Infinite powers are kept finite for that product.
__device__ __forceinline__ float exp_neg(float z) {
    const float t = z * -1.4426950216293335f;
    const float lost = fmaf(z, -1.9259629911266175e-8f, fmaf(z, -1.4426950216293335f, -t));
    const float e = fminf(ex2(t), 3.0e38f);
    return fmaf(e, fabsf(lost) < 1.0f ? lost * 0.6931471805599453f : 0.0f, e);   // infinite z lose nothing
}
// 1 / (1 + e^-z); 0 where the power is infinite.
template <bool kFast> __device__ __forceinline__ float sigmoid(float z) {
    return rcp(1.0f + (kFast ? ex2(-1.4426950408889634f * z) : exp_neg(z)));
}
// Phi(-x), the normal distribution's tail, for x >= 0, as 2^S(x): S = log2 Phi(-x) is smooth and
// nearly a parabola, here a polynomial of degree 10 (minimax in the error of the power, by
// iteratively reweighted least squares in double): in float 4e-6 relative for x <= 4, 2e-5 at 9, where
// Phi is 1e-19 and the polynomial ends. One special function and no division: the rational form it
// replaces (1 / (1 + c x) and exp(-x^2 / 2)) took two and four instructions more.
__device__ __forceinline__ float normal_tail(float x) {
    float s = -1.87925829e-09f;
    s = fmaf(s, x, 8.08722736e-08f);
    s = fmaf(s, x, -1.3956618e-06f);
    s = fmaf(s, x, 1.1034977e-05f);
    s = fmaf(s, x, -8.45205791e-06f);
    s = fmaf(s, x, -0.000698472729f);
    s = fmaf(s, x, 0.00804607337f);
    s = fmaf(s, x, -0.0534383855f);
    s = fmaf(s, x, -0.458760105f);
    s = fmaf(s, x, -1.15118688f);
    s = fmaf(s, x, -0.999997556f);
    return ex2(s);
}
// Phi(-x) and e = exp(-x^2 / 2) for float results: Phi(-x) = e R(x), R(x) = erfcx(x / sqrt 2) / 2 fitted by
// t P(t), t = 1 / (1 + 0.27 x), P of degree 8 (by the same means; 7e-8 on [0, 14] with these constants
// as floats); e makes up for the rounding of x^2.
__device__ __forceinline__ float normal_tail(float x, float& e) {
    const float t = rcp(fmaf(0.27f, x, 1.0f));
    const float xx = fminf(x * x, 400.0f), lost = fmaf(x, x, -x * x);   // past 14 both factors vanish
    e = exp_neg(0.5f * xx);
    e = fmaf(e, fabsf(lost) < 1.0f ? -0.5f * lost : 0.0f, e);
    float p = 0.0289153096f;
    p = fmaf(t, p, -0.126255433f);
    p = fmaf(t, p, 0.169291745f);
    p = fmaf(t, p, -0.068621354f);
    p = fmaf(t, p, 0.107399681f);
    p = fmaf(t, p, 0.0722401889f);
    p = fmaf(t, p, 0.10175919f);
    p = fmaf(t, p, 0.107550503f);
    p = fmaf(t, p, 0.107720181f);
    return p * t * e;
}
// act(z).
template <int ACT, bool kFast> __device__ __forceinline__ float act(float z) {
    if (ACT == STG_ACT_RELU) return relu(z);
    if (ACT == STG_ACT_SILU) return z * sigmoid<kFast>(z);
    if (ACT == STG_ACT_GELU) {   // z Phi(z) = max(z, 0) - |z| Phi(-|z|)
        float e;
        const float u = fminf(fabsf(z), kFast ? 9.0f : 100.0f);
        return fmaf(-u, kFast ? normal_tail(u) : normal_tail(u, e), relu(z));
    }
    if (ACT == STG_ACT_SIGMOID) return sigmoid<kFast>(z);
    return z;
}
// act(z) and its derivative.
template <int ACT, bool kFast> __device__ __forceinline__ void act_both(float z, float& a, float& d) {
    if (ACT == STG_ACT_RELU) {
        a = relu(z);
        d = z > 0.0f ? 1.0f : (z <= 0.0f ? 0.0f : z);
    } else if (ACT == STG_ACT_SILU) {
        const float s = sigmoid<kFast>(z);
        a = z * s;
        d = fmaf(a, 1.0f - s, s);
    } else if (ACT == STG_ACT_GELU) {
        float e;
        const float u = fminf(fabsf(z), kFast ? 9.0f : 100.0f), tail = kFast ? normal_tail(u) : normal_tail(u, e);
        if (kFast) e = ex2(-0.72134752044448170f * z * z);
        a = fmaf(-u, tail, relu(z));
        d = fmaf(0.3989422804014327f * z, e, z < 0.0f ? tail : 1.0f - tail);
    } else if (ACT == STG_ACT_SIGMOID) {
        a = sigmoid<kFast>(z);
        d = a * (1.0f - a);
    } else {
        a = z;
        d = 1.0f;
    }
}
template <int ACT, bool kFast> __device__ __forceinline__ float act_grad(float z) {
    float a, d;
    act_both<ACT, kFast>(z, a, d);
    return d;
}

// ---- pairs: two floats to an instruction --------------------------------------------------------
struct f2 { uint64_t v; };
__device__ __forceinline__ f2 make_f2(float x, float y) { f2 r; asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(x), "f"(y)); return r; }
// A constant for both, kept in registers: left to the compiler it is made again at each use, which
// costs as much as the packed instruction saves.
__device__ __forceinline__ f2 held_f2(float x) { f2 r; asm volatile("mov.b64 %0, {%1, %1};" : "=l"(r.v) : "f"(x)); return r; }
__device__ __forceinline__ float2 split(f2 a) { float2 r; asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v)); return r; }
__device__ __forceinline__ f2 operator+(f2 a, f2 b) { f2 r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v)); return r; }
__device__ __forceinline__ f2 operator*(f2 a, f2 b) { f2 r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v)); return r; }
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) { f2 r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v)); return r; }
template <class Fn> __device__ __forceinline__ f2 each(f2 a, Fn&& fn) { const float2 v = split(a); return make_f2(fn(v.x), fn(v.y)); }

// Pair i of a vector as floats, and back. A vector of one is a pair with nothing beside it.
template <class T, int V> __device__ __forceinline__ f2 get(const Pack<T, V>& v, int i) {
    if constexpr (V == 1) return make_f2(to_float(v.v[0]), 0.0f);
    else if constexpr (std::is_same<T, __nv_bfloat16>::value) {   // a bf16 is the upper half of a float
        const uint32_t u = reinterpret_cast<const uint32_t*>(&v)[i];
        return make_f2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
    } else if constexpr (std::is_same<T, __half>::value) {
        const float2 f = __half22float2(reinterpret_cast<const __half2*>(&v)[i]);
        return make_f2(f.x, f.y);
    } else return make_f2(v.v[2 * i], v.v[2 * i + 1]);
}
template <class T, int V> __device__ __forceinline__ void put(Pack<T, V>& v, int i, f2 a) {
    const float2 f = split(a);
    if constexpr (V == 1) v.v[0] = from_float<T>(f.x);
    else if constexpr (std::is_same<T, __nv_bfloat16>::value) reinterpret_cast<__nv_bfloat162*>(&v)[i] = __floats2bfloat162_rn(f.x, f.y);
    else if constexpr (std::is_same<T, __half>::value) reinterpret_cast<__half2*>(&v)[i] = __floats2half2_rn(f.x, f.y);
    else { v.v[2 * i] = f.x; v.v[2 * i + 1] = f.y; }
}

// sigmoid<false> of a pair. Past 88 either way the power or its reciprocal vanishes, and up to there all is
// finite: no tests for infinite values. (Mask head, 2 x 2 x 62 BS bands x 87 at hidden 250 f16: 22.3 us, with
// sigmoid<false> 22.9, sigmoid<true> 22.0; 60 mel bands x 801 at 1536 67 us, 67.4 and 67.)
__device__ __forceinline__ f2 sigmoid(f2 z) {
    const f2 x = each(z, [](float v) {   // NaN stays
        asm("max.NaN.f32 %0, %0, 0fC2B00000;\nmin.NaN.f32 %0, %0, 0f42B00000;" : "+f"(v));
        return v;
    });
    const f2 t = x * make_f2(-1.4426950216293335f, -1.4426950216293335f);
    const f2 over = fma2(x, make_f2(1.9259629911266175e-8f, 1.9259629911266175e-8f), fma2(x, make_f2(1.4426950216293335f, 1.4426950216293335f), t));
    const f2 e = each(t, ex2);
    return each(fma2(e, over * make_f2(-0.6931471805599453f, -0.6931471805599453f), e) + make_f2(1.0f, 1.0f), rcp);
}

// act() and act_grad() of pairs. Float results go through the plain functions; 16-bit ones keep their
// constants in registers.
template <int ACT, bool kFast> struct PairAct {
    __device__ __forceinline__ f2 value(f2 z) const { return each(z, [](float x) { return act<ACT, kFast>(x); }); }
    __device__ __forceinline__ f2 slope(f2 z) const { return each(z, [](float x) { return act_grad<ACT, kFast>(x); }); }
};
template <> struct PairAct<STG_ACT_NONE, true> {
    __device__ __forceinline__ f2 value(f2 z) const { return z; }
    __device__ __forceinline__ f2 slope(f2) const { return make_f2(1.0f, 1.0f); }
};
template <> struct PairAct<STG_ACT_NONE, false> : PairAct<STG_ACT_NONE, true> {};
struct PairSigmoid {
    f2 log2e = held_f2(-1.4426950408889634f), one = held_f2(1.0f);
    __device__ __forceinline__ f2 sigmoid(f2 z) const { return each(each(z * log2e, ex2) + one, rcp); }
    __device__ __forceinline__ f2 rest(f2 s) const { return each(s, [](float x) { return 1.0f - x; }); }
};
template <> struct PairAct<STG_ACT_SILU, true> : PairSigmoid {
    __device__ __forceinline__ f2 value(f2 z) const { return z * sigmoid(z); }
    __device__ __forceinline__ f2 slope(f2 z) const {
        const f2 s = sigmoid(z);
        return fma2(z * s, rest(s), s);
    }
};
template <> struct PairAct<STG_ACT_SIGMOID, true> : PairSigmoid {
    __device__ __forceinline__ f2 value(f2 z) const { return sigmoid(z); }
    __device__ __forceinline__ f2 slope(f2 z) const {
        const f2 s = sigmoid(z);
        return s * rest(s);
    }
};
template <> struct PairAct<STG_ACT_GELU, true> {   // normal_tail's polynomial in -|z|
    f2 c[11] = {held_f2(-0.999997556f),
               held_f2(1.15118688f),
               held_f2(-0.458760105f),
               held_f2(0.0534383855f),
               held_f2(0.00804607337f),
               held_f2(0.000698472729f),
               held_f2(-8.45205791e-06f),
               held_f2(-1.1034977e-05f),
               held_f2(-1.3956618e-06f),
               held_f2(-8.08722736e-08f),
               held_f2(-1.87925829e-09f)};
    // w = max(-|z|, -9); Phi(w)
    __device__ __forceinline__ f2 tail(f2 z, f2& w) const {
        w = each(z, [](float x) { return fmaxf(-fabsf(x), -9.0f); });
        f2 s = c[10];
#pragma unroll
        for (int i = 9; i >= 0; i--) s = fma2(s, w, c[i]);
        return each(s, ex2);
    }
    __device__ __forceinline__ f2 value(f2 z) const {
        f2 w;
        const f2 t = tail(z, w);
        return fma2(w, t, each(z, relu));
    }
    __device__ __forceinline__ f2 slope(f2 z) const {
        f2 w;
        const float2 t = split(tail(z, w)), x = split(z);
        const f2 phi = make_f2(x.x < 0.0f ? t.x : 1.0f - t.x, x.y < 0.0f ? t.y : 1.0f - t.y);
        const f2 e = each(z * z, [](float v) { return 0.3989422804014327f * ex2(-0.72134752044448170f * v); });
        return fma2(z, e, phi);
    }
};

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
