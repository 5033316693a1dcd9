// groupnorm.cu -- group norm with an activation, channels last, and its backward pass
// (include/stems_gpu_v1.h: stg_group_norm, stg_group_norm_backward).
//
// x [batch][positions][channels]; a group is channels / groups neighbouring channels of every
// position of a batch item. Forward: mean and variance per (item, group), then
// y = act((x - mean) rstd gamma + beta). Backward, with xh = (x - mean) rstd,
// z = gamma xh + beta, dz = dy act'(z), over the m elements of a group:
//   dbeta = sum dz,  dgamma = sum dz xh  (over items and positions),
//   dx = rstd (d - sum(d) / m - xh sum(d xh) / m),  d = gamma dz.
//
// Three kernels each way. A block of the first takes a range of positions with all channels:
// its threads stand side by side along the channels (16-byte vectors, whole rows, so every
// sector is used whatever the group size) and step down the positions, each with sums of its
// own channels. The second joins the blocks' parts in a fixed order. The third reads x again.
#include "layers.h"

namespace stg {

namespace {

constexpr int kThreads = 256;
constexpr int kMaxChannels = 8192;

struct NormParams {
    const void *x, *dy, *gamma, *beta;
    void *y, *dx, *dgamma, *dbeta;
    float *mean, *rstd;              // [batch][groups]
    float2* part;                    // forward [batch][groups][chunks] (mean, M2); backward [batch][chunks][channels]
    float2* sums;                    // backward [batch][channels]: sum dz, sum dz xh
    int64_t positions, xb, xp, yb, yp, db, dp;
    int channels, groups, cpg;       // cpg: channels of a group
    int batch, chunks, rows;         // chunks per item, positions of a chunk (the last may have fewer)
    int columns;                     // vectors of a row
    FastDiv columns_div;             // by min(columns, kThreads)
    float eps;
    int param_float;
};

// ---- activations: float for f32 with CUDA's accurate functions, the fast ones (about 2^-21
// relative) where the result is rounded to 16 bits anyway -----------------------------------------
template <bool kFast> __device__ __forceinline__ float sigmoid(float z) {
    return kFast ? sigmoidf(z) : 1.0f / (1.0f + expf(-z));
}
template <int ACT, bool kFast> __device__ __forceinline__ float act(float z) {
    if (ACT == STG_ACT_RELU) return z < 0.0f ? 0.0f : z;   // keeps NaN
    if (ACT == STG_ACT_SILU) return z * sigmoid<kFast>(z);
    if (ACT == STG_ACT_GELU) return 0.5f * z * erfcf(-z * 0.70710678118654752f);
    if (ACT == STG_ACT_SIGMOID) return sigmoid<kFast>(z);
    return z;
}
template <int ACT, bool kFast> __device__ __forceinline__ float act_grad(float z) {
    if (ACT == STG_ACT_RELU) return z > 0.0f ? 1.0f : (z <= 0.0f ? 0.0f : z);
    if (ACT == STG_ACT_SILU) { const float s = sigmoid<kFast>(z); return s * fmaf(z, 1.0f - s, 1.0f); }
    if (ACT == STG_ACT_GELU) {
        const float e = kFast ? __expf(-0.5f * z * z) : expf(-0.5f * z * z);
        return fmaf(0.3989422804014327f * z, e, 0.5f * erfcf(-z * 0.70710678118654752f));
    }
    if (ACT == STG_ACT_SIGMOID) { const float s = sigmoid<kFast>(z); return s * (1.0f - s); }
    return 1.0f;
}

// Mean and sum of squared deviations of n values, joined pairwise (Chan, Golub, LeVeque 1979).
struct Moments { float n, mean, m2; };
__device__ __forceinline__ void join(Moments& a, const Moments& b) {
    if (b.n == 0.0f) return;
    if (a.n == 0.0f) { a = b; return; }
    const float n = a.n + b.n, d = b.mean - a.mean, w = b.n / n;
    a.mean = fmaf(d, w, a.mean);
    a.m2 = a.m2 + b.m2 + d * d * a.n * w;
    a.n = n;
}
__device__ __forceinline__ void warp_join(Moments& a) {
    for (int o = 16; o > 0; o >>= 1) {
        Moments b;
        b.n = __shfl_xor_sync(~0u, a.n, o);
        b.mean = __shfl_xor_sync(~0u, a.mean, o);
        b.m2 = __shfl_xor_sync(~0u, a.m2, o);
        // both partners compute the same bits: the lower lane's part comes first
        if (threadIdx.x & o) { Moments t = b; b = a; a = t; }
        join(a, b);
    }
}

__device__ __forceinline__ float param(const void* p, int i, bool f32, float none, const float*) { return p ? static_cast<const float*>(p)[i] : none; }
template <class T> __device__ __forceinline__ float param(const void* p, int i, bool f32, float none, const T*) {
    if (!p) return none;
    return f32 ? static_cast<const float*>(p)[i] : to_float(static_cast<const T*>(p)[i]);
}
__device__ __forceinline__ void set_param(void* p, int i, bool f32, float v, const float*) { static_cast<float*>(p)[i] = v; }
template <class T> __device__ __forceinline__ void set_param(void* p, int i, bool f32, float v, const T*) {
    if (f32) static_cast<float*>(p)[i] = v;
    else static_cast<T*>(p)[i] = from_float<T>(v);
}

// The thread's place in a block: column vector `col` of the current column tile and one of
// `step` positions taken side by side.
struct Place { int width, step, r, col; };
__device__ __forceinline__ Place place(const NormParams& p) {
    Place q;
    q.width = (int)p.columns_div.d;
    q.step = kThreads / q.width;
    q.r = (int)p.columns_div.div(threadIdx.x);
    q.col = threadIdx.x - q.r * q.width;
    return q;
}

// Moments of a chunk's groups. Each thread sums its channels' differences from the first value
// it meets, so that a mean far from zero costs no digits.
template <class T, int V>
__global__ void __launch_bounds__(kThreads) moments_kernel(const __grid_constant__ NormParams p) {
    __shared__ float2 part[kThreads * V];       // [r][col][V]: mean, M2
    const int b = blockIdx.y, chunk = blockIdx.x;
    const int64_t l0 = (int64_t)chunk * p.rows;
    const int n = (int)min((int64_t)p.rows, p.positions - l0);
    const Place q = place(p);
    const T* x = static_cast<const T*>(p.x) + b * p.xb + l0 * p.xp;
    extern __shared__ Moments group[];          // [groups], joined over column tiles
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int c0 = 0; c0 < p.columns; c0 += q.width) {
        const int cols = min(q.width, p.columns - c0);
        const bool on = q.r < q.step && q.col < cols;
        if (on) {
            float pivot[V], s[V], s2[V];
            float cnt = 0.0f;
#pragma unroll
            for (int j = 0; j < V; j++) pivot[j] = s[j] = s2[j] = 0.0f;
            if (q.r < n) {
                const Pack<T, V> v = *reinterpret_cast<const Pack<T, V>*>(x + (int64_t)q.r * p.xp + (int64_t)(c0 + q.col) * V);
#pragma unroll
                for (int j = 0; j < V; j++) pivot[j] = to_float(v.v[j]);
                cnt = (float)((n - q.r + q.step - 1) / q.step);
            }
#pragma unroll 4
            for (int l = q.r + q.step; l < n; l += q.step) {
                const Pack<T, V> v = *reinterpret_cast<const Pack<T, V>*>(x + (int64_t)l * p.xp + (int64_t)(c0 + q.col) * V);
#pragma unroll
                for (int j = 0; j < V; j++) {
                    const float d = to_float(v.v[j]) - pivot[j];
                    s[j] += d;
                    s2[j] = fmaf(d, d, s2[j]);
                }
            }
#pragma unroll
            for (int j = 0; j < V; j++) {
                const float m = cnt > 0.0f ? s[j] / cnt : 0.0f;
                part[(q.r * q.width + q.col) * V + j] = make_float2(pivot[j] + m, fmaxf(fmaf(-s[j], m, s2[j]), 0.0f) + 0.0f * s[j]);
            }
        }
        __syncthreads();
        // a warp per group of this tile: lanes join every 32nd of its (position, channel) parts
        const int ch0 = c0 * V, ch1 = ch0 + cols * V;
        for (int g = ch0 / p.cpg + warp; g * p.cpg < ch1; g += kThreads / 32) {
            const int a = max(g * p.cpg, ch0) - ch0, w = min((g + 1) * p.cpg, ch1) - ch0 - a;
            const int rows = min(q.step, n);
            Moments m{0.0f, 0.0f, 0.0f};
            for (int i = lane; i < rows * w; i += 32) {
                const int r = i / w, c = a + i - r * w;
                const float2 v = part[r * q.width * V + c];
                join(m, Moments{(float)((n - r + q.step - 1) / q.step), v.x, v.y});
            }
            warp_join(m);
            if (lane == 0) {
                if (g * p.cpg < ch0) { Moments t = group[g]; join(t, m); m = t; }   // began in the tile before
                group[g] = m;
            }
        }
        __syncthreads();
    }
    for (int g = threadIdx.x; g < p.groups; g += kThreads)
        p.part[((int64_t)b * p.groups + g) * p.chunks + chunk] = make_float2(group[g].mean, group[g].m2);
}

// One warp per (item, group): its chunks' moments, joined.
__global__ void __launch_bounds__(128) moments_join(const __grid_constant__ NormParams p) {
    const int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (i >= (int64_t)p.batch * p.groups) return;
    Moments m{0.0f, 0.0f, 0.0f};
    for (int c = lane; c < p.chunks; c += 32) {
        const float2 v = p.part[i * p.chunks + c];
        const float n = (float)min((int64_t)p.rows, p.positions - (int64_t)c * p.rows) * (float)p.cpg;
        join(m, Moments{n, v.x, v.y});
    }
    warp_join(m);
    if (lane == 0) {
        p.mean[i] = m.mean;
        p.rstd[i] = 1.0f / sqrtf(m.m2 / ((float)p.positions * (float)p.cpg) + p.eps);
    }
}

template <class T, int V, int ACT>
__global__ void __launch_bounds__(kThreads) apply_kernel(const __grid_constant__ NormParams p) {
    const int b = blockIdx.y, chunk = blockIdx.x;
    const int64_t l0 = (int64_t)chunk * p.rows;
    const int n = (int)min((int64_t)p.rows, p.positions - l0);
    const Place q = place(p);
    if (q.r >= q.step) return;
    constexpr bool fast = sizeof(T) == 2;
    for (int col = q.col; col < p.columns; col += q.width) {
        const int ch = col * V;
        float mu[V], a[V], sh[V];
#pragma unroll
        for (int j = 0; j < V; j++) {
            const int g = (ch + j) / p.cpg;
            mu[j] = p.mean[(int64_t)b * p.groups + g];
            a[j] = p.rstd[(int64_t)b * p.groups + g] * param(p.gamma, ch + j, p.param_float, 1.0f, (const T*)nullptr);
            sh[j] = param(p.beta, ch + j, p.param_float, 0.0f, (const T*)nullptr);
        }
        const T* x = static_cast<const T*>(p.x) + b * p.xb + l0 * p.xp + ch;
        T* y = static_cast<T*>(p.y) + b * p.yb + l0 * p.yp + ch;
#pragma unroll 4
        for (int l = q.r; l < n; l += q.step) {
            Pack<T, V> v = *reinterpret_cast<const Pack<T, V>*>(x + (int64_t)l * p.xp);
#pragma unroll
            for (int j = 0; j < V; j++) v.v[j] = from_float<T>(act<ACT, fast>(fmaf(to_float(v.v[j]) - mu[j], a[j], sh[j])));
            *reinterpret_cast<Pack<T, V>*>(y + (int64_t)l * p.yp) = v;
        }
    }
}

// ---- backward --------------------------------------------------------------------------------

// A chunk's sums of dz and dz xh per channel.
template <class T, int V, int ACT>
__global__ void __launch_bounds__(kThreads) grad_sums_kernel(const __grid_constant__ NormParams p) {
    __shared__ float2 part[kThreads * V];
    const int b = blockIdx.y, chunk = blockIdx.x;
    const int64_t l0 = (int64_t)chunk * p.rows;
    const int n = (int)min((int64_t)p.rows, p.positions - l0);
    const Place q = place(p);
    constexpr bool fast = sizeof(T) == 2;
    for (int c0 = 0; c0 < p.columns; c0 += q.width) {
        const int cols = min(q.width, p.columns - c0);
        if (q.r < q.step && q.col < cols) {
            const int ch = (c0 + q.col) * V;
            float mu[V], rs[V], ga[V], be[V], s1[V], s2[V];
#pragma unroll
            for (int j = 0; j < V; j++) {
                const int g = (ch + j) / p.cpg;
                mu[j] = p.mean[(int64_t)b * p.groups + g];
                rs[j] = p.rstd[(int64_t)b * p.groups + g];
                ga[j] = param(p.gamma, ch + j, p.param_float, 1.0f, (const T*)nullptr);
                be[j] = param(p.beta, ch + j, p.param_float, 0.0f, (const T*)nullptr);
                s1[j] = s2[j] = 0.0f;
            }
            const T* x = static_cast<const T*>(p.x) + b * p.xb + l0 * p.xp + ch;
            const T* dy = static_cast<const T*>(p.dy) + b * p.yb + l0 * p.yp + ch;
#pragma unroll 2
            for (int l = q.r; l < n; l += q.step) {
                const Pack<T, V> v = *reinterpret_cast<const Pack<T, V>*>(x + (int64_t)l * p.xp);
                const Pack<T, V> w = *reinterpret_cast<const Pack<T, V>*>(dy + (int64_t)l * p.yp);
#pragma unroll
                for (int j = 0; j < V; j++) {
                    const float xh = (to_float(v.v[j]) - mu[j]) * rs[j];
                    const float dz = to_float(w.v[j]) * act_grad<ACT, fast>(fmaf(xh, ga[j], be[j]));
                    s1[j] += dz;
                    s2[j] = fmaf(dz, xh, s2[j]);
                }
            }
#pragma unroll
            for (int j = 0; j < V; j++) part[(q.r * q.width + q.col) * V + j] = make_float2(s1[j], s2[j]);
        }
        __syncthreads();
        for (int c = threadIdx.x; c < cols * V; c += kThreads) {
            float2 t = make_float2(0.0f, 0.0f);
            for (int r = 0; r < q.step; r++) {
                const float2 v = part[r * q.width * V + c];
                t.x += v.x;
                t.y += v.y;
            }
            p.part[((int64_t)b * p.chunks + chunk) * p.channels + c0 * V + c] = t;
        }
        __syncthreads();
    }
}

// A warp per channel: every item's sums over its chunks, and their sums, dbeta and dgamma.
template <class T>
__global__ void __launch_bounds__(128) grad_join(const __grid_constant__ NormParams p) {
    const int c = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (c >= p.channels) return;
    float db = 0.0f, dg = 0.0f;
    for (int b = 0; b < p.batch; b++) {
        float s1 = 0.0f, s2 = 0.0f;
        for (int k = lane; k < p.chunks; k += 32) {
            const float2 v = p.part[((int64_t)b * p.chunks + k) * p.channels + c];
            s1 += v.x;
            s2 += v.y;
        }
        for (int o = 16; o > 0; o >>= 1) {
            s1 += __shfl_xor_sync(~0u, s1, o);
            s2 += __shfl_xor_sync(~0u, s2, o);
        }
        if (lane == 0) p.sums[(int64_t)b * p.channels + c] = make_float2(s1, s2);
        db += s1;
        dg += s2;
    }
    if (lane == 0) {
        if (p.dbeta) set_param(p.dbeta, c, p.param_float, db, (const T*)nullptr);
        if (p.dgamma) set_param(p.dgamma, c, p.param_float, dg, (const T*)nullptr);
    }
}

template <class T, int V, int ACT>
__global__ void __launch_bounds__(kThreads) grad_apply_kernel(const __grid_constant__ NormParams p) {
    extern __shared__ float2 mean_of[];   // [groups]: sum(d) / m, sum(d xh) / m
    const int b = blockIdx.y, chunk = blockIdx.x;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const float m = (float)p.positions * (float)p.cpg;
    for (int g = warp; g < p.groups; g += kThreads / 32) {
        float a = 0.0f, c = 0.0f;
        for (int k = lane; k < p.cpg; k += 32) {
            const int ch = g * p.cpg + k;
            const float2 s = p.sums[(int64_t)b * p.channels + ch];
            const float ga = param(p.gamma, ch, p.param_float, 1.0f, (const T*)nullptr);
            a = fmaf(ga, s.x, a);
            c = fmaf(ga, s.y, c);
        }
        for (int o = 16; o > 0; o >>= 1) {
            a += __shfl_xor_sync(~0u, a, o);
            c += __shfl_xor_sync(~0u, c, o);
        }
        if (lane == 0) mean_of[g] = make_float2(a / m, c / m);
    }
    __syncthreads();
    const int64_t l0 = (int64_t)chunk * p.rows;
    const int n = (int)min((int64_t)p.rows, p.positions - l0);
    const Place q = place(p);
    if (q.r >= q.step) return;
    constexpr bool fast = sizeof(T) == 2;
    for (int col = q.col; col < p.columns; col += q.width) {
        const int ch = col * V;
        float mu[V], rs[V], ga[V], be[V];
        float2 mo[V];
#pragma unroll
        for (int j = 0; j < V; j++) {
            const int g = (ch + j) / p.cpg;
            mu[j] = p.mean[(int64_t)b * p.groups + g];
            rs[j] = p.rstd[(int64_t)b * p.groups + g];
            ga[j] = param(p.gamma, ch + j, p.param_float, 1.0f, (const T*)nullptr);
            be[j] = param(p.beta, ch + j, p.param_float, 0.0f, (const T*)nullptr);
            mo[j] = mean_of[g];
        }
        const T* x = static_cast<const T*>(p.x) + b * p.xb + l0 * p.xp + ch;
        const T* dy = static_cast<const T*>(p.dy) + b * p.yb + l0 * p.yp + ch;
        T* dx = static_cast<T*>(p.dx) + b * p.db + l0 * p.dp + ch;
#pragma unroll 2
        for (int l = q.r; l < n; l += q.step) {
            const Pack<T, V> v = *reinterpret_cast<const Pack<T, V>*>(x + (int64_t)l * p.xp);
            const Pack<T, V> w = *reinterpret_cast<const Pack<T, V>*>(dy + (int64_t)l * p.yp);
            Pack<T, V> o;
#pragma unroll
            for (int j = 0; j < V; j++) {
                const float xh = (to_float(v.v[j]) - mu[j]) * rs[j];
                const float d = to_float(w.v[j]) * act_grad<ACT, fast>(fmaf(xh, ga[j], be[j])) * ga[j];
                o.v[j] = from_float<T>(rs[j] * (d - mo[j].x - xh * mo[j].y));
            }
            *reinterpret_cast<Pack<T, V>*>(dx + (int64_t)l * p.dp) = o;
        }
    }
}

// ---- host -------------------------------------------------------------------------------------

void check_config(const stg_group_norm_config* c) {
    check_sized(c, "group norm");
    check(valid_dtype(c->dtype), "group norm: unknown dtype");
    check(c->param_dtype == c->dtype || c->param_dtype == STG_F32, "group norm: param_dtype must be dtype or STG_F32");
    check(valid_activation(c->activation), "group norm: unknown activation");
    check(c->batch >= 0 && c->positions >= 0, "group norm: negative size");
    check(c->channels >= 1 && c->groups >= 1 && c->channels % c->groups == 0, "group norm: groups must divide channels");
    check(c->eps >= 0.0 && c->eps <= 1e30, "group norm: eps must not be negative");
    check(c->x_batch >= 0 && c->x_position >= 0 && c->y_batch >= 0 && c->y_position >= 0 && c->dx_batch >= 0 && c->dx_position >= 0,
          "group norm: negative stride");
    if (c->channels > kMaxChannels) fail(STG_UNSUPPORTED, "group norm: more than 8192 channels");
    if (c->batch > 65535) fail(STG_UNSUPPORTED, "group norm: more than 65535 items");
    if (c->positions > ((int64_t)1 << 40) / c->channels) fail(STG_UNSUPPORTED, "group norm: an item of more than 2^40 elements");
}

// An item's positions are cut so that the whole call has about four blocks per SM, each with at
// least 16 positions, and at most 1024 parts to join.
int chunks_of(const stg_group_norm_config& c) {
    const int64_t per_item = (148 * 4 + c.batch - 1) / std::max<int64_t>(c.batch, 1);
    const int64_t n = std::min<int64_t>({std::max<int64_t>(per_item, 1), (c.positions + 15) / 16, 1024});
    const int64_t rows = (c.positions + n - 1) / std::max<int64_t>(n, 1);
    return (int)((c.positions + rows - 1) / std::max<int64_t>(rows, 1));
}

struct NormLayout { size_t part = 0, sums = 0, stats = 0, bytes = 0; };
size_t up(size_t n) { return (n + 255) / 256 * 256; }
NormLayout layout_of(const stg_group_norm_config& c, bool backward) {
    NormLayout l;
    if (!c.batch || !c.positions) return l;
    const size_t chunks = (size_t)chunks_of(c);
    if (backward) {
        l.sums = up(sizeof(float2) * (size_t)c.batch * chunks * c.channels);
        l.bytes = l.sums + up(sizeof(float2) * (size_t)c.batch * c.channels);
    } else {
        l.stats = up(sizeof(float2) * (size_t)c.batch * chunks * c.groups);
        l.bytes = l.stats + 2 * up(sizeof(float) * (size_t)c.batch * c.groups);
    }
    return l;
}

NormParams params_of(const stg_group_norm_config& c) {
    NormParams p{};
    p.positions = c.positions;
    p.xb = c.x_batch; p.xp = c.x_position;
    p.yb = c.y_batch; p.yp = c.y_position;
    p.db = c.dx_batch; p.dp = c.dx_position;
    p.channels = c.channels;
    p.groups = c.groups;
    p.cpg = c.channels / c.groups;
    p.batch = (int)c.batch;
    p.eps = (float)c.eps;
    p.param_float = c.param_dtype == STG_F32;
    if (c.batch && c.positions) {
        p.chunks = chunks_of(c);
        const int64_t rows = (c.positions + p.chunks - 1) / p.chunks;
        if (rows > (1 << 30)) fail(STG_UNSUPPORTED, "group norm: too many positions");
        p.rows = (int)rows;
        p.chunks = (int)((c.positions + rows - 1) / rows);
    }
    return p;
}

template <class Fn> void with_activation(int a, Fn&& fn) {
    switch (a) {
        case STG_ACT_RELU: return fn(std::integral_constant<int, STG_ACT_RELU>{});
        case STG_ACT_SILU: return fn(std::integral_constant<int, STG_ACT_SILU>{});
        case STG_ACT_GELU: return fn(std::integral_constant<int, STG_ACT_GELU>{});
        case STG_ACT_SIGMOID: return fn(std::integral_constant<int, STG_ACT_SIGMOID>{});
        default: return fn(std::integral_constant<int, STG_ACT_NONE>{});
    }
}
// Widest (16 bytes) or scalar vectors, as sizes, strides and addresses allow.
template <class T, class Fn> void with_width(bool wide, NormParams& p, Fn&& fn) {
    constexpr int W = 16 / sizeof(T);
    p.columns = wide ? p.channels / W : p.channels;
    p.columns_div = FastDiv((uint32_t)std::min(p.columns, kThreads));
    if (wide) fn(std::integral_constant<int, W>{});
    else fn(std::integral_constant<int, 1>{});
}
bool wide_fits(const stg_group_norm_config& c, std::initializer_list<const void*> ptrs, std::initializer_list<int64_t> strides) {
    const int w = 16 / (int)elem_size(c.dtype);
    if (c.channels % w) return false;
    for (const void* q : ptrs) if (!aligned(q, 16)) return false;
    for (int64_t s : strides) if (s % w) return false;
    return true;
}
void check_output_strides(int64_t batch, int64_t positions, const stg_group_norm_config& c) {
    check((batch >= c.channels || c.batch <= 1) && (positions >= c.channels || c.positions <= 1), "group norm: an output's rows overlap");
}

} // namespace

} // namespace stg

extern "C" {

STG_API stg_status stg_group_norm_workspace(const stg_group_norm_config* c, int32_t backward, size_t* bytes) {
    return guard(nullptr, [&] {
        check_config(c);
        check(bytes && (backward == 0 || backward == 1), "group norm: null buffer");
        *bytes = layout_of(*c, backward != 0).bytes;
    });
}

STG_API stg_status stg_group_norm(stg_engine* e, const stg_group_norm_config* c, const void* d_x, const void* d_gamma,
                                  const void* d_beta, void* d_y, float* d_mean, float* d_rstd, void* d_ws, size_t ws_bytes,
                                  void* stream) {
    if (!e) return STG_INVALID_ARGUMENT;
    return guard(e, [&] {
        check_config(c);
        const size_t es = elem_size(c->dtype), ps = elem_size(c->param_dtype);
        check(!d_mean == !d_rstd, "group norm: mean and rstd go together");
        check(aligned(d_gamma, ps) && aligned(d_beta, ps) && aligned(d_mean, 4) && aligned(d_rstd, 4) && aligned(d_x, es) && aligned(d_y, es),
              "group norm: a buffer is not aligned to its elements");
        check_output_strides(c->y_batch, c->y_position, *c);
        if (!c->batch || !c->positions) return;
        check(d_x && d_y, "group norm: null buffer");
        const NormLayout lay = layout_of(*c, false);
        check(d_ws && aligned(d_ws, 256) && ws_bytes >= lay.bytes, "group norm: workspace is missing, unaligned or too small");
        NormParams p = params_of(*c);
        char* ws = static_cast<char*>(d_ws);
        p.x = d_x; p.y = d_y; p.gamma = d_gamma; p.beta = d_beta;
        p.part = reinterpret_cast<float2*>(ws);
        p.mean = d_mean ? d_mean : reinterpret_cast<float*>(ws + lay.stats);
        p.rstd = d_rstd ? d_rstd : p.mean + up(sizeof(float) * (size_t)c->batch * c->groups) / sizeof(float);
        const bool wide = wide_fits(*c, {d_x, d_y}, {c->x_batch, c->x_position, c->y_batch, c->y_position});
        DeviceScope scope(e);
        const cudaStream_t st = static_cast<cudaStream_t>(stream);
        const dim3 grid((unsigned)p.chunks, (unsigned)p.batch);
        with_dtype(c->dtype, [&](auto* tag) {
            using T = std::remove_pointer_t<decltype(tag)>;
            with_width<T>(wide, p, [&](auto v) {
                constexpr int V = decltype(v)::value;
                const size_t smem = sizeof(Moments) * (size_t)p.groups;
                if (smem + sizeof(float2) * kThreads * V > 48 * 1024)
                    cuda_check(cudaFuncSetAttribute(moments_kernel<T, V>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem), "group norm kernel");
                moments_kernel<T, V><<<grid, kThreads, smem, st>>>(p);
                moments_join<<<(unsigned)(((int64_t)p.batch * p.groups + 3) / 4), 128, 0, st>>>(p);
                with_activation(c->activation, [&](auto a) { apply_kernel<T, V, decltype(a)::value><<<grid, kThreads, 0, st>>>(p); });
            });
        });
        cuda_check(cudaGetLastError(), "group norm kernel");
    });
}

STG_API stg_status stg_group_norm_backward(stg_engine* e, const stg_group_norm_config* c, const void* d_dy, const void* d_x,
                                           const void* d_gamma, const void* d_beta, const float* d_mean, const float* d_rstd,
                                           void* d_dx, void* d_dgamma, void* d_dbeta, void* d_ws, size_t ws_bytes, void* stream) {
    if (!e) return STG_INVALID_ARGUMENT;
    return guard(e, [&] {
        check_config(c);
        const size_t es = elem_size(c->dtype), ps = elem_size(c->param_dtype);
        check(aligned(d_gamma, ps) && aligned(d_beta, ps) && aligned(d_dgamma, ps) && aligned(d_dbeta, ps) && aligned(d_mean, 4) &&
                  aligned(d_rstd, 4) && aligned(d_x, es) && aligned(d_dy, es) && aligned(d_dx, es),
              "group norm: a buffer is not aligned to its elements");
        check_output_strides(c->dx_batch, c->dx_position, *c);
        DeviceScope scope(e);
        const cudaStream_t st = static_cast<cudaStream_t>(stream);
        if (!c->batch || !c->positions) {   // sums over nothing
            if (d_dgamma) cuda_check(cudaMemsetAsync(d_dgamma, 0, ps * c->channels, st), "group norm memset");
            if (d_dbeta) cuda_check(cudaMemsetAsync(d_dbeta, 0, ps * c->channels, st), "group norm memset");
            return;
        }
        check(d_x && d_dy && d_mean && d_rstd, "group norm: null buffer");
        if (!d_dx && !d_dgamma && !d_dbeta) return;
        const NormLayout lay = layout_of(*c, true);
        check(d_ws && aligned(d_ws, 256) && ws_bytes >= lay.bytes, "group norm: workspace is missing, unaligned or too small");
        NormParams p = params_of(*c);
        char* ws = static_cast<char*>(d_ws);
        p.x = d_x; p.dy = d_dy; p.dx = d_dx; p.gamma = d_gamma; p.beta = d_beta;
        p.dgamma = d_dgamma; p.dbeta = d_dbeta;
        p.mean = const_cast<float*>(d_mean);
        p.rstd = const_cast<float*>(d_rstd);
        p.part = reinterpret_cast<float2*>(ws);
        p.sums = reinterpret_cast<float2*>(ws + lay.sums);
        const bool wide = wide_fits(*c, {d_x, d_dy, d_dx}, {c->x_batch, c->x_position, c->y_batch, c->y_position, c->dx_batch, c->dx_position});
        const dim3 grid((unsigned)p.chunks, (unsigned)p.batch);
        with_dtype(c->dtype, [&](auto* tag) {
            using T = std::remove_pointer_t<decltype(tag)>;
            with_width<T>(wide, p, [&](auto v) {
                constexpr int V = decltype(v)::value;
                with_activation(c->activation, [&](auto a) {
                    constexpr int A = decltype(a)::value;
                    grad_sums_kernel<T, V, A><<<grid, kThreads, 0, st>>>(p);
                    grad_join<T><<<(unsigned)((p.channels + 3) / 4), 128, 0, st>>>(p);
                    if (p.dx) {
                        const size_t smem = sizeof(float2) * (size_t)p.groups;
                        if (smem > 48 * 1024)
                            cuda_check(cudaFuncSetAttribute(grad_apply_kernel<T, V, A>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem), "group norm kernel");
                        grad_apply_kernel<T, V, A><<<grid, kThreads, smem, st>>>(p);
                    }
                });
            });
        });
        cuda_check(cudaGetLastError(), "group norm kernel");
    });
}

} // extern "C"
