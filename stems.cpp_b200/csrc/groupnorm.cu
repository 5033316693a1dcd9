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
// The floor is one read of x (and dy) and one write, so what a block has read for the statistics
// it keeps in shared memory for the second look, and one launch does both: the positions of
// an item are dealt to a set of blocks, each takes the moments of its share, the set meets, joins
// the moments in a fixed order and applies them.
//   - An item that fits the shared memory of up to eight blocks is a cluster's, which
//     meets in hardware and reads each other's moments there; items do not wait for each other.
//   - Larger items take all SMs (as many items at a time as fit the GPU's shared memory, at
//     least one) in a cooperative launch; what does not fit is read again, from L2 where it can be.
//   - Very many groups or channels, whose moments would themselves be much to exchange, take
//     three launches: moments, their joining, a second reading.
// A block's threads stand side by side along the channels (16-byte vectors, whole rows, so every
// sector is used whatever the group size) and step down the positions.
#include "layers.h"

#include <cooperative_groups.h>

namespace cg = cooperative_groups;

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
    int used;                        // chunks of an item that have a position: fewer only in a cluster
    int columns;                     // vectors of a row
    FastDiv columns_div;             // by min(columns, kThreads)
    float eps;
    int param_float;
    // one-launch kernels: items at a time, steps a thread keeps, blocks of an item (= chunks)
    int at_once, kept;
    int mono;                        // a vector's channels are of one group
};

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
        for (int k = lane; k < p.used; k += 32) {
            const float2 v = p.part[((int64_t)b * p.chunks + k) * p.channels + c];
            s1 += v.x;
            s2 += v.y;
        }
        for (int o = 16; o > 0; o >>= 1) {
            s1 += __shfl_xor_sync(~0u, s1, o);
            s2 += __shfl_xor_sync(~0u, s2, o);
        }
        if (lane == 0 && p.sums) p.sums[(int64_t)b * p.channels + c] = make_float2(s1, s2);
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

// ---- one launch -------------------------------------------------------------------------------

constexpr int kFused = 512;          // threads: with 1024 the registers do not hold a vector's sums
constexpr int kFusedGroups = 2048;   // most groups
constexpr int kClusterMost = 8;

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// The 8 bytes at the same place in another block of the cluster.
__device__ __forceinline__ float2 peer_read(const float2* p, int rank) {
    uint32_t a;
    float2 v;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(a) : "memory");
    return v;
}

struct Share { int item, chunk, n; int64_t l0; };
template <bool GRID> __device__ __forceinline__ Share share_of(const NormParams& p, int round) {
    Share s;
    const int slot = blockIdx.x / p.chunks;
    s.chunk = blockIdx.x - slot * p.chunks;
    s.item = GRID ? (slot < p.at_once ? round * p.at_once + slot : p.batch) : slot;
    s.l0 = (int64_t)s.chunk * p.rows;
    s.n = s.item < p.batch ? (int)min((int64_t)p.rows, p.positions - s.l0) : 0;
    return s;
}

// Moments of the block's groups from its threads' parts: [step][row] of them, of `per` channels each,
// mean and M2 of the rows that place r has. The mean of the means first, then the deviations from
// it, both from the group's first part on; several warps to a group when groups are few.
__device__ __forceinline__ void block_moments(const NormParams& p, const Place& q, int n, const float2* part, int vec, float2* group, float2* red) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = kFused / 32;
    const int per = p.mono ? vec : 1, row = p.channels / per, w = p.cpg / per;   // parts of a row, of a group in a row
    const int rows = min(q.step, n), team = max(1, warps / p.groups);
    const int base = n / q.step, more = n - base * q.step;       // place r has base rows, and one more below `more`
    const int member = warp % team, lead = member * 32 + lane;
    const int r0 = lead / w, c0 = lead - r0 * w, dr = team * 32 / w, dc = team * 32 - dr * w;
    const float inv = 1.0f / ((float)n * (float)p.cpg);
    for (int g0 = 0; g0 < p.groups; g0 += warps / team) {
        const int g = g0 + warp / team;
        const bool live = g < p.groups && warp < warps / team * team;
        const float2* at = part + g * w;
        const float from = live ? at[0].x : 0.0f;
        float mean = 0.0f;
        for (int pass = 0; pass < 2; pass++) {
            float sum = 0.0f;
            if (live)
                for (int r = r0, c = c0; r < rows;) {
                    const float2 v = at[r * row + c];
                    const float cnt = (float)((base + (r < more)) * per), d = v.x - from - mean;
                    sum += pass ? fmaf(cnt * d, d, v.y) : cnt * d;
                    r += dr;
                    if ((c += dc) >= w) { c -= w; r++; }
                }
            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
            if (team > 1) {   // then every group has its team at once: one round
                if (lane == 0) reinterpret_cast<float*>(red)[warp] = sum;
                __syncthreads();
                sum = 0.0f;
                if (live)
                    for (int k = 0; k < team; k++) sum += reinterpret_cast<float*>(red)[warp - member + k];
                __syncthreads();
            }
            if (pass == 0) mean = sum * inv;
            else if (live && member == 0 && lane == 0) group[g] = make_float2(from + mean, sum);
        }
    }
    __syncthreads();
}

template <class T, int V, int ACT, bool GRID>
__global__ void __launch_bounds__(kFused, 1) norm_fused(const __grid_constant__ NormParams p) {
    constexpr bool fast = sizeof(T) == 2;
    constexpr int U = 8, N = (V + 1) / 2;       // positions in flight per thread, pairs of a vector
    using P = Pack<T, V>;
    extern __shared__ __align__(16) uint8_t smem[];
    P* keep = reinterpret_cast<P*>(smem);       // [kept][threads]
    float2* part = reinterpret_cast<float2*>(smem + (size_t)p.kept * kFused * sizeof(P));
    float2* group = part + kFused * (p.mono ? 1 : V);   // [groups]: the block's moments
    float2* stat = group + p.groups;                    // [groups]: the item's mean and rstd
    __shared__ float2 red[kFused / 64];
    Place q;
    q.width = p.columns;
    q.step = kFused / q.width;
    q.r = (int)p.columns_div.div(threadIdx.x);
    q.col = threadIdx.x - q.r * q.width;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, ch = q.col * V;
    const bool on = q.r < q.step;
    const int rounds = GRID ? (p.batch + p.at_once - 1) / p.at_once : 1;
    for (int round = 0; round < rounds; round++) {
        const Share s = share_of<GRID>(p, round);
        const T* x = static_cast<const T*>(p.x) + s.item * p.xb + s.l0 * p.xp + ch;
        if (s.n > 0) {
            if (on && q.r < s.n) {
                // differences from the first value met, so that a mean far from zero costs no digits
                f2 pivot[N], a[N], b[N];
                const T* at = x + (int64_t)q.r * p.xp;
                {
                    const P first = *reinterpret_cast<const P*>(at);
#pragma unroll
                    for (int i = 0; i < N; i++) {
                        const float2 f = split(get(first, i)), f0 = split(get(first, 0));
                        pivot[i] = p.mono ? make_f2(-f0.x, -f0.x) : make_f2(-f.x, -f.y);
                        a[i] = b[i] = make_f2(0.0f, 0.0f);
                    }
                }
                const int64_t step = (int64_t)q.step * p.xp;
                const int mine = (s.n - q.r + q.step - 1) / q.step;
                auto take = [&](const P& v) {
#pragma unroll
                    for (int i = 0; i < N; i++) {
                        const f2 d = get(v, i) + pivot[i];
                        a[i] = a[i] + d;
                        b[i] = fma2(d, d, b[i]);
                    }
                };
                int it = 0;
                P* k = keep + threadIdx.x;
                for (; it + U <= min(mine, p.kept); it += U, k += U * kFused) {
                    P v[U];
#pragma unroll
                    for (int u = 0; u < U; u++, at += step) v[u] = *reinterpret_cast<const P*>(at);
#pragma unroll
                    for (int u = 0; u < U; u++) {
                        k[u * kFused] = v[u];
                        take(v[u]);
                    }
                }
                for (; it < mine; it += U) {
                    P v[U];
#pragma unroll
                    for (int u = 0; u < U; u++, at += step)
                        if (it + u < mine) v[u] = *reinterpret_cast<const P*>(at);
#pragma unroll
                    for (int u = 0; u < U; u++) {
                        if (it + u >= mine) break;
                        if (it + u < p.kept) keep[(it + u) * kFused + threadIdx.x] = v[u];
                        take(v[u]);
                    }
                }
                auto moments = [&](float sum, float sq, float n, float neg) {   // + 0 sum: a NaN stays one
                    const float m = sum / n;
                    return make_float2(m - neg, fmaxf(fmaf(-sum, m, sq), 0.0f) + 0.0f * sum);
                };
                if (V == 1) {
                    part[q.r * q.width + q.col] = moments(split(a[0]).x, split(b[0]).x, (float)mine, split(pivot[0]).x);
                } else if (p.mono) {
#pragma unroll
                    for (int i = 1; i < N; i++) { a[0] = a[0] + a[i]; b[0] = b[0] + b[i]; }
                    const float2 sa = split(a[0]), sb = split(b[0]);
                    part[q.r * q.width + q.col] = moments(sa.x + sa.y, sb.x + sb.y, (float)mine * V, split(pivot[0]).x);
                } else {
#pragma unroll
                    for (int i = 0; i < N; i++) {
                        const float2 sa = split(a[i]), sb = split(b[i]), sp = split(pivot[i]);
                        float2* to = part + (q.r * q.width + q.col) * V + 2 * i;
                        to[0] = moments(sa.x, sb.x, (float)mine, sp.x);
                        to[1] = moments(sa.y, sb.y, (float)mine, sp.y);
                    }
                }
            }
            __syncthreads();
            block_moments(p, q, s.n, part, V, group, red);
            if (GRID)
                for (int g = threadIdx.x; g < p.groups; g += kFused) p.part[((int64_t)s.item * p.groups + g) * p.chunks + s.chunk] = group[g];
        }
        __syncwarp();
        if (GRID) cg::this_grid().sync();
        else {
            cluster_arrive();
            cluster_wait();
        }
        if (s.n > 0) {
            for (int g = warp; g < p.groups; g += kFused / 32) {
                Moments m{0.0f, 0.0f, 0.0f};
                for (int c = lane; c < p.used; c += 32) {
                    const float n = (float)min((int64_t)p.rows, p.positions - (int64_t)c * p.rows) * (float)p.cpg;
                    const float2 v = GRID ? __ldcg(p.part + ((int64_t)s.item * p.groups + g) * p.chunks + c) : peer_read(group + g, c);
                    join(m, Moments{n, v.x, v.y});
                }
                warp_join(m);
                if (lane == 0) {
                    const float r = 1.0f / sqrtf(m.m2 / ((float)p.positions * (float)p.cpg) + p.eps);
                    stat[g] = make_float2(m.mean, r);
                    if (s.chunk == 0 && p.mean) {
                        p.mean[(int64_t)s.item * p.groups + g] = m.mean;
                        p.rstd[(int64_t)s.item * p.groups + g] = r;
                    }
                }
            }
        }
        __syncwarp();
        if (!GRID) cluster_arrive();   // waited for below: no block goes while others still read its moments
        __syncthreads();
        if (s.n > 0 && on) {
            // z = (x - mu) a + sh. For 16-bit x as x a + (sh - mu a): what that rounds, 2^-24 of mu a, is far
            // below the 2^-9 (2^-12) of mu a that x itself was rounded by.
            f2 mu[N], a[N], sh[N];
#pragma unroll
            for (int i = 0; i < N; i++) {
                float m[2], s1[2], s0[2];
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    const int c = V == 1 ? ch : ch + 2 * i + k;
                    const float2 st = stat[c / p.cpg];
                    m[k] = -st.x;
                    s1[k] = st.y * param(p.gamma, c, p.param_float, 1.0f, (const T*)nullptr);
                    s0[k] = param(p.beta, c, p.param_float, 0.0f, (const T*)nullptr);
                    if (fast) s0[k] = fmaf(m[k], s1[k], s0[k]);
                }
                mu[i] = make_f2(m[0], m[1]);
                a[i] = make_f2(s1[0], s1[1]);
                sh[i] = make_f2(s0[0], s0[1]);
            }
            const PairAct<ACT, fast> fn;
            const int64_t sx = (int64_t)q.step * p.xp, sy = (int64_t)q.step * p.yp;
            auto one = [&](P v, T* y) {
#pragma unroll
                for (int i = 0; i < N; i++) {
                    const f2 f = get(v, i);
                    put(v, i, fn.value(fma2(fast ? f : f + mu[i], a[i], sh[i])));
                }
                *reinterpret_cast<P*>(y) = v;
            };
            const int mine = q.r < s.n ? (s.n - q.r + q.step - 1) / q.step : 0;
            // what was read last and not kept is in L2 yet: from the end
            int it = mine - 1;
            const T* at = x + (q.r + (int64_t)it * q.step) * p.xp;
            T* y = static_cast<T*>(p.y) + s.item * p.yb + s.l0 * p.yp + ch + (q.r + (int64_t)it * q.step) * p.yp;
            constexpr int W = 4;
            for (; it >= p.kept; it -= W) {
                P v[W];
#pragma unroll
                for (int u = 0; u < W; u++, at -= sx)
                    if (it - u >= p.kept) v[u] = *reinterpret_cast<const P*>(at);
#pragma unroll
                for (int u = 0; u < W; u++)
                    if (it - u >= p.kept) {
                        one(v[u], y);
                        y -= sy;
                    }
            }
            const P* k = keep + min(mine, p.kept) * kFused + threadIdx.x;
#pragma unroll 2
            for (it = min(mine, p.kept); it > 0; it--, y -= sy) one(*(k -= kFused), y);
        }
        if (GRID) __syncthreads();   // stat and the kept values are the next round's
        else {
            __syncwarp();
            cluster_wait();
        }
    }
}

// Backward: the block's sums of dz and dz xh per channel, of gamma times them per group; the set's
// blocks meet over the group sums. Channel sums go out per block for dgamma and dbeta.
template <class T, int V, int ACT, bool GRID>
__global__ void __launch_bounds__(kFused, 1) norm_grad_fused(const __grid_constant__ NormParams p) {
    constexpr bool fast = sizeof(T) == 2;
    constexpr int U = 4, N = (V + 1) / 2;
    const PairAct<ACT, fast> fn;
    using P = Pack<T, V>;
    extern __shared__ __align__(16) uint8_t smem[];
    P* keep = reinterpret_cast<P*>(smem);       // [kept][x, dy][threads]
    float2* part = reinterpret_cast<float2*>(smem + (size_t)p.kept * 2 * kFused * sizeof(P));   // [step][channels]
    float2* chan = part + kFused * V;           // [channels]
    float2* group = chan + p.channels;          // [groups]: the block's sums
    float2* stat = group + p.groups;            // [groups]: the item's means of d and d xh
    Place q;
    q.width = p.columns;
    q.step = kFused / q.width;
    q.r = (int)p.columns_div.div(threadIdx.x);
    q.col = threadIdx.x - q.r * q.width;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, ch = q.col * V;
    const bool on = q.r < q.step;
    const int rounds = GRID ? (p.batch + p.at_once - 1) / p.at_once : 1;
    for (int round = 0; round < rounds; round++) {
        const Share s = share_of<GRID>(p, round);
        const T* x = static_cast<const T*>(p.x) + s.item * p.xb + s.l0 * p.xp + ch;
        const T* dy = static_cast<const T*>(p.dy) + s.item * p.yb + s.l0 * p.yp + ch;
        // z = (x - mu) za + zb; the sums are of dz and dz (x - mu), the latter scaled by rstd at the end
        f2 mu[N], za[N], zb[N];
        const int mine = q.r < s.n ? (s.n - q.r + q.step - 1) / q.step : 0;
        const int64_t sx = (int64_t)q.step * p.xp, sd = (int64_t)q.step * p.yp;
        if (s.n > 0) {
            if (on) {
                f2 a[N], b[N];
                float rs[2 * N];
#pragma unroll
                for (int i = 0; i < N; i++) {
                    float m[2], s1[2], s0[2];
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        const int c = V == 1 ? ch : ch + 2 * i + k;
                        const int64_t g = (int64_t)s.item * p.groups + c / p.cpg;
                        m[k] = -p.mean[g];
                        rs[2 * i + k] = p.rstd[g];
                        s1[k] = rs[2 * i + k] * param(p.gamma, c, p.param_float, 1.0f, (const T*)nullptr);
                        s0[k] = param(p.beta, c, p.param_float, 0.0f, (const T*)nullptr);
                    }
                    mu[i] = make_f2(m[0], m[1]);
                    za[i] = make_f2(s1[0], s1[1]);
                    zb[i] = make_f2(s0[0], s0[1]);
                    a[i] = b[i] = make_f2(0.0f, 0.0f);
                }
                auto take = [&](const P& v, const P& w) {
#pragma unroll
                    for (int i = 0; i < N; i++) {
                        const f2 xm = get(v, i) + mu[i];
                        const f2 dz = get(w, i) * fn.slope(fma2(xm, za[i], zb[i]));
                        a[i] = a[i] + dz;
                        b[i] = fma2(dz, xm, b[i]);
                    }
                };
                const T *ax = x + (int64_t)q.r * p.xp, *ad = dy + (int64_t)q.r * p.yp;
                int it = 0;
                P* k = keep + threadIdx.x;
                for (; it + U <= min(mine, p.kept); it += U, k += U * 2 * kFused) {
                    P v[U], w[U];
#pragma unroll
                    for (int u = 0; u < U; u++, ax += sx, ad += sd) {
                        v[u] = *reinterpret_cast<const P*>(ax);
                        w[u] = *reinterpret_cast<const P*>(ad);
                    }
#pragma unroll
                    for (int u = 0; u < U; u++) {
                        k[u * 2 * kFused] = v[u];
                        k[u * 2 * kFused + kFused] = w[u];
                        take(v[u], w[u]);
                    }
                }
                for (; it < mine; it++, ax += sx, ad += sd) {
                    const P v = *reinterpret_cast<const P*>(ax), w = *reinterpret_cast<const P*>(ad);
                    if (it < p.kept) {
                        keep[it * 2 * kFused + threadIdx.x] = v;
                        keep[it * 2 * kFused + kFused + threadIdx.x] = w;
                    }
                    take(v, w);
                }
#pragma unroll
                for (int j = 0; j < V; j++) {
                    const float2 sa = split(a[j / 2]), sb = split(b[j / 2]);
                    part[(q.r * q.width + q.col) * V + j] = make_float2(j & 1 ? sa.y : sa.x, (j & 1 ? sb.y : sb.x) * rs[j]);
                }
            }
            __syncthreads();
            for (int c = threadIdx.x; c < p.channels; c += kFused) {
                float2 t = make_float2(0.0f, 0.0f);
                for (int r = 0; r < q.step; r++) {
                    const float2 v = part[r * p.channels + c];
                    t.x += v.x;
                    t.y += v.y;
                }
                chan[c] = t;
                p.part[((int64_t)s.item * p.chunks + s.chunk) * p.channels + c] = t;
            }
            __syncthreads();
            for (int g = warp; g < p.groups; g += kFused / 32) {
                float a = 0.0f, b = 0.0f;
                for (int k = lane; k < p.cpg; k += 32) {
                    const int c = g * p.cpg + k;
                    const float gc = param(p.gamma, c, p.param_float, 1.0f, (const T*)nullptr);
                    a = fmaf(gc, chan[c].x, a);
                    b = fmaf(gc, chan[c].y, b);
                }
                for (int o = 16; o > 0; o >>= 1) {
                    a += __shfl_xor_sync(~0u, a, o);
                    b += __shfl_xor_sync(~0u, b, o);
                }
                if (lane == 0) {
                    group[g] = make_float2(a, b);
                    if (GRID) p.sums[((int64_t)s.item * p.groups + g) * p.chunks + s.chunk] = make_float2(a, b);
                }
            }
        }
        __syncwarp();
        if (GRID) cg::this_grid().sync();
        else {
            cluster_arrive();
            cluster_wait();
        }
        if (s.n > 0 && p.dx) {
            const float m = (float)p.positions * (float)p.cpg;
            for (int g = warp; g < p.groups; g += kFused / 32) {
                float a = 0.0f, b = 0.0f;
                for (int c = lane; c < p.used; c += 32) {
                    const float2 v = GRID ? __ldcg(p.sums + ((int64_t)s.item * p.groups + g) * p.chunks + c) : peer_read(group + g, c);
                    a += v.x;
                    b += v.y;
                }
                for (int o = 16; o > 0; o >>= 1) {
                    a += __shfl_xor_sync(~0u, a, o);
                    b += __shfl_xor_sync(~0u, b, o);
                }
                if (lane == 0) stat[g] = make_float2(a / m, b / m);
            }
        }
        __syncwarp();
        if (!GRID) cluster_arrive();
        __syncthreads();
        if (s.n > 0 && p.dx && on) {
            // dx = rstd gamma dz - (x - mu) rstd^2 mean(d xh) - rstd mean(d)
            f2 c1[N], c2[N];
#pragma unroll
            for (int i = 0; i < N; i++) {
                float u1[2], u2[2];
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    const int g = (V == 1 ? ch : ch + 2 * i + k) / p.cpg;
                    const float r = p.rstd[(int64_t)s.item * p.groups + g];
                    u1[k] = -r * stat[g].x;
                    u2[k] = -r * r * stat[g].y;
                }
                c1[i] = make_f2(u1[0], u1[1]);
                c2[i] = make_f2(u2[0], u2[1]);
            }
            auto one = [&](const P& v, const P& w, T* dx) {
                P o;
#pragma unroll
                for (int i = 0; i < N; i++) {
                    const f2 xm = get(v, i) + mu[i];
                    const f2 dz = get(w, i) * fn.slope(fma2(xm, za[i], zb[i]));
                    put(o, i, fma2(dz, za[i], fma2(xm, c2[i], c1[i])));
                }
                *reinterpret_cast<P*>(dx) = o;
            };
            int it = mine - 1;
            const int64_t last = q.r + (int64_t)it * q.step, so = (int64_t)q.step * p.dp;
            const T *ax = x + last * p.xp, *ad = dy + last * p.yp;
            T* dx = static_cast<T*>(p.dx) + s.item * p.db + (s.l0 + last) * p.dp + ch;
            constexpr int W = 2;
            for (; it >= p.kept; it -= W) {
                P v[W], w[W];
#pragma unroll
                for (int u = 0; u < W; u++, ax -= sx, ad -= sd)
                    if (it - u >= p.kept) {
                        v[u] = *reinterpret_cast<const P*>(ax);
                        w[u] = *reinterpret_cast<const P*>(ad);
                    }
#pragma unroll
                for (int u = 0; u < W; u++)
                    if (it - u >= p.kept) {
                        one(v[u], w[u], dx);
                        dx -= so;
                    }
            }
            const P* k = keep + min(mine, p.kept) * 2 * kFused + threadIdx.x;
            for (it = min(mine, p.kept); it > 0; it--, dx -= so) {
                k -= 2 * kFused;
                one(k[0], k[kFused], dx);
            }
        }
        if (GRID) __syncthreads();
        else {
            __syncwarp();
            cluster_wait();
        }
    }
    if (GRID && (p.dgamma || p.dbeta)) {   // every item's parts were complete at the last meeting
        const int all = (int)gridDim.x * (kFused / 32);
        for (int c = blockIdx.x * (kFused / 32) + warp; c < p.channels; c += all) {
            float a = 0.0f, b = 0.0f;
            for (int k = lane; k < p.batch * p.chunks; k += 32) {
                const float2 v = __ldcg(p.part + (int64_t)k * p.channels + c);
                a += v.x;
                b += v.y;
            }
            for (int o = 16; o > 0; o >>= 1) {
                a += __shfl_xor_sync(~0u, a, o);
                b += __shfl_xor_sync(~0u, b, o);
            }
            if (lane == 0) {
                if (p.dbeta) set_param(p.dbeta, c, p.param_float, a, (const T*)nullptr);
                if (p.dgamma) set_param(p.dgamma, c, p.param_float, b, (const T*)nullptr);
            }
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

size_t up(size_t n) { return (n + 255) / 256 * 256; }

enum Path { THREE_LAUNCHES, CLUSTER, GRID };
// How a call runs with vectors of `vec` channels on `sms` SMs, and the scratch it takes.
struct NormPlan {
    Path path = THREE_LAUNCHES;
    int chunks = 0, at_once = 1, kept = 0;
    int64_t rows = 0;
    size_t smem = 0;
    size_t second = 0, third = 0, bytes = 0;   // offsets of the scratch's parts
};
NormPlan plan_of(const stg_group_norm_config& c, bool backward, int vec, int sms) {
    NormPlan r;
    if (!c.batch || !c.positions) return r;
    const int columns = c.channels / vec, cpg = c.channels / c.groups;
    const size_t vb = (size_t)vec * elem_size(c.dtype) * (backward ? 2 : 1), block_step = vb * kFused;
    const bool mono = cpg % vec == 0;
    // shared memory besides the kept values: the threads' parts, channel and group sums
    const size_t other = backward ? sizeof(float2) * ((size_t)kFused * vec + c.channels + 2 * (size_t)c.groups)
                                  : sizeof(float2) * ((size_t)kFused * (mono ? 1 : vec) + 2 * (size_t)c.groups);
    const size_t most = 225 * 1024;
    if (columns <= kFused && c.groups <= kFusedGroups && other + 8 * block_step <= most) {
        const int64_t step = kFused / columns, room = (int64_t)((most - other) / block_step);   // steps a block can keep
        const int64_t item_steps = (c.positions + step - 1) / step;
        int64_t blocks = (item_steps + room - 1) / room;
        if (blocks <= kClusterMost) {
            // as many blocks as fill the GPU once, each with at least four steps
            int64_t size = 1;
            while (size < kClusterMost && (size < blocks || (size * 2 * c.batch <= sms && size * 8 <= item_steps))) size *= 2;
            r.path = CLUSTER;
            r.chunks = (int)size;
            r.rows = (c.positions + size - 1) / size;
            r.kept = (int)((r.rows + step - 1) / step);
        } else {
            r.at_once = (int)std::max<int64_t>(1, std::min<int64_t>(c.batch, sms * room / item_steps));
            const int64_t per = sms / r.at_once;
            if (per * c.groups <= 32768) {   // what every block reads of the others' sums: at most 256 KB
                r.path = GRID;
                r.rows = (c.positions + per - 1) / per;
                r.chunks = (int)((c.positions + r.rows - 1) / r.rows);
                r.kept = (int)std::min<int64_t>(room, (r.rows + step - 1) / step);
            }
        }
        if (r.path != THREE_LAUNCHES && r.rows <= (1 << 30)) {
            r.smem = other + (size_t)r.kept * block_step;
            const size_t sets = (size_t)c.batch * r.chunks;
            if (backward) {
                r.second = up(sizeof(float2) * sets * c.channels);
                r.bytes = r.second + (r.path == GRID ? up(sizeof(float2) * sets * c.groups) : 0);
            } else r.bytes = r.path == GRID ? up(sizeof(float2) * sets * c.groups) : 0;
            return r;
        }
    }
    r = NormPlan{};
    r.chunks = chunks_of(c);
    r.rows = (c.positions + r.chunks - 1) / r.chunks;
    if (r.rows > (1 << 30)) fail(STG_UNSUPPORTED, "group norm: too many positions");
    if (backward) {
        r.second = up(sizeof(float2) * (size_t)c.batch * r.chunks * c.channels);
        r.bytes = r.second + up(sizeof(float2) * (size_t)c.batch * c.channels);
    } else {
        r.second = up(sizeof(float2) * (size_t)c.batch * r.chunks * c.groups);
        r.third = r.second + up(sizeof(float) * (size_t)c.batch * c.groups);
        r.bytes = r.third + up(sizeof(float) * (size_t)c.batch * c.groups);
    }
    return r;
}
constexpr int kSms = 148;
// Enough for either vector width: which one a call can use its buffers' addresses decide.
size_t workspace_of(const stg_group_norm_config& c, bool backward) {
    size_t n = plan_of(c, backward, 1, kSms).bytes;
    const int w = 16 / (int)elem_size(c.dtype);
    if (c.channels % w == 0) n = std::max(n, plan_of(c, backward, w, kSms).bytes);
    return n;
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
    return p;
}

// Widest (16 bytes) or scalar vectors, as sizes, strides and addresses allow.
template <class T, class Fn> void with_width(bool wide, Fn&& fn) {
    if (wide) fn(std::integral_constant<int, 16 / (int)sizeof(T)>{});
    else fn(std::integral_constant<int, 1>{});
}
void set_plan(NormParams& p, const NormPlan& plan, int vec, int fused) {
    p.columns = p.channels / vec;
    p.columns_div = FastDiv((uint32_t)std::min(p.columns, plan.path == THREE_LAUNCHES ? kThreads : fused));
    p.chunks = plan.chunks;
    p.rows = (int)plan.rows;
    p.used = (int)((p.positions + plan.rows - 1) / plan.rows);
    p.at_once = plan.at_once;
    p.kept = plan.kept;
    p.mono = p.cpg % vec == 0;
}
template <class K> void launch_fused(K kernel, const NormParams& p, const NormPlan& plan, int threads, cudaStream_t st) {
    cuda_check(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)plan.smem), "group norm kernel");
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr[1];
    const int64_t blocks = plan.path == GRID ? (int64_t)plan.at_once * plan.chunks : (int64_t)p.batch * plan.chunks;
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = plan.smem;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (plan.path == GRID) {
        attr[0].id = cudaLaunchAttributeCooperative;
        attr[0].val.cooperative = 1;
    } else {
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = plan.chunks;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    }
    cuda_check(cudaLaunchKernelEx(&cfg, kernel, p), "group norm kernel");
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
        *bytes = workspace_of(*c, backward != 0);
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
        const bool wide = wide_fits(*c, {d_x, d_y}, {c->x_batch, c->x_position, c->y_batch, c->y_position});
        const NormPlan plan = plan_of(*c, false, wide ? 16 / (int)es : 1, std::min(e->sms, kSms));
        check(!plan.bytes || (d_ws && aligned(d_ws, 256) && ws_bytes >= plan.bytes), "group norm: workspace is missing, unaligned or too small");
        NormParams p = params_of(*c);
        char* ws = static_cast<char*>(d_ws);
        p.x = d_x; p.y = d_y; p.gamma = d_gamma; p.beta = d_beta;
        p.part = reinterpret_cast<float2*>(ws);
        p.mean = d_mean;
        p.rstd = d_rstd;
        DeviceScope scope(e);
        const cudaStream_t st = static_cast<cudaStream_t>(stream);
        with_dtype(c->dtype, [&](auto* tag) {
            using T = std::remove_pointer_t<decltype(tag)>;
            with_width<T>(wide, [&](auto v) {
                constexpr int V = decltype(v)::value;
                set_plan(p, plan, V, kFused);
                with_activation(c->activation, [&](auto a) {
                    constexpr int A = decltype(a)::value;
                    if (plan.path == CLUSTER) return launch_fused(norm_fused<T, V, A, false>, p, plan, kFused, st);
                    if (plan.path == GRID) return launch_fused(norm_fused<T, V, A, true>, p, plan, kFused, st);
                    if (!p.mean) {
                        p.mean = reinterpret_cast<float*>(ws + plan.second);
                        p.rstd = reinterpret_cast<float*>(ws + plan.third);
                    }
                    const dim3 grid((unsigned)p.chunks, (unsigned)p.batch);
                    const size_t smem = sizeof(Moments) * (size_t)p.groups;
                    if (smem + sizeof(float2) * kThreads * V > 48 * 1024)
                        cuda_check(cudaFuncSetAttribute(moments_kernel<T, V>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem), "group norm kernel");
                    moments_kernel<T, V><<<grid, kThreads, smem, st>>>(p);
                    moments_join<<<(unsigned)(((int64_t)p.batch * p.groups + 3) / 4), 128, 0, st>>>(p);
                    apply_kernel<T, V, A><<<grid, kThreads, 0, st>>>(p);
                });
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
        const bool wide = wide_fits(*c, {d_x, d_dy, d_dx}, {c->x_batch, c->x_position, c->y_batch, c->y_position, c->dx_batch, c->dx_position});
        const NormPlan plan = plan_of(*c, true, wide ? 16 / (int)es : 1, std::min(e->sms, kSms));
        check(d_ws && aligned(d_ws, 256) && ws_bytes >= plan.bytes, "group norm: workspace is missing, unaligned or too small");
        NormParams p = params_of(*c);
        char* ws = static_cast<char*>(d_ws);
        p.x = d_x; p.dy = d_dy; p.dx = d_dx; p.gamma = d_gamma; p.beta = d_beta;
        p.dgamma = d_dgamma; p.dbeta = d_dbeta;
        p.mean = const_cast<float*>(d_mean);
        p.rstd = const_cast<float*>(d_rstd);
        p.part = reinterpret_cast<float2*>(ws);
        p.sums = plan.path == CLUSTER ? nullptr : reinterpret_cast<float2*>(ws + plan.second);
        with_dtype(c->dtype, [&](auto* tag) {
            using T = std::remove_pointer_t<decltype(tag)>;
            with_width<T>(wide, [&](auto v) {
                constexpr int V = decltype(v)::value;
                set_plan(p, plan, V, kFused);
                with_activation(c->activation, [&](auto a) {
                    constexpr int A = decltype(a)::value;
                    const unsigned join_blocks = (unsigned)((p.channels + 3) / 4);
                    if (plan.path == CLUSTER) {
                        launch_fused(norm_grad_fused<T, V, A, false>, p, plan, kFused, st);
                        if (p.dgamma || p.dbeta) grad_join<T><<<join_blocks, 128, 0, st>>>(p);
                        return;
                    }
                    if (plan.path == GRID) return launch_fused(norm_grad_fused<T, V, A, true>, p, plan, kFused, st);
                    const dim3 grid((unsigned)p.chunks, (unsigned)p.batch);
                    grad_sums_kernel<T, V, A><<<grid, kThreads, 0, st>>>(p);
                    grad_join<T><<<join_blocks, 128, 0, st>>>(p);
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
