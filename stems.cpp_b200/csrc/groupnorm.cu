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
// The floor is one read of x (and dy) and one write.
//   - An item that fits the shared memory of up to eight blocks is a cluster's: each block keeps
//     its positions in shared memory, the blocks meet in hardware and read each other's moments
//     there. One launch, one read, and items do not wait for each other.
//   - Larger items take three launches: moments by block, their joining, and a second reading in the
//     opposite order, so that what the first left in L2 is met there. A cooperative launch that
//     kept 26 MB in the SMs' shared memory instead stood still at each item's meeting: 121 us for
//     4 x 172032 x 96 bf16.
// Measured: 4 x 172032 x 96 bf16 with GELU 88 us (264 MB at least; read twice, the second time half from
// L2, 326 MB): moments 30 us at 4.7 TB/s, the second reading 58 us, which issues in 52 % of its cycles
// (14 instructions a value, mostly the activation's) and waits about evenly for the arithmetic and
// for loads in the rest, with 14 warps per SM. Its backward pass at 2 x 43008 x 192 f32 with SiLU 64 us
// (198 MB at least; both readings at 4.7 TB/s and 40 % issue, waiting for loads), one row of 336 x 48 f32 7.7 us.
// A block's threads stand side by side along the channels (16-byte vectors, whole rows, so every
// sector is used whatever the group size) and step down the positions. Each takes the differences
// from a pivot near its mean (Sums), so that neither a mean far from zero nor an outlier costs digits.
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
    int used;                        // chunks of an item that have a position: fewer only in a cluster
    int columns;                     // vectors of a row
    FastDiv columns_div;             // by min(columns, kThreads)
    float eps;
    int param_float;
    int kept;                        // cluster: steps a thread keeps
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
template <int LANES = 32> __device__ __forceinline__ void warp_join(Moments& a) {
    for (int o = LANES / 2; o > 0; o >>= 1) {
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
__device__ __forceinline__ Place place(const NormParams& p, int threads) {
    Place q;
    q.width = (int)p.columns_div.d;
    q.step = threads / q.width;
    q.r = (int)p.columns_div.div(threadIdx.x);
    q.col = threadIdx.x - q.r * q.width;
    return q;
}
// Positions of n that place q has.
__device__ __forceinline__ int mine_of(const Place& q, int n) { return q.r < n ? (n - q.r + q.step - 1) / q.step : 0; }

template <class P> struct Two { P x, dy; };

// A thread's sums of its channels: of the differences from a pivot, and of their squares. The pivot is
// the first value met, then, after U, 4U, 16U ... positions, the mean of what has been met: were the first
// value k deviations from the rest, n positions' squares would be n k^2 and what cancels of them at the
// end n times the outlier's own share of the variance (rstd 14 % off at n = 5376, k = 10^5).
template <class T, int V, int U> struct Sums {
    static constexpr int N = (V + 1) / 2;
    f2 pivot[N], a[N], b[N];
    static constexpr uint32_t kTurns = U * 0x55555555u;   // the bits U, 4U, 16U ...
    uint32_t met = 0;
    // after every U positions: to pivot + h, sum - n h, squares - h (sum + new sum)
    __device__ __forceinline__ void batch(bool mono) {
        met += U;
        if ((met & (met - 1)) || !(met & kTurns)) return;
        const float n = (float)met, each = __uint_as_float(0x7f000000u - __float_as_uint(n));   // 1 / n: a power of two
        const f2 less = make_f2(-n, -n);
        f2 all = a[0];
        if (V > 1 && mono) {   // one pivot for all the vector's channels
#pragma unroll
            for (int i = 1; i < N; i++) all = all + a[i];
            const float2 s = split(all);
            all = make_f2((s.x + s.y) * (1.0f / V), (s.x + s.y) * (1.0f / V));
        }
#pragma unroll
        for (int i = 0; i < N; i++) {
            const f2 from = pivot[i], h0 = (V > 1 && mono ? all : a[i]) * make_f2(each, each);
            pivot[i] = from + h0 * make_f2(-1.0f, -1.0f);
            const f2 h = from + pivot[i] * make_f2(-1.0f, -1.0f);   // the step as it was rounded
            const f2 s = fma2(less, h, a[i]);
            b[i] = fma2(h * make_f2(-1.0f, -1.0f), a[i] + s, b[i]);
            a[i] = s;
        }
    }
    __device__ __forceinline__ void start(const Pack<T, V>& first, bool mono) {
#pragma unroll
        for (int i = 0; i < N; i++) {
            const float2 f = split(get(first, i)), f0 = split(get(first, 0));
            pivot[i] = mono ? make_f2(-f0.x, -f0.x) : make_f2(-f.x, -f.y);
            a[i] = b[i] = make_f2(0.0f, 0.0f);
        }
    }
    __device__ __forceinline__ void take(const Pack<T, V>& v) {
#pragma unroll
        for (int i = 0; i < N; i++) {
            const f2 d = get(v, i) + pivot[i];
            a[i] = a[i] + d;
            b[i] = fma2(d, d, b[i]);
        }
    }
    // Mean and M2 of the `mine` positions: one part for the vector when its channels are of one
    // group, else one for each channel.
    __device__ __forceinline__ void finish(int mine, bool mono, float2* part, int at) {
        auto moments = [](float sum, float sq, float n, float neg) {   // + 0 sum: a NaN stays one
            const float m = sum / n;
            return make_float2(m - neg, fmaxf(fmaf(-sum, m, sq), 0.0f) + 0.0f * sum);
        };
        if (V == 1) {
            part[at] = moments(split(a[0]).x, split(b[0]).x, (float)mine, split(pivot[0]).x);
        } else if (mono) {
#pragma unroll
            for (int i = 1; i < N; i++) { a[0] = a[0] + a[i]; b[0] = b[0] + b[i]; }
            const float2 sa = split(a[0]), sb = split(b[0]);
            part[at] = moments(sa.x + sa.y, sb.x + sb.y, (float)mine * V, split(pivot[0]).x);
        } else {
#pragma unroll
            for (int i = 0; i < N; i++) {
                const float2 sa = split(a[i]), sb = split(b[i]), sp = split(pivot[i]);
                part[at * V + 2 * i] = moments(sa.x, sb.x, (float)mine, sp.x);
                part[at * V + 2 * i + 1] = moments(sa.y, sb.y, (float)mine, sp.y);
            }
        }
    }
};

// Moments of the groups with channels in [ch0, ch1) from a block's parts of them: [step][row],
// mean and M2 of the positions that place r has. The mean of the means first, then the deviations
// from it, both from the group's first part on. All threads are shared out to the groups at once,
// several warps to one or, with more groups than warps, down to one lane (a warp to each in turn:
// 542 us where this takes 43 for 2 x 16 x 4096 with 4096 groups). A group that began before ch0 is
// joined to what group[] has of it.
__device__ __forceinline__ void block_moments(const NormParams& p, int threads, const Place& q, int n, int vec, int ch0, int ch1, const float2* part, float2* group,
                                              float* red) {
    const int per = p.mono ? vec : 1, row = q.width * vec / per, rows = min(q.step, n);
    const int base = n / q.step, more = n - base * q.step;       // place r has base positions, and one more below `more`
    const int first = ch0 / p.cpg, count = (ch1 - 1) / p.cpg + 1 - first;
    int lanes = 32;
    while (lanes > 1 && count * lanes > threads) lanes >>= 1;
    const int team = max(1, threads / 32 / count), share = lanes * team, at_once = threads / share;
    const int slot = threadIdx.x / share, lead = threadIdx.x - slot * share;
    for (int g0 = 0; g0 < count; g0 += at_once) {
        const int g = first + g0 + slot;
        const bool live = g - first < count && slot < at_once;
        const int from_ch = max(g * p.cpg, ch0), w = live ? (min((g + 1) * p.cpg, ch1) - from_ch) / per : 1;
        const float2* at = part + (from_ch - ch0) / per;
        const int r0 = lead / w, c0 = lead - r0 * w, dr = share / w, dc = share - dr * w;
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
            for (int o = lanes / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
            if (team > 1) {   // then every group has its team at once: one round
                if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = sum;
                __syncthreads();
                sum = 0.0f;
                if (live)
                    for (int k = 0; k < team; k++) sum += red[slot * team + k];
                __syncthreads();
            }
            if (pass == 0) mean = sum / ((float)n * (float)(w * per));
            else if (live && lead == 0) {
                Moments m{(float)n * (float)(w * per), from + mean, sum};
                if (g * p.cpg < ch0) {
                    Moments t{(float)n * (float)(ch0 - g * p.cpg), group[g].x, group[g].y};
                    join(t, m);
                    m = t;
                }
                group[g] = make_float2(m.mean, m.m2);
            }
        }
    }
    __syncthreads();
}

// z = (x + mu) a + sh for a thread's channels, mu the negative mean: the difference first, so that
// values near the mean, a constant group's above all, keep their digits.
template <class T, int V, int ACT> struct Affine {
    static constexpr int N = (V + 1) / 2;
    f2 mu[N], a[N], sh[N];
    PairAct<ACT, sizeof(T) == 2> fn;
    // stat(g): mean and rstd of a group
    template <class Fn> __device__ __forceinline__ void start(const NormParams& p, int ch, Fn&& stat) {
#pragma unroll
        for (int i = 0; i < N; i++) {
            float m[2], s1[2], s0[2];
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const int c = V == 1 ? ch : ch + 2 * i + k;
                const float2 st = stat(c / p.cpg);
                m[k] = -st.x;
                s1[k] = st.y * param(p.gamma, c, p.param_float, 1.0f, (const T*)nullptr);
                s0[k] = param(p.beta, c, p.param_float, 0.0f, (const T*)nullptr);
            }
            mu[i] = make_f2(m[0], m[1]);
            a[i] = make_f2(s1[0], s1[1]);
            sh[i] = make_f2(s0[0], s0[1]);
        }
    }
    __device__ __forceinline__ void put_at(T* y, Pack<T, V> v) const {
#pragma unroll
        for (int i = 0; i < N; i++) put(v, i, fn.value(fma2(get(v, i) + mu[i], a[i], sh[i])));
        store_stream(y, v);
    }
};

// Backward: z = (x + mu) za + zb; the sums are of dz and dz (x + mu), the latter scaled by rstd at the end;
// dx = dz za + (x + mu) c2 + c1, c2 = -rstd^2 mean(d xh), c1 = -rstd mean(d).
template <class T, int V, int ACT> struct Slope {
    static constexpr int N = (V + 1) / 2;
    f2 mu[N], za[N], zb[N];
    float rs[2 * N];
    PairAct<ACT, sizeof(T) == 2> fn;
    __device__ __forceinline__ void start(const NormParams& p, int item, int ch) {
#pragma unroll
        for (int i = 0; i < N; i++) {
            float m[2], s1[2], s0[2];
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const int c = V == 1 ? ch : ch + 2 * i + k;
                const int64_t g = (int64_t)item * p.groups + c / p.cpg;
                m[k] = -p.mean[g];
                rs[2 * i + k] = p.rstd[g];
                s1[k] = rs[2 * i + k] * param(p.gamma, c, p.param_float, 1.0f, (const T*)nullptr);
                s0[k] = param(p.beta, c, p.param_float, 0.0f, (const T*)nullptr);
            }
            mu[i] = make_f2(m[0], m[1]);
            za[i] = make_f2(s1[0], s1[1]);
            zb[i] = make_f2(s0[0], s0[1]);
        }
    }
    __device__ __forceinline__ void take(const Pack<T, V>& v, const Pack<T, V>& w, f2 (&a)[N], f2 (&b)[N]) const {
#pragma unroll
        for (int i = 0; i < N; i++) {
            const f2 xm = get(v, i) + mu[i];
            const f2 dz = get(w, i) * fn.slope(fma2(xm, za[i], zb[i]));
            a[i] = a[i] + dz;
            b[i] = fma2(dz, xm, b[i]);
        }
    }
    __device__ __forceinline__ void parts(const f2 (&a)[N], const f2 (&b)[N], float2* part) const {
#pragma unroll
        for (int j = 0; j < V; j++) {
            const float2 sa = split(a[j / 2]), sb = split(b[j / 2]);
            part[j] = make_float2(j & 1 ? sa.y : sa.x, (j & 1 ? sb.y : sb.x) * rs[j]);
        }
    }
    // means(g): the group's means of d and d xh
    template <class Fn> __device__ __forceinline__ void ends(const NormParams& p, int ch, f2 (&c1)[N], f2 (&c2)[N], Fn&& means) const {
#pragma unroll
        for (int i = 0; i < N; i++) {
            float u1[2], u2[2];
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const float2 m = means((V == 1 ? ch : ch + 2 * i + k) / p.cpg);
                const float r = rs[2 * i + k];
                u1[k] = -r * m.x;
                u2[k] = -r * r * m.y;
            }
            c1[i] = make_f2(u1[0], u1[1]);
            c2[i] = make_f2(u2[0], u2[1]);
        }
    }
    __device__ __forceinline__ void put_at(T* dx, const Pack<T, V>& v, const Pack<T, V>& w, const f2 (&c1)[N], const f2 (&c2)[N]) const {
        Pack<T, V> o;
#pragma unroll
        for (int i = 0; i < N; i++) {
            const f2 xm = get(v, i) + mu[i];
            const f2 dz = get(w, i) * fn.slope(fma2(xm, za[i], zb[i]));
            put(o, i, fma2(dz, za[i], fma2(xm, c2[i], c1[i])));
        }
        store_stream(dx, o);
    }
};

// ---- three launches -----------------------------------------------------------------------------

// A launch of these may begin before the one it depends on has ended: nothing it reads of that one's
// is read before this.
__device__ __forceinline__ void after_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void next_may_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

struct Range { int item, chunk, n; int64_t l0; };
// Blocks take the chunks in order, or (the second reading) from the last.
__device__ __forceinline__ Range range_of(const NormParams& p, bool reverse) {
    Range s;
    s.item = reverse ? gridDim.y - 1 - blockIdx.y : blockIdx.y;
    s.chunk = reverse ? gridDim.x - 1 - blockIdx.x : blockIdx.x;
    s.l0 = (int64_t)s.chunk * p.rows;
    s.n = (int)min((int64_t)p.rows, p.positions - s.l0);
    return s;
}

// Moments of a chunk's groups.
template <class T, int V>
__global__ void __launch_bounds__(kThreads, 2) moments_kernel(const __grid_constant__ NormParams p) {
    constexpr int U = 8;
    using P = Pack<T, V>;
    __shared__ float2 part[kThreads * V];
    __shared__ float red[kThreads / 32];
    extern __shared__ float2 group[];          // [groups]
    next_may_start();
    const Range s = range_of(p, false);
    const Place q = place(p, kThreads);
    const int mine = mine_of(q, s.n);
    for (int c0 = 0; c0 < p.columns; c0 += q.width) {
        const int cols = min(q.width, p.columns - c0);
        if (q.r < q.step && q.col < cols && mine) {
            const T* at = static_cast<const T*>(p.x) + s.item * p.xb + (s.l0 + q.r) * p.xp + (int64_t)(c0 + q.col) * V;
            const int64_t step = (int64_t)q.step * p.xp;
            Sums<T, V, U> sums;
            sums.start(*reinterpret_cast<const P*>(at), p.mono);
            stream<P, U>(mine, [&](P& v) { v = *reinterpret_cast<const P*>(at); at += step; }, [&](const P& v) { sums.take(v); },
                         [&] { sums.batch(p.mono); });
            sums.finish(mine, p.mono, part, q.r * q.width + q.col);
        }
        __syncthreads();
        block_moments(p, kThreads, q, s.n, V, c0 * V, (c0 + cols) * V, part, group, red);
    }
    for (int g = threadIdx.x; g < p.groups; g += kThreads) p.part[((int64_t)s.item * p.groups + g) * p.chunks + s.chunk] = group[g];
}

// One warp per (item, group): its chunks' moments, joined.
__global__ void __launch_bounds__(128) moments_join(const __grid_constant__ NormParams p) {
    const int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    next_may_start();
    after_previous();
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
__global__ void __launch_bounds__(kThreads, 2) apply_kernel(const __grid_constant__ NormParams p) {
    constexpr int U = 4;
    using P = Pack<T, V>;
    const Range s = range_of(p, true);
    const Place q = place(p, kThreads);
    after_previous();
    const int mine = mine_of(q, s.n);
    if (q.r >= q.step || !mine) return;
    for (int col = q.col; col < p.columns; col += q.width) {
        const int ch = col * V;
        Affine<T, V, ACT> f;
        f.start(p, ch, [&](int g) { return make_float2(p.mean[(int64_t)s.item * p.groups + g], p.rstd[(int64_t)s.item * p.groups + g]); });
        const int64_t last = s.l0 + q.r + (int64_t)(mine - 1) * q.step, sx = (int64_t)q.step * p.xp, sy = (int64_t)q.step * p.yp;
        const T* at = static_cast<const T*>(p.x) + s.item * p.xb + last * p.xp + ch;
        T* y = static_cast<T*>(p.y) + s.item * p.yb + last * p.yp + ch;
        stream<P, U>(mine, [&](P& v) { v = load_stream<P>(at); at -= sx; }, [&](const P& v) { f.put_at(y, v); y -= sy; });
    }
}

// Backward: a chunk's sums of dz and dz xh per channel.
template <class T, int V, int ACT>
__global__ void __launch_bounds__(kThreads, 2) grad_sums_kernel(const __grid_constant__ NormParams p) {
    constexpr int U = V == 8 ? 2 : 4, N = (V + 1) / 2;   // what the registers hold beside the channels' sums
    using P = Pack<T, V>;
    __shared__ float2 part[kThreads * V];
    next_may_start();
    const Range s = range_of(p, false);
    const Place q = place(p, kThreads);
    const int mine = mine_of(q, s.n);
    for (int c0 = 0; c0 < p.columns; c0 += q.width) {
        const int cols = min(q.width, p.columns - c0);
        if (q.r < q.step && q.col < cols) {
            const int ch = (c0 + q.col) * V;
            Slope<T, V, ACT> f;
            f.start(p, s.item, ch);
            f2 a[N], b[N];
#pragma unroll
            for (int i = 0; i < N; i++) a[i] = b[i] = make_f2(0.0f, 0.0f);
            const T* ax = static_cast<const T*>(p.x) + s.item * p.xb + (s.l0 + q.r) * p.xp + ch;
            const T* ad = static_cast<const T*>(p.dy) + s.item * p.yb + (s.l0 + q.r) * p.yp + ch;
            const int64_t sx = (int64_t)q.step * p.xp, sd = (int64_t)q.step * p.yp;
            stream<Two<P>, U>(mine, [&](Two<P>& v) { v.x = *reinterpret_cast<const P*>(ax); v.dy = *reinterpret_cast<const P*>(ad); ax += sx; ad += sd; },
                              [&](const Two<P>& v) { f.take(v.x, v.dy, a, b); });
            f.parts(a, b, part + (q.r * q.width + q.col) * V);
        }
        __syncthreads();
        for (int c = threadIdx.x; c < cols * V; c += kThreads) {
            float2 t = make_float2(0.0f, 0.0f);
            for (int r = 0; r < q.step; r++) {
                const float2 v = part[r * q.width * V + c];
                t.x += v.x;
                t.y += v.y;
            }
            p.part[((int64_t)s.item * p.chunks + s.chunk) * p.channels + c0 * V + c] = t;
        }
        __syncthreads();
    }
}

// Channels side by side, 32 to a block of 32 x 8 threads: an item's sums over its chunks, and, of one
// block per 32 channels, their sums over the items, dbeta and dgamma. With a grid row to each item
// those are items_join's.
template <class T>
__global__ void __launch_bounds__(256) grad_join(const __grid_constant__ NormParams p) {
    __shared__ float2 red[8][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    const bool each = gridDim.y > 1;
    next_may_start();
    after_previous();
    float2 all = make_float2(0.0f, 0.0f);
    for (int b = blockIdx.y; b < (each ? (int)blockIdx.y + 1 : p.batch); b++) {
        float2 s = make_float2(0.0f, 0.0f);
        if (c < p.channels)
#pragma unroll 4
            for (int k = warp; k < p.used; k += 8) {
                const float2 v = p.part[((int64_t)b * p.chunks + k) * p.channels + c];
                s.x += v.x;
                s.y += v.y;
            }
        red[warp][lane] = s;
        __syncthreads();
        if (warp == 0) {
            for (int w = 1; w < 8; w++) { s.x += red[w][lane].x; s.y += red[w][lane].y; }
            if (c < p.channels) p.sums[(int64_t)b * p.channels + c] = s;
            all.x += s.x;
            all.y += s.y;
        }
        __syncthreads();
    }
    if (warp == 0 && c < p.channels && !each) {
        if (p.dbeta) set_param(p.dbeta, c, p.param_float, all.x, (const T*)nullptr);
        if (p.dgamma) set_param(p.dgamma, c, p.param_float, all.y, (const T*)nullptr);
    }
}

// The same over `count` rows of channel sums in one list, `every` rows apart, `run` of them to a grid
// row: their sum goes to the first one's place in `to` (which may be `from`), or, with one grid row,
// to dbeta and dgamma. The loads of a warp do not wait for each other: the backward pass of 3000 x 7 x 75
// f32 takes 23 us, 1391 when the items were added up one after the other.
template <class T>
__global__ void __launch_bounds__(1024) items_join(const __grid_constant__ NormParams p, const float2* from, float2* to, int64_t count, int64_t every,
                                                   int64_t run) {
    __shared__ float2 red[32][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    const int64_t i0 = blockIdx.y * run, i1 = min(count, i0 + run);
    next_may_start();
    after_previous();
    float2 s = make_float2(0.0f, 0.0f);
    if (c < p.channels)
#pragma unroll 8
        for (int64_t i = i0 + warp; i < i1; i += 32) {
            const float2 v = from[i * every * p.channels + c];
            s.x += v.x;
            s.y += v.y;
        }
    red[warp][lane] = s;
    __syncthreads();
    if (warp || c >= p.channels) return;
    for (int w = 1; w < 32; w++) { s.x += red[w][lane].x; s.y += red[w][lane].y; }
    if (gridDim.y > 1) {
        to[i0 * every * p.channels + c] = s;
        return;
    }
    if (p.dbeta) set_param(p.dbeta, c, p.param_float, s.x, (const T*)nullptr);
    if (p.dgamma) set_param(p.dgamma, c, p.param_float, s.y, (const T*)nullptr);
}

// Sums over a group's channels of gamma times their sums: s(c) -> out(g).
template <class T, class S, class Out>
__device__ __forceinline__ void group_sums(const NormParams& p, int threads, S&& s, Out&& out) {
    int lanes = 32;   // of a group: all threads at once, as in block_moments
    while (lanes > 1 && p.groups * lanes > threads) lanes >>= 1;
    const int lead = threadIdx.x & (lanes - 1);
    for (int g0 = 0; g0 < p.groups; g0 += threads / lanes) {
        const int g = g0 + threadIdx.x / lanes;
        float a = 0.0f, b = 0.0f;
        for (int k = lead; k < p.cpg && g < p.groups; k += lanes) {
            const int c = g * p.cpg + k;
            const float2 v = s(c);
            const float gc = param(p.gamma, c, p.param_float, 1.0f, (const T*)nullptr);
            a = fmaf(gc, v.x, a);
            b = fmaf(gc, v.y, b);
        }
        for (int o = lanes / 2; o > 0; o >>= 1) {
            a += __shfl_xor_sync(~0u, a, o);
            b += __shfl_xor_sync(~0u, b, o);
        }
        if (lead == 0 && g < p.groups) out(g, a, b);
    }
}

template <class T, int V, int ACT>
__global__ void __launch_bounds__(kThreads, 2) grad_apply_kernel(const __grid_constant__ NormParams p) {
    constexpr int U = V == 8 ? 2 : 4, N = (V + 1) / 2;
    using P = Pack<T, V>;
    extern __shared__ float2 group[];   // [groups]: means of d and d xh
    const Range s = range_of(p, true);
    const Place q = place(p, kThreads);
    after_previous();
    const float m = (float)p.positions * (float)p.cpg;
    group_sums<T>(p, kThreads, [&](int c) { return p.sums[(int64_t)s.item * p.channels + c]; },
                            [&](int g, float a, float b) { group[g] = make_float2(a / m, b / m); });
    __syncthreads();
    const int mine = mine_of(q, s.n);
    if (q.r >= q.step || !mine) return;
    for (int col = q.col; col < p.columns; col += q.width) {
        const int ch = col * V;
        Slope<T, V, ACT> f;
        f.start(p, s.item, ch);
        f2 c1[N], c2[N];
        f.ends(p, ch, c1, c2, [&](int g) { return group[g]; });
        const int64_t last = s.l0 + q.r + (int64_t)(mine - 1) * q.step;
        const int64_t sx = (int64_t)q.step * p.xp, sd = (int64_t)q.step * p.yp, so = (int64_t)q.step * p.dp;
        const T* ax = static_cast<const T*>(p.x) + s.item * p.xb + last * p.xp + ch;
        const T* ad = static_cast<const T*>(p.dy) + s.item * p.yb + last * p.yp + ch;
        T* dx = static_cast<T*>(p.dx) + s.item * p.db + last * p.dp + ch;
        stream<Two<P>, U>(mine, [&](Two<P>& v) { v.x = load_stream<P>(ax); v.dy = load_stream<P>(ad); ax -= sx; ad -= sd; },
                          [&](const Two<P>& v) { f.put_at(dx, v.x, v.dy, c1, c2); dx -= so; });
    }
}

// ---- clusters -----------------------------------------------------------------------------------

constexpr int kFused = 512;          // threads: with 1024 the registers do not hold a vector's sums
constexpr int kFusedGroups = 2048;   // most groups
constexpr int kClusterMost = 8;
constexpr size_t kClusterSmem = 225 * 1024;   // dynamic shared memory of a block

__device__ __forceinline__ void cluster_arrive() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// The 8 bytes at the same place in another block of the cluster.
__device__ __forceinline__ float2 peer_read(const float2* p, int rank) {
    uint32_t a;
    float2 v;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(a) : "memory");
    return v;
}

__device__ __forceinline__ Range cluster_range(const NormParams& p) {
    Range s;
    s.item = blockIdx.x / p.chunks;
    s.chunk = blockIdx.x - s.item * p.chunks;
    s.l0 = (int64_t)s.chunk * p.rows;
    s.n = (int)max((int64_t)0, min((int64_t)p.rows, p.positions - s.l0));
    return s;
}

template <class T, int V, int ACT>
__global__ void __launch_bounds__(kFused, 1) norm_cluster(const __grid_constant__ NormParams p) {
    constexpr int U = 4;                        // positions in flight per thread
    using P = Pack<T, V>;
    extern __shared__ __align__(16) uint8_t smem[];
    const int threads = blockDim.x;             // kFused at most
    P* keep = reinterpret_cast<P*>(smem);       // [kept][threads]
    float2* part = reinterpret_cast<float2*>(smem + (size_t)p.kept * threads * sizeof(P));
    float2* group = part + threads * (p.mono ? 1 : V);   // [groups]: the block's moments
    float2* stat = group + p.groups;                    // [groups]: the item's mean and rstd
    __shared__ float red[kFused / 32];
    const Range s = cluster_range(p);
    const Place q = place(p, threads);
    const int ch = q.col * V;
    const int mine = q.r < q.step ? mine_of(q, s.n) : 0;
    if (s.n > 0) {
        if (mine) {
            const T* at = static_cast<const T*>(p.x) + s.item * p.xb + (s.l0 + q.r) * p.xp + ch;
            const int64_t step = (int64_t)q.step * p.xp;
            Sums<T, V, U> sums;
            sums.start(*reinterpret_cast<const P*>(at), p.mono);
            P* k = keep + threadIdx.x;
            stream<P, U>(mine, [&](P& v) { v = *reinterpret_cast<const P*>(at); at += step; }, [&](const P& v) {
                *k = v;
                k += threads;
                sums.take(v);
            }, [&] { sums.batch(p.mono); });
            sums.finish(mine, p.mono, part, q.r * q.width + q.col);
        }
        __syncthreads();
        block_moments(p, threads, q, s.n, V, 0, p.channels, part, group, red);
    }
    cluster_arrive();
    cluster_wait();
    if (s.n > 0) {
        for (int g0 = 0; g0 < p.groups; g0 += threads / kClusterMost) {   // a lane to a block
            const int g = g0 + threadIdx.x / kClusterMost, c = threadIdx.x % kClusterMost;
            Moments m{0.0f, 0.0f, 0.0f};
            if (g < p.groups && c < p.used) {
                const float2 v = peer_read(group + g, c);
                m = Moments{(float)min((int64_t)p.rows, p.positions - (int64_t)c * p.rows) * (float)p.cpg, v.x, v.y};
            }
            warp_join<kClusterMost>(m);
            if (g < p.groups && c == 0) {
                const float r = 1.0f / sqrtf(m.m2 / ((float)p.positions * (float)p.cpg) + p.eps);
                stat[g] = make_float2(m.mean, r);
                if (s.chunk == 0 && p.mean) {
                    p.mean[(int64_t)s.item * p.groups + g] = m.mean;
                    p.rstd[(int64_t)s.item * p.groups + g] = r;
                }
            }
        }
    }
    cluster_arrive();   // waited for below: no block goes while others still read its moments
    __syncthreads();
    if (mine) {
        Affine<T, V, ACT> f;
        f.start(p, ch, [&](int g) { return stat[g]; });
        T* y = static_cast<T*>(p.y) + s.item * p.yb + (s.l0 + q.r) * p.yp + ch;
        const int64_t sy = (int64_t)q.step * p.yp;
        const P* k = keep + threadIdx.x;
        for (int it = 0; it < mine; it++, k += threads, y += sy) f.put_at(y, *k);
    }
    __syncwarp();
    cluster_wait();
}

// Backward: the blocks meet over their groups' sums; channel sums go out per block for grad_join.
template <class T, int V, int ACT>
__global__ void __launch_bounds__(kFused, 1) norm_grad_cluster(const __grid_constant__ NormParams p) {
    constexpr int U = 2, N = (V + 1) / 2;
    using P = Pack<T, V>;
    extern __shared__ __align__(16) uint8_t smem[];
    const int threads = blockDim.x;             // kFused at most
    P* keep = reinterpret_cast<P*>(smem);       // [kept][x, dy][threads]
    float2* part = reinterpret_cast<float2*>(smem + (size_t)p.kept * 2 * threads * sizeof(P));   // [step][channels]
    float2* chan = part + threads * V;           // [channels]
    float2* group = chan + p.channels;          // [groups]: the block's sums
    float2* stat = group + p.groups;            // [groups]: the item's means of d and d xh
    next_may_start();
    const Range s = cluster_range(p);
    const Place q = place(p, threads);
    const int ch = q.col * V;
    const bool on = q.r < q.step && s.n > 0;
    const int mine = on ? mine_of(q, s.n) : 0;
    Slope<T, V, ACT> f;
    if (s.n > 0) {
        if (on) {
            f.start(p, s.item, ch);
            f2 a[N], b[N];
#pragma unroll
            for (int i = 0; i < N; i++) a[i] = b[i] = make_f2(0.0f, 0.0f);
            const T* ax = static_cast<const T*>(p.x) + s.item * p.xb + (s.l0 + q.r) * p.xp + ch;
            const T* ad = static_cast<const T*>(p.dy) + s.item * p.yb + (s.l0 + q.r) * p.yp + ch;
            const int64_t sx = (int64_t)q.step * p.xp, sd = (int64_t)q.step * p.yp;
            P* k = keep + threadIdx.x;
            stream<Two<P>, U>(mine, [&](Two<P>& v) { v.x = *reinterpret_cast<const P*>(ax); v.dy = *reinterpret_cast<const P*>(ad); ax += sx; ad += sd; },
                              [&](const Two<P>& v) {
                                  k[0] = v.x;
                                  k[threads] = v.dy;
                                  k += 2 * threads;
                                  f.take(v.x, v.dy, a, b);
                              });
            f.parts(a, b, part + (q.r * q.width + q.col) * V);
        }
        __syncthreads();
        for (int c = threadIdx.x; c < p.channels; c += threads) {
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
        group_sums<T>(p, threads, [&](int c) { return chan[c]; }, [&](int g, float a, float b) { group[g] = make_float2(a, b); });
    } else {
        for (int c = threadIdx.x; c < p.channels; c += threads) p.part[((int64_t)s.item * p.chunks + s.chunk) * p.channels + c] = make_float2(0.0f, 0.0f);
    }
    cluster_arrive();
    cluster_wait();
    if (s.n > 0 && p.dx) {
        const float m = (float)p.positions * (float)p.cpg;
        for (int g0 = 0; g0 < p.groups; g0 += threads / kClusterMost) {   // a lane to a block
            const int g = g0 + threadIdx.x / kClusterMost, c = threadIdx.x % kClusterMost;
            float2 v = g < p.groups && c < p.used ? peer_read(group + g, c) : make_float2(0.0f, 0.0f);
            for (int o = kClusterMost / 2; o > 0; o >>= 1) {
                v.x += __shfl_xor_sync(~0u, v.x, o);
                v.y += __shfl_xor_sync(~0u, v.y, o);
            }
            if (g < p.groups && c == 0) stat[g] = make_float2(v.x / m, v.y / m);
        }
    }
    cluster_arrive();
    __syncthreads();
    if (mine && p.dx) {
        f2 c1[N], c2[N];
        f.ends(p, ch, c1, c2, [&](int g) { return stat[g]; });
        T* dx = static_cast<T*>(p.dx) + s.item * p.db + (s.l0 + q.r) * p.dp + ch;
        const int64_t so = (int64_t)q.step * p.dp;
        const P* k = keep + threadIdx.x;
        for (int it = 0; it < mine; it++, k += 2 * threads, dx += so) f.put_at(dx, k[0], k[threads], c1, c2);
    }
    __syncwarp();
    cluster_wait();
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

// An item's positions are cut so that the whole call has two blocks per SM, what the registers
// allow at a time, each with at least 16 positions: a block's joining at its end reads nothing, so few
// long blocks beat more short ones (moments of 132 MB: 30 us with two per SM, 34 with four, 43 with
// eight).
int chunks_of(const stg_group_norm_config& c) {
    const int64_t per_item = (148 * 2 + c.batch - 1) / std::max<int64_t>(c.batch, 1);
    const int64_t n = std::min<int64_t>({std::max<int64_t>(per_item, 1), (c.positions + 15) / 16});
    const int64_t rows = (c.positions + n - 1) / std::max<int64_t>(n, 1);
    return (int)((c.positions + rows - 1) / std::max<int64_t>(rows, 1));
}

size_t up(size_t n) { return (n + 255) / 256 * 256; }

enum Path { THREE_LAUNCHES, CLUSTER };
// How a call runs with vectors of `vec` channels on `sms` SMs, and the scratch it takes.
struct NormPlan {
    Path path = THREE_LAUNCHES;
    int chunks = 0, kept = 0, threads = 0;      // threads: a cluster's blocks
    int64_t rows = 0;
    size_t smem = 0;
    size_t second = 0, third = 0, bytes = 0;   // offsets of the scratch's parts
};
NormPlan plan_of(const stg_group_norm_config& c, bool backward, int vec, int sms) {
    NormPlan r;
    if (!c.batch || !c.positions) return r;
    const int columns = c.channels / vec, cpg = c.channels / c.groups;
    // Items that a smaller block reads in eight steps, more of them than SMs: such blocks, of which an SM
    // holds several (9000 x 16 x 16 f32: 35 us, 281 with kFused threads each; 3000 x 7 x 75 20 and 97).
    int threads = kFused;
    while (threads > 32 && columns <= threads / 2 && c.positions <= 8 * (threads / 2 / columns) && c.batch > sms) threads /= 2;
    r.threads = threads;
    const size_t vb = (size_t)vec * elem_size(c.dtype) * (backward ? 2 : 1), block_step = vb * threads;
    const bool mono = cpg % vec == 0;
    // shared memory besides the kept values: the threads' parts, channel and group sums
    const size_t other = backward ? sizeof(float2) * ((size_t)threads * vec + c.channels + 2 * (size_t)c.groups)
                                  : sizeof(float2) * ((size_t)threads * (mono ? 1 : vec) + 2 * (size_t)c.groups);
    const size_t most = kClusterSmem;
    if (columns <= threads && c.groups <= kFusedGroups && other + 8 * block_step <= most) {
        const int64_t step = threads / columns, room = (int64_t)((most - other) / block_step);   // steps a block can keep
        const int64_t item_steps = (c.positions + step - 1) / step;
        auto steps = [&](int64_t size) { return ((c.positions + size - 1) / size + step - 1) / step; };   // of one of `size` blocks
        // as many blocks as fill the GPU once, each with at least four steps
        int64_t size = 1;
        while (size < kClusterMost && (steps(size) > room || (size * 2 * c.batch <= sms && size * 8 <= item_steps))) size *= 2;
        if (steps(size) <= room) {
            r.path = CLUSTER;
            r.chunks = (int)size;
            r.rows = (c.positions + size - 1) / size;
            r.kept = (int)steps(size);
            r.smem = other + (size_t)r.kept * block_step;
            if (backward) r.bytes = up(sizeof(float2) * (size_t)c.batch * r.chunks * c.channels);
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
void set_plan(NormParams& p, const NormPlan& plan, int vec) {
    p.columns = p.channels / vec;
    p.columns_div = FastDiv((uint32_t)std::min(p.columns, plan.path == THREE_LAUNCHES ? kThreads : plan.threads));
    p.chunks = plan.chunks;
    p.rows = (int)plan.rows;
    p.used = (int)((p.positions + plan.rows - 1) / plan.rows);
    p.kept = plan.kept;
    p.mono = p.cpg % vec == 0;
}
// A launch that may begin while the one before it ends (see after_previous).
template <class K, class... More> void launch_after(K kernel, dim3 grid, int threads, size_t smem, cudaStream_t st, const NormParams& p, More... more) {
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr[1];
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cuda_check(cudaLaunchKernelEx(&cfg, kernel, p, more...), "group norm kernel");
}
// Up to here grad_join adds the items up as it goes, one launch less; past it a grid row has an item each and
// items_join adds them up. N x 3000 x 384 f32, whole backward pass, in turn and each: 24 items 127 and 110 us,
// 64 315 and 285; but also 16 85 and 74, 4 21 and 17.
constexpr int kItemsInTurn = 16;
// Rows of channel sums of one run; more rows are joined in runs first, into p.part (a launch more). N x 7 x 75 f32, whole
// backward pass, in runs of 512, of 128 and in one: 600 items 9.4, 9.0 and 9.6 us, 3000 23, 22 and 32; 60000 x 4 x 16
// 212, 215 and 396.
constexpr int64_t kJoinRun = 512;
// dbeta and dgamma from `count` rows of channel sums.
template <class T> void join_items(const NormParams& p, const float2* from, int64_t count, cudaStream_t st) {
    if (!p.dgamma && !p.dbeta) return;
    const unsigned columns = (unsigned)((p.channels + 31) / 32);
    const int64_t runs = (count + kJoinRun - 1) / kJoinRun;
    if (runs > 1) launch_after(items_join<T>, dim3(columns, (unsigned)runs), 1024, 0, st, p, from, p.part, count, (int64_t)1, kJoinRun);
    if (runs > 1) launch_after(items_join<T>, dim3(columns), 1024, 0, st, p, (const float2*)p.part, p.part, runs, kJoinRun, runs);
    else launch_after(items_join<T>, dim3(columns), 1024, 0, st, p, from, p.part, count, (int64_t)1, count);
}
// The limit belongs to the function on the device, not to the call: it is only ever set to the kernel's `most`, so
// that another host thread's smaller call cannot lower it between this one's setting and its launch.
template <class K> void allow_smem(K kernel, size_t smem, size_t most, size_t fixed = 0) {
    if (smem + fixed > 48 * 1024) cuda_check(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most), "group norm kernel");
}
template <class K> void launch_cluster(K kernel, const NormParams& p, const NormPlan& plan, cudaStream_t st) {
    allow_smem(kernel, plan.smem, kClusterSmem, 256);
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr[1];
    cfg.gridDim = dim3((unsigned)(p.batch * plan.chunks));
    cfg.blockDim = dim3(plan.threads);
    cfg.dynamicSmemBytes = plan.smem;
    cfg.stream = st;
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = plan.chunks;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
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
                set_plan(p, plan, V);
                with_activation(c->activation, [&](auto a) {
                    constexpr int A = decltype(a)::value;
                    if (plan.path == CLUSTER) return launch_cluster(norm_cluster<T, V, A>, p, plan, st);
                    if (!p.mean) {
                        p.mean = reinterpret_cast<float*>(ws + plan.second);
                        p.rstd = reinterpret_cast<float*>(ws + plan.third);
                    }
                    const dim3 grid((unsigned)p.chunks, (unsigned)p.batch);
                    const size_t smem = sizeof(float2) * (size_t)p.groups;
                    allow_smem(moments_kernel<T, V>, smem, sizeof(float2) * kMaxChannels, sizeof(float2) * kThreads * V + 256);
                    moments_kernel<T, V><<<grid, kThreads, smem, st>>>(p);
                    launch_after(moments_join, dim3((unsigned)(((int64_t)p.batch * p.groups + 3) / 4)), 128, 0, st, p);
                    launch_after(apply_kernel<T, V, A>, grid, kThreads, 0, st, p);
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
        if (d_dx) check_output_strides(c->dx_batch, c->dx_position, *c);
        DeviceScope scope(e);
        const cudaStream_t st = static_cast<cudaStream_t>(stream);
        if (!c->batch || !c->positions) {   // sums over nothing
            if (d_dgamma) cuda_check(cudaMemsetAsync(d_dgamma, 0, ps * c->channels, st), "group norm memset");
            if (d_dbeta) cuda_check(cudaMemsetAsync(d_dbeta, 0, ps * c->channels, st), "group norm memset");
            return;
        }
        check(d_x && d_dy && d_mean && d_rstd, "group norm: null buffer");
        if (!d_dx && !d_dgamma && !d_dbeta) return;
        const bool wide = wide_fits(*c, {d_x, d_dy}, {c->x_batch, c->x_position, c->y_batch, c->y_position}) &&
                          (!d_dx || wide_fits(*c, {d_dx}, {c->dx_batch, c->dx_position}));
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
                set_plan(p, plan, V);
                with_activation(c->activation, [&](auto a) {
                    constexpr int A = decltype(a)::value;
                    const unsigned columns = (unsigned)((p.channels + 31) / 32);
                    if (plan.path == CLUSTER) {
                        launch_cluster(norm_grad_cluster<T, V, A>, p, plan, st);
                        join_items<T>(p, p.part, (int64_t)p.batch * p.chunks, st);
                        return;
                    }
                    const dim3 grid((unsigned)p.chunks, (unsigned)p.batch);
                    grad_sums_kernel<T, V, A><<<grid, kThreads, 0, st>>>(p);
                    const bool each = p.batch > kItemsInTurn;
                    launch_after(grad_join<T>, dim3(columns, each ? (unsigned)p.batch : 1), 256, 0, st, p);
                    if (each) join_items<T>(p, p.sums, p.batch, st);
                    if (p.dx) {
                        const size_t smem = sizeof(float2) * (size_t)p.groups;
                        allow_smem(grad_apply_kernel<T, V, A>, smem, sizeof(float2) * kMaxChannels);
                        launch_after(grad_apply_kernel<T, V, A>, grid, kThreads, smem, st, p);
                    }
                });
            });
        });
        cuda_check(cudaGetLastError(), "group norm kernel");
    });
}

} // extern "C"
