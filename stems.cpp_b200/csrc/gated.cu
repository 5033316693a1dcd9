// gated.cu -- the gated projection, its backward pass and RoFormer's mask head
// (include/stems_gpu_v1.h: stg_gated, stg_gated_backward, stg_mask_head): entry points and the
// kernels on the CUDA cores.
//
// With g = x Wg^T + bg and u = x Wu^T + bu: y = act(g) u. Backward:
//   dg = dy u act'(g), du = dy act(g);  dx = dg Wg + du Wu;  dWg = dg^T x, dWu = du^T x;
//   dbg, dbu = column sums of dg, du.
#include "gated.h"

namespace stg {

namespace {

constexpr int kThreads = 256;
constexpr int kTileK = 16;

__device__ __forceinline__ void gate_both(int kind, float z, float& a, float& d) {
    switch (kind) {
        case STG_ACT_RELU: return act_both<STG_ACT_RELU, false>(z, a, d);
        case STG_ACT_SILU: return act_both<STG_ACT_SILU, false>(z, a, d);
        case STG_ACT_GELU: return act_both<STG_ACT_GELU, false>(z, a, d);
        case STG_ACT_SIGMOID: return act_both<STG_ACT_SIGMOID, false>(z, a, d);
        default: return act_both<STG_ACT_NONE, false>(z, a, d);
    }
}

template <bool kFast> __device__ __forceinline__ float gate_value(int kind, float z) {
    switch (kind) {
        case STG_ACT_RELU: return act<STG_ACT_RELU, kFast>(z);
        case STG_ACT_SILU: return act<STG_ACT_SILU, kFast>(z);
        case STG_ACT_GELU: return act<STG_ACT_GELU, kFast>(z);
        case STG_ACT_SIGMOID: return act<STG_ACT_SIGMOID, kFast>(z);
        default: return z;
    }
}

// An S x 16 tile of an operand on its way to shared memory, [k][S]. KMAJOR: element (i, k) is at
// p[i * ld + k], otherwise at p[k * ld + i]. A thread takes its neighbours in memory.
template <class T, bool KMAJOR, int S> struct TileLoad {
    static constexpr int N = S / 16, PER_ROW = KMAJOR ? kTileK / N : S / N;   // elements of a thread, threads of a memory row
    static constexpr int kPitch = S + 4;
    float v[N];
    // the row of the operand, within the tile, that the thread carries when KMAJOR
    __device__ __forceinline__ static int row() { return threadIdx.x / PER_ROW; }
    __device__ __forceinline__ void fetch(const T* p, int64_t ld, int64_t i0, int64_t ni, int64_t k0, int64_t nk) {
        const int t = threadIdx.x;
        const int64_t r = KMAJOR ? i0 : k0 + t / PER_ROW;      // KMAJOR: the caller adds row()
        const int64_t c = (KMAJOR ? k0 : i0) + t % PER_ROW * N;
        const bool row_ok = r < (KMAJOR ? ni : nk);
        const int64_t nc = KMAJOR ? nk : ni;
        const T* q = p + r * ld + c;
        constexpr int W = 16 / sizeof(T) < N ? 16 / sizeof(T) : N;
        if (row_ok && c + N <= nc && reinterpret_cast<uintptr_t>(q) % (W * sizeof(T)) == 0) {
#pragma unroll
            for (int j = 0; j < N; j += W) {
                const Pack<T, W> w = *reinterpret_cast<const Pack<T, W>*>(q + j);
#pragma unroll
                for (int e = 0; e < W; e++) v[j + e] = to_float(w.v[e]);
            }
        } else {
#pragma unroll
            for (int j = 0; j < N; j++) v[j] = row_ok && c + j < nc ? to_float(q[j]) : 0.0f;
        }
    }
    __device__ __forceinline__ void store(float* s) const {
        const int t = threadIdx.x;
        if (KMAJOR) {
#pragma unroll
            for (int j = 0; j < N; j++) s[(t % PER_ROW * N + j) * kPitch + t / PER_ROW] = v[j];
        } else {
#pragma unroll
            for (int j = 0; j < N; j += 4)
                *reinterpret_cast<float4*>(s + t / PER_ROW * kPitch + t % PER_ROW * N + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
        }
    }
};

__device__ __forceinline__ void fma2(uint64_t& d, uint64_t a, uint64_t b) {
    asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(d) : "l"(a), "l"(b));
}
__device__ __forceinline__ uint64_t twice(float a) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %1};" : "=l"(r) : "f"(a));
    return r;
}
__device__ __forceinline__ float2 halves(uint64_t a) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a));
    return r;
}

// S x S outputs per block: 128 with 8 x 8 per thread (rows 4 ty + {0..3} and 64 + that, columns 4 tx +
// {0..3} and 64 + that), or 64 with 4 x 4, for products with too few tiles for the GPU. In the dual
// modes half of the columns are the up projection of the same outputs as the other half, placed
// so that a thread holds both factors of its outputs: at 128 the second 64 columns, at 64 the
// second two of each thread's four. Products and sums are float with one rounding each (packed in
// pairs); K runs in order. Bound by the float units: 48 TFLOP/s at 48060 x 384 x 1408; the
// backward pass at 777 x 301 x 515 in float takes 31, 24 and 27 us and 8 us of joining.
template <class T, int MODE, int S>
__global__ void __launch_bounds__(kThreads) gated_simt(const __grid_constant__ GatedParams p) {
    constexpr bool DUAL = MODE == GATED_FWD || MODE == GATED_HEAD || MODE == GATED_PRE;
    constexpr bool AK = MODE != GATED_DW, BK = DUAL;   // contraction contiguous in memory
    constexpr int G = S / 64, R = 4 * G, CP = 2 * G, kPitch = S + 4;   // rows and column pairs of a thread
    constexpr int kTileM = S, kTileOut = DUAL ? S / 2 : S;
    __shared__ __align__(16) float As[2][kTileK * kPitch], Bs[2][kTileK * kPitch];
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;

    // the tile
    int64_t m0, ni, nk, nj;           // first row, rows, contraction, columns of an operand
    int n0;
    const T *a = nullptr, *b0 = nullptr, *b1 = nullptr, *a2 = nullptr;
    int64_t lda, ldb0, ldb1;
    HeadTile ht{};
    int64_t head_row = 0, bias0 = 0;  // mask head: first frame of the tile's band in x; row of the band's first weight
    int64_t kbeg = 0;
    if (MODE == GATED_HEAD) {
        ht = p.tiles[blockIdx.x % p.n_tiles];
        const int64_t rest = blockIdx.x / p.n_tiles, mt = (p.frames + kTileM - 1) / kTileM;
        const int64_t cs = rest / mt;                    // chunk * stems + stem
        m0 = (rest - cs * mt) * kTileM;
        n0 = ht.n0;
        ni = p.frames; nk = p.k; nj = ht.din;
        head_row = (cs * p.bands + ht.band) * p.frames;
        a = static_cast<const T*>(p.x) + head_row * p.k;
        lda = p.k;
        bias0 = (cs % p.stems) * 2 * p.band_cols + 2 * (int64_t)ht.off;
        b0 = static_cast<const T*>(p.wg) + bias0 * p.k;
        b1 = b0 + (int64_t)ht.din * p.k;
        ldb0 = ldb1 = p.k;
        head_row = cs;                                   // for the output
    } else if (DUAL) {
        const int nt = (p.n + kTileOut - 1) / kTileOut;
        m0 = (int64_t)(blockIdx.x / nt) * kTileM;
        n0 = (int)(blockIdx.x % nt) * kTileOut;
        ni = p.m; nk = p.k; nj = p.n;
        a = static_cast<const T*>(p.x);
        b0 = static_cast<const T*>(p.wg);
        b1 = static_cast<const T*>(p.wu);
        lda = p.x_row; ldb0 = p.wg_row; ldb1 = p.wu_row;
    } else if (MODE == GATED_DX) {
        const int nt = (p.k + S - 1) / S;
        m0 = (int64_t)(blockIdx.x / nt) * kTileM;
        n0 = (int)(blockIdx.x % nt) * S;
        ni = p.m; nk = p.n; nj = p.k;
        a = static_cast<const T*>(p.dg);
        a2 = static_cast<const T*>(p.du);
        b0 = static_cast<const T*>(p.wg);
        b1 = static_cast<const T*>(p.wu);
        lda = p.pre_row; ldb0 = p.wg_row; ldb1 = p.wu_row;
    } else {
        const int nt = (p.k + S - 1) / S;
        m0 = (int64_t)(blockIdx.x / nt) * kTileM;
        n0 = (int)(blockIdx.x % nt) * S;
        const bool up = blockIdx.y & 1;
        kbeg = (int64_t)(blockIdx.y >> 1) * p.split_rows;
        ni = p.n; nk = min(p.m, kbeg + p.split_rows); nj = p.k;
        a = static_cast<const T*>(up ? p.du : p.dg);
        b0 = static_cast<const T*>(p.x);
        lda = p.pre_row; ldb0 = ldb1 = p.x_row;
    }

    uint64_t acc[R][CP];
#pragma unroll
    for (int i = 0; i < R; i++)
#pragma unroll
        for (int j = 0; j < CP; j++) acc[i][j] = 0;

    // dx runs through Wg's rows, then Wu's; its splits share out the steps of both
    const int64_t steps1 = (nk - kbeg + kTileK - 1) / kTileK, all = steps1 * (MODE == GATED_DX ? 2 : 1);
    const int64_t share = MODE == GATED_DX ? (all + p.dx_splits - 1) / p.dx_splits : all;
    const int64_t first = MODE == GATED_DX ? min(all, blockIdx.y * share) : 0, steps = min(all, first + share);
    TileLoad<T, AK, S> la;
    TileLoad<T, BK, S> lb;
    auto fetch = [&](int64_t s) {
        const bool second = MODE == GATED_DX && s >= steps1;
        const int64_t k0 = kbeg + (second ? s - steps1 : s) * kTileK;
        la.fetch(second ? a2 : a, lda, m0 + (AK ? la.row() : 0), ni, k0, nk);
        if (DUAL) {
            const int r = lb.row();   // the tile's row the thread carries: which weight, which output
            const bool up = S == 128 ? r >= 64 : r & 2;
            lb.fetch(up ? b1 : b0, up ? ldb1 : ldb0, n0 + (S == 128 ? r & 63 : (r >> 2) * 2 + (r & 1)), nj, k0, nk);
        } else {
            lb.fetch(second ? b1 : b0, second ? ldb1 : ldb0, n0, nj, k0, nk);
        }
    };
    if (first < steps) {
        fetch(first);
        la.store(As[0]);
        lb.store(Bs[0]);
    }
    __syncthreads();
    for (int64_t s = first; s < steps; s++) {
        const int cur = (int)((s - first) & 1);
        if (s + 1 < steps) fetch(s + 1);
        const float *pa = As[cur] + 4 * ty, *pb = Bs[cur] + 4 * tx;
#pragma unroll
        for (int k = 0; k < kTileK; k++) {
            float av[R];
            uint64_t bv[CP];
#pragma unroll
            for (int g = 0; g < G; g++) {
                const float4 x = *reinterpret_cast<const float4*>(pa + k * kPitch + 64 * g);
                const ulonglong2 y = *reinterpret_cast<const ulonglong2*>(pb + k * kPitch + 64 * g);
                av[4 * g] = x.x; av[4 * g + 1] = x.y; av[4 * g + 2] = x.z; av[4 * g + 3] = x.w;
                bv[2 * g] = y.x; bv[2 * g + 1] = y.y;
            }
#pragma unroll
            for (int i = 0; i < R; i++) {
                const uint64_t d = twice(av[i]);
#pragma unroll
                for (int j = 0; j < CP; j++) fma2(acc[i][j], d, bv[j]);
            }
        }
        if (s + 1 < steps) {
            la.store(As[cur ^ 1]);
            lb.store(Bs[cur ^ 1]);
        }
        __syncthreads();
    }

    float v[R][2 * CP];
#pragma unroll
    for (int i = 0; i < R; i++)
#pragma unroll
        for (int j = 0; j < CP; j++) {
            const float2 h = halves(acc[i][j]);
            v[i][2 * j] = h.x;
            v[i][2 * j + 1] = h.y;
        }
    auto row_of = [&](int i) { return m0 + 4 * ty + (i & 3) + (i >> 2) * 64; };

    if (DUAL) {
        constexpr int O = CP;   // outputs of a thread, the gate's columns before the up projection's
        float bg[O], bu[O];
#pragma unroll
        for (int j = 0; j < O; j++) {
            const int c = n0 + O * tx + j;
            bg[j] = bu[j] = 0.0f;
            if (p.bg && c < nj) {
                bg[j] = to_float(static_cast<const T*>(p.bg)[bias0 + c]);
                if (MODE == GATED_HEAD) bu[j] = to_float(static_cast<const T*>(p.bg)[bias0 + ht.din + c]);
            }
            if (MODE != GATED_HEAD && p.bu && c < nj) bu[j] = to_float(static_cast<const T*>(p.bu)[c]);
        }
        float sg[O] = {}, su[O] = {};
#pragma unroll
        for (int i = 0; i < R; i++) {
            const int64_t r = row_of(i);
            if (r >= ni) continue;
#pragma unroll
            for (int j = 0; j < O; j++) {
                const int c = n0 + O * tx + j;
                if (c >= nj) continue;
                const float g = v[i][j] + bg[j], u = v[i][O + j] + bu[j];
                float a, d;
                if (MODE != GATED_HEAD) gate_both(p.act, g, a, d);
                if (MODE == GATED_FWD) {
                    static_cast<T*>(p.y)[r * p.y_row + c] = from_float<T>(a * u);
                } else if (MODE == GATED_HEAD) {   // value rows come first: g is the value, u its gate
                    p.masks[(head_row * p.band_cols + ht.off) * p.frames + r * ht.din + c] = g * sigmoid<false>(u);
                } else {
                    const float dy = to_float(static_cast<const T*>(p.dy)[r * p.y_row + c]);
                    const float dg = dy * u * d, du = dy * a;
                    static_cast<T*>(p.dg)[r * p.pre_row + c] = from_float<T>(dg);
                    static_cast<T*>(p.du)[r * p.pre_row + c] = from_float<T>(du);
                    sg[j] += dg;
                    su[j] += du;
                }
            }
        }
        if (MODE == GATED_PRE && p.col_sums) {
            // the 16 threads of a column group, through shared memory in a fixed order
            float* red = As[0];   // [ty][2][S / 2]
#pragma unroll
            for (int j = 0; j < O; j++) {
                red[ty * S + O * tx + j] = sg[j];
                red[ty * S + S / 2 + O * tx + j] = su[j];
            }
            __syncthreads();
            if (threadIdx.x < S) {
                float t = 0.0f;
                for (int r = 0; r < 16; r++) t += red[r * S + threadIdx.x];
                const int up = threadIdx.x >= S / 2, c = n0 + threadIdx.x - up * (S / 2);
                if (c < p.n) p.col_sums[((m0 / kTileM) * 2 + up) * p.n + c] = t;
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < R; i++) {
            const int64_t r = row_of(i);
            if (r >= ni) continue;
#pragma unroll
            for (int j = 0; j < 2 * CP; j++) {
                const int c = n0 + 4 * tx + (j & 3) + (j >> 2) * 64;
                if (c >= nj) continue;
                if (MODE == GATED_DX) {
                    if (p.dx_splits > 1) p.dx_part[(blockIdx.y * ni + r) * p.k + c] = v[i][j];
                    else static_cast<T*>(p.dx)[r * p.dx_row + c] = from_float<T>(v[i][j]);
                } else if (p.splits > 1) p.dw_part[((int64_t)blockIdx.y * p.n + r) * p.k + c] = v[i][j];
                else if (T* d = static_cast<T*>(p.dw[blockIdx.y])) d[r * p.dw_row[blockIdx.y] + c] = from_float<T>(v[i][j]);
            }
        }
    }
}

// A few rows: y, or dg and du, for M rows at a time, by streaming the weights once. A warp has O outputs, both weight
// rows of each, and steps along the features with all lanes (V of them to an access); the rows of x
// come from L1, where the block's warps share them. With few outputs, S warps share one and add up
// through shared memory. Bound by reading the weights, each once: one row at 5461 x 2048 bf16 (45 MB)
// takes 7.4 us, 6.0 TB/s. More rows than M go in groups of M.
constexpr int kFewRows = 8;
template <class T, int MODE, int M, int V>
__global__ void __launch_bounds__(kThreads) gated_rows(const __grid_constant__ GatedParams p) {
    constexpr bool fast = sizeof(T) == 2;
    constexpr int O = M > 2 ? 2 : 1, U = M > 2 ? 2 : 4;
    using P = Pack<T, V>;
    __shared__ float red[kThreads / 32][2 * O * M], parts[2][MODE == GATED_PRE ? kThreads / 32 * O * M : 1];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, share = p.splits, slice = warp % share;
    // blocks next to one another take the same outputs for the groups of M rows: their weights come from L2
    const int groups = (int)((p.m + M - 1) / M), block = blockIdx.x / groups;
    const int64_t m0 = (int64_t)(blockIdx.x - block * groups) * M;
    const int n0 = (block * (kThreads / 32 / share) + warp / share) * O;
    const T *w[2 * O], *x[M];
#pragma unroll
    for (int o = 0; o < O; o++) {   // an output past the last reads the last
        const int64_t n = min(n0 + o, p.n - 1);
        w[2 * o] = static_cast<const T*>(p.wg) + n * p.wg_row;
        w[2 * o + 1] = static_cast<const T*>(p.wu) + n * p.wu_row;
    }
#pragma unroll
    for (int m = 0; m < M; m++) x[m] = static_cast<const T*>(p.x) + min(m0 + m, p.m - 1) * p.x_row;
    float acc[2 * O][M];
#pragma unroll
    for (int i = 0; i < 2 * O; i++)
#pragma unroll
        for (int m = 0; m < M; m++) acc[i][m] = 0.0f;
    auto take = [&](const P (&v)[2 * O], int k) {
#pragma unroll
        for (int m = 0; m < M; m++) {
            const P xv = *reinterpret_cast<const P*>(x[m] + k);
#pragma unroll
            for (int i = 0; i < 2 * O; i++)
#pragma unroll
                for (int j = 0; j < V; j++) acc[i][m] = fmaf(to_float(v[i].v[j]), to_float(xv.v[j]), acc[i][m]);
        }
    };
    const int step = 32 * V * share, whole = p.k / V * V;
    int k = (slice * 32 + lane) * V;
    for (; k + (U - 1) * step < whole; k += U * step) {
        P v[U][2 * O];
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int i = 0; i < 2 * O; i++) v[u][i] = *reinterpret_cast<const P*>(w[i] + k + u * step);
#pragma unroll
        for (int u = 0; u < U; u++) take(v[u], k + u * step);
    }
    for (; k < whole; k += step) {
        P v[2 * O];
#pragma unroll
        for (int i = 0; i < 2 * O; i++) v[i] = *reinterpret_cast<const P*>(w[i] + k);
        take(v, k);
    }
    for (int e = whole + lane; slice == 0 && e < p.k; e += 32)   // the features past the last whole vector
#pragma unroll
        for (int m = 0; m < M; m++)
#pragma unroll
            for (int i = 0; i < 2 * O; i++) acc[i][m] = fmaf(to_float(w[i][e]), to_float(x[m][e]), acc[i][m]);
#pragma unroll
    for (int i = 0; i < 2 * O; i++)
#pragma unroll
        for (int m = 0; m < M; m++) {
            float s = acc[i][m];
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
            if (lane == 0) red[warp][i * M + m] = s;
        }
    __syncthreads();
    // one thread to an output and row
    for (int e = threadIdx.x; e < kThreads / 32 / share * O * M; e += kThreads) {
        const int out = e / M, m = e - out * M, n = block * (kThreads / 32 / share) * O + out;
        if (MODE == GATED_PRE) parts[0][e] = parts[1][e] = 0.0f;
        if (n >= p.n || m0 + m >= p.m) continue;
        float g = 0.0f, u = 0.0f;
        for (int q = 0; q < share; q++) {
            g += red[out / O * share + q][(out % O * 2) * M + m];
            u += red[out / O * share + q][(out % O * 2 + 1) * M + m];
        }
        if (p.bg) g += to_float(static_cast<const T*>(p.bg)[n]);
        if (p.bu) u += to_float(static_cast<const T*>(p.bu)[n]);
        if (MODE == GATED_FWD) {
            static_cast<T*>(p.y)[(m0 + m) * p.y_row + n] = from_float<T>(gate_value<fast>(p.act, g) * u);
        } else {
            float a, d;
            gate_both(p.act, g, a, d);
            const float dy = to_float(static_cast<const T*>(p.dy)[(m0 + m) * p.y_row + n]);
            parts[0][e] = dy * u * d;
            parts[1][e] = dy * a;
            static_cast<T*>(p.dg)[(m0 + m) * p.pre_row + n] = from_float<T>(parts[0][e]);
            static_cast<T*>(p.du)[(m0 + m) * p.pre_row + n] = from_float<T>(parts[1][e]);
        }
    }
    if (MODE == GATED_PRE && p.col_sums) {   // of the group's rows, in order
        __syncthreads();
        const int outs = kThreads / 32 / share * O, out = threadIdx.x >> 1, up = threadIdx.x & 1, n = block * outs + out;
        if (out >= outs || n >= p.n) return;
        float t = 0.0f;
        for (int m = 0; m < M; m++) t += parts[up][out * M + m];
        p.col_sums[((m0 / M) * 2 + up) * p.n + n] = t;
    }
}

// The biases' gradients from the column sums [sums][2][n] (the first sum_blocks blocks, 32 columns
// each) and dW from its partial sums [splits][2][n][k], both added in a fixed order.
template <class T>
__global__ void __launch_bounds__(kThreads) join_parts(const __grid_constant__ GatedParams p, int64_t sums, unsigned sum_blocks, T* dwg,
                                                       int64_t dwg_row, T* dwu, int64_t dwu_row, T* dbg, T* dbu) {
    if (blockIdx.x < sum_blocks) {
        __shared__ float red[8][33];
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        const int64_t i = (int64_t)blockIdx.x * 32 + lane, n2 = 2 * (int64_t)p.n;
        float s = 0.0f;
        if (i < n2)
#pragma unroll 4
            for (int64_t t = warp; t < sums; t += 8) s += p.col_sums[t * n2 + i];
        red[warp][lane] = s;
        __syncthreads();
        if (warp || i >= n2) return;
        for (int w = 1; w < 8; w++) s += red[w][lane];
        T* d = i < p.n ? dbg : dbu;
        if (d) d[i < p.n ? i : i - p.n] = from_float<T>(s);
        return;
    }
    const int64_t total = 2 * (int64_t)p.n * p.k, blocks = gridDim.x - sum_blocks;
    const bool wide = p.k % 4 == 0;
    for (int64_t i = ((blockIdx.x - sum_blocks) * (int64_t)kThreads + threadIdx.x) * 4; i < total; i += blocks * kThreads * 4) {
        float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int q = 0; q < p.splits; q++) {
            const float* from = p.dw_part + q * total + i;
            if (wide) {
                const float4 v = *reinterpret_cast<const float4*>(from);
                s[0] += v.x; s[1] += v.y; s[2] += v.z; s[3] += v.w;
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (i + e < total) s[e] += from[e];
            }
        }
        const int64_t row4 = i / p.k;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            if (i + e >= total) break;
            const int64_t row = wide ? row4 : (i + e) / p.k, c = i + e - row * p.k;   // row of [dWg; dWu]
            const bool up = row >= p.n;
            T* d = up ? dwu : dwg;
            if (d) d[(up ? row - p.n : row) * (up ? dwu_row : dwg_row) + c] = from_float<T>(s[e]);
        }
    }
}

// dx from its partial sums, added in order.
template <class T> __global__ void __launch_bounds__(kThreads) join_dx(const __grid_constant__ GatedParams p) {
    const int64_t total = p.m * p.k;
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < total; i += (int64_t)gridDim.x * kThreads) {
        float s = 0.0f;
        for (int q = 0; q < p.dx_splits; q++) s += p.dx_part[q * total + i];
        const int64_t r = i / p.k;
        static_cast<T*>(p.dx)[r * p.dx_row + i - r * p.k] = from_float<T>(s);
    }
}

// Copies of up to three matrices of one width, their rows `pitch` elements apart, for operands
// whose rows are no whole 16 bytes. A thread makes 16 bytes of a copy; elements past the width are 0.
struct RepackParams {
    const void* src[3];
    void* dst[3];
    int64_t row[3], rows[3];
    int cols;
    FastDiv pieces;      // of 16 bytes in a row
};
template <class T>
__global__ void __launch_bounds__(kThreads) repack(const __grid_constant__ RepackParams p) {
    const int z = blockIdx.y;
    const int64_t total = p.rows[z] * p.pieces.d;
    const T* src = static_cast<const T*>(p.src[z]);
    const bool pairs = p.row[z] % 2 == 0 && reinterpret_cast<uintptr_t>(src) % 4 == 0;
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < total; i += (int64_t)gridDim.x * kThreads) {
        const int64_t r = total < (1ll << 31) ? p.pieces.div((uint32_t)i) : i / p.pieces.d;
        const int c = (int)(i - r * p.pieces.d) * 8;
        const T* from = src + r * p.row[z] + c;
        Pack<T, 8> v;
        if (pairs && c + 8 <= p.cols) {
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                const Pack<T, 2> w = *reinterpret_cast<const Pack<T, 2>*>(from + e);
                v.v[e] = w.v[0];
                v.v[e + 1] = w.v[1];
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) v.v[e] = c + e < p.cols ? from[e] : from_float<T>(0.0f);
        }
        *reinterpret_cast<Pack<T, 8>*>(static_cast<T*>(p.dst[z]) + i * 8) = v;
    }
}

// ---- host -------------------------------------------------------------------------------------

size_t up256(size_t n) { return (n + 255) / 256 * 256; }
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// The kernels' 32-bit positions along features and outputs reach a tile, or gated_rows' steps, past the last one.
constexpr int kMostSpan = INT32_MAX - 65535;
void check_span(int n, const char* what) {
    if (n > kMostSpan) fail(STG_UNSUPPORTED, std::string(what) + " above 2^31 - 2^16");
}

void check_config(const stg_gated_config* c, bool backward) {
    check_sized(c, "gated");
    check(valid_dtype(c->dtype), "gated: unknown dtype");
    check(valid_activation(c->activation), "gated: unknown activation");
    check(c->features >= 1 && c->width >= 1 && c->rows >= 0, "gated: features and width must be at least 1, rows at least 0");
    if (c->rows > INT32_MAX) fail(STG_UNSUPPORTED, "gated: too many rows");
    check_span(c->features, "gated: features");
    check_span(c->width, "gated: width");
    // operands broadcast by strides of 0 make such sizes possible: the scratch's bytes must not pass 64 bits
    const int64_t most = 1ll << 50, rows = std::max<int64_t>(c->rows, 1);
    if (c->width > most / rows || c->features > most / rows || c->features > most / c->width)
        fail(STG_UNSUPPORTED, "gated: a matrix of more than 2^50 elements");
    check(c->x_row >= 0 && c->wg_row >= 0 && c->wu_row >= 0 && c->y_row >= 0, "gated: negative stride");
    check((c->y_row >= c->width || c->rows <= 1) || backward, "gated: the output's rows overlap");
}

// Which operands the tensor-core path needs a repacked copy of (bytes, 0: none): it reads by
// TMA, whose rows are a multiple of 16 bytes apart and do not overlap (as a broadcast's do).
struct Copies { size_t x = 0, wg = 0, wu = 0; size_t bytes() const { return x + wg + wu; } };
size_t copy_bytes(int64_t rows, int64_t row, int cols) {
    return rows <= 1 || (row % 8 == 0 && row >= cols) ? 0 : up256((size_t)rows * (size_t)(ceil_div(cols, 8) * 8) * 2);
}
Copies copies_of(const stg_gated_config& c, bool backward) {
    Copies r;
    if (c.dtype == STG_F32 || !c.rows || (!backward && c.rows <= kFewRows)) return r;
    r.x = copy_bytes(c.rows, c.x_row, c.features);
    r.wg = copy_bytes(c.width, c.wg_row, c.features);
    r.wu = copy_bytes(c.width, c.wu_row, c.features);
    return r;
}
// Makes the copies in ws and points p at them.
template <class T> void copy_operands(GatedParams& p, const Copies& copies, int64_t x_rows, int64_t w_rows, char* ws, cudaStream_t st) {
    if (!copies.bytes()) return;
    RepackParams r{};
    r.cols = p.k;
    r.pieces = FastDiv((uint32_t)ceil_div(p.k, 8));
    int n = 0;
    int64_t most = 0;
    auto add = [&](const void*& src, int64_t& row, size_t bytes, int64_t rows) {
        if (!bytes) return;
        r.src[n] = src;
        r.dst[n] = ws;
        r.row[n] = row;
        r.rows[n] = rows;
        n++;
        most = std::max(most, rows);
        src = ws;
        row = ceil_div(p.k, 8) * 8;
        ws += bytes;
    };
    add(p.x, p.x_row, copies.x, x_rows);
    add(p.wg, p.wg_row, copies.wg, w_rows);
    add(p.wu, p.wu_row, copies.wu, w_rows);
    const unsigned blocks = (unsigned)std::min<int64_t>(ceil_div(most * r.pieces.d, kThreads), 148 * 16);
    repack<T><<<dim3(blocks, n), kThreads, 0, st>>>(r);
}

dim3 tile_grid(int64_t tiles, int64_t y = 1) {
    if (tiles > INT32_MAX || y > 65535) fail(STG_UNSUPPORTED, "gated: too many tiles");
    return dim3((unsigned)tiles, (unsigned)y);
}

// A product of float tiles, as 128 x 128 ones or, when those number fewer than one and a half per SM, 64 x 64
// ones, of which an SM holds three or four where it holds two of the large ones (one in dx and the mask head, whose f32
// kernels have 132 and 134 registers). f32, 64 and 128 wide in us: y of 384 x 1408 at 1000 rows (176 large tiles)
// 71 and 77, at 1300 (242) 96 and 78; dx there at 4000 rows (96) 285 and 271; dW at 1300 rows (330) 84 and 64, at
// 777 x 301 x 515 (90) 27 and 88. Not the better one everywhere below the border: y of 1024 x 1024 at 1000 rows (128) 146 and 111.
// out: columns of a 128-wide tile.
template <class T, int MODE> int launch_simt(const GatedParams& p, int64_t rows, int64_t cols, int out, int64_t y, cudaStream_t st) {
    auto tiles = [&](int s) { return ceil_div(rows, s) * ceil_div(cols, out * s / 128); };
    if (MODE == GATED_HEAD || tiles(128) * y >= 222) {
        gated_simt<T, MODE, 128><<<tile_grid(MODE == GATED_HEAD ? rows : tiles(128), y), kThreads, 0, st>>>(p);
        return 128;
    }
    if constexpr (MODE != GATED_HEAD) gated_simt<T, MODE, 64><<<tile_grid(tiles(64), y), kThreads, 0, st>>>(p);
    return 64;
}

// Off the tensor cores gated_rows also takes more rows than eight, in groups of eight, up to 32 rows or
// while gated_simt's tiles of 64 rows x 32 outputs would leave half the SMs idle: each such tile walks
// all features alone, 43 ns a feature. float, features x outputs, gated_rows against gated_simt in us:
// 2048 x 5461 at 16 rows 50 and 142, at 32 88 and 143, at 64 167 and 146; 1024 x 1024 at 64 rows 21 and
// 47, at 128 37 and 47, at 192 52 and 47; 4096 x 1000 at 128 rows 107 and 176.
// So does the backward pass with its projections: whole, at 2048 x 5461 and 8 rows 217 us for 318, at
// 1024 x 1024 and 32 rows 43 for 78.
bool few_tiles(int64_t rows, int64_t width) {
    return rows <= 4 * kFewRows || ceil_div(rows, 64) * ceil_div(width, 32) <= 148 / 2;
}

struct GatedLayout { size_t dg = 0, du = 0, sums = 0, dw = 0, dx = 0, copies = 0, bytes = 0; int64_t pre_row = 0; int splits = 1, dx_splits = 1; int64_t split_rows = 0; };

GatedLayout backward_layout(const stg_gated_config& c) {
    GatedLayout l;
    const size_t es = elem_size(c.dtype);
    l.pre_row = ceil_div(c.width, 8) * 8;
    l.du = up256((size_t)c.rows * l.pre_row * es);
    l.sums = l.du + up256((size_t)c.rows * l.pre_row * es);
    // dW has 2 width x features outputs and a sum over all rows: rows are split until the tiles
    // fill the GPU, while a part keeps at least 256 rows, into at most 64 parts
    // (f32: 128 x 128 tiles, two blocks per SM; else pairs of SMs and their 256 x 224 tiles).
    // bf16, product and joining in us with parts of at least 64, 256 and 1024 rows: 2000 x 64 x 64 10.4, 10.0 and
    // 11.6; 2000 x 384 x 136 16.2, 12.7 and 12.9; 777 x 301 x 515 23.8, 18.8 and 17.0; f32 there 29 and 31.
    // With one part the product writes dW itself: the backward pass at 5461 x 2048 bf16 and 256 rows
    // takes 109 us, with float sums (89 MB) and a kernel that converts them 184.
    const bool f32 = c.dtype == STG_F32;
    const int64_t tiles = 2 * ceil_div(c.width, f32 ? 128 : 256) * ceil_div(c.features, f32 ? 128 : 224);
    const int64_t want = f32 ? ceil_div(2 * 148, tiles) : std::max<int64_t>(1, 74 / tiles);
    l.splits = (int)std::max<int64_t>(1, std::min<int64_t>({want, c.rows / 256, 64}));
    // float: sums in order of at most 4096 terms, while 64 parts (in dx 32) are enough for that: longer ones lose
    // digits to a library's
    if (f32) l.splits = (int)std::max<int64_t>(l.splits, std::min<int64_t>(64, ceil_div(c.rows, 4096)));
    l.split_rows = std::max<int64_t>(64, ceil_div(ceil_div(c.rows, l.splits), 64) * 64);
    l.splits = (int)std::max<int64_t>(1, ceil_div(c.rows, l.split_rows));
    l.dw = l.sums + up256(sizeof(float) * (size_t)std::max<int64_t>(ceil_div(c.rows, few_tiles(c.rows, c.width) ? kFewRows : 64), l.splits * ceil_div(c.features, 64)) * 2 * c.width);
    if (f32) {   // dx likewise: its sums are 2 width long, its tiles few when rows and features are
        const int64_t tiles128 = ceil_div(c.rows, 128) * ceil_div(c.features, 128), tiles64 = ceil_div(c.rows, 64) * ceil_div(c.features, 64);
        const int64_t more = tiles128 >= 222 ? 1 : std::min<int64_t>(ceil_div(296, tiles64), 2 * (int64_t)c.width / 256);
        l.dx_splits = (int)std::min<int64_t>(32, std::max<int64_t>({1, more, ceil_div(2 * (int64_t)c.width, 4096)}));
    }
    l.dx = l.dw + (l.splits > 1 ? up256(sizeof(float) * (size_t)l.splits * 2 * c.width * c.features) : 0);
    l.copies = l.dx + (l.dx_splits > 1 ? up256(sizeof(float) * (size_t)l.dx_splits * c.rows * c.features) : 0);
    l.bytes = l.copies + copies_of(c, true).bytes();
    return l;
}

GatedParams params_of(const stg_gated_config& c) {
    GatedParams p{};
    p.m = c.rows; p.n = c.width; p.k = c.features;
    p.act = c.activation;
    p.x_row = c.x_row; p.wg_row = c.wg_row; p.wu_row = c.wu_row; p.y_row = c.y_row; p.dx_row = c.dx_row;
    return p;
}

// f16 and bf16 go to the tensor cores where the operands that are not copied start on 16 bytes.
bool on_tensor_cores(const stg_gated_config& c, const Copies& copies, const GatedParams& p) {
    return c.dtype != STG_F32 && (copies.x || aligned(p.x, 16)) && (copies.wg || aligned(p.wg, 16)) && (copies.wu || aligned(p.wu, 16));
}

// A few rows (gated_rows): below that the tensor cores' 256-row tiles are nearly empty, and at 5461 x
// 2048 bf16 they read the weights at 1.2 TB/s. Vectors of 16 bytes where every row starts on 16.
template <class T, int MODE, int M> void launch_rows(GatedParams p, cudaStream_t st) {
    constexpr int O = M > 2 ? 2 : 1, W = 16 / (int)sizeof(T);
    // warps to an output: more while that gives fewer than eight warps per SM
    p.splits = 1;
    while (p.splits < kThreads / 32 && ceil_div(p.n, O) * ceil_div(p.m, M) * p.splits < 148 * 8 && p.k > 32 * W * p.splits) p.splits *= 2;
    const unsigned blocks = (unsigned)(ceil_div(ceil_div(p.n, O), kThreads / 32 / p.splits) * ceil_div(p.m, M));
    const bool wide = aligned(p.x, 16) && aligned(p.wg, 16) && aligned(p.wu, 16) && (p.x_row % W == 0 || p.m == 1) &&
                      (p.wg_row % W == 0 || p.n == 1) && (p.wu_row % W == 0 || p.n == 1);
    if (wide) gated_rows<T, MODE, M, W><<<blocks, kThreads, 0, st>>>(p);
    else gated_rows<T, MODE, M, 1><<<blocks, kThreads, 0, st>>>(p);
}

} // namespace

} // namespace stg

extern "C" {

STG_API stg_status stg_gated_workspace(const stg_gated_config* c, int32_t backward, size_t* bytes) {
    return guard(nullptr, [&] {
        check_config(c, backward != 0);
        check(bytes && (backward == 0 || backward == 1), "gated: null buffer");
        *bytes = !c->rows ? 0 : backward ? backward_layout(*c).bytes : copies_of(*c, false).bytes();
    });
}

STG_API stg_status stg_gated(stg_engine* e, const stg_gated_config* c, const void* d_x, const void* d_wg, const void* d_wu,
                             const void* d_bg, const void* d_bu, void* d_y, void* d_ws, size_t ws_bytes, void* stream) {
    if (!e) return STG_INVALID_ARGUMENT;
    return guard(e, [&] {
        check_config(c, false);
        const size_t es = elem_size(c->dtype);
        for (const void* q : {d_x, d_wg, d_wu, d_bg, d_bu, (const void*)d_y}) check(aligned(q, es), "gated: a buffer is not aligned to its elements");
        if (!c->rows) return;
        check(d_x && d_wg && d_wu && d_y, "gated: null buffer");
        GatedParams p = params_of(*c);
        p.x = d_x; p.wg = d_wg; p.wu = d_wu; p.bg = d_bg; p.bu = d_bu; p.y = d_y;
        DeviceScope scope(e);
        const cudaStream_t st = static_cast<cudaStream_t>(stream);
        const Copies copies = copies_of(*c, false);
        check(!copies.bytes() || (d_ws && aligned(d_ws, 256) && ws_bytes >= copies.bytes()), "gated: workspace is missing, unaligned or too small");
        with_dtype(c->dtype, [&](auto* tag) {
            using T = std::remove_pointer_t<decltype(tag)>;
            if (p.m == 1) return launch_rows<T, GATED_FWD, 1>(p, st);
            if (p.m == 2) return launch_rows<T, GATED_FWD, 2>(p, st);
            if (p.m <= 4) return launch_rows<T, GATED_FWD, 4>(p, st);
            if (p.m <= kFewRows) return launch_rows<T, GATED_FWD, kFewRows>(p, st);
            if (on_tensor_cores(*c, copies, p)) {
                copy_operands<T>(p, copies, p.m, p.n, static_cast<char*>(d_ws), st);
                return launch_gated_mma(GATED_FWD, c->dtype == STG_BF16, p, 0, e->sms, st);
            }
            if (few_tiles(p.m, p.n)) return launch_rows<T, GATED_FWD, kFewRows>(p, st);
            launch_simt<T, GATED_FWD>(p, p.m, p.n, 64, 1, st);
        });
        cuda_check(cudaGetLastError(), "gated kernel");
    });
}

STG_API stg_status stg_gated_backward(stg_engine* e, const stg_gated_config* c, const void* d_dy, const void* d_x, const void* d_wg,
                                      const void* d_wu, const void* d_bg, const void* d_bu, void* d_dx, void* d_dwg, void* d_dwu,
                                      void* d_dbg, void* d_dbu, void* d_ws, size_t ws_bytes, void* stream) {
    if (!e) return STG_INVALID_ARGUMENT;
    return guard(e, [&] {
        check_config(c, true);
        const size_t es = elem_size(c->dtype);
        for (const void* q : {d_dy, d_x, d_wg, d_wu, d_bg, d_bu, (const void*)d_dx, (const void*)d_dwg, (const void*)d_dwu, (const void*)d_dbg, (const void*)d_dbu})
            check(aligned(q, es), "gated: a buffer is not aligned to its elements");
        check(!d_dx || c->dx_row >= c->features || c->rows <= 1, "gated: the rows of dx overlap");
        check((!d_dwg || c->dwg_row >= c->features || c->width == 1) && (!d_dwu || c->dwu_row >= c->features || c->width == 1),
              "gated: the rows of a weight's gradient overlap");
        DeviceScope scope(e);
        const cudaStream_t st = static_cast<cudaStream_t>(stream);
        if (!c->rows) {   // sums over no rows
            auto zero = [&](void* d, int64_t row, int64_t w, int64_t h) {
                if (d) cuda_check(cudaMemset2DAsync(d, (size_t)std::max(row, w) * es, 0, (size_t)w * es, (size_t)h, st), "gated memset");
            };
            zero(d_dwg, c->dwg_row, c->features, c->width);
            zero(d_dwu, c->dwu_row, c->features, c->width);
            zero(d_dbg, c->width, c->width, 1);
            zero(d_dbu, c->width, c->width, 1);
            return;
        }
        check(d_dy && d_x && d_wg && d_wu, "gated: null buffer");
        if (!d_dx && !d_dwg && !d_dwu && !d_dbg && !d_dbu) return;
        const GatedLayout lay = backward_layout(*c);
        check(d_ws && aligned(d_ws, 256) && ws_bytes >= lay.bytes, "gated: workspace is missing, unaligned or too small");
        char* ws = static_cast<char*>(d_ws);
        GatedParams p = params_of(*c);
        p.dy = d_dy; p.x = d_x; p.wg = d_wg; p.wu = d_wu; p.bg = d_bg; p.bu = d_bu; p.dx = d_dx;
        p.dg = ws;
        p.du = ws + lay.du;
        p.pre_row = lay.pre_row;
        p.col_sums = d_dbg || d_dbu ? reinterpret_cast<float*>(ws + lay.sums) : nullptr;
        p.dw[0] = d_dwg; p.dw[1] = d_dwu;
        p.dw_row[0] = c->dwg_row; p.dw_row[1] = c->dwu_row;
        p.dw_part = reinterpret_cast<float*>(ws + lay.dw);
        p.splits = lay.splits;
        p.dx_part = reinterpret_cast<float*>(ws + lay.dx);
        p.dx_splits = lay.dx_splits;
        p.split_rows = lay.split_rows;
        auto join = [&](auto* tag, int64_t sums) {   // the partial sums of dW and of the biases' gradients
            using T = std::remove_pointer_t<decltype(tag)>;
            const bool dw = p.splits > 1 && (d_dwg || d_dwu);
            if (!dw && !p.col_sums) return;
            const unsigned sum_blocks = p.col_sums ? (unsigned)ceil_div(2 * (int64_t)p.n, 32) : 0;
            const unsigned dw_blocks = dw ? (unsigned)std::min<int64_t>(ceil_div(2 * (int64_t)p.n * p.k, 4 * kThreads), 148 * 8) : 0;
            join_parts<T><<<sum_blocks + dw_blocks, kThreads, 0, st>>>(p, sums, sum_blocks, static_cast<T*>(d_dwg), c->dwg_row, static_cast<T*>(d_dwu),
                                                                       c->dwu_row, static_cast<T*>(d_dbg), static_cast<T*>(d_dbu));
        };
        with_dtype(c->dtype, [&](auto* tag) {
            using T = std::remove_pointer_t<decltype(tag)>;
            const Copies copies = copies_of(*c, true);
            if (on_tensor_cores(*c, copies, p)) {
                copy_operands<T>(p, copies, p.m, p.n, ws + lay.copies, st);
                auto product = [&](GatedMode mode) { launch_gated_mma(mode, c->dtype == STG_BF16, p, 0, e->sms, st); };
                product(GATED_PRE);
                if (d_dx) product(GATED_DX);
                if (d_dwg || d_dwu || p.col_sums) product(GATED_DW);
                join((T*)nullptr, gated_col_sums(p, e->sms));
                return;
            }
            int pre = kFewRows;   // rows to a column sum
            if (few_tiles(p.m, p.n)) launch_rows<T, GATED_PRE, kFewRows>(p, st);
            else pre = launch_simt<T, GATED_PRE>(p, p.m, p.n, 64, 1, st);
            if (d_dx) {
                launch_simt<T, GATED_DX>(p, p.m, p.k, 128, p.dx_splits, st);
                if (p.dx_splits > 1) join_dx<T><<<(unsigned)std::min<int64_t>(ceil_div(p.m * p.k, kThreads), 148 * 8), kThreads, 0, st>>>(p);
            }
            if (d_dwg || d_dwu) launch_simt<T, GATED_DW>(p, p.n, p.k, 128, 2 * p.splits, st);
            join((T*)nullptr, ceil_div(p.m, pre));
        });
        cuda_check(cudaGetLastError(), "gated kernel");
    });
}

STG_API stg_status stg_engine_status(stg_engine* e) {
    if (!e) return STG_INVALID_ARGUMENT;
    return guard(e, [&] {
        DeviceScope scope(e);
        if (gated_gave_up()) fail(STG_INTERNAL_ERROR, "a kernel of the gated projection gave up a wait: its result is incomplete");
    });
}

static void check_head(const stg_plan* p, const stg_mask_head_config* c) {
    check_sized(c, "mask head");
    check(p->H.arch == ARCH_ROFORMER && !p->H.band_din.empty(), "mask head: not a RoFormer plan");
    check(valid_dtype(c->dtype), "mask head: unknown dtype");
    check(c->hidden >= 1 && c->n_chunks >= 0, "mask head: hidden must be at least 1, n_chunks at least 0");
    check_span(c->hidden, "mask head: hidden");
}

static int64_t head_rows(const stg_plan* p, const stg_mask_head_config* c) {
    return (int64_t)c->n_chunks * p->H.S * (int64_t)p->H.band_din.size() * p->H.g.T;
}
static Copies head_copies(const stg_plan* p, const stg_mask_head_config* c) {
    Copies r;
    if (c->dtype == STG_F32 || !c->n_chunks) return r;
    r.x = copy_bytes(head_rows(p, c), c->hidden, c->hidden);
    r.wg = copy_bytes(p->H.S * 2 * (p->H.stem_stride / p->H.g.T), c->hidden, c->hidden);
    return r;
}

STG_API stg_status stg_mask_head_sizes(const stg_plan* p, int32_t* stems, int32_t* bands, int32_t* frames, int64_t* columns) {
    if (!p) return STG_INVALID_ARGUMENT;
    return guard(p->engine, [&] {
        check(p->H.arch == ARCH_ROFORMER && !p->H.band_din.empty(), "mask head: not a RoFormer plan");
        check(stems && bands && frames && columns, "mask head: null buffer");
        *stems = p->H.S;
        *bands = (int32_t)p->H.band_din.size();
        *frames = p->H.g.T;
        *columns = p->H.stem_stride / p->H.g.T;
    });
}

STG_API stg_status stg_mask_head_workspace(const stg_plan* p, const stg_mask_head_config* c, size_t* bytes) {
    if (!p) return STG_INVALID_ARGUMENT;
    return guard(p->engine, [&] {
        check_head(p, c);
        check(bytes, "mask head: null buffer");
        *bytes = head_copies(p, c).bytes();
    });
}

STG_API stg_status stg_mask_head(stg_plan* plan, const stg_mask_head_config* c, const void* d_hidden, const void* d_weight,
                                 const void* d_bias, float* d_masks, void* d_ws, size_t ws_bytes, void* stream) {
    if (!plan) return STG_INVALID_ARGUMENT;
    return guard(plan->engine, [&] {
        check_head(plan, c);
        const size_t es = elem_size(c->dtype);
        for (const void* q : {d_hidden, d_weight, d_bias}) check(aligned(q, es), "mask head: a buffer is not aligned to its elements");
        if (!c->n_chunks) return;
        check(d_hidden && d_weight && d_masks, "mask head: null buffer");
        plan->H.check_mask(d_masks);
        GatedParams p{};
        p.x = d_hidden; p.wg = d_weight; p.bg = d_bias; p.masks = d_masks;
        p.k = c->hidden;
        p.frames = plan->H.g.T;
        p.bands = (int)plan->H.band_din.size();
        p.stems = plan->H.S;
        p.band_cols = plan->H.stem_stride / plan->H.g.T;
        p.tiles = plan->d_head.as<HeadTile>();
        p.n_tiles = plan->head_tiles;
        DeviceScope scope(plan->engine);
        const cudaStream_t st = static_cast<cudaStream_t>(stream);
        const Copies copies = head_copies(plan, c);
        check(!copies.bytes() || (d_ws && aligned(d_ws, 256) && ws_bytes >= copies.bytes()), "mask head: workspace is missing, unaligned or too small");
        const int64_t rows = head_rows(plan, c);
        with_dtype(c->dtype, [&](auto* tag) {
            using T = std::remove_pointer_t<decltype(tag)>;
            if (c->dtype != STG_F32 && rows <= INT32_MAX && (copies.x || aligned(d_hidden, 16)) && (copies.wg || aligned(d_weight, 16))) {
                p.x_row = p.wg_row = p.k;
                copy_operands<T>(p, copies, rows, p.stems * 2 * p.band_cols, static_cast<char*>(d_ws), st);
                p.tiles += plan->head_tiles;
                p.n_tiles = plan->head_wide;
                return launch_gated_mma(GATED_HEAD, c->dtype == STG_BF16, p, rows, plan->engine->sms, st);
            }
            launch_simt<T, GATED_HEAD>(p, (int64_t)c->n_chunks * p.stems * ceil_div(p.frames, kGatedTileM) * p.n_tiles, 0, 64, 1, st);
        });
        cuda_check(cudaGetLastError(), "mask head kernel");
    });
}

} // extern "C"
