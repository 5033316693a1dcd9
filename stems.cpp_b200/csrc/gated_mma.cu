// gated_mma.cu -- the gated projection's products on the tensor cores, f16 and bf16
// (gated.h: GatedMode; the mathematics is in gated.cu).
//
// One persistent block per SM walks 128-row output tiles. A producer thread brings 64-deep
// slices of the operands into a ring of shared-memory stages by TMA (128-byte swizzle); one
// thread issues tcgen05.mma with float accumulators in TMEM; eight warps read finished
// accumulators back, apply the epilogue and store. Two accumulator sets let the epilogue of a
// tile run under the products of the next. In the forward modes a stage holds Wg's and Wu's
// rows of the same output columns one behind the other, so one instruction computes both
// projections and a thread of the epilogue finds g and u of an output in its own TMEM lane: the
// projections never leave the SM.
//
// Where an operand's contraction is not its contiguous axis (W in dx = dg Wg + du Wu; all of
// dW = dg^T x), the tile goes to shared memory as it lies and the instruction reads it
// MN-major, so nothing is transposed in memory.
#include "gated.h"

#include <cuda.h>

namespace stg {

namespace {

constexpr int kThreads = 384;      // warp 0 TMA, warp 1 MMA, warp 2 TMEM, warps 4..11 epilogue
constexpr int kEpilogueWarps = 8;
constexpr int kDepth = 64;         // contraction per stage: 128 bytes, one swizzle row
constexpr int kABytes = kGatedTileM * kDepth * 2;

// Kernels that gave up a wait (never, unless a copy or a product failed): see wait().
__device__ unsigned int g_gave_up;

struct MmaParams {
    GatedParams g;
    CUtensorMap a[2], b[2], c[2];
    int64_t tiles;
    int tiles_n;                   // column tiles of a row of tiles
    int cols;                      // columns of a tile (the instruction's N; outputs x 2 in the forward modes)
    int store_by_tma;
};

// ---- PTX -------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void bar_init(uint64_t* b, uint32_t n) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_addr(b)), "r"(n));
}
__device__ __forceinline__ void bar_expect(uint64_t* b, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_addr(b)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint64_t* b) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(b)) : "memory");
}
__device__ __forceinline__ bool bar_try(uint64_t* b, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}"
                 : "=r"(ok) : "r"(smem_addr(b)), "r"(parity) : "memory");
    return ok != 0;
}
__device__ __forceinline__ uint64_t now_ns() {
    uint64_t t;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
    return t;
}
// Waits for a barrier's phase; gives up after ten seconds, or when another thread of the block
// has, so that no failure leaves the GPU spinning. After that every wait fails at once, the
// block runs out its loops without work and frees what it holds.
__device__ __noinline__ bool wait_slow(uint64_t* b, uint32_t parity, volatile int* dead) {
    const uint64_t t0 = now_ns();
    for (uint32_t i = 0;; i++) {
        if (bar_try(b, parity)) return true;
        if ((i & 63) == 63 && (*dead || now_ns() - t0 > 10000000000ull)) break;
    }
    if (!*dead) {
        *dead = 1;
        atomicExch(&g_gave_up, 1u);
    }
    return false;
}
__device__ __forceinline__ bool wait(uint64_t* b, uint32_t parity, volatile int* dead) {
#pragma unroll 1
    for (int i = 0; i < 16; i++)
        if (bar_try(b, parity)) return true;
    return wait_slow(b, parity, dead);
}
__device__ __forceinline__ void tma_load(void* dst, const CUtensorMap* m, int x, int y, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
                     smem_addr(dst)), "l"(m), "r"(x), "r"(y), "r"(smem_addr(bar)) : "memory");
}
__device__ __forceinline__ void tma_store(const CUtensorMap* m, int x, int y, const void* src) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(m), "r"(x), "r"(y), "r"(
                     smem_addr(src)) : "memory");
}
__device__ __forceinline__ void store_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
__device__ __forceinline__ void stores_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d), "l"(a),
                 "l"(b), "r"(idesc), "r"((uint32_t)add) : "memory");
}
// The barrier's phase completes when the products issued so far have.
__device__ __forceinline__ void mma_commit(uint64_t* b) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(b)) : "memory");
}
__device__ __forceinline__ void tmem_load32(uint32_t (&v)[32], uint32_t addr) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, "
        "%20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
          "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]),
          "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]),
          "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(addr));
}
__device__ __forceinline__ void tmem_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }

// Shared-memory matrix descriptor, 128-byte swizzle: address and offsets in 16-byte units, bit
// 46 the descriptor's version, layout 2 in bits 61..63. K-major: rows of 128 bytes, groups of
// eight 1024 bytes apart. MN-major: the same rows run along m or n, 64 of them; `lead` is the distance
// of the next 64.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lead) {
    return (uint64_t)((addr & 0x3ffff) >> 4) | (uint64_t)(lead >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | 1ull << 46 | 2ull << 61;
}

template <class T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}

// ---- activations: results are rounded to 16 bits, so the fast exponential and division do -----------
template <int ACT> __device__ __forceinline__ float act(float z) {
    if (ACT == STG_ACT_RELU) return z < 0.0f ? 0.0f : z;
    if (ACT == STG_ACT_SILU) return z * sigmoidf(z);
    if (ACT == STG_ACT_GELU) return 0.5f * z * erfcf(-z * 0.70710678118654752f);
    if (ACT == STG_ACT_SIGMOID) return sigmoidf(z);
    return z;
}
// act(z) and its derivative.
template <int ACT> __device__ __forceinline__ void act_both(float z, float& a, float& d) {
    if (ACT == STG_ACT_RELU) {
        a = z < 0.0f ? 0.0f : z;
        d = z > 0.0f ? 1.0f : (z <= 0.0f ? 0.0f : z);
    } else if (ACT == STG_ACT_SILU) {
        const float s = sigmoidf(z);
        a = z * s;
        d = fmaf(a, 1.0f - s, s);
    } else if (ACT == STG_ACT_GELU) {
        const float h = 0.5f * erfcf(-z * 0.70710678118654752f);
        a = z * h;
        d = fmaf(0.3989422804014327f * z, __expf(-0.5f * z * z), h);
    } else if (ACT == STG_ACT_SIGMOID) {
        a = sigmoidf(z);
        d = a * (1.0f - a);
    } else {
        a = z;
        d = 1.0f;
    }
}

// Where a tile lies.
struct Tile {
    int64_t m0;      // first output row
    int n0;          // first output column
    int a_y, b_y;    // coordinates of the operands' rows
    int up_y;
    int kb;          // stages
    int part;        // DW: gate or up, and split
    HeadTile h;
    int64_t cs;      // mask head: chunk * stems + stem
};

template <int MODE> __device__ __forceinline__ Tile tile_at(const MmaParams& p, int64_t t) {
    Tile r{};
    const GatedParams& g = p.g;
    if (MODE == GATED_HEAD) {
        // frames first: a band's rows and its weights are then read by neighbours in time
        const int64_t mt = (g.frames + kGatedTileM - 1) / kGatedTileM, rest = t / mt;
        r.m0 = (t - rest * mt) * kGatedTileM;
        r.cs = rest / g.n_tiles;
        r.h = g.tiles[rest - r.cs * g.n_tiles];
        r.n0 = r.h.n0;
        r.a_y = (int)((r.cs * g.bands + r.h.band) * g.frames + r.m0);
        r.b_y = (int)((r.cs % g.stems) * 2 * g.band_cols + 2 * (int64_t)r.h.off + r.n0);
        r.up_y = r.b_y + r.h.din;
        r.kb = (g.k + kDepth - 1) / kDepth;
    } else if (MODE == GATED_FWD || MODE == GATED_PRE) {
        const int64_t mt = t / p.tiles_n;
        r.m0 = mt * kGatedTileM;
        r.n0 = (int)(t - mt * p.tiles_n) * (p.cols / 2);
        r.a_y = (int)r.m0;
        r.b_y = r.up_y = r.n0;
        r.kb = (g.k + kDepth - 1) / kDepth;
    } else if (MODE == GATED_DX) {
        const int64_t mt = t / p.tiles_n;
        r.m0 = mt * kGatedTileM;
        r.n0 = (int)(t - mt * p.tiles_n) * p.cols;
        r.a_y = (int)r.m0;
        r.kb = 2 * ((g.n + kDepth - 1) / kDepth);
    } else {
        const int tm = (g.n + kGatedTileM - 1) / kGatedTileM;
        const int64_t q = t / p.tiles_n;
        r.n0 = (int)(t - q * p.tiles_n) * p.cols;
        r.part = (int)(q / tm);                          // 2 split + (gate, up)
        r.m0 = (q - (int64_t)r.part * tm) * kGatedTileM;
        const int64_t beg = (r.part >> 1) * g.split_rows;
        r.a_y = (int)beg;
        r.kb = (int)((min(g.m, beg + g.split_rows) - beg + kDepth - 1) / kDepth);
    }
    return r;
}

template <int MODE> __host__ __device__ constexpr int b_bytes() { return MODE == GATED_HEAD ? 128 * kDepth * 2 : 256 * kDepth * 2; }
// Per epilogue warp: 32 rows x 32 columns of output, for dg and du each (float in the mask head,
// rows 33 apart), and 64 floats of each bias.
template <int MODE> __host__ __device__ constexpr int out_bytes() {
    return MODE == GATED_PRE ? 4096 : MODE == GATED_HEAD ? 32 * 33 * 4 : MODE == GATED_DW ? 0 : 2048;
}
template <int MODE> __host__ __device__ constexpr int stages() { return MODE == GATED_HEAD ? 5 : MODE == GATED_PRE ? 3 : 4; }
template <int MODE> constexpr size_t smem_bytes() {
    return (size_t)stages<MODE>() * (kABytes + b_bytes<MODE>()) + (size_t)kEpilogueWarps * (out_bytes<MODE>() + 512) + 256;
}

template <class T, int MODE, int ACT>
__global__ void __launch_bounds__(kThreads, 1) gated_mma(const __grid_constant__ MmaParams p) {
    constexpr bool DUAL = MODE == GATED_FWD || MODE == GATED_HEAD || MODE == GATED_PRE;
    constexpr int kStages = stages<MODE>();
    constexpr int kStageBytes = kABytes + b_bytes<MODE>();
    constexpr int kAccCols = MODE == GATED_HEAD ? 128 : 256;   // TMEM columns of an accumulator set
    extern __shared__ __align__(1024) uint8_t base[];   // the swizzle counts from 1024-byte boundaries
    uint8_t* out_stage = base + kStages * kStageBytes;
    float* bias_stage = reinterpret_cast<float*>(out_stage + kEpilogueWarps * out_bytes<MODE>());
    uint64_t* bars = reinterpret_cast<uint64_t*>(bias_stage + kEpilogueWarps * 128);
    uint64_t *full = bars, *empty = bars + kStages, *acc_full = bars + 2 * kStages, *acc_empty = acc_full + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
    volatile int* dead = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const GatedParams& g = p.g;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; s++) { bar_init(full + s, 1); bar_init(empty + s, 1); }
        for (int s = 0; s < 2; s++) { bar_init(acc_full + s, 1); bar_init(acc_empty + s, kEpilogueWarps); }
        *dead = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 2) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)), "r"(2 * kAccCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp == 0 && lane == 0) {
        // ---- producer ----------------------------------------------------------------------------
        int s = 0;
        uint32_t phase = 0;
        int64_t issued = 0;
        const int nb = (p.cols + 63) / 64;
        for (int64_t t = blockIdx.x; t < p.tiles; t += gridDim.x) {
            const Tile q = tile_at<MODE>(p, t);
            for (int k = 0; k < q.kb; k++) {
                if (issued >= kStages && !wait(empty + s, phase ^ 1, dead)) break;
                uint8_t* a = base + s * kStageBytes;
                uint8_t* b = a + kABytes;
                if (DUAL) {
                    bar_expect(full + s, kABytes + (uint32_t)p.cols * kDepth * 2);
                    tma_load(a, &p.a[0], k * kDepth, q.a_y, full + s);
                    tma_load(b, &p.b[0], k * kDepth, q.b_y, full + s);
                    tma_load(b + (p.cols / 2) * kDepth * 2, &p.b[1], k * kDepth, q.up_y, full + s);
                } else if (MODE == GATED_DX) {
                    const int half = q.kb / 2, up = k >= half, j = (up ? k - half : k) * kDepth;
                    bar_expect(full + s, kABytes + (uint32_t)nb * 8192);
                    tma_load(a, &p.a[up], j, q.a_y, full + s);
                    for (int c = 0; c < nb; c++) tma_load(b + c * 8192, &p.b[up], q.n0 + c * 64, j, full + s);
                } else {
                    const int r = q.a_y + k * kDepth;
                    bar_expect(full + s, kABytes + (uint32_t)nb * 8192);
                    tma_load(a, &p.a[q.part & 1], (int)q.m0, r, full + s);
                    tma_load(a + 8192, &p.a[q.part & 1], (int)q.m0 + 64, r, full + s);
                    for (int c = 0; c < nb; c++) tma_load(b + c * 8192, &p.b[0], q.n0 + c * 64, r, full + s);
                }
                issued++;
                if (++s == kStages) { s = 0; phase ^= 1; }
            }
        }
        // after a failed wait: let the copies in flight land before the block goes
        if (*dead)
            for (int i = 0; i < kStages && i < issued; i++) {
                const int64_t n = issued - 1 - i;
                for (int tries = 0; tries < 1000000 && !bar_try(full + n % kStages, (uint32_t)(n / kStages) & 1); tries++) {}
            }
    } else if (warp == 1 && lane == 0) {
        // ---- products ----------------------------------------------------------------------------
        constexpr uint32_t kType = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
        constexpr uint32_t kAMn = MODE == GATED_DW, kBMn = !DUAL;
        // D float; A and B types; majors; N / 8; M / 16
        const uint32_t idesc = 1u << 4 | kType << 7 | kType << 10 | kAMn << 15 | kBMn << 16 | (uint32_t)(p.cols >> 3) << 17 | (uint32_t)(kGatedTileM >> 4) << 24;
        int s = 0, acc = 0;
        uint32_t phase = 0;
        int64_t n = 0;
        for (int64_t t = blockIdx.x; t < p.tiles; t += gridDim.x, n++) {
            const Tile q = tile_at<MODE>(p, t);
            if (n >= 2 && !wait(acc_empty + acc, (uint32_t)((n >> 1) - 1) & 1, dead)) break;
            fence_after();
            const uint32_t d = tmem + acc * kAccCols;
            bool ok = true;
            for (int k = 0; k < q.kb; k++) {
                if (!(ok = wait(full + s, phase, dead))) break;
                fence_after();
                const uint32_t a = smem_addr(base + s * kStageBytes), b = a + kABytes;
#pragma unroll
                for (int i = 0; i < kDepth / 16; i++)
                    mma(d, smem_desc(a + i * (kAMn ? 2048 : 32), kAMn ? 8192 : 16), smem_desc(b + i * (kBMn ? 2048 : 32), kBMn ? 8192 : 16), idesc,
                        k > 0 || i > 0);
                mma_commit(empty + s);
                if (++s == kStages) { s = 0; phase ^= 1; }
            }
            if (!ok) break;
            mma_commit(acc_full + acc);
            acc ^= 1;
        }
    } else if (warp >= 4) {
        // ---- epilogue ----------------------------------------------------------------------------
        const int e = warp - 4, quad = warp & 3, half = e >> 2;   // TMEM lanes 32 quad.., half of the columns
        uint8_t* stage = out_stage + e * out_bytes<MODE>();
        float* bias = bias_stage + e * 128;
        int64_t n = 0;
        for (int64_t t = blockIdx.x; t < p.tiles; t += gridDim.x, n++) {
            const Tile q = tile_at<MODE>(p, t);
            const int acc = (int)(n & 1);
            const int width = DUAL ? p.cols / 2 : p.cols;         // outputs of the tile's row
            // two warps share a quadrant: 32-column pieces, the first half of them to one
            const int pieces = (width + 31) / 32, mine0 = half ? (pieces + 1) / 2 : 0, mine1 = half ? pieces : (pieces + 1) / 2;
            const int64_t row = q.m0 + quad * 32 + lane;
            if (DUAL) {
                const int nj = MODE == GATED_HEAD ? q.h.din : g.n;
                __syncwarp();
                for (int i = lane; i < 64; i += 32) {
                    const int c = q.n0 + mine0 * 32 + i;
                    float bg = 0.0f, bu = 0.0f;
                    if (c < nj) {
                        if (MODE == GATED_HEAD) {
                            const int64_t at = (q.cs % g.stems) * 2 * g.band_cols + 2 * (int64_t)q.h.off + c;
                            if (g.bg) { bg = to_float(static_cast<const T*>(g.bg)[at]); bu = to_float(static_cast<const T*>(g.bg)[at + nj]); }
                        } else {
                            if (g.bg) bg = to_float(static_cast<const T*>(g.bg)[c]);
                            if (g.bu) bu = to_float(static_cast<const T*>(g.bu)[c]);
                        }
                    }
                    bias[i] = bg;
                    bias[64 + i] = bu;
                }
                __syncwarp();
            }
            if (!wait(acc_full + acc, (uint32_t)(n >> 1) & 1, dead)) break;
            fence_after();
            const uint32_t lanes = tmem + acc * kAccCols + ((uint32_t)(quad * 32) << 16);
            for (int c = mine0; c < mine1; c++) {
                uint32_t v[32], w[32];
                tmem_load32(v, lanes + c * 32);
                if (DUAL) tmem_load32(w, lanes + width + c * 32);
                tmem_wait();
                if (c + 1 == mine1) {   // the accumulators are in registers: the next products may have them
                    fence_before();
                    __syncwarp();
                    if (lane == 0) bar_arrive(acc_empty + acc);
                }
                const int j0 = q.n0 + c * 32, lc = (c - mine0) * 32;
                if (MODE == GATED_DW) {
                    // 32 floats of the row: whole 128-byte lines where the rows are aligned
                    if (row < g.n) {
                        float* o = g.dw_part + ((int64_t)q.part * g.n + row) * g.k + j0;
                        if ((g.k & 3) == 0 && j0 + 32 <= g.k) {
#pragma unroll
                            for (int i = 0; i < 32; i += 4) *reinterpret_cast<uint4*>(o + i) = make_uint4(v[i], v[i + 1], v[i + 2], v[i + 3]);
                        } else {
#pragma unroll
                            for (int i = 0; i < 32; i++)
                                if (j0 + i < g.k) o[i] = __uint_as_float(v[i]);
                        }
                    }
                    continue;
                }
                if (MODE == GATED_HEAD) {
                    float* sm = reinterpret_cast<float*>(stage);
#pragma unroll
                    for (int i = 0; i < 32; i += 4) {
                        const float4 bv = *reinterpret_cast<const float4*>(bias + lc + i), bw = *reinterpret_cast<const float4*>(bias + 64 + lc + i);
                        const float bva[4] = {bv.x, bv.y, bv.z, bv.w}, bwa[4] = {bw.x, bw.y, bw.z, bw.w};
#pragma unroll
                        for (int k = 0; k < 4; k++)
                            sm[lane * 33 + i + k] = (__uint_as_float(v[i + k]) + bva[k]) * sigmoidf(__uint_as_float(w[i + k]) + bwa[k]);
                    }
                    __syncwarp();
                    const int64_t r0 = q.m0 + quad * 32;
                    const int rows = (int)min((int64_t)32, g.frames - r0);
                    float* o = g.masks + (q.cs * g.band_cols + q.h.off) * g.frames + r0 * q.h.din + j0 + lane;
                    if (j0 + lane < q.h.din)
                        for (int r = 0; r < rows; r++) o[(int64_t)r * q.h.din] = sm[r * 33 + lane];
                    __syncwarp();
                    continue;
                }
                uint32_t o[16], o2[16];
                if (MODE == GATED_FWD) {
#pragma unroll
                    for (int i = 0; i < 32; i += 4) {
                        const float4 bv = *reinterpret_cast<const float4*>(bias + lc + i), bw = *reinterpret_cast<const float4*>(bias + 64 + lc + i);
                        const float y0 = act<ACT>(__uint_as_float(v[i]) + bv.x) * (__uint_as_float(w[i]) + bw.x);
                        const float y1 = act<ACT>(__uint_as_float(v[i + 1]) + bv.y) * (__uint_as_float(w[i + 1]) + bw.y);
                        const float y2 = act<ACT>(__uint_as_float(v[i + 2]) + bv.z) * (__uint_as_float(w[i + 2]) + bw.z);
                        const float y3 = act<ACT>(__uint_as_float(v[i + 3]) + bv.w) * (__uint_as_float(w[i + 3]) + bw.w);
                        o[i / 2] = pack2<T>(y0, y1);
                        o[i / 2 + 1] = pack2<T>(y2, y3);
                    }
                } else if (MODE == GATED_PRE) {
                    // dg and du in place of g and u, then their sums over the warp's rows
                    const T* dy = static_cast<const T*>(g.dy) + row * g.y_row + j0;
                    const bool row_ok = row < g.m;
                    const bool vec = row_ok && j0 + 32 <= g.n && (reinterpret_cast<uintptr_t>(dy) & 15) == 0;
#pragma unroll
                    for (int i = 0; i < 32; i += 8) {
                        float d[8];
                        if (vec) {
                            const Pack<T, 8> x = *reinterpret_cast<const Pack<T, 8>*>(dy + i);
#pragma unroll
                            for (int k = 0; k < 8; k++) d[k] = to_float(x.v[k]);
                        } else {
#pragma unroll
                            for (int k = 0; k < 8; k++) d[k] = row_ok && j0 + i + k < g.n ? to_float(dy[i + k]) : 0.0f;
                        }
#pragma unroll
                        for (int k = 0; k < 8; k++) {
                            const float gg = __uint_as_float(v[i + k]) + bias[lc + i + k], uu = __uint_as_float(w[i + k]) + bias[64 + lc + i + k];
                            float a, s;
                            act_both<ACT>(gg, a, s);
                            // a row or column past the end has d = 0, but its g and u are not defined
                            const bool in = row_ok && j0 + i + k < g.n;
                            v[i + k] = __float_as_uint(in ? d[k] * uu * s : 0.0f);
                            w[i + k] = __float_as_uint(in ? d[k] * a : 0.0f);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        o[i] = pack2<T>(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]));
                        o2[i] = pack2<T>(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
                    }
                    if (g.col_sums) {
                        // Sums of 32 columns over 32 lanes in 31 steps each: a lane and its partner split
                        // the columns between them and add, until a lane holds one column: its own number's.
#pragma unroll
                        for (int h = 16; h > 0; h >>= 1) {
                            const bool hi = lane & h;
#pragma unroll
                            for (int i = 0; i < 16; i++) {
                                if (i >= h) break;
                                const float kv = __uint_as_float(hi ? v[i + h] : v[i]), sv = __uint_as_float(hi ? v[i] : v[i + h]);
                                const float kw = __uint_as_float(hi ? w[i + h] : w[i]), sw = __uint_as_float(hi ? w[i] : w[i + h]);
                                v[i] = __float_as_uint(kv + __shfl_xor_sync(~0u, sv, h));
                                w[i] = __float_as_uint(kw + __shfl_xor_sync(~0u, sw, h));
                            }
                        }
                        if (j0 + lane < g.n) {
                            float* sums = g.col_sums + ((q.m0 / 32 + quad) * 2) * g.n + j0 + lane;
                            sums[0] = __uint_as_float(v[0]);
                            sums[g.n] = __uint_as_float(w[0]);
                        }
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 16; i++) o[i] = pack2<T>(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]));
                }
                T* out = static_cast<T*>(MODE == GATED_FWD ? g.y : MODE == GATED_PRE ? g.dg : g.dx);
                const int64_t pitch = MODE == GATED_FWD ? g.y_row : MODE == GATED_PRE ? g.pre_row : g.dx_row;
                const int nj = MODE == GATED_DX ? g.k : g.n;
                if (p.store_by_tma) {
                    // 32 rows of 64 bytes as the 64-byte swizzle has them: 16-byte piece c of row r at c ^ (r / 2 & 3)
                    if (lane == 0) stores_read();
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int to = lane * 64 + ((i ^ ((lane >> 1) & 3)) << 4);
                        *reinterpret_cast<uint4*>(stage + to) = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                        if (MODE == GATED_PRE)
                            *reinterpret_cast<uint4*>(stage + 2048 + to) = make_uint4(o2[4 * i], o2[4 * i + 1], o2[4 * i + 2], o2[4 * i + 3]);
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    const int64_t y = q.m0 + quad * 32;
                    if (lane == 0 && j0 < nj && y < g.m) {
                        tma_store(&p.c[0], j0, (int)y, stage);
                        if (MODE == GATED_PRE) tma_store(&p.c[1], j0, (int)y, stage + 2048);
                        store_commit();
                    }
                } else if (row < g.m) {
#pragma unroll
                    for (int i = 0; i < 32; i++) {
                        if (j0 + i >= nj) break;
                        const T* s = reinterpret_cast<const T*>(&o[i / 2]);
                        out[row * pitch + j0 + i] = s[i & 1];
                        if (MODE == GATED_PRE) static_cast<T*>(g.du)[row * pitch + j0 + i] = reinterpret_cast<const T*>(&o2[i / 2])[i & 1];
                    }
                }
            }
            if (mine0 == mine1 && lane == 0) bar_arrive(acc_empty + acc);   // no piece of this tile
        }
        if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    if (warp == 2) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2 * kAccCols));
}

// ---- host -------------------------------------------------------------------------------------

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                              const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn encoder() {
    static const EncodeFn fn = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult r;
        cuda_check(cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &r), "cuTensorMapEncodeTiled");
        if (r != cudaDriverEntryPointSuccess || !f) fail(STG_INTERNAL_ERROR, "cuTensorMapEncodeTiled is not available");
        return reinterpret_cast<EncodeFn>(f);
    }();
    return fn;
}

// A 16-bit matrix [rows][cols], rows `pitch` elements apart, in boxes of box_cols x box_rows;
// elements past its sides read as zeros and are not written.
void encode(CUtensorMap* m, bool bf16, const void* p, int64_t rows, int64_t cols, int64_t pitch, int box_cols, int box_rows, bool store = false) {
    if (rows == 1) pitch = (cols + 7) / 8 * 8;   // of no consequence, but it must be a multiple of 16 bytes
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)pitch * 2};
    const cuuint32_t box[2] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows}, one[2] = {1, 1};
    const CUresult r = encoder()(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void*>(p), dims, strides,
                                 box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, store ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
                                 CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) fail(STG_INTERNAL_ERROR, "cuTensorMapEncodeTiled failed with " + std::to_string((int)r));
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

template <class T, int MODE, int ACT> void launch(const MmaParams& p, int sms, cudaStream_t st) {
    const auto kernel = gated_mma<T, MODE, ACT>;
    cuda_check(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem_bytes<MODE>()), "gated kernel");
    kernel<<<(unsigned)std::min<int64_t>(p.tiles, sms), kThreads, smem_bytes<MODE>(), st>>>(p);
    cuda_check(cudaGetLastError(), "gated kernel");
}

template <class T, int MODE> void launch_act(const MmaParams& p, int sms, cudaStream_t st) {
    switch (p.g.act) {
        case STG_ACT_RELU: return launch<T, MODE, STG_ACT_RELU>(p, sms, st);
        case STG_ACT_SILU: return launch<T, MODE, STG_ACT_SILU>(p, sms, st);
        case STG_ACT_GELU: return launch<T, MODE, STG_ACT_GELU>(p, sms, st);
        case STG_ACT_SIGMOID: return launch<T, MODE, STG_ACT_SIGMOID>(p, sms, st);
        default: return launch<T, MODE, STG_ACT_NONE>(p, sms, st);
    }
}

} // namespace

void launch_gated_mma(GatedMode mode, bool bf16, const GatedParams& g, int64_t head_rows, int sms, cudaStream_t st) {
    MmaParams p{};
    p.g = g;
    const int64_t mt = ceil_div(mode == GATED_HEAD ? g.frames : g.m, kGatedTileM);
    if (mode == GATED_HEAD) {
        p.cols = 2 * kGatedTileN;
        p.tiles = head_rows / g.frames / g.bands * mt * g.n_tiles;
        encode(&p.a[0], bf16, g.x, head_rows, g.k, g.x_row, kDepth, kGatedTileM);
        encode(&p.b[0], bf16, g.wg, g.stems * 2 * g.band_cols, g.k, g.wg_row, kDepth, kGatedTileN);
        p.b[1] = p.b[0];
    } else if (mode == GATED_FWD || mode == GATED_PRE) {
        // 128 outputs to a tile; 64 when that would leave SMs without a tile
        const int n = mt * ceil_div(g.n, 128) < sms ? 64 : 128;
        p.cols = 2 * n;
        p.tiles_n = (int)ceil_div(g.n, n);
        p.tiles = mt * p.tiles_n;
        encode(&p.a[0], bf16, g.x, g.m, g.k, g.x_row, kDepth, kGatedTileM);
        encode(&p.b[0], bf16, g.wg, g.n, g.k, g.wg_row, kDepth, n);
        encode(&p.b[1], bf16, g.wu, g.n, g.k, g.wu_row, kDepth, n);
        if (mode == GATED_FWD) {
            p.store_by_tma = aligned(g.y, 16) && (g.y_row % 8 == 0 || g.m == 1);
            if (p.store_by_tma) encode(&p.c[0], bf16, g.y, g.m, g.n, g.y_row, 32, 32, true);
        } else {
            p.store_by_tma = 1;
            encode(&p.c[0], bf16, g.dg, g.m, g.n, g.pre_row, 32, 32, true);
            encode(&p.c[1], bf16, g.du, g.m, g.n, g.pre_row, 32, 32, true);
        }
    } else {
        // the fewest column tiles of at most 256, of one width: whole 32-column pieces, as the epilogue
        // stores them, so that no piece reaches into the next tile
        p.tiles_n = (int)ceil_div(g.k, 256);
        p.cols = (int)ceil_div(ceil_div(g.k, p.tiles_n), 32) * 32;
        p.tiles_n = (int)ceil_div(g.k, p.cols);
        if (mode == GATED_DX) {
            p.tiles = mt * p.tiles_n;
            encode(&p.a[0], bf16, g.dg, g.m, g.n, g.pre_row, kDepth, kGatedTileM);
            encode(&p.a[1], bf16, g.du, g.m, g.n, g.pre_row, kDepth, kGatedTileM);
            encode(&p.b[0], bf16, g.wg, g.n, g.k, g.wg_row, 64, kDepth);
            encode(&p.b[1], bf16, g.wu, g.n, g.k, g.wu_row, 64, kDepth);
            p.store_by_tma = aligned(g.dx, 16) && (g.dx_row % 8 == 0 || g.m == 1);
            if (p.store_by_tma) encode(&p.c[0], bf16, g.dx, g.m, g.k, g.dx_row, 32, 32, true);
        } else {
            p.tiles = 2 * g.splits * ceil_div(g.n, kGatedTileM) * p.tiles_n;
            encode(&p.a[0], bf16, g.dg, g.m, g.n, g.pre_row, 64, kDepth);
            encode(&p.a[1], bf16, g.du, g.m, g.n, g.pre_row, 64, kDepth);
            encode(&p.b[0], bf16, g.x, g.m, g.k, g.x_row, 64, kDepth);
        }
    }
    auto go = [&](auto* tag) {
        using T = std::remove_pointer_t<decltype(tag)>;
        if (mode == GATED_HEAD) launch<T, GATED_HEAD, STG_ACT_SIGMOID>(p, sms, st);
        else if (mode == GATED_FWD) launch_act<T, GATED_FWD>(p, sms, st);
        else if (mode == GATED_PRE) launch_act<T, GATED_PRE>(p, sms, st);
        else if (mode == GATED_DX) launch<T, GATED_DX, STG_ACT_NONE>(p, sms, st);
        else launch<T, GATED_DW, STG_ACT_NONE>(p, sms, st);
    };
    if (bf16) go((__nv_bfloat16*)nullptr);
    else go((__half*)nullptr);
}

int gated_gave_up() {
    unsigned int v = 0;
    cuda_check(cudaMemcpyFromSymbol(&v, g_gave_up, sizeof(v)), "gated status");
    return (int)v;
}

} // namespace stg
