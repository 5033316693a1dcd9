// gated_mma.cu -- the gated projection's products on the tensor cores, f16 and bf16
// (gated.h: GatedMode; the mathematics is in gated.cu).
//
// Two neighbouring SMs work as a pair (a cluster of two blocks, tcgen05 cta_group::2) and walk
// 256-row output tiles: each block holds its own 128 rows of A and half the columns of B, so
// a slice of the contraction costs an SM 32 KB of loads for the work of a 128 x 256 tile where a
// block alone would load 48 KB (alone, the products waited for the loads and reached half the
// tensor cores' rate). A producer thread brings 64-deep slices into a ring of shared-memory
// stages by TMA (128-byte swizzle); one thread of the pair issues the products, float
// accumulators in TMEM; sixteen warps per block read finished accumulators back, apply the
// epilogue and store. In the forward modes one block of the pair loads Wg's rows and the other
// Wu's rows of the same outputs, so one instruction computes both projections and an epilogue
// thread finds g and u of an output in its own TMEM lane: the projections never leave the SM.
//
// Where an operand's contraction is not its contiguous axis (W in dx = dg Wg + du Wu; all of
// dW = dg^T x), the tile goes to shared memory as it lies and the instruction reads it
// MN-major, so nothing is transposed in memory.
//
// Measured (bf16, kernel time): gated 48060 x K x 1408 at K 1536 254 us, 1.64 PFLOP/s (97 % of the
// measured cuBLAS rate), at 768 132 us, at 384 86 us, 1.21 PFLOP/s: there a tile is six slices and the
// epilogue of 128 x 128 outputs per block is what bounds it (60 us with the products left out; the tensor cores
// are active in 64 % of the cycles). The backward products at 24030 x 384 x 1408: dg and du 65 us (the
// epilogue reads dy too; tensor cores active in 41 %), dx 56 and dW 56 us (52 and 56 %): the SMs take in 50 and
// 46 bytes a cycle of operands, dx 24 KB per slice and block for its 128-column tiles (282 in four rounds of
// 74 pairs), dW 32 KB for its 192-column ones (72 in one round), of which a block loads boxes of 128 columns for
// its 96. The mask head of 60 mel bands x 801 frames at hidden 1536 67 us (220 MB at least; 45 %): one
// accumulator set, so a tile's epilogue runs alone, in 5.3 rounds of tiles.
#include "gated.h"

#include <cuda.h>

namespace stg {

namespace {

constexpr int kEpilogueWarps = 16;
constexpr int kThreads = 128 + 32 * kEpilogueWarps;   // warp 0 TMA, warp 1 products, warp 2 TMEM, warps 4.. epilogue
constexpr int kDepth = 64;         // contraction per stage: 128 bytes, one swizzle row
constexpr int kPairM = 256;        // rows of a pair's tile
constexpr int kABytes = 128 * kDepth * 2, kBBytes = 128 * kDepth * 2;   // of one block
constexpr int kStageBytes = kABytes + kBBytes;
constexpr int kAccCols = 256;      // TMEM columns of an accumulator set
constexpr int kSumCol = 240;       // dW: the column of the set that sums dg over the rows

// Kernels that gave up a wait (never, unless a copy or a product failed): see wait().
__device__ unsigned int g_gave_up;

struct MmaParams {
    GatedParams g;
    CUtensorMap a[2], b[2], c[2];
    int tiles;
    FastDiv tiles_n;               // column tiles of a row of tiles (mask head: row tiles of a band)
    FastDiv rest_n;                // row tiles of a part in dW, column tiles of a stem in the mask head
    int cols;                      // columns of a tile (the instruction's N; outputs x 2 in the forward modes)
    int sums;                      // dW: also sum dg and du over the rows
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
// The address of a barrier (or anything at the same place) in the pair's first block.
__device__ __forceinline__ uint32_t in_leader(const void* p) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(smem_addr(p)));
    return r;
}
__device__ __forceinline__ void bar_arrive_cluster(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
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
// Called by whole warps; all lanes get the same answer.
__device__ __forceinline__ bool wait(uint64_t* b, uint32_t parity, volatile int* dead) {
    bool ok = bar_try(b, parity);
    if (!ok) ok = wait_slow(b, parity, dead);
    return __all_sync(~0u, ok);
}
// Into this block's shared memory; the bytes count at a barrier of the pair's first block.
__device__ __forceinline__ void tma_load(void* dst, const CUtensorMap* m, int x, int y, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], [%4];" ::"r"(
                     smem_addr(dst)), "l"(m), "r"(x), "r"(y), "r"(bar) : "memory");
}
__device__ __forceinline__ void tma_store(const CUtensorMap* m, int x, int y, const void* src) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(m), "r"(x), "r"(y), "r"(
                     smem_addr(src)) : "memory");
}
__device__ __forceinline__ void store_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
__device__ __forceinline__ void stores_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d), "l"(a),
                 "l"(b), "r"(idesc), "r"((uint32_t)add) : "memory");
}
// The barrier at this place in both blocks: its phase completes when the products issued so far have.
__device__ __forceinline__ void mma_commit(uint64_t* b) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_addr(b)),
                 "h"((uint16_t)3) : "memory");
}
__device__ __forceinline__ void tmem_load16(uint32_t (&v)[16], uint32_t addr) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
          "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(addr));
}
__device__ __forceinline__ void tmem_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.aligned;\nbarrier.cluster.wait.aligned;" ::: "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }

// One lane of a converged warp, the same one each time.
__device__ __forceinline__ bool elect() {
    uint32_t r;
    asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(r));
    return r != 0;
}

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

// a += x, b += y in one packed instruction.
__device__ __forceinline__ void add2(uint32_t& a, uint32_t& b, float x, float y) {
    asm("{\n.reg .b64 u, v;\nmov.b64 u, {%0, %1};\nmov.b64 v, {%2, %3};\nadd.rn.f32x2 u, u, v;\nmov.b64 {%0, %1}, u;\n}"
        : "+r"(a), "+r"(b) : "f"(x), "f"(y));
}

// Where a pair's tile lies.
struct Tile {
    int64_t m0;      // first output row
    int n0;          // first output column
    int cols;        // the instruction's N
    int a_y;         // A: first row (of the contraction, in dW)
    int b_y, up_y;   // forward modes: first rows of the two weights
    int kb;          // slices of the contraction
    int part;        // dW: 2 split + (0 gate, 1 up)
    int tile_n;      // dW: number of the column tile
    HeadTile h;
    int64_t cs;      // mask head: chunk * stems + stem
};

template <int MODE> __device__ __forceinline__ Tile tile_at(const MmaParams& p, uint32_t t) {
    Tile r{};
    const GatedParams& g = p.g;
    r.cols = p.cols;
    if (MODE == GATED_HEAD) {
        // frames first: a band's rows and its weights are then read by neighbours in time
        const uint32_t rest = p.tiles_n.div(t), cs = p.rest_n.div(rest);
        r.m0 = (int64_t)(t - rest * p.tiles_n.d) * kPairM;
        r.cs = cs;
        r.h = g.tiles[rest - cs * p.rest_n.d];
        r.n0 = r.h.n0;
        r.cols = 2 * ((min(kHeadWideN, r.h.din - r.n0) + 31) / 32 * 32);
        r.a_y = (int)((r.cs * g.bands + r.h.band) * g.frames + r.m0);
        r.b_y = (int)(((uint32_t)r.cs % (uint32_t)g.stems) * 2 * g.band_cols + 2 * (int64_t)r.h.off + r.n0);
        r.up_y = r.b_y + r.h.din;
        r.kb = (g.k + kDepth - 1) / kDepth;
    } else if (MODE == GATED_FWD || MODE == GATED_PRE) {
        const uint32_t mt = p.tiles_n.div(t);
        r.m0 = (int64_t)mt * kPairM;
        r.n0 = (int)(t - mt * p.tiles_n.d) * (p.cols / 2);
        r.a_y = (int)r.m0;
        r.b_y = r.up_y = r.n0;
        r.kb = (g.k + kDepth - 1) / kDepth;
    } else if (MODE == GATED_DX) {
        const uint32_t mt = p.tiles_n.div(t);
        r.m0 = (int64_t)mt * kPairM;
        r.n0 = (int)(t - mt * p.tiles_n.d) * p.cols;
        r.a_y = (int)r.m0;
        r.kb = 2 * ((g.n + kDepth - 1) / kDepth);
    } else {
        const uint32_t q = p.tiles_n.div(t), part = p.rest_n.div(q);
        r.tile_n = (int)(t - q * p.tiles_n.d);
        r.n0 = r.tile_n * p.cols;
        r.part = (int)part;
        r.m0 = (int64_t)(q - part * p.rest_n.d) * kPairM;
        const int64_t beg = (r.part >> 1) * g.split_rows;
        r.a_y = (int)beg;
        r.kb = (int)((min(g.m, beg + g.split_rows) - beg + kDepth - 1) / kDepth);
    }
    return r;
}

// Per epilogue warp: 32 rows x 32 columns of output, for dg and du each (in the mask head 16 columns of
// float, rows 17 apart), and 64 floats of each bias.
template <int MODE> __host__ __device__ constexpr int out_bytes() {
    return MODE == GATED_PRE ? 4096 : MODE == GATED_HEAD ? 32 * 17 * 4 : MODE == GATED_DW ? 0 : 2048;
}
template <int MODE> __host__ __device__ constexpr int stages() { return MODE == GATED_PRE ? 4 : 5; }
// dW: a tile of ones, 16 columns
template <int MODE> __host__ __device__ constexpr int ones_bytes() { return MODE == GATED_DW ? 64 * kDepth * 2 : 0; }
template <int MODE> constexpr size_t smem_bytes() {
    return (size_t)stages<MODE>() * kStageBytes + ones_bytes<MODE>() + (size_t)kEpilogueWarps * (out_bytes<MODE>() + 512) + 256;
}

template <class T, int MODE, int ACT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1) gated_mma(const __grid_constant__ MmaParams p) {
    constexpr bool DUAL = MODE == GATED_FWD || MODE == GATED_HEAD || MODE == GATED_PRE;
    constexpr int kStages = stages<MODE>();
    // Two accumulator sets let the epilogue of a tile run under the products of the next. The mask
    // head's float results see the accumulators' roundings (the tensor cores cut, so they add up
    // along a sum: 1.5e-6 of the result at hidden 1536): its two sets are instead two partial
    // sums of one tile, of alternate slices (0.7e-6).
    constexpr int kSets = MODE == GATED_HEAD ? 1 : 2;
    extern __shared__ __align__(1024) uint8_t base[];   // the swizzle counts from 1024-byte boundaries
    uint8_t* ones = base + kStages * kStageBytes;
    uint8_t* out_stage = ones + ones_bytes<MODE>();
    float* bias_stage = reinterpret_cast<float*>(out_stage + kEpilogueWarps * out_bytes<MODE>());
    uint64_t* bars = reinterpret_cast<uint64_t*>(bias_stage + kEpilogueWarps * 128);
    // full and acc_empty are used in the pair's first block, empty and acc_full in both
    uint64_t *full = bars, *empty = bars + kStages, *acc_full = bars + 2 * kStages, *acc_empty = acc_full + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
    volatile int* dead = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const int warp = __shfl_sync(~0u, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;   // the warp's number, known to be uniform
    const int rank = blockIdx.x & 1;
    const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    const GatedParams& g = p.g;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; s++) { bar_init(full + s, 1); bar_init(empty + s, 1); }
        for (int s = 0; s < 2; s++) { bar_init(acc_full + s, 1); bar_init(acc_empty + s, MODE == GATED_FWD || MODE == GATED_PRE ? kEpilogueWarps : 2 * kEpilogueWarps); }
        *dead = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (MODE == GATED_DW)   // the same value everywhere: no layout to mind
        for (int i = threadIdx.x; i < ones_bytes<MODE>() / 4; i += kThreads) reinterpret_cast<uint32_t*>(ones)[i] = pack2<T>(1.0f, 1.0f);
    if (warp == 2) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)), "r"(2 * kAccCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    fence_before();
    __syncthreads();
    cluster_sync();
    fence_after();
    const uint32_t tmem = *tmem_slot;

    // The producer and the product warp run converged with one lane issuing: their addresses and
    // descriptors then stay in uniform registers. (With one diverged lane the per-slice arithmetic
    // took about 550 cycles and the tensor cores waited for it.)
    if (warp == 0) {
        // ---- producer: this block's rows of A, and its half of B ------------------------------------
        const bool one = elect();
        int s = 0;
        uint32_t phase = 0;
        int issued = 0;      // saturates at kStages
        for (int t = pair; t < p.tiles; t += pairs) {
            const Tile q = tile_at<MODE>(p, t);
            const int nb = DUAL ? 1 : (q.cols / 2 + 63) / 64;
            const uint32_t bytes = kABytes + (DUAL ? (uint32_t)q.cols / 2 * kDepth * 2 : (uint32_t)nb * 8192);
            for (int k = 0; k < q.kb; k++) {
                if (issued >= kStages && !wait(empty + s, phase ^ 1, dead)) break;
                uint8_t* a = base + s * kStageBytes;
                uint8_t* b = a + kABytes;
                const uint32_t bar = in_leader(full + s);
                if (one && rank == 0) bar_expect(full + s, 2 * bytes);
                if (!one) {
                } else if (DUAL) {
                    tma_load(a, &p.a[0], k * kDepth, q.a_y + rank * 128, bar);
                    const int y = rank ? q.up_y : q.b_y;
                    if (MODE == GATED_HEAD)
                        for (int c = 0; c < q.cols / 2; c += 32) tma_load(b + c * kDepth * 2, &p.b[0], k * kDepth, y + c, bar);
                    else tma_load(b, &p.b[rank], k * kDepth, y, bar);
                } else if (MODE == GATED_DX) {
                    const int half = q.kb / 2, up = k >= half, j = (up ? k - half : k) * kDepth;
                    tma_load(a, &p.a[up], j, q.a_y + rank * 128, bar);
                    for (int c = 0; c < nb; c++) tma_load(b + c * 8192, &p.b[up], q.n0 + rank * (q.cols / 2) + c * 64, j, bar);
                } else {
                    const int r = q.a_y + k * kDepth;
                    tma_load(a, &p.a[q.part & 1], (int)q.m0 + rank * 128, r, bar);
                    tma_load(a + 8192, &p.a[q.part & 1], (int)q.m0 + rank * 128 + 64, r, bar);
                    for (int c = 0; c < nb; c++) tma_load(b + c * 8192, &p.b[0], q.n0 + rank * (q.cols / 2) + c * 64, r, bar);
                }
                issued = min(issued + 1, kStages);
                if (++s == kStages) { s = 0; phase ^= 1; }
            }
        }
        // after a failed wait: time for the copies in flight to land before the block goes
        if (*dead) {
            const uint64_t t0 = now_ns();
            while (now_ns() - t0 < 10000000) {}
        }
    } else if (warp == 1 && rank == 0) {
        // ---- products, for both blocks ---------------------------------------------------------------
        constexpr uint32_t kType = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
        constexpr uint32_t kAMn = MODE == GATED_DW, kBMn = !DUAL;
        // D float; A and B types; majors; M / 16. N / 8 is added per tile
        constexpr uint32_t idesc0 = 1u << 4 | kType << 7 | kType << 10 | kAMn << 15 | kBMn << 16 | (uint32_t)(kPairM >> 4) << 24;
        // descriptors of the first stage; a stage or a step of 16 further on adds to the address field
        const uint64_t a0 = smem_desc(smem_addr(base), kAMn ? 8192 : 16), b0 = smem_desc(smem_addr(base) + kABytes, kBMn ? 8192 : 16);
        const uint64_t ones0 = MODE == GATED_DW ? smem_desc(smem_addr(ones), 8192) : 0;
        constexpr uint32_t a_step = (kAMn ? 2048 : 32) >> 4, b_step = (kBMn ? 2048 : 32) >> 4;
        const bool one = elect();
        int s = 0;
        uint32_t phase = 0;
        int n = 0;
        for (int t = pair; t < p.tiles; t += pairs, n++) {
            const Tile q = tile_at<MODE>(p, t);
            const int set = n % kSets;
            if (n >= kSets && !wait(acc_empty + set, (uint32_t)(n / kSets - 1) & 1, dead)) break;
            fence_after();
            const uint32_t d0 = tmem + set * kAccCols, idesc = idesc0 | (uint32_t)(q.cols >> 3) << 17;
            bool ok = true;
            for (int k = 0; k < q.kb; k++) {
                if (!(ok = wait(full + s, phase, dead))) break;
                fence_after();
                const uint64_t a = a0 + (uint32_t)(s * (kStageBytes >> 4)), b = b0 + (uint32_t)(s * (kStageBytes >> 4));
                const uint32_t d = MODE == GATED_HEAD ? d0 + (k & 1) * kAccCols : d0;
                const bool add = k > (MODE == GATED_HEAD ? 1 : 0);
                // The sums dg^T 1 of a slice, shared between the column tiles, which read the same dg. (Adding
                // across lanes in GATED_PRE's epilogue, or there by mma.sync, took 12 and 16 us more at 24030 x
                // 1408; here it is 8.)
                const bool sum = MODE == GATED_DW && p.sums && (uint32_t)k % p.tiles_n.d == (uint32_t)q.tile_n;
                if (one) {
#pragma unroll
                    for (int i = 0; i < kDepth / 16; i++) {
                        mma(d, a + i * a_step, b + i * b_step, idesc, add || i > 0);
                        if (MODE == GATED_DW && sum)
                            mma(d + kSumCol, a + i * a_step, ones0 + i * b_step, idesc0 | 2u << 17, k >= (int)p.tiles_n.d || i > 0);
                    }
                    mma_commit(empty + s);
                }
                if (++s == kStages) { s = 0; phase ^= 1; }
            }
            if (!ok) break;
            if (one) mma_commit(acc_full + set);
        }
    } else if (warp >= 4) {
        // ---- epilogue --------------------------------------------------------------------------------
        // A warp reads TMEM lanes 32 quad.. and every kStep-th 32-column piece. In gated and its
        // first backward product, whose tiles are short, eight warps take the even tiles and
        // eight the odd ones, so that the waits of one half run under the work of the other (gated
        // 48060 x 384 x 1408: 86 us; with plain stores in place of TMA's 88; all sixteen on each
        // tile, 32 columns in registers at a time, 102, and 117 with TMA's).
        constexpr int kHalves = MODE == GATED_FWD || MODE == GATED_PRE ? 2 : 1, kStep = 4 / kHalves;
        const int e = warp - 4, quad = warp & 3, group = (e >> 2) % kStep;
        const bool store = MODE != GATED_DW && MODE != GATED_HEAD && p.store_by_tma;
        // dy of the next 16 columns of this warp, on its way while the present ones are used; 0 past the sides
        Pack<T, 8> dy[2], ahead[2];
        auto ahead_of = [&](int64_t r, int j, Pack<T, 8> (&to)[2]) {
            const T* from = static_cast<const T*>(g.dy) + r * g.y_row + j;
            if (r < g.m && j + 16 <= g.n && (reinterpret_cast<uintptr_t>(from) & 15) == 0) {
                to[0] = *reinterpret_cast<const Pack<T, 8>*>(from);
                to[1] = *reinterpret_cast<const Pack<T, 8>*>(from + 8);
            } else {
#pragma unroll
                for (int i = 0; i < 16; i++) to[i / 8].v[i % 8] = r < g.m && j + i < g.n ? from[i] : from_float<T>(0.0f);
            }
        };
        if (MODE == GATED_PRE) {
            const int first = pair + (e >> 3) * pairs;   // this warp's first tile
            if (first < p.tiles) {
                const Tile q = tile_at<MODE>(p, first);
                ahead_of(q.m0 + rank * 128 + quad * 32 + lane, q.n0 + group * 32, ahead);
            }
        }
        uint8_t* stage = out_stage + e * out_bytes<MODE>();
        float* bias = bias_stage + e * 128;
        int n = 0;
        for (int t = pair; t < p.tiles; t += pairs, n++) {
            if (kHalves == 2 && (n & 1) != (e >> 3)) continue;
            const Tile q = tile_at<MODE>(p, t);
            const int set = n % kSets;
            const int width = DUAL ? q.cols / 2 : q.cols;         // outputs of the tile's row
            const int pieces = (width + 31) / 32;
            const int64_t row0 = q.m0 + rank * 128 + quad * 32, row = row0 + lane;
            if (DUAL) {   // at most four pieces to a tile, so kHalves to a warp
                const int nj = MODE == GATED_HEAD ? q.h.din : g.n;
                float bg[kHalves], bu[kHalves];
#pragma unroll
                for (int i = 0; i < kHalves; i++) {
                    const int c = q.n0 + (group + i * kStep) * 32 + lane;
                    bg[i] = bu[i] = 0.0f;
                    if (c >= nj) continue;
                    if (MODE == GATED_HEAD) {
                        const int64_t at = ((uint32_t)q.cs % (uint32_t)g.stems) * 2 * g.band_cols + 2 * (int64_t)q.h.off + c;
                        if (g.bg) { bg[i] = to_float(static_cast<const T*>(g.bg)[at]); bu[i] = to_float(static_cast<const T*>(g.bg)[at + nj]); }
                    } else {
                        if (g.bg) bg[i] = to_float(static_cast<const T*>(g.bg)[c]);
                        if (g.bu) bu[i] = to_float(static_cast<const T*>(g.bu)[c]);
                    }
                }
                __syncwarp();
#pragma unroll
                for (int i = 0; i < kHalves; i++) {
                    bias[64 * i + lane] = bg[i];
                    bias[64 * i + 32 + lane] = bu[i];
                }
                __syncwarp();
            }
            if (!wait(acc_full + set, (uint32_t)(n / kSets) & 1, dead)) break;
            fence_after();
            const uint32_t lanes = tmem + set * kAccCols + ((uint32_t)(quad * 32) << 16);
            if (MODE == GATED_DW && p.sums && group == 3) {
                uint32_t sum;
                asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(sum) : "r"(lanes + kSumCol));
                tmem_wait();
                // a column tile past the slices has summed none
                if (row < g.n)
                    g.col_sums[((int64_t)((q.part >> 1) * (int)p.tiles_n.d + q.tile_n) * 2 + (q.part & 1)) * g.n + row] = q.tile_n < q.kb ? __uint_as_float(sum) : 0.0f;
            }
            // 16 columns of a piece, bias added, through the epilogue to the stage or to memory
            auto half = [&](uint32_t (&v)[16], uint32_t (&w)[16], int c, int hh) {
                const int lc = hh * 16, j = q.n0 + c * 32 + lc;
                if (MODE == GATED_DW) {
                    if (g.splits == 1) {
                        T* o = static_cast<T*>(g.dw[q.part]);
                        if (row >= g.n || !o) return;
                        o += row * g.dw_row[q.part] + j;
                        Pack<T, 8> out[2];
#pragma unroll
                        for (int i = 0; i < 16; i++) out[i / 8].v[i % 8] = from_float<T>(__uint_as_float(v[i]));
                        if (g.dw_row[q.part] % 8 == 0 && j + 16 <= g.k && (reinterpret_cast<uintptr_t>(g.dw[q.part]) & 15) == 0) {
                            reinterpret_cast<Pack<T, 8>*>(o)[0] = out[0];
                            reinterpret_cast<Pack<T, 8>*>(o)[1] = out[1];
                        } else {
#pragma unroll
                            for (int i = 0; i < 16; i++)
                                if (j + i < g.k) o[i] = out[i / 8].v[i % 8];
                        }
                    } else if (row < g.n) {
                        float* o = g.dw_part + ((int64_t)q.part * g.n + row) * g.k + j;
                        if ((g.k & 3) == 0 && j + 16 <= g.k) {
#pragma unroll
                            for (int i = 0; i < 16; i += 4) *reinterpret_cast<uint4*>(o + i) = make_uint4(v[i], v[i + 1], v[i + 2], v[i + 3]);
                        } else {
#pragma unroll
                            for (int i = 0; i < 16; i++)
                                if (j + i < g.k) o[i] = __uint_as_float(v[i]);
                        }
                    }
                    return;
                }
                if (DUAL) {
                    const float* pb = bias + (c - group) / kStep * 64 + lc;
#pragma unroll
                    for (int i = 0; i < 16; i += 4) {
                        const float4 x = *reinterpret_cast<const float4*>(pb + i), y = *reinterpret_cast<const float4*>(pb + 32 + i);
                        add2(v[i], v[i + 1], x.x, x.y);
                        add2(v[i + 2], v[i + 3], x.z, x.w);
                        add2(w[i], w[i + 1], y.x, y.y);
                        add2(w[i + 2], w[i + 3], y.z, y.w);
                    }
                }
                if (MODE == GATED_HEAD) {
                    // through shared memory, so that a row's 16 floats are stored side by side
                    float* sm = reinterpret_cast<float*>(stage);
#pragma unroll
                    for (int i = 0; i < 16; i += 2) {
                        const float2 m = split(make_f2(__uint_as_float(v[i]), __uint_as_float(v[i + 1])) *
                                               sigmoid(make_f2(__uint_as_float(w[i]), __uint_as_float(w[i + 1]))));
                        sm[lane * 17 + i] = m.x;
                        sm[lane * 17 + i + 1] = m.y;
                    }
                    __syncwarp();
                    const int rows = (int)max((int64_t)0, min((int64_t)32, g.frames - row0)), col = j + (lane & 15);
                    float* o = g.masks + (q.cs * g.band_cols + q.h.off) * g.frames + row0 * q.h.din + col;
                    if (col < q.h.din) {
#pragma unroll 8
                        for (int r = lane >> 4; r < rows; r += 2) o[(int64_t)r * q.h.din] = sm[r * 17 + (lane & 15)];
                    }
                    __syncwarp();
                    return;
                }
                uint32_t o[8], o2[8];
                if (MODE == GATED_FWD) {
#pragma unroll
                    for (int i = 0; i < 16; i += 2)
                        o[i / 2] = pack2<T>(act<ACT, true>(__uint_as_float(v[i])) * __uint_as_float(w[i]),
                                            act<ACT, true>(__uint_as_float(v[i + 1])) * __uint_as_float(w[i + 1]));
                } else if (MODE == GATED_PRE) {
                    // rounded to the type: the next products' operands have 16 bits (dx and dW are 2.4e-3
                    // off for it in bf16, 1.7e-3 by their own rounding alone)
#pragma unroll
                    for (int i = 0; i < 16; i += 2) {
                        float dg[2], du[2];
#pragma unroll
                        for (int k = 0; k < 2; k++) {
                            const float x = to_float(dy[(i + k) / 8].v[(i + k) % 8]);
                            float a, s;
                            act_both<ACT, true>(__uint_as_float(v[i + k]), a, s);
                            dg[k] = x * __uint_as_float(w[i + k]) * s;
                            du[k] = x * a;
                        }
                        o[i / 2] = pack2<T>(dg[0], dg[1]);
                        o2[i / 2] = pack2<T>(du[0], du[1]);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 8; i++) o[i] = pack2<T>(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]));
                }
                if (store) {
                    if (hh == 0) {   // the stage's last store has read it
                        if (lane == 0) stores_read();
                        __syncwarp();
                    }
                    // rows of 64 bytes as the 64-byte swizzle has them: 16-byte piece c of row r at c ^ (r / 2 & 3)
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        const int to = lane * 64 + (((2 * hh + i) ^ ((lane >> 1) & 3)) << 4);
                        *reinterpret_cast<uint4*>(stage + to) = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                        if (MODE == GATED_PRE)
                            *reinterpret_cast<uint4*>(stage + 2048 + to) = make_uint4(o2[4 * i], o2[4 * i + 1], o2[4 * i + 2], o2[4 * i + 3]);
                    }
                } else if (MODE != GATED_PRE && row < g.m) {
                    T* out = static_cast<T*>(MODE == GATED_FWD ? g.y : g.dx);
                    const int64_t pitch = MODE == GATED_FWD ? g.y_row : g.dx_row;
                    const int nj = MODE == GATED_DX ? g.k : g.n;
#pragma unroll
                    for (int i = 0; i < 16; i++)
                        if (j + i < nj) out[row * pitch + j + i] = reinterpret_cast<const T*>(&o[i / 2])[i & 1];
                }
            };
            auto load = [&](uint32_t (&v)[16], uint32_t (&w)[16], int c, int hh) {
                tmem_load16(v, lanes + c * 32 + hh * 16);
                if (DUAL) tmem_load16(w, lanes + width + c * 32 + hh * 16);
            };
            auto loaded = [&](uint32_t (&v)[16], uint32_t (&w)[16], int c, int hh) {
                tmem_wait();
                if (MODE == GATED_HEAD && q.kb > 1) {   // the other partial sum
                    uint32_t x[16];
#pragma unroll
                    for (int which = 0; which < 2; which++) {
                        tmem_load16(x, lanes + kAccCols + which * width + c * 32 + hh * 16);
                        tmem_wait();
#pragma unroll
                        for (int i = 0; i < 16; i++) {
                            uint32_t& y = which ? w[i] : v[i];
                            y = __float_as_uint(__uint_as_float(y) + __uint_as_float(x[i]));
                        }
                    }
                }
            };
            // The next 16 columns are on their way from TMEM while these go through the epilogue. (Not in
            // GATED_PRE, which has dy ahead instead: both together spill.)
            constexpr bool kAhead = MODE != GATED_PRE;
            uint32_t v0[16], w0[16], v1[16], w1[16];
            if (kAhead && group < pieces) {
                load(v0, w0, group, 0);
                loaded(v0, w0, group, 0);
            }
            for (int c = group; c < pieces; c += kStep) {
                const int j0 = q.n0 + c * 32;
                const bool last = c + kStep >= pieces;
                if (kAhead) load(v1, w1, c, 1);
                else {
                    load(v0, w0, c, 0);
                    loaded(v0, w0, c, 0);
                }
                if (MODE == GATED_PRE) {
                    dy[0] = ahead[0];
                    dy[1] = ahead[1];
                    ahead_of(row, j0 + 16, ahead);
                }
                half(v0, w0, c, 0);
                if (!kAhead) load(v1, w1, c, 1);
                loaded(v1, w1, c, 1);
                if (!last) {
                    if (kAhead) load(v0, w0, c + kStep, 0);
                } else {   // all in registers: the next products may have the set
                    fence_before();
                    __syncwarp();
                    if (lane == 0) bar_arrive_cluster(in_leader(acc_empty + set));
                }
                if (MODE == GATED_PRE) {
                    dy[0] = ahead[0];
                    dy[1] = ahead[1];
                    if (!last) ahead_of(row, j0 + kStep * 32, ahead);
                    else if (t + 2 * pairs < p.tiles) {   // of this warp's next tile
                        const Tile nq = tile_at<MODE>(p, t + 2 * pairs);
                        ahead_of(nq.m0 + rank * 128 + quad * 32 + lane, nq.n0 + group * 32, ahead);
                    }
                }
                half(v1, w1, c, 1);
                if (kAhead && !last) loaded(v0, w0, c + kStep, 0);
                if (store) {
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0 && j0 < (MODE == GATED_DX ? g.k : g.n) && row0 < g.m) {
                        tma_store(&p.c[0], j0, (int)row0, stage);
                        if (MODE == GATED_PRE) tma_store(&p.c[1], j0, (int)row0, stage + 2048);
                        store_commit();
                    }
                }
            }
            if (group >= pieces) {   // no piece of this tile
                fence_before();
                __syncwarp();
                if (lane == 0) bar_arrive_cluster(in_leader(acc_empty + set));
            }
        }
        if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    cluster_sync();   // neither block goes while the other may still signal or read it
    if (warp == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2 * kAccCols));
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
    kernel<<<2 * (unsigned)std::min<int64_t>(p.tiles, sms / 2), kThreads, smem_bytes<MODE>(), st>>>(p);
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

// The width of dx's and dW's column tiles: whole 32-column pieces as the epilogue stores them (so that
// no piece reaches into the next tile), of the tile count that takes the fewest column steps per
// pair, counting 32 more per tile for the rows of A that each tile loads again. dW's
// sums over the rows have the accumulators' last columns.
int column_tile(int k, int64_t rest, int64_t pairs, bool sums) {
    const int most = sums ? kSumCol / 32 * 32 : 256;
    int64_t best = INT64_MAX, width = 0;
    const int64_t few = ceil_div(k, most);
    for (int64_t t = few; t <= std::min(ceil_div(k, 64), few + 16); t++) {
        const int64_t cols = ceil_div(ceil_div(k, t), 32) * 32, cost = ceil_div(rest * ceil_div(k, cols), pairs) * (cols + 32);
        if (cost < best) { best = cost; width = cols; }
    }
    return (int)width;
}

} // namespace

int64_t gated_col_sums(const GatedParams& g, int sms) {
    return g.splits * ceil_div(g.k, column_tile(g.k, 2 * g.splits * ceil_div(g.n, kPairM), sms / 2, true));
}

void launch_gated_mma(GatedMode mode, bool bf16, const GatedParams& g, int64_t head_rows, int sms, cudaStream_t st) {
    MmaParams p{};
    p.g = g;
    const int64_t mt = ceil_div(mode == GATED_HEAD ? g.frames : g.m, kPairM), pairs = sms / 2;
    int64_t tiles = 0, tiles_n = 1, rest_n = 1;
    if (mode == GATED_HEAD) {
        tiles_n = mt;
        rest_n = g.n_tiles;
        tiles = head_rows / g.frames / g.bands * mt * g.n_tiles;
        encode(&p.a[0], bf16, g.x, head_rows, g.k, g.x_row, kDepth, 128);
        encode(&p.b[0], bf16, g.wg, g.stems * 2 * g.band_cols, g.k, g.wg_row, kDepth, 32);
    } else if (mode == GATED_FWD || mode == GATED_PRE) {
        // 128 outputs to a tile; 64 when that would leave SMs without a tile (384 x 1408 bf16, 64 and 128: 256
        // rows 6.6 and 8.2 us, 1500 8.4 and 8.7, 3000 12.1 and 11.1)
        const int n = mt * ceil_div(g.n, 128) < pairs ? 64 : 128;
        p.cols = 2 * n;
        tiles_n = ceil_div(g.n, n);
        tiles = mt * tiles_n;
        encode(&p.a[0], bf16, g.x, g.m, g.k, g.x_row, kDepth, 128);
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
        const int64_t rest = mode == GATED_DX ? mt : 2 * g.splits * ceil_div(g.n, kPairM);
        p.sums = mode == GATED_DW && g.col_sums;
        p.cols = column_tile(g.k, rest, pairs, p.sums);
        tiles_n = ceil_div(g.k, p.cols);
        rest_n = ceil_div(g.n, kPairM);
        tiles = rest * tiles_n;
        if (mode == GATED_DX) {
            encode(&p.a[0], bf16, g.dg, g.m, g.n, g.pre_row, kDepth, 128);
            encode(&p.a[1], bf16, g.du, g.m, g.n, g.pre_row, kDepth, 128);
            encode(&p.b[0], bf16, g.wg, g.n, g.k, g.wg_row, 64, kDepth);
            encode(&p.b[1], bf16, g.wu, g.n, g.k, g.wu_row, 64, kDepth);
            p.store_by_tma = aligned(g.dx, 16) && (g.dx_row % 8 == 0 || g.m == 1);
            if (p.store_by_tma) encode(&p.c[0], bf16, g.dx, g.m, g.k, g.dx_row, 32, 32, true);
        } else {
            encode(&p.a[0], bf16, g.dg, g.m, g.n, g.pre_row, 64, kDepth);
            encode(&p.a[1], bf16, g.du, g.m, g.n, g.pre_row, 64, kDepth);
            encode(&p.b[0], bf16, g.x, g.m, g.k, g.x_row, 64, kDepth);
        }
    }
    if (tiles > INT32_MAX) fail(STG_UNSUPPORTED, "gated: too many tiles");
    p.tiles = (int)tiles;
    p.tiles_n = FastDiv((uint32_t)tiles_n);
    p.rest_n = FastDiv((uint32_t)rest_n);
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
    cuda_check(cudaDeviceSynchronize(), "gated status");   // the copy alone does not wait for streams that do not block
    cuda_check(cudaMemcpyFromSymbol(&v, g_gave_up, sizeof(v)), "gated status");
    return (int)v;
}

} // namespace stg
