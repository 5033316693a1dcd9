// rotary.cu -- rotary positions for queries and keys (include/stems_gpu_v1.h: stg_rotary).
//
// Pair i of a token at position p turns by a = p f_i: (x0, x1) -> m (x0 cos a - x1 sin a,
// x1 cos a + x0 sin a). The work is one read and one write of the tensors; what could spoil it
// is the sines and cosines, which every head of a token shares. A block therefore takes a few
// tokens with all their heads, of queries and keys together, computes the tokens' table of
// (cos, sin) once into shared memory and streams the heads past it in 16-byte vectors. 60 x 801
// tokens of 8 query and 8 key heads of 64, bf16: 38 us, 5.2 TB/s.
#include "layers.h"

#include <cmath>

namespace stg {

namespace {

constexpr int kThreads = 256;
constexpr int kMaxHalf = 256;      // rotary_dim at most 512
constexpr size_t kSmem = 32 * 1024;   // a block's tables at most

struct RotaryTensor {
    const void* x;
    void* y;
    int64_t xb, xt, xh, yb, yt, yh;
};

struct RotaryParams {
    RotaryTensor t[2];
    int heads0, heads;              // of the first tensor, of both
    int half, rotary, dim;
    int64_t tokens, n;              // a batch item's tokens, all tokens
    int tokens_per_block, heads_per_block;
    int copy_tail;
    FastDiv per_head;               // items of a head: rotated ones, then copied ones
    int rot_items, tail_items;
    FastDiv half_div;
    const int32_t* pos;
    int64_t pos_batch;
    int offset;
    float magnitude;
    double turns[kMaxHalf];         // f_i / 2 pi, negative for the inverse
};

// cos and sin of 2 pi t, t in turns. The fraction r in [-1/2, 1/2] is exact in double; it goes to
// float as a leading part and a rest, and the rest's effect is added to first order, so the
// result is good to about one unit of the last place, and past positions of 2^28 to what the product
// p f_i loses in double (2^-52 of it: 5e-7 at 2^31).
__device__ __forceinline__ float2 cos_sin_turns(double t) {
    const double r = 2.0 * (t - rint(t));   // half turns
    const float hi = (float)r;
    const float lo = (float)(r - (double)hi) * 3.14159265358979f;
    float s, c;
    sincospif(hi, &s, &c);
    return make_float2(fmaf(-s, lo, c), fmaf(c, lo, s));
}

// V elements per access. LAYOUT 0: an item is a run of max(V, 2) neighbouring elements, whole
// pairs; LAYOUT 1: V elements of the first half and their partners in the second. Tail items
// are V elements past the rotated part. A thread keeps to one place of the heads (or a few) and walks
// the block's tokens, so that an item costs it an offset from shared memory and an addition.
template <class T, int V, int LAYOUT>
__global__ void __launch_bounds__(kThreads, 4) rotary_kernel(const __grid_constant__ RotaryParams p) {
    constexpr int E = LAYOUT == 0 && V < 2 ? 2 : V;          // elements of an item's run
    constexpr int R = LAYOUT == 0 ? E / V : 2;               // accesses of an item
    constexpr int U = 4 / R;
    using P = Pack<T, V>;
    struct Item { P v[R]; };
    extern __shared__ __align__(16) uint8_t smem[];
    longlong2* at = reinterpret_cast<longlong2*>(smem);      // [tensor][token]: offsets into x and y
    double* turns = reinterpret_cast<double*>(at + 2 * p.tokens_per_block);
    float2* table = reinterpret_cast<float2*>(turns + p.half);
    int32_t* where = reinterpret_cast<int32_t*>(table + p.tokens_per_block * p.half);   // [token]: positions
    const int64_t tok0 = (int64_t)blockIdx.x * p.tokens_per_block;
    const int n_tok = (int)min((int64_t)p.tokens_per_block, p.n - tok0);
    const int head0 = blockIdx.y * p.heads_per_block;
    const int columns = min(p.heads_per_block, p.heads - head0) * (int)p.per_head.d;

    for (int e = threadIdx.x; e < 2 * n_tok; e += kThreads) {
        const int k = e >= n_tok, tk = e - k * n_tok;
        const int64_t tok = tok0 + tk, b = tok / p.tokens, t = tok - b * p.tokens;
        if (!k) where[tk] = p.pos ? p.pos[b * p.pos_batch + t] : p.offset + (int32_t)t;
        at[k * p.tokens_per_block + tk] = make_longlong2(b * p.t[k].xb + t * p.t[k].xt, b * p.t[k].yb + t * p.t[k].yt);
    }
    for (int i = threadIdx.x; i < p.half; i += kThreads) turns[i] = p.turns[i];
    __syncthreads();
    for (int e = threadIdx.x; e < n_tok * p.half; e += kThreads) {
        const int tk = (int)p.half_div.div((uint32_t)e), i = e - tk * p.half;
        float2 cs = cos_sin_turns((double)where[tk] * turns[i]);
        cs.x *= p.magnitude;
        cs.y *= p.magnitude;
        table[e] = cs;
    }
    __syncthreads();

    auto turn = [](Item& i, const float2* w) {
        if (LAYOUT == 0) {
#pragma unroll
            for (int j = 0; j < E; j += 2) {
                const float2 t = w[j >> 1];
                T &x0 = i.v[j / V].v[j % V], &x1 = i.v[(j + 1) / V].v[(j + 1) % V];
                const float a = to_float(x0), b = to_float(x1);
                x0 = from_float<T>(fmaf(a, t.x, -b * t.y));
                x1 = from_float<T>(fmaf(b, t.x, a * t.y));
            }
        } else {
#pragma unroll
            for (int j = 0; j < V; j++) {
                const float2 t = w[j];
                const float a = to_float(i.v[0].v[j]), b = to_float(i.v[R - 1].v[j]);
                i.v[0].v[j] = from_float<T>(fmaf(a, t.x, -b * t.y));
                i.v[R - 1].v[j] = from_float<T>(fmaf(b, t.x, a * t.y));
            }
        }
    };
    const int width = min(columns, kThreads), step = kThreads / width, r = threadIdx.x / width;
    if (r >= step) return;
    for (int c = threadIdx.x - r * width; c < columns; c += width) {
        const int hd = (int)p.per_head.div((uint32_t)c), item = c - hd * (int)p.per_head.d;
        const int h = head0 + hd, k = h >= p.heads0, hh = k ? h - p.heads0 : h;
        const bool tail = item >= p.rot_items;
        const int run = tail ? p.rotary + (item - p.rot_items) * V : item * E;
        const T* x = static_cast<const T*>(k ? p.t[1].x : p.t[0].x) + hh * (k ? p.t[1].xh : p.t[0].xh) + run;
        T* y = static_cast<T*>(k ? p.t[1].y : p.t[0].y) + hh * (k ? p.t[1].yh : p.t[0].yh) + run;
        const longlong2* to = at + k * p.tokens_per_block;
        const float2* cs = table + (LAYOUT == 0 ? run >> 1 : run);
        constexpr int other = LAYOUT == 0 ? V : 0;
        const int second = LAYOUT == 0 ? other : p.half;
        for (int t0 = r; t0 < n_tok; t0 += U * step) {
            Item i[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int tk = t0 + u * step;
                if (tk >= n_tok) break;
                const T* q = x + to[tk].x;
                i[u].v[0] = load_stream<P>(q);
                if (R == 2 && !tail) i[u].v[R - 1] = load_stream<P>(q + second);
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int tk = t0 + u * step;
                if (tk >= n_tok) break;
                T* q = y + to[tk].y;
                if (!tail) {
                    turn(i[u], cs + tk * p.half);
                    if (R == 2) store_stream(q + second, i[u].v[R - 1]);
                }
                store_stream(q, i[u].v[0]);
            }
        }
    }
}

template <class T, int V>
void launch(RotaryParams& p, int layout, cudaStream_t st) {
    const int e = layout == 0 && V < 2 ? 2 : V;
    p.rot_items = (layout == 0 ? p.rotary : p.half) / e;
    p.tail_items = p.copy_tail ? (p.dim - p.rotary) / V : 0;
    const int per_head = p.rot_items + p.tail_items;
    // tokens so that a thread has about sixteen items, while the table fits and the GPU has two blocks
    // per SM; heads split over blocks only when so few tokens would leave most of it idle (then
    // each part repeats the table)
    p.heads_per_block = p.heads;
    p.tokens_per_block = 1;
    auto smem_of = [&](int tokens) { return (size_t)tokens * (sizeof(float2) * p.half + 2 * sizeof(longlong2) + sizeof(int32_t)) + sizeof(double) * p.half; };
    while ((int64_t)p.tokens_per_block * per_head * p.heads < 16 * kThreads && smem_of(2 * p.tokens_per_block) <= kSmem &&
           p.n / (2 * p.tokens_per_block) >= 296)
        p.tokens_per_block *= 2;
    const int64_t blocks = (p.n + p.tokens_per_block - 1) / p.tokens_per_block;
    if (blocks < 148) {
        const int want = (int)std::min<int64_t>((296 + blocks - 1) / blocks, ((int64_t)per_head * p.heads + kThreads - 1) / kThreads);
        p.heads_per_block = std::max(1, (p.heads + want - 1) / std::max(1, want));
    }
    // a block's items stay far below 2^31
    while ((int64_t)p.tokens_per_block * per_head * p.heads_per_block >= (1 << 30)) p.heads_per_block = (p.heads_per_block + 1) / 2;
    const int parts = (p.heads + p.heads_per_block - 1) / p.heads_per_block;
    p.per_head = FastDiv((uint32_t)per_head);
    p.half_div = FastDiv((uint32_t)p.half);
    if (blocks > INT32_MAX || parts > 65535) fail(STG_UNSUPPORTED, "rotary: too many tokens or heads");
    const dim3 grid((unsigned)blocks, (unsigned)parts);
    const size_t smem = smem_of(p.tokens_per_block);
    if (layout == 0) rotary_kernel<T, V, 0><<<grid, kThreads, smem, st>>>(p);
    else rotary_kernel<T, V, 1><<<grid, kThreads, smem, st>>>(p);
    cuda_check(cudaGetLastError(), "rotary kernel");
}

template <class T, int V>
void launch_widest(RotaryParams& p, int layout, int width, cudaStream_t st) {
    if constexpr (V > 1) {
        if (width < V) return launch_widest<T, V / 2>(p, layout, width, st);
    }
    launch<T, V>(p, layout, st);
}

void check_config(const stg_rotary_config* c) {
    check_sized(c, "rotary");
    check(valid_dtype(c->dtype), "rotary: unknown dtype");
    check(c->layout == 0 || c->layout == 1, "rotary: layout must be 0 or 1");
    check(c->inverse == 0 || c->inverse == 1, "rotary: inverse must be 0 or 1");
    check(c->batch >= 0 && c->tokens >= 0, "rotary: negative size");
    check(c->head_dim >= 1 && c->head_dim <= 65536, "rotary: head_dim must be 1..65536");
    const int r = c->rotary_dim ? c->rotary_dim : c->head_dim;
    check(r >= 2 && r % 2 == 0 && r <= c->head_dim, "rotary: rotary_dim must be even and at most head_dim");
    if (r > 2 * kMaxHalf) fail(STG_UNSUPPORTED, "rotary: rotary_dim above 512");
    check(c->scaling >= 0 && c->scaling <= 3, "rotary: unknown scaling");
    check(c->base == 0.0 || (c->base > 0.0 && c->base != 1.0 && std::isfinite(c->base)), "rotary: base must be positive and not 1");
    check(std::isfinite(c->magnitude), "rotary: magnitude must be finite");
    if (c->scaling != 0) check(c->factor >= 1.0 && std::isfinite(c->factor), "rotary: factor must be at least 1");
    if (c->scaling == 2) check(r > 2, "rotary: NTK scaling needs rotary_dim above 2");
    if (c->scaling == 3) {
        check(c->original_length > 0.0 && std::isfinite(c->original_length), "rotary: original_length must be positive");
        const bool none = c->beta_fast == 0.0 && c->beta_slow == 0.0;
        check(none || (c->beta_slow > 0.0 && c->beta_fast > c->beta_slow && std::isfinite(c->beta_fast)),
              "rotary: beta_fast must be above beta_slow, both positive");
    }
    if (c->batch > 0 && c->tokens > INT64_MAX / 2 / c->batch) fail(STG_UNSUPPORTED, "rotary: too many tokens");
}

// f_i and m of a checked configuration.
double frequencies(const stg_rotary_config& c, double* f) {
    const int r = c.rotary_dim ? c.rotary_dim : c.head_dim, half = r / 2;
    double base = c.base == 0.0 ? 10000.0 : c.base, m = 1.0;
    const double s = c.factor;
    if (c.scaling == 2) base *= std::pow(s, (double)r / (r - 2));
    for (int i = 0; i < half; i++) f[i] = std::pow(base, -2.0 * i / r);
    if (c.scaling == 1)
        for (int i = 0; i < half; i++) f[i] /= s;
    if (c.scaling == 3) {
        const bool none = c.beta_fast == 0.0 && c.beta_slow == 0.0;
        const double fast = none ? 32.0 : c.beta_fast, slow = none ? 1.0 : c.beta_slow;
        auto dim_of = [&](double turns) { return r * std::log(c.original_length / (turns * 2.0 * M_PI)) / (2.0 * std::log(base)); };
        const double lo = std::max(std::floor(dim_of(fast)), 0.0);
        // the ramp may end past the last pair (half - 1): then every pair turns more than `slow` times
        const double hi = std::min(std::ceil(dim_of(slow)), (double)(r - 1));
        for (int i = 0; i < half; i++) {
            const double g = std::min(std::max((i - lo) / std::max(hi - lo, 0.001), 0.0), 1.0);
            f[i] = (1.0 - g) * f[i] + g * f[i] / s;
        }
        m = 0.1 * std::log(s) + 1.0;
    }
    return c.magnitude != 0.0 ? c.magnitude : m;
}

} // namespace

} // namespace stg

extern "C" {

STG_API stg_status stg_rotary_frequencies(const stg_rotary_config* c, double* f, double* magnitude) {
    return guard(nullptr, [&] {
        check_config(c);
        check(f && magnitude, "rotary: null buffer");
        *magnitude = frequencies(*c, f);
    });
}

STG_API stg_status stg_rotary(stg_engine* e, const stg_rotary_config* c, const stg_rotary_tensor* tensors,
                              int32_t n_tensors, const int32_t* d_positions, int64_t position_batch_stride, void* stream) {
    if (!e) return STG_INVALID_ARGUMENT;
    return guard(e, [&] {
        check_config(c);
        check(tensors && (n_tensors == 1 || n_tensors == 2), "rotary: one or two tensors");
        check(position_batch_stride >= 0, "rotary: negative stride");
        check(aligned(d_positions, 4), "rotary: positions are not aligned");
        if (!d_positions && c->tokens > 0)
            check(c->offset + (c->tokens - 1) <= INT32_MAX, "rotary: a position does not fit 32 bits");
        RotaryParams p{};
        const size_t es = elem_size(c->dtype);
        p.dim = c->head_dim;
        p.rotary = c->rotary_dim ? c->rotary_dim : c->head_dim;
        p.half = p.rotary / 2;
        p.tokens = c->tokens;
        p.n = c->batch * c->tokens;
        int64_t heads = 0;
        // the widest vector that the sizes, strides and addresses allow
        int width = (int)(16 / es);
        auto fit = [&](int64_t n) { while (n % width) width /= 2; };
        fit(c->layout == 0 ? p.rotary : p.half);
        bool in_place = true;
        for (int k = 0; k < n_tensors; k++) {
            const stg_rotary_tensor& t = tensors[k];
            check(t.heads >= 0 && t.heads <= (1 << 20), "rotary: heads must be 0..2^20");
            check(t.x_batch >= 0 && t.x_token >= 0 && t.x_head >= 0 && t.y_batch >= 0 && t.y_token >= 0 && t.y_head >= 0,
                  "rotary: negative stride");
            p.t[k] = RotaryTensor{t.d_x, t.d_y, t.x_batch, t.x_token, t.x_head, t.y_batch, t.y_token, t.y_head};
            if (k == 0) p.heads0 = (int)t.heads;
            heads += t.heads;
            if (!t.heads || !p.n) continue;
            check(t.d_x && t.d_y, "rotary: null buffer");
            check(aligned(t.d_x, es) && aligned(t.d_y, es), "rotary: a buffer is not aligned to its elements");
            check((t.y_batch || c->batch == 1) && (t.y_token || c->tokens == 1) && (t.y_head || t.heads == 1),
                  "rotary: an output stride of 0");
            if (t.d_x != t.d_y || t.x_batch != t.y_batch || t.x_token != t.y_token || t.x_head != t.y_head) in_place = false;
            for (int64_t s : {t.x_batch, t.x_token, t.x_head, t.y_batch, t.y_token, t.y_head}) fit(s);
            while (!aligned(t.d_x, width * es) || !aligned(t.d_y, width * es)) width /= 2;
        }
        p.heads = (int)heads;
        if (!p.n || !heads) return;
        p.copy_tail = p.rotary < p.dim && !in_place;
        if (p.copy_tail) { fit(p.dim - p.rotary); fit(p.rotary); }
        p.pos = d_positions;
        p.pos_batch = position_batch_stride;
        p.offset = c->offset;
        p.magnitude = (float)frequencies(*c, p.turns);
        for (int i = 0; i < p.half; i++) p.turns[i] *= (c->inverse ? -1.0 : 1.0) / (2.0 * M_PI);
        DeviceScope scope(e);
        const cudaStream_t st = static_cast<cudaStream_t>(stream);
        with_dtype(c->dtype, [&](auto* tag) {
            using T = std::remove_pointer_t<decltype(tag)>;
            launch_widest<T, (int)(16 / sizeof(T))>(p, c->layout, width, st);
        });
    });
}

} // extern "C"
