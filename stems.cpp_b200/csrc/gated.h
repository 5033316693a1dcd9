// gated.h -- what the gated projection's entry points (gated.cu) and its kernels share.
#pragma once
#include "layers.h"

namespace stg {

constexpr int kGatedTileM = 128;   // rows of a tile on the CUDA cores

// The four products of the gated projection. Rows of x are m, outputs n, features k.
enum GatedMode : int {
    GATED_FWD,    // y = act(x Wg^T + bg) (x Wu^T + bu)
    GATED_HEAD,   // the same per band, the sigmoid on the second factor, float output
    GATED_PRE,    // dg = dy u act'(g) and du = dy act(g), and their column sums
    GATED_DX,     // dx = dg Wg + du Wu
    GATED_DW,     // dWg = dg^T x, dWu = du^T x
};

struct GatedParams {
    int64_t m;
    int n, k;
    int act;
    const void *x, *wg, *wu, *bg, *bu, *dy;
    int64_t x_row, wg_row, wu_row, y_row, dx_row;
    void *y, *dx;
    // backward scratch: dg and du [m][pre_row] in the element type, column sums [row tiles of 128, 64 or 8, or gated_col_sums][2][n]
    void *dg, *du;
    int64_t pre_row;
    float* col_sums;
    // dWg and dWu (either may be null): written by their product when `splits` is 1, else partial sums
    // over that many ranges of rows, [splits][2][n][k] float
    void* dw[2];
    int64_t dw_row[2];
    float* dw_part;
    int splits;
    int64_t split_rows;
    // dx on the CUDA cores: partial sums over dx_splits ranges of the widths, [dx_splits][m][k] float, when more than one
    float* dx_part;
    int dx_splits;
    // mask head: tiles over the bands' columns
    const HeadTile* tiles;
    int n_tiles;                       // tiles of one stem
    int64_t frames;                    // rows of a band
    int bands, stems;
    int64_t band_cols;                 // sum of din
    float* masks;
};

// One of the products on the tensor cores (gated_mma.cu), f16 or bf16. Matrices of g that are
// read or written by TMA (x, Wg, Wu, dg, du) start on 16 bytes with rows a multiple of 16 bytes apart.
// head_rows: rows of x in the mask head, below 2^31.
void launch_gated_mma(GatedMode mode, bool bf16, const GatedParams& g, int64_t head_rows, int sms, cudaStream_t st);
// How many partial column sums GATED_DW leaves: one per split and column tile, at most splits * ceil(k / 64).
int64_t gated_col_sums(const GatedParams& g, int sms);
// Whether a kernel of launch_gated_mma gave up a wait since the library was loaded (it then
// returned with its result incomplete). Waits for the device.
int gated_gave_up();

} // namespace stg
