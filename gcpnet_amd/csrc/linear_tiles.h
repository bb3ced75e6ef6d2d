// How a product C[m][n] = sum_k A[m][k] B[n][k] of linear_act.hip is cut into workgroups.
#pragma once
#include "common.h"

struct GcpLinearPlan {
    int shape;  // 0: 64 x 64, 1: 128 x 128, 2: 256 x 256 tiles
    int64_t tiles_m, tiles_n;
    int splits;
    int64_t k_per, floats;  // k of a split; workspace
};

// The largest tile that still gives every CU (256) two workgroups: a large tile reads its operands fewer times, but idle CUs cost more.
// With fewer workgroups than CUs even so, k is split, in pieces of at least eight tiles of 128 bytes.  (fp32 takes the matrix pipe 16
// times as long per byte: 128 x 128 tiles feed it.)
inline GcpLinearPlan gcp_linear_plan(int64_t m, int64_t n, int64_t k, int size) {
    const int64_t ke = 128 / size, steps = (k + ke - 1) / ke;
    GcpLinearPlan p = {};
    for (p.shape = size == 4 ? 1 : 2; p.shape >= 0; --p.shape) {
        const int64_t bm = 64 << p.shape, bn = bm;
        p.tiles_m = (m + bm - 1) / bm;
        p.tiles_n = (n + bn - 1) / bn;
        if (p.tiles_m * p.tiles_n >= 256 || p.shape == 0) break;
    }
    const int64_t tiles = p.tiles_m * p.tiles_n;
    int64_t s = tiles > 0 ? 512 / tiles : 1, most = steps / 8;
    s = s < most ? s : most;
    if (tiles >= 256 || s < 2) s = 1;
    const int64_t per = s > 0 && steps > 0 ? (steps + s - 1) / s : 1;
    p.splits = steps > 0 ? (int)((steps + per - 1) / per) : 1;
    p.k_per = per * ke;
    p.floats = p.splits > 1 ? (int64_t)p.splits * m * n : 0;
    return p;
}

// Block -> tile of C.  Blocks go round the eight XCDs: consecutive ones of an XCD get consecutive tiles (its L2 holds what they share), and
// tiles are numbered through bands of eight rows of tiles, column by column.
__device__ __forceinline__ void gcp_tile_of_block(int block, int total, int tiles_m, int tiles_n, int& tm, int& tn) {
    const int xcd = block & 7, at = block >> 3, each = total >> 3, more = total & 7;
    const int id = xcd * each + (xcd < more ? xcd : more) + at;
    const int band = 8 * tiles_n, first = id / band * 8, in = id % band;
    const int high = tiles_m - first < 8 ? tiles_m - first : 8;
    tm = first + in % high;
    tn = in / high;
}

// out[q][c] = sum over `blocks` of part[b][q][c], in a fixed order, for `sets` <= 5 rows of d columns (block_norm.hip)
int gcp_column_sums(const float* part, int blocks, int sets, int d, void* const* out, const int* type, hipStream_t stream);
