// How a product C[m][n] = sum_k A[m][k] B[n][k] of linear_act.hip is cut into workgroups.
#pragma once
#include "common.h"

struct GcpLinearPlan {
    int shape;  // 0: 64 x 64, 1: 128 x 128, 2: 256 x 256 tiles
    int64_t tiles_m, tiles_n;
    int splits;
    int64_t k_per, floats;  // k of a split; workspace
};

// A forward of up to so many rows reads W once, straight into the fragments (4096 x 4096 bf16: 32 rows 14.9 us, in tiles 17.6; 64 rows would
// be 23.2).
#define GCP_FEW_ROWS 32

// The largest tile that still gives every CU (256) a workgroup: a large tile reads its operands fewer times, but idle CUs cost more.
// With few workgroups even so, k is split (up to 512 of them, or 256 of the largest), in pieces of at least eight tiles of 128 bytes, where that
// saves 16 tiles' time or more: the second launch takes as long as some 12 of them (1000 x 1024 x 1024 bf16, 16 tiles along k: 9.8 us in one piece, 14.6 in two;
// 200 x 4096 x 4096, 64 tiles: 25.5 and 22.4 us).
inline GcpLinearPlan gcp_linear_plan(int64_t m, int64_t n, int64_t k, int size) {
    const int64_t ke = 128 / size, steps = (k + ke - 1) / ke;
    GcpLinearPlan p = {};
    for (p.shape = size == 4 ? 1 : 2; p.shape >= 0; --p.shape) {
        const int64_t b = 64 << p.shape;
        p.tiles_m = (m + b - 1) / b;
        p.tiles_n = (n + b - 1) / b;
        if (p.tiles_m * p.tiles_n >= 256 || p.shape == 0) break;
    }
    const int64_t tiles = p.tiles_m * p.tiles_n, most = steps / 8;
    int64_t s = tiles > 0 ? (p.shape == 2 ? 256 : 512) / tiles : 1;
    s = s < most ? s : most;
    if (s < 2 || steps - steps / s < 16) s = 1;
    const int64_t per = steps > 0 ? (steps + s - 1) / s : 1;
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
