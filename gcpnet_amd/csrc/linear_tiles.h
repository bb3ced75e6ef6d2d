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

// Which tile, and into how many pieces k is split: the least of the estimated times
//     rounds over the 256 CUs x (products of a tile / rate + what a tile takes besides) [+ joining the pieces]
// with the rates that the tiles reach on one CU (TFLOP/s; one, two, more workgroups of it on a CU: one alone cannot hide the memory's latency),
// fitted to these measurements (us, bf16 unless said; 64 / 128 / 256 tile): 2048^3 27 / 23 / 53, 500 x 4096 x 4096 31 / 37 / 94,
// 1537 x 1000 x 777 11 / 13 / 32, 200 x 4096 x 4096 25 / 36 / 92 and 64 in two pieces 22, 4096 x 8192 x 2048 177 / 127 / 178,
// 10000 x 128 x 512 fp32 20 / 26, 2048^3 fp32 141 / 144.
inline GcpLinearPlan gcp_linear_plan(int64_t m, int64_t n, int64_t k, int size) {
    static const double RATE[2][3][3] = {{{1.35, 2.2, 2.5}, {3.3, 4.1, 4.1}, {4.9, 4.9, 4.9}}, {{0.345, 0.43, 0.48}, {0.47, 0.53, 0.55}, {}}};
    static const double BESIDES[3] = {1.5, 3.0, 6.0};
    const int64_t ke = 128 / size, steps = (k + ke - 1) / ke;
    GcpLinearPlan best = {};
    double least = 0.0;
    for (int shape = 0; shape < (size == 4 ? 2 : 3); ++shape) {
        const int64_t b = 64 << shape, tm = (m + b - 1) / b, tn = (n + b - 1) / b, tiles = tm * tn;
        for (int64_t s = 1; s <= 32 && (s == 1 || (steps >= 8 * s && tiles * s <= 1024)); s += s < 4 ? 1 : s < 8 ? 2 : 4) {
            const int64_t per = steps > 0 ? (steps + s - 1) / s : 1, pieces = steps > 0 ? (steps + per - 1) / per : 1;
            const int64_t rounds = (tiles * pieces + 255) / 256;
            const double work = 2e-6 * (double)(b * b) * (double)(per * ke);
            double t = (double)rounds * (work / RATE[size == 4][shape][rounds < 3 ? (rounds > 0 ? rounds - 1 : 0) : 2] + BESIDES[shape]);
            if (pieces > 1) t += 3.0 + 2e-6 * (double)(pieces * m) * (double)n;  // (8 bytes a value at 4 TB/s)
            if (best.tiles_m && t >= least) continue;
            least = t;
            best.shape = shape;
            best.tiles_m = tm;
            best.tiles_n = tn;
            best.splits = (int)pieces;
            best.k_per = per * ke;
            best.floats = pieces > 1 ? pieces * m * n : 0;
        }
    }
    return best;
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
