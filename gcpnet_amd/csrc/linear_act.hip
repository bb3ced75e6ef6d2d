// y = act(x W^T + b) + r and its backward for fp32, bf16 and fp16, every length and stride.
//
//   z = x W^T + b;  y = act(z) + r;     dz = dy act'(z);  dx = dz W;  dW = dz^T x;  db = column sums of dz;  dr = dy
//
// All three products are C[m][n] = sum_k A[m][k] B[n][k] with operands whose k runs along memory or across it (W in dx; dz and x in
// dW), in one kernel template:
//   * a workgroup owns a BM x BN tile of C, a wave a part of it in 16 x 16 MFMA tiles (16-bit: v_mfma_f32_16x16x32, fp32:
//     v_mfma_f32_16x16x4_f32; sums in fp32);
//   * tiles of 128 bytes of k travel from memory into a ring of LDS buffers by direct loads (no registers); the 16-byte pieces of an LDS
//     row are permuted (by the row) so that fragment reads spread over the banks;
//   * a tile is two steps of the 16-bit matrix instructions; while one step's fragments are multiplied the next step's are read, B's into
//     a second set of registers, A's into the registers of the row of products just issued; the waves meet once a tile, and the direct loads
//     of the next free buffer are spread between the rows of products (all at once they held the matrix pipe up: 8192 x 4096 x 4096 bf16
//     240 us, spread 223.5 = 1.23 PFLOP/s; in training, the median of 24 launches in two runs, 265 - 275 us with SiLU, residual and z, 241 - 253 us dx, 220 - 237 us dW);
//   * an operand with k across memory keeps its layout in LDS, [k][m]; 16-bit fragments come out of it through the transposing LDS
//     read, fp32 ones element by element;
//   * operands whose rows are not whole 16-byte pieces are first copied into the workspace, rows filled up with zeros (one launch for all of
//     them); where k ends inside a tile, the places behind it are set to zero;
//   * a forward with few rows reads W once, straight into registers (few_rows_kernel);
//   * few tiles of C: k is split over workgroups, which leave fp32 partial sums for a second launch that adds them in a fixed order and
//     applies the epilogue (no atomics: results repeat bit for bit).
// The epilogue adds the bias, applies the activation, adds the residual and rounds once; in training it also stores z.  The accumulators go
// through LDS first, so that a lane holds 16 bytes of a row and a wave reads and writes whole rows of its part of the tile.
#include <type_traits>

#include "elem_types.h"
#include "linear_tiles.h"

namespace {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int KROW = 128;  // bytes of k in a tile

struct Epilogue {
    const void *bias, *residual;
    int64_t r_ld;
    int act, bias_f32;
    float slope;
    void *y, *z;  // contiguous [m, n]
};

struct Gemm {
    int64_t m, n, k;
    const void *a, *b;
    int64_t a_ld, b_ld;
    int64_t a_rows, b_rows;  // rows of A and B that are there to be read: m and n, or more where k is across and rows are filled up
    int tiles_m, tiles_n, splits;
    int64_t k_per;       // k per split, a multiple of the tile's
    float* part;         // [splits, m, n] or NULL
    Epilogue e;
};

// V columns of one row from n on, `count` of them there: bias, z, activation, residual (`r`, loaded before), y
template <class E, int V>
__device__ __forceinline__ void finish(const Epilogue& e, int64_t m, int64_t n, int64_t N, int count, const float (&bias)[V], const Raw<E, V>& r, float (&v)[V]) {
    const int64_t at = m * N + n;
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] += bias[j];
    if (e.z) {
        // z past the type's range: silu'(-inf) would be -inf * 0, while every activation's slope has reached its constant at the largest number
        float z[V];
#pragma unroll
        for (int j = 0; j < V; ++j) z[j] = elem_in_range<E>(v[j]);
        elem_store<E, V>(e.z, at, z, count);
    }
    float none[V];
    elem_act<V, false>(e.act, e.slope, v, v, none);
    if (e.residual)
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] += r[j];
    elem_store<E, V>(e.y, at, v, count);
}

template <class E, int V>
__device__ __forceinline__ void bias_load(const Epilogue& e, int64_t n, int count, float (&bias)[V]) {
#pragma unroll
    for (int j = 0; j < V; ++j) bias[j] = 0.f;
    if (e.bias && count > 0) param_load<E, V>(e.bias, n, count, e.bias_f32).unpack(e.bias_f32, bias);
}

// 16 bytes per lane from memory (uniform base + offset) to LDS (lane l to base + 16 l), counted by vmcnt.  In asm, because the compiler would
// otherwise wait for it before every later LDS read, which is of the other buffer; m0 it sets itself before each use.  (A write of m0 needs one wait state before its use.)
__device__ __forceinline__ void to_lds(const char* from, unsigned offset, const char* lds) {
    const unsigned base = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)(const __attribute__((address_space(3))) char*)lds);
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(base), "v"(offset), "s"(from) : "memory");
}

// One operand's tile in LDS: R rows of C's side (m or n), KROW bytes of k.
//   k along memory: [R][8 pieces], piece p of row i at place p ^ (i >> 1 & 7)
//   k across memory: [KE][R * size / 16 pieces], piece p of row kk at place p ^ spread(kk)
template <class E, bool ACROSS, int R, int THREADS>
struct Tile {
    typedef typename E::type T;
    static constexpr int S = (int)sizeof(T), PE = 16 / S, KE = KROW / S, BYTES = R * KROW;
    static constexpr int ROWP = ACROSS ? R / PE : 8;        // pieces of an LDS row
    static constexpr int PIECES = BYTES / 16, TURNS = PIECES / THREADS;
    static_assert(PIECES % THREADS == 0, "a whole number of turns");

    __device__ static __forceinline__ int place(int row, int piece) {
        if constexpr (!ACROSS) return piece ^ ((row >> 1) & 7);
        else if constexpr (S == 2) return piece ^ (((row & 3) << 1 | (row & 8)) & (ROWP - 1));  // 32-byte columns of rows 8 q + 0..3 apart
        else return piece ^ ((row & 12) & (ROWP - 1));                                          // 64-byte columns of rows 4 q + j apart
    }

    // piece number `id` of the tile -> its row and logical piece (the lane's piece is fixed by the LDS place it fills)
    __device__ static __forceinline__ void where(int id, int& row, int& piece) {
        row = id / ROWP;
        piece = place(row, id % ROWP);  // (an involution)
    }

    // the tile's first element in memory (uniform), and the piece's bytes from there (the host has seen that they fit 32 bits); rows past the
    // end are clamped (their products are never stored)
    __device__ static __forceinline__ const char* origin(const void* base, int64_t ld, int64_t first, int64_t k0) {
        return (const char*)base + (ACROSS ? k0 * ld + first : first * ld + k0) * S;
    }
    __device__ static __forceinline__ unsigned offset(int64_t ld, int64_t first, int64_t rows, int id) {
        int row, piece;
        where(id, row, piece);
        const int64_t left = rows - first;  // (at least one row or piece)
        if constexpr (!ACROSS) return (unsigned)(((row < left ? row : left - 1) * ld + piece * PE) * S);
        else return (unsigned)((row * ld + (piece * PE < left ? piece * PE : left - PE)) * S);
    }

    // turn t of the tile from memory; WHOLE: k does not end in it, else `left` is k from its start on
    template <bool WHOLE>
    __device__ static __forceinline__ void stage(char* lds, const char* from, unsigned offset, int t, int64_t left) {
        const int wave = threadIdx.x >> 6;
        if constexpr (WHOLE) {
            to_lds(from, offset, lds + (t * THREADS + wave * 64) * 16);
        } else {
            int row, piece;
            where(t * THREADS + (int)threadIdx.x, row, piece);
            if ((ACROSS ? row : piece * PE) < left) to_lds(from, offset, lds + (t * THREADS + wave * 64) * 16);
            else *(u32x4*)(lds + (t * THREADS + (int)threadIdx.x) * 16) = u32x4{0, 0, 0, 0};
        }
    }

    // fragment of MFMA rows i0 .. i0 + 15 for step kk: 16 bytes per lane, lane l = 16 q + i: row i0 + i, piece 4 kk + q of its k
    __device__ static __forceinline__ u32x4 fragment(const char* lds, int i0, int kk, int lane) {
        const int i = lane & 15, q = lane >> 4;
        if constexpr (!ACROSS) {
            return *(const u32x4*)(lds + ((i0 + i) * 8 + place(i0 + i, kk * 4 + q)) * 16);
        } else if constexpr (S == 2) {
            // two transposing reads: of 16 lanes, lane s names row s / 4 of four rows of k and columns 4 (s % 4) .. + 3; lane i gets column i
            u32x4 f;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int row = kk * 32 + q * 8 + h * 4 + (i >> 2), col = i0 + 4 * (i & 3);
                const char* p = lds + (row * ROWP + place(row, col / PE)) * 16 + (col % PE) * S;
                const u32x2 v = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p));
                f[2 * h] = v[0];
                f[2 * h + 1] = v[1];
            }
            return f;
        } else {
            u32x4 f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int row = kk * 16 + q * 4 + j, col = i0 + i;
                f[j] = *(const unsigned*)(lds + (row * ROWP + place(row, col / PE)) * 16 + (col % PE) * S);
            }
            return f;
        }
    }
};

template <class E>
__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    if constexpr (E::code == GCP_TYPE_BF16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else if constexpr (E::code == GCP_TYPE_F16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else {
#pragma unroll
        for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[j]), __uint_as_float(b[j]), c, 0, 0, 0);
        return c;
    }
}

template <int N>
__device__ __forceinline__ void wait_loads_and_meet() {  // this wave's direct loads but the last N, and its LDS traffic; then all waves
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

template <int BM, int BN, int RING>
constexpr int ring_bytes() { return RING * (BM + BN) * KROW; }

// One tile of C: tile number `block` of the product, piece `piece` of k.
template <class E, bool AC, bool BC, int BM, int BN, int WM, int WN, int RING>
__device__ __forceinline__ void gemm_tile(const Gemm& g, int block, int piece, char* lds) {
    constexpr int THREADS = WM * WN * 64, TM = BM / WM / 16, TN = BN / WN / 16;
    typedef Tile<E, AC, BM, THREADS> TA;
    typedef Tile<E, BC, BN, THREADS> TB;
    constexpr int STAGE = TA::BYTES + TB::BYTES, LOADS = TA::TURNS + TB::TURNS;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = wave / WN, wn = wave % WN;

    const int total = g.tiles_m * g.tiles_n;
    int tm, tn;
    gcp_tile_of_block(block, total, g.tiles_m, g.tiles_n, tm, tn);
    const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BN;
    const int64_t k0 = (int64_t)piece * g.k_per, k1 = k0 + g.k_per < g.k ? k0 + g.k_per : g.k;
    const int steps = k1 > k0 ? (int)((k1 - k0 + TA::KE - 1) / TA::KE) : 0;
    const int whole = steps > 0 ? (int)((k1 - k0) / TA::KE) : 0;  // tiles that do not reach past the end of k

    const char *pa = TA::origin(g.a, g.a_ld, m0, k0), *pb = TB::origin(g.b, g.b_ld, n0, k0);
    unsigned oa[TA::TURNS], ob[TB::TURNS];
#pragma unroll
    for (int t = 0; t < TA::TURNS; ++t) oa[t] = TA::offset(g.a_ld, m0, g.a_rows, t * THREADS + tid);
#pragma unroll
    for (int t = 0; t < TB::TURNS; ++t) ob[t] = TB::offset(g.b_ld, n0, g.b_rows, t * THREADS + tid);
    const int64_t da = (AC ? g.a_ld * TA::KE : TA::KE) * TA::S, db = (BC ? g.b_ld * TB::KE : TB::KE) * TB::S;

    auto stage = [&](int step, char* buf) {
        if (step < whole) {
#pragma unroll
            for (int t = 0; t < TA::TURNS; ++t) TA::template stage<true>(buf, pa + step * da, oa[t], t, 0);
#pragma unroll
            for (int t = 0; t < TB::TURNS; ++t) TB::template stage<true>(buf + TA::BYTES, pb + step * db, ob[t], t, 0);
        } else {
            const int64_t left = k1 - k0 - (int64_t)step * TA::KE;
#pragma unroll
            for (int t = 0; t < TA::TURNS; ++t) TA::template stage<false>(buf, pa + step * da, oa[t], t, left);
#pragma unroll
            for (int t = 0; t < TB::TURNS; ++t) TB::template stage<false>(buf + TA::BYTES, pb + step * db, ob[t], t, left);
        }
    };

    f32x4 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    u32x4 fa[TM], fb[2][TN];
    auto read_b = [&](const char* buf, auto kk) {
#pragma unroll
        for (int j = 0; j < TN; ++j) fb[kk][j] = TB::fragment(buf + TA::BYTES, (wn * TN + j) * 16, kk, lane);
    };
    auto read_a = [&](const char* buf, int kk, int i) { fa[i] = TA::fragment(buf, (wm * TM + i) * 16, kk, lane); };
    // the products of step kk; meanwhile fragments of A for step `then` of buf and, between the rows of products, the direct loads of tile `ahead`
    auto multiply = [&](auto kk, const char* buf, int then, auto loads, int ahead, char* into) {
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int j = 0; j < TN; ++j) acc[i][j] = mfma<E>(fb[kk][j], fa[i], acc[i][j]);  // (transposed: a lane gets four n of one m)
            __builtin_amdgcn_sched_barrier(0);  // (not before: the registers are the products')
            read_a(buf, then, i);
            if constexpr (decltype(loads)::value) {
#pragma unroll
                for (int t = i * TA::TURNS / TM; t < (i + 1) * TA::TURNS / TM; ++t) TA::template stage<true>(into, pa + ahead * da, oa[t], t, 0);
#pragma unroll
                for (int t = i * TB::TURNS / TM; t < (i + 1) * TB::TURNS / TM; ++t) TB::template stage<true>(into + TA::BYTES, pb + ahead * db, ob[t], t, 0);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    std::integral_constant<int, 0> first;
    std::integral_constant<int, 1> second;
#pragma unroll 1
    for (int t = 0; t < RING && t < steps; ++t) stage(t, lds + t * STAGE);
    if (RING <= whole) wait_loads_and_meet<(RING - 1) * LOADS>();
    else wait_loads_and_meet<0>();
    char* buf = lds;
    read_b(buf, first);
#pragma unroll
    for (int i = 0; i < TM; ++i) read_a(buf, 0, i);
    auto turn = [&](int s, auto ahead) {  // ahead: the tile that follows the ring is whole
        char* next = buf + STAGE == lds + RING * STAGE ? lds : buf + STAGE;
        read_b(buf, second);
        multiply(first, buf, 1, std::false_type(), 0, nullptr);
        // everybody has all of this tile's fragments, and the next tile is there: those after it may still be under way
        if constexpr (decltype(ahead)::value) {
            wait_loads_and_meet<(RING - 2) * LOADS>();
        } else {
            if (s + RING <= whole) wait_loads_and_meet<(RING - 2) * LOADS>();
            else wait_loads_and_meet<0>();
        }
        read_b(next, first);  // (behind the last tile: what is there is read, and not used)
        if constexpr (!decltype(ahead)::value)
            if (s + RING < steps) stage(s + RING, buf);
        multiply(second, next, 0, ahead, s + RING, buf);
        buf = next;
    };
    int s = 0;
#pragma unroll 1
    for (; s + RING < whole; ++s) turn(s, std::true_type());
#pragma unroll 1
    for (; s < steps; ++s) turn(s, std::false_type());
    __syncthreads();  // (the epilogue writes over the ring)

    // A wave's part of C goes through its own LDS, PH rows at a time: [PH][COLS] fp32 in pieces of 16 bytes, piece p of row r at p ^ (r & mask)
    constexpr int COLS = TN * 16, P = COLS / 4, OWN = RING * STAGE / (WM * WN), ROWS = TM * 16;
    constexpr int PH = ROWS * COLS * 4 <= OWN ? ROWS : OWN / (COLS * 4) / 16 * 16;
    constexpr int V = E::vec, LPR = COLS / V, RPP = 64 / LPR;  // lanes per row, rows per pass
    constexpr int AT_ONCE = PH / RPP < 4 ? PH / RPP : 4;
    static_assert(PH >= 16 && ROWS % PH == 0 && PH % (RPP * AT_ONCE) == 0, "whole phases");
    f32x4* own = (f32x4*)(lds + wave * OWN);
    const int64_t n = n0 + wn * COLS + (lane % LPR) * V;
    const int count = g.n - n < V ? (int)(g.n - n) : V;
    float bias[V];
    bias_load<E, V>(g.e, n, count, bias);
#pragma unroll
    for (int ph = 0; ph < ROWS / PH; ++ph) {
        gcp_wave_lds_sync();  // (lanes exchange: what the phase before read has been read)
#pragma unroll
        for (int i = 0; i < PH / 16; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j) {
                const int r = i * 16 + (lane & 15);
                own[r * P + ((4 * j + (lane >> 4)) ^ (r & (P - 1)))] = acc[ph * (PH / 16) + i][j];
            }
        gcp_wave_lds_sync();
#pragma unroll 1
        for (int r0 = 0; r0 < PH; r0 += RPP * AT_ONCE) {
            // (the residual of several passes is requested before the first is finished)
            Raw<E, V> res[AT_ONCE];
            if (g.e.residual && !g.part)
#pragma unroll
                for (int u = 0; u < AT_ONCE; ++u) {
                    const int64_t m = m0 + wm * ROWS + ph * PH + r0 + u * RPP + lane / LPR;
                    if (m < g.m) res[u] = elem_load<E, V>(g.e.residual, m * g.e.r_ld + n, count);
                }
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u) {
                const int r = r0 + u * RPP + lane / LPR;
                const int64_t m = m0 + wm * ROWS + ph * PH + r;
                float v[V];
#pragma unroll
                for (int h = 0; h < V / 4; ++h) {
                    const f32x4 x = own[r * P + (((lane % LPR) * (V / 4) + h) ^ (r & (P - 1)))];
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[4 * h + j] = x[j];
                }
                if (m >= g.m || count <= 0) continue;
                if (g.part) {
#pragma unroll
                    for (int h = 0; h < V; h += 4) {
                        const float four[4] = {v[h], v[h + 1], v[h + 2], v[h + 3]};
                        elem_store<ElemF32, 4>(g.part, ((int64_t)piece * g.m + m) * g.n + n + h, four, count - h < 4 ? count - h : 4);
                    }
                } else {
                    finish<E, V>(g.e, m, n, g.n, count, bias, res[u], v);
                }
            }
        }
    }
}

template <class E, bool AC, bool BC, int BM, int BN, int WM, int WN, int RING>
__global__ __launch_bounds__(WM * WN * 64, 2) void gemm_kernel(Gemm g) {
    __shared__ __attribute__((aligned(16))) char lds[ring_bytes<BM, BN, RING>()];
    gemm_tile<E, AC, BC, BM, BN, WM, WN, RING>(g, (int)blockIdx.x, (int)blockIdx.y, lds);
}

// Both products of a backward in one launch: dx = dz W in the first workgroups, dW = dz^T x in the others, so that small ones run side by side.
template <class E, int BM, int BN, int WM, int WN, int RING>
__global__ __launch_bounds__(WM * WN * 64, 2) void gemm_pair_kernel(Gemm dx, Gemm dw) {
    __shared__ __attribute__((aligned(16))) char lds[ring_bytes<BM, BN, RING>()];
    const int tiles = dx.tiles_m * dx.tiles_n, first = tiles * dx.splits, block = (int)blockIdx.x;
    if (block < first) {
        gemm_tile<E, false, true, BM, BN, WM, WN, RING>(dx, block % tiles, block / tiles, lds);
    } else {
        const int other = dw.tiles_m * dw.tiles_n;
        gemm_tile<E, true, true, BM, BN, WM, WN, RING>(dw, (block - first) % other, (block - first) / other, lds);
    }
}

// The partial sums of a split product, added in order, and the epilogue.
template <class E>
__global__ __launch_bounds__(256) void join_kernel(const float* __restrict__ part, int splits, int64_t m, int64_t n, Epilogue e) {
    constexpr int V = E::vec;
    const int64_t vecs = (n + V - 1) / V, all = m * vecs, step = m * n;
    for (int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x; id < all; id += (int64_t)gridDim.x * 256) {
        const int64_t row = id / vecs, col = (id - row * vecs) * V;
        const int count = n - col < V ? (int)(n - col) : V;
        float v[V], bias[V];
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = 0.f;
        bias_load<E, V>(e, col, count, bias);
        Raw<E, V> res;
        if (e.residual) res = elem_load<E, V>(e.residual, row * e.r_ld + col, count);
#pragma unroll 4
        for (int s = 0; s < splits; ++s)
#pragma unroll
            for (int h = 0; h < V; h += 4) {
                const Raw<ElemF32, 4> x = elem_load<ElemF32, 4>(part, s * step + row * n + col + h, count - h < 4 ? count - h : 4);
#pragma unroll
                for (int j = 0; j < 4; ++j) v[h + j] += x[j];
            }
        finish<E, V>(e, row, col, n, count, bias, res, v);
    }
}

static_assert(GCP_FEW_ROWS == 32, "two forms of few_rows_kernel");
// Few rows (up to 16 MT): bound by the read of W, which goes from memory straight into the fragments of the matrix instructions, 512
// consecutive bytes of each of 16 rows per wave and turn (4 rows, 4096 -> 8192 bf16: 13.4 us, 5.0 TB/s).  A workgroup takes 16 columns of y,
// its eight waves take turns along k; their sums meet in LDS.  x comes from the caches.  Loads at any alignment: nothing is copied.
struct FewRows {
    int rows, k, n;
    const void *x, *w;
    int64_t x_ld, w_ld;
    Epilogue e;
};

template <class E, int MT>
__global__ __launch_bounds__(512) void few_rows_kernel(FewRows a) {
    typedef typename E::type T;
    constexpr int PE = 16 / (int)sizeof(T), U = 8, WAVES = 8, STEP = 4 * PE;  // k of one fragment
    __shared__ f32x4 part[WAVES][MT][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, q = lane >> 4;
    const int n0 = blockIdx.x * 16, row = n0 + i < a.n ? n0 + i : a.n - 1;  // (past the end: the last row again, not stored)
    const T* w = (const T*)a.w + row * a.w_ld + q * PE;
    const T* x[MT];
    f32x4 acc[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int m = t * 16 + i < a.rows ? t * 16 + i : a.rows - 1;
        x[t] = (const T*)a.x + m * a.x_ld + q * PE;
        acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    for (int k = wave * U * STEP; k < a.k; k += WAVES * U * STEP) {
        Raw<E, PE> fw[U];
        if (k + U * STEP <= a.k) {
#pragma unroll
            for (int u = 0; u < U; ++u) fw[u] = elem_load<E, PE>(w, k + u * STEP);
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int t = 0; t < MT; ++t) {
                    const Raw<E, PE> fx = elem_load<E, PE>(x[t], k + u * STEP);
                    acc[t] = mfma<E>(__builtin_bit_cast(u32x4, fw[u]), __builtin_bit_cast(u32x4, fx), acc[t]);
                }
        } else {
            for (int u = 0; u < U; ++u) {
                const int left = a.k - (k + u * STEP + q * PE), count = left < 0 ? 0 : left < PE ? left : PE;
                const Raw<E, PE> f = elem_load<E, PE>(w, k + u * STEP, count);
#pragma unroll
                for (int t = 0; t < MT; ++t) {
                    const Raw<E, PE> fx = elem_load<E, PE>(x[t], k + u * STEP, count);
                    acc[t] = mfma<E>(__builtin_bit_cast(u32x4, f), __builtin_bit_cast(u32x4, fx), acc[t]);
                }
            }
        }
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) part[wave][t][i * 4 + q] = acc[t];  // (a lane: columns 4 q .. + 3 of row i)
    __syncthreads();
    for (int id = threadIdx.x; id < MT * 256; id += 512) {
        const int t = id >> 8, r = id >> 4 & 15, c = id & 15, m = t * 16 + r, n = n0 + c;
        if (m >= a.rows || n >= a.n) continue;
        float v = 0.f;
#pragma unroll
        for (int y = 0; y < WAVES; ++y) v += ((const float*)part[y][t])[r * 16 + c];
        if (a.e.bias) v += (E::code != GCP_TYPE_F32 && a.e.bias_f32) ? ((const float*)a.e.bias)[n] : (float)((const T*)a.e.bias)[n];
        const int64_t at = (int64_t)m * a.n + n;
        if (a.e.z) ((T*)a.e.z)[at] = (T)elem_in_range<E>(v);
        float one[1] = {v}, none[1];
        elem_act<1, false>(a.e.act, a.e.slope, one, one, none);
        if (a.e.residual) one[0] += (float)((const T*)a.e.residual)[m * a.e.r_ld + n];
        ((T*)a.e.y)[at] = (T)one[0];
    }
}

// dz = dy act'(z) and the partial column sums of the unrounded dz.  dz is rounded to the rows' type, since the matrix pipe takes 16-bit operands, and z
// was stored in it, which halves its bytes (67 MB each way at 8192 x 4096).  Errors of dx and dW in bf16, SiLU: 1.66e-3 by the rounding of the
// results alone, 1.76e-3 with that of z, 2.35e-3 with that of dz, 2.42e-3 with both.
// Threads of a workgroup: TX over vectors of columns, 256 / TX over rows; the rows of a workgroup are every gridDim.y-th group of them.
struct DzArgs {
    int64_t rows;
    int n, tx, act;
    float slope;
    const void *z, *dy;
    int64_t dy_ld;
    void* dz;     // [rows, dz_ld] or NULL; dz_ld: n rounded up to whole pieces, which are filled up with zeros
    int dz_ld;
    float* part;  // [gridDim.y, n] or NULL
};

template <class E>
__global__ __launch_bounds__(256) void dz_kernel(DzArgs a) {
    constexpr int V = E::vec;
    __shared__ float cols[256 * V];
    const int tx = threadIdx.x % a.tx, ty = threadIdx.x / a.tx, TY = 256 / a.tx;
    const int64_t c = ((int64_t)blockIdx.x * a.tx + tx) * V;
    const int count = a.n - c < V ? (int)(a.n - c) : V;  // (0 or less: nothing to do)
    float sum[V];
#pragma unroll
    for (int j = 0; j < V; ++j) sum[j] = 0.f;
    const int64_t step = (int64_t)gridDim.y * TY;
    if (count > 0)
        for (int64_t r0 = (int64_t)blockIdx.y * TY + ty; r0 < a.rows; r0 += 4 * step) {  // four rows requested at a time
            Raw<E, V> dy[4], zr[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int64_t r = r0 + u * step;
                if (r >= a.rows) continue;
                dy[u] = elem_load<E, V>(a.dy, r * a.dy_ld + c, count);
                if (a.act != GCP_ACT_NONE) zr[u] = elem_load<E, V>(a.z, r * a.n + c, count);
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int64_t r = r0 + u * step;
                if (r >= a.rows) continue;
                float v[V];
#pragma unroll
                for (int j = 0; j < V; ++j) v[j] = dy[u][j];
                if (a.act != GCP_ACT_NONE) {
                    float z[V], act[V], d[V];
#pragma unroll
                    for (int j = 0; j < V; ++j) z[j] = zr[u][j];
                    elem_act<V, true>(a.act, a.slope, z, act, d);
#pragma unroll
                    for (int j = 0; j < V; ++j) v[j] = j < count ? v[j] * d[j] : 0.f;
                }
#pragma unroll
                for (int j = 0; j < V; ++j) sum[j] += v[j];
                if (a.dz) elem_store<E, V>(a.dz, r * a.dz_ld + c, v);  // (whole pieces: dz_ld is a multiple of them)
            }
        }
    if (!a.part) return;
#pragma unroll
    for (int j = 0; j < V; ++j) cols[threadIdx.x * V + j] = sum[j];
    __syncthreads();
    if (ty == 0 && count > 0) {
        for (int y = 1; y < TY; ++y)
#pragma unroll
            for (int j = 0; j < V; ++j) sum[j] += cols[(y * a.tx + tx) * V + j];
#pragma unroll
        for (int h = 0; h < V; h += 4) {
            const float four[4] = {sum[h], sum[h + 1], sum[h + 2], sum[h + 3]};
            elem_store<ElemF32, 4>(a.part, (int64_t)blockIdx.y * a.n + c + h, four, count - h < 4 ? count - h : 4);
        }
    }
}

template <class F>
int by_type(int type, F f) {
    if (type == GCP_TYPE_F32) return f(ElemF32());
    if (type == GCP_TYPE_BF16) return f(ElemBf16());
    return f(ElemF16());
}

// Copies of up to three matrices whose rows are not whole 16-byte pieces, filled up with zeros.  A workgroup takes rows in turn.
struct CopyArgs {
    const void* from[3];
    void* to[3];
    int64_t ld[3], rows[3];
    int cols[3], wide[3];
};
template <class E>
__global__ __launch_bounds__(256) void copy_kernel(CopyArgs a) {
    typedef typename E::type T;
    const int q = blockIdx.y;
    const T* from = (const T*)a.from[q];
    T* to = (T*)a.to[q];
    const int wide = a.wide[q], pieces = wide / E::vec;
    const int64_t all = a.rows[q] * pieces;
    for (int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x; id < all; id += (int64_t)gridDim.x * 256) {
        const int64_t r = id / pieces;
        const int c = (int)(id - r * pieces) * E::vec;
        const Raw<E, E::vec> x = elem_load<E, E::vec>(from, r * a.ld[q] + c, a.cols[q] - c < E::vec ? a.cols[q] - c : E::vec);
        __builtin_memcpy(to + r * wide + c, x.u, 16);
    }
}

// ---- host -------------------------------------------------------------------------------------------------------------------------
// A matrix as the products read it: rows of `cols` elements in whole 16-byte pieces (`wide` of them there to be read)
struct Mat { const void* p; int64_t ld, rows; int cols, wide; };

int wide_of(int cols, int size) { return gcp_round_up(cols, 16 / size); }
bool in_pieces(const void* p, int64_t ld, int cols, int size) {
    // (a stride so long that the offsets within a tile of 256 rows pass 32 bits is shortened by the copy, too)
    return aligned16(p) && ld % (16 / size) == 0 && cols % (16 / size) == 0 && ld < (int64_t)1 << 21;
}
int64_t copy_floats(int64_t rows, int cols, int size) { return (rows * wide_of(cols, size) * size + 15) / 16 * 4; }

// Gives every matrix that needs it a copy in `space`, which moves on behind them.
template <class E>
int put_in_pieces(Mat* const* mats, int n, float*& space, hipStream_t stream) {
    constexpr int size = (int)sizeof(typename E::type);
    CopyArgs a = {};
    int count = 0;
    int64_t most = 0;
    for (int i = 0; i < n; ++i) {
        Mat& x = *mats[i];
        x.wide = x.cols;
        if (x.rows == 0 || in_pieces(x.p, x.ld, x.cols, size)) continue;
        if (!space) return GCPNET_E_BADARG;
        a.from[count] = x.p; a.ld[count] = x.ld; a.rows[count] = x.rows; a.cols[count] = x.cols;
        x.wide = wide_of(x.cols, size);
        x.p = space; x.ld = x.wide;
        a.to[count] = space; a.wide[count++] = x.wide;
        space += copy_floats(x.rows, x.cols, size);
        const int64_t blocks = (x.rows * (x.wide / E::vec) + 255) / 256;
        most = blocks > most ? blocks : most;
    }
    if (!count) return 0;
    hipLaunchKernelGGL(HIP_KERNEL_NAME(copy_kernel<E>), dim3((unsigned)(most < 2048 ? most : 2048), (unsigned)count), dim3(256), 0, stream, a);
    GCP_HIP_CHECK_LAUNCH();
    return 0;
}

// A longer ring hides more of the memory's latency, a shorter one lets more workgroups reside: few of them take the longer (2048^3 bf16, 256
// tiles of 128: 23.3 us with three, 26.4 with two; 500 x 4096 x 4096, 512 tiles of 64: 30.7 us with four, 36.0 with two; 3000 x 500 x 2001,
// 384 tiles of 128: 25.9 us with three, 22.9 with two; 2048^3 in 1024 tiles of 64: 35.0 with four, 27.2 with two).
int form_of(int shape, int64_t groups) { return shape == 0 ? (groups <= 512 ? 0 : 1) : shape == 1 ? (groups <= 256 ? 2 : 3) : 4; }

template <class F>
void by_form(int form, F f) {
#define FORM(bm, wn, ring) f(std::integral_constant<int, bm>(), std::integral_constant<int, wn>(), std::integral_constant<int, ring>())
    switch (form) {
        case 0: FORM(64, 2, 4); break;
        case 1: FORM(64, 2, 2); break;
        case 2: FORM(128, 4, 3); break;
        case 3: FORM(128, 4, 2); break;
        default: FORM(256, 4, 2);
    }
#undef FORM
}

// Workgroups of one product: two products of one launch at 512 threads stay below the 2^32 that a launch can have.
constexpr int64_t MAX_GROUPS = (1 << 22) - 1;

// C[m][n] = sum_k A[m][k] B[n][k] with the epilogue; A and B in pieces, as [m][k] and [n][k] or, across, [k][m] and [k][n].
template <class E>
int describe(Gemm& g, int& shape, int64_t m, int64_t n, int64_t k, const Mat& a, bool a_across, const Mat& b, bool b_across, const Epilogue& e, float*& ws) {
    const GcpLinearPlan plan = gcp_linear_plan(m, n, k, (int)sizeof(typename E::type));
    if (plan.tiles_m * plan.splits > MAX_GROUPS / plan.tiles_n) return GCPNET_E_UNSUPPORTED;
    if (plan.splits > 1 && !ws) return GCPNET_E_BADARG;
    shape = plan.shape;
    g = {};
    g.m = m; g.n = n; g.k = k;
    g.a = a.p; g.a_ld = a.ld; g.b = b.p; g.b_ld = b.ld;
    g.a_rows = a_across ? a.wide : m;
    g.b_rows = b_across ? b.wide : n;
    g.tiles_m = (int)plan.tiles_m; g.tiles_n = (int)plan.tiles_n; g.splits = plan.splits; g.k_per = plan.k_per;
    if (plan.splits > 1) {
        g.part = ws;
        ws += (plan.floats + 3) / 4 * 4;
    }
    g.e = e;
    return 0;
}

template <class E>
int join(const Gemm& g, hipStream_t stream) {
    if (g.splits == 1) return 0;
    const int64_t vecs = g.m * ((g.n + E::vec - 1) / E::vec), blocks = (vecs + 255) / 256;
    hipLaunchKernelGGL(HIP_KERNEL_NAME(join_kernel<E>), dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(256), 0, stream, g.part, g.splits, g.m, g.n, g.e);
    GCP_HIP_CHECK_LAUNCH();
    return 0;
}

template <class E, bool AC, bool BC>
int launch(const Gemm& g, int shape, hipStream_t stream) {
    const dim3 grid((unsigned)(g.tiles_m * g.tiles_n), (unsigned)g.splits);
    by_form(form_of(shape, (int64_t)grid.x * grid.y), [&](auto b, auto wn, auto ring) {
        constexpr int B = b.value, WN = wn.value;
        if constexpr (B < 256 || E::code != GCP_TYPE_F32)
            hipLaunchKernelGGL(HIP_KERNEL_NAME(gemm_kernel<E, AC, BC, B, B, 2, WN, ring.value>), grid, dim3(128 * WN), 0, stream, g);
    });
    GCP_HIP_CHECK_LAUNCH();
    return join<E>(g, stream);
}

constexpr int DZ_GROUPS = 512;

int check_desc(const gcp_linear_t* l) {
    if (!l || l->rows < 0 || l->k < 1 || l->n < 1 || !elem_type_ok(l->type) || l->act < 0 || l->act > GCP_ACT_SIGMOID) return GCPNET_E_BADARG;
    if (l->bias_type != GCP_TYPE_F32 && l->bias_type != l->type) return GCPNET_E_BADARG;
    if (l->rows > 0 && (!l->x || l->x_ld < 0)) return GCPNET_E_BADARG;
    if (!l->w || l->w_ld < 0) return GCPNET_E_BADARG;
    if (l->rows > INT32_MAX || l->k >= 1 << 21 || l->n >= 1 << 21) return GCPNET_E_UNSUPPORTED;
    return 0;
}

int64_t larger(int64_t a, int64_t b) { return a > b ? a : b; }

}  // namespace

extern "C" int64_t gcpnet_linear_act_workspace(const gcp_linear_t* l, int backward) {
    if (int rc = check_desc(l)) return rc;
    const int size = elem_bytes(l->type);
    const int64_t rows = l->rows;
    int64_t copies = 0;
    if (!backward && rows <= GCP_FEW_ROWS) return 0;
    if (rows > 0 && !in_pieces(l->x, l->x_ld, l->k, size)) copies += copy_floats(rows, l->k, size);
    if (rows > 0 && !in_pieces(l->w, l->w_ld, l->k, size)) copies += copy_floats(l->n, l->k, size);
    if (!backward) return copies + (gcp_linear_plan(rows, l->n, l->k, size).floats + 3) / 4 * 4;
    copies += copy_floats(rows, l->n, size);  // dz, or a copy of dy
    const int64_t parts = (gcp_linear_plan(rows, l->k, l->n, size).floats + 3) / 4 * 4 + (gcp_linear_plan(l->n, l->k, rows, size).floats + 3) / 4 * 4;
    return copies + larger(parts, (int64_t)DZ_GROUPS * l->n);
}

extern "C" int gcpnet_linear_act_forward(const gcp_linear_t* l, const void* residual, int64_t r_ld, void* y, void* z, float* workspace, void* stream) {
    if (int rc = check_desc(l)) return rc;
    if (l->rows == 0) return 0;
    if (!y || r_ld < 0 || !aligned16(workspace)) return GCPNET_E_BADARG;
    Epilogue e = {};
    e.bias = l->bias; e.bias_f32 = l->bias_type == GCP_TYPE_F32;
    e.residual = residual; e.r_ld = r_ld;
    e.act = l->act; e.slope = l->slope;
    e.y = y; e.z = z;
    return by_type(l->type, [&](auto t) {
        typedef decltype(t) E;
        if (l->rows <= GCP_FEW_ROWS) {
            const FewRows f = {(int)l->rows, l->k, l->n, l->x, l->w, l->x_ld, l->w_ld, e};
            const dim3 grid((unsigned)gcp_cdiv(l->n, 16));
            if (l->rows <= 16) hipLaunchKernelGGL(HIP_KERNEL_NAME(few_rows_kernel<E, 1>), grid, dim3(512), 0, (hipStream_t)stream, f);
            else hipLaunchKernelGGL(HIP_KERNEL_NAME(few_rows_kernel<E, 2>), grid, dim3(512), 0, (hipStream_t)stream, f);
            GCP_HIP_CHECK_LAUNCH();
            return 0;
        }
        Mat x = {l->x, l->x_ld, l->rows, l->k, 0}, w = {l->w, l->w_ld, l->n, l->k, 0};
        Mat* const both[2] = {&x, &w};
        if (int rc = put_in_pieces<E>(both, 2, workspace, (hipStream_t)stream)) return rc;
        Gemm g;
        int shape;
        if (int rc = describe<E>(g, shape, l->rows, l->n, l->k, x, false, w, false, e, workspace)) return rc;
        return launch<E, false, false>(g, shape, (hipStream_t)stream);
    });
}

extern "C" int gcpnet_linear_act_backward(const gcp_linear_t* l, const void* z, const void* dy, int64_t dy_ld, void* dx, void* dw, void* db,
                                          float* workspace, void* stream) {
    if (int rc = check_desc(l)) return rc;
    const bool act = l->act != GCP_ACT_NONE;
    if (dy_ld < 0 || (l->rows > 0 && (!dy || (act && !z))) || !aligned16(workspace)) return GCPNET_E_BADARG;
    if ((db || (act && l->rows > 0)) && !workspace) return GCPNET_E_BADARG;
    const int size = elem_bytes(l->type);
    const hipStream_t st = (hipStream_t)stream;
    return by_type(l->type, [&](auto t) {
        typedef decltype(t) E;
        Mat x = {l->x, l->x_ld, l->rows, l->k, 0}, w = {l->w, l->w_ld, l->n, l->k, 0}, g = {dy, dy_ld, l->rows, l->n, 0};
        Mat* mats[3];
        int count = 0;
        if (dw) mats[count++] = &x;
        if (dx && l->rows > 0) mats[count++] = &w;
        if (!act && (dw || dx)) mats[count++] = &g;
        if (int rc = put_in_pieces<E>(mats, count, workspace, st)) return rc;
        if (db || (act && l->rows > 0 && (dw || dx))) {
            DzArgs a = {};
            a.rows = l->rows; a.n = l->n; a.act = l->act; a.slope = l->slope;
            a.z = z; a.dy = dy; a.dy_ld = dy_ld;
            a.dz_ld = wide_of(l->n, size);
            if (act && (dw || dx)) {
                a.dz = workspace;
                g.p = workspace; g.ld = g.wide = a.dz_ld;
                workspace += copy_floats(l->rows, l->n, size);
            }
            a.part = db ? workspace : nullptr;
            const int64_t across = a.dz_ld / E::vec;
            a.tx = 8;
            while (a.tx < 256 && a.tx < across) a.tx *= 2;
            const int64_t bx = (across + a.tx - 1) / a.tx, ty = 256 / a.tx;
            // (four workgroups per CU in all; a thread takes four rows or more before there are more groups of rows)
            int64_t by = (l->rows + 4 * ty - 1) / (4 * ty), most = (1024 + bx - 1) / bx;
            by = by < most ? by : most;
            by = by < DZ_GROUPS ? by : DZ_GROUPS;
            if (by > 0) {
                hipLaunchKernelGGL(HIP_KERNEL_NAME(dz_kernel<E>), dim3((unsigned)bx, (unsigned)by), dim3(256), 0, st, a);
                GCP_HIP_CHECK_LAUNCH();
            }
            if (db)
                if (const int rc = gcp_column_sums(workspace, (int)by, 1, l->n, &db, &l->bias_type, st)) return rc;
        }
        Epilogue e = {};
        Gemm one, two;
        int shape1 = -1, shape2 = -1;
        if (dx && l->rows > 0) {
            e.y = dx;
            if (int rc = describe<E>(one, shape1, l->rows, l->k, l->n, g, false, w, true, e, workspace)) return rc;
        }
        if (dw) {
            e.y = dw;
            if (int rc = describe<E>(two, shape2, l->n, l->k, l->rows, g, true, x, true, e, workspace)) return rc;
        }
        if (shape1 >= 0 && shape1 == shape2 && shape1 < 2) {  // (the largest tiles fill the chip one product at a time)
            const int64_t groups = (int64_t)one.tiles_m * one.tiles_n * one.splits + (int64_t)two.tiles_m * two.tiles_n * two.splits;
            by_form(form_of(shape1, groups), [&](auto b, auto wn, auto ring) {
                constexpr int B = b.value, WN = wn.value;
                if constexpr (B < 256)
                    hipLaunchKernelGGL(HIP_KERNEL_NAME(gemm_pair_kernel<E, B, B, 2, WN, ring.value>), dim3((unsigned)groups), dim3(128 * WN), 0, st, one, two);
            });
            GCP_HIP_CHECK_LAUNCH();
            if (int rc = join<E>(one, st)) return rc;
            return join<E>(two, st);
        }
        if (shape1 >= 0)
            if (int rc = launch<E, false, true>(one, shape1, st)) return rc;
        if (shape2 >= 0) return launch<E, true, true>(two, shape2, st);
        return 0;
    });
}
