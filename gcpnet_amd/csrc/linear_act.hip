// y = act(x W^T + b) + r and its backward for fp32, bf16 and fp16, every length and stride.
//
//   z = x W^T + b;  y = act(z) + r;     dz = dy act'(z);  dx = dz W;  dW = dz^T x;  db = column sums of dz;  dr = dy
//
// All three products are C[m][n] = sum_k A[m][k] B[n][k] with operands whose k runs along memory or across it (W in dx; dz and x in
// dW), in one kernel template:
//   * a workgroup owns a BM x BN tile of C, a wave a part of it in 16 x 16 MFMA tiles (16-bit: v_mfma_f32_16x16x32, fp32:
//     v_mfma_f32_16x16x4_f32; sums in fp32);
//   * tiles of 128 bytes of k travel from memory into one of two LDS buffers by direct loads (no registers), one tile ahead of the
//     products; the 16-byte pieces of an LDS row are permuted (by the row) so that fragment reads spread over the banks;
//   * an operand with k across memory keeps its layout in LDS, [k][m]; 16-bit fragments come out of it through the transposing LDS
//     read, fp32 ones element by element;
//   * operands whose rows do not start at multiples of 16 bytes, and the tile in which k ends, go through registers element by element
//     into the same places, zeros where there is no data;
//   * few tiles of C: k is split over workgroups, which leave fp32 partial sums for a second launch that adds them in a fixed order and
//     applies the epilogue (no atomics: results repeat bit for bit).
// The epilogue adds the bias, applies the activation, adds the residual and rounds once; in training it also stores z.
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
    int act, bias_f32, whole;  // whole: four columns at a time (all rows of y, z, residual allow it)
    float slope;
    void *y, *z;  // contiguous [m, n]
};

struct Gemm {
    int64_t m, n, k;
    const void *a, *b;
    int64_t a_ld, b_ld;
    int a_fast, b_fast;  // 16-byte pieces
    int tiles_m, tiles_n, splits;
    int64_t k_per;       // k per split, a multiple of the tile's
    float* part;         // [splits, m, n] or NULL
    Epilogue e;
};

template <class E>
__device__ __forceinline__ void epilogue4(const Epilogue& e, int64_t m, int64_t n, int64_t N, f32x4 v) {
    typedef typename E::type T;
    const int64_t at = m * N + n;
    float out[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) out[j] = v[j];
    const int cols = N - n < 4 ? (int)(N - n) : 4;
    if (e.bias) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j < cols) out[j] += (E::code != GCP_TYPE_F32 && e.bias_f32) ? ((const float*)e.bias)[n + j] : (float)((const T*)e.bias)[n + j];
    }
    typedef T T4 __attribute__((ext_vector_type(4)));
    if (e.z) {
        if (e.whole) {
            T4 q;
#pragma unroll
            for (int j = 0; j < 4; ++j) q[j] = (T)out[j];
            *(T4*)((T*)e.z + at) = q;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (j < cols) ((T*)e.z)[at + j] = (T)out[j];
        }
    }
    if (e.act != GCP_ACT_NONE) {
#pragma unroll
        for (int j = 0; j < 4; ++j) out[j] = gcp_act(e.act, out[j], e.slope);
    }
    if (e.whole) {
        if (e.residual) {
            const T4 r = *(const T4*)((const T*)e.residual + m * e.r_ld + n);
#pragma unroll
            for (int j = 0; j < 4; ++j) out[j] += (float)r[j];
        }
        T4 q;
#pragma unroll
        for (int j = 0; j < 4; ++j) q[j] = (T)out[j];
        *(T4*)((T*)e.y + at) = q;
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j < cols) {
                if (e.residual) out[j] += (float)((const T*)e.residual)[m * e.r_ld + n + j];
                ((T*)e.y)[at + j] = (T)out[j];
            }
    }
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

    // address of the piece in memory at k = 0 of the tile; rows past the end are clamped (their products are never stored)
    __device__ static __forceinline__ const char* address(const void* base, int64_t ld, int64_t first, int64_t rows, int64_t k0, int id) {
        int row, piece;
        where(id, row, piece);
        if constexpr (!ACROSS) {
            int64_t i = first + row;
            i = i < rows ? i : rows - 1;
            return (const char*)base + (i * ld + k0 + piece * PE) * S;
        } else {
            int64_t i = first + piece * PE;
            i = i < rows ? i : rows - PE;
            return (const char*)base + ((k0 + row) * ld + i) * S;
        }
    }

    // element by element through registers: any address, any end
    __device__ static void slow(char* lds, const void* base, int64_t ld, int64_t first, int64_t rows, int64_t k0, int64_t k_end) {
#pragma unroll 1
        for (int t = 0; t < TURNS; ++t) {
            const int id = t * THREADS + (int)threadIdx.x;
            int row, piece;
            where(id, row, piece);
            T x[PE];
#pragma unroll
            for (int j = 0; j < PE; ++j) {
                const int64_t i = ACROSS ? first + piece * PE + j : first + row, k = ACROSS ? k0 + row : k0 + piece * PE + j;
                x[j] = i < rows && k < k_end ? ((const T*)base)[ACROSS ? k * ld + i : i * ld + k] : (T)0.f;
            }
            u32x4 q;
            __builtin_memcpy(&q, x, 16);
            *(u32x4*)(lds + id * 16) = q;
        }
    }

    // fragment of MFMA rows i0 .. i0 + 15 and k step `kk` (64 bytes of k each): 16 bytes per lane, lane l = 16 q + i: row i0 + i,
    // k = (4 kk + q) pieces
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

// 16 bytes per lane from memory to LDS (lane l to base + 16 l, the base uniform), counted by vmcnt.  In asm, because the compiler would
// otherwise wait for it before every later LDS read, which is of the other buffer; m0 it sets itself before each use.  (A write of m0 needs one wait state before its use.)
__device__ __forceinline__ void to_lds(const char* from, const char* lds) {
    const unsigned base = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)(const __attribute__((address_space(3))) char*)lds);
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(base), "v"(from) : "memory");
}

template <class E, bool AC, bool BC, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(WM * WN * 64) void gemm_kernel(Gemm g) {
    constexpr int THREADS = WM * WN * 64, TM = BM / WM / 16, TN = BN / WN / 16;
    typedef Tile<E, AC, BM, THREADS> TA;
    typedef Tile<E, BC, BN, THREADS> TB;
    __shared__ __attribute__((aligned(16))) char lds[2][TA::BYTES + TB::BYTES];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = wave / WN, wn = wave % WN;

    const int total = g.tiles_m * g.tiles_n;
    int tm, tn;
    gcp_tile_of_block((int)blockIdx.x, total, g.tiles_m, g.tiles_n, tm, tn);
    const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BN;
    const int64_t k0 = (int64_t)blockIdx.y * g.k_per, k1 = k0 + g.k_per < g.k ? k0 + g.k_per : g.k;
    const int steps = k1 > k0 ? (int)((k1 - k0 + TA::KE - 1) / TA::KE) : 0;

    const char *pa[TA::TURNS], *pb[TB::TURNS];
    if (g.a_fast)
#pragma unroll
        for (int t = 0; t < TA::TURNS; ++t) pa[t] = TA::address(g.a, g.a_ld, m0, g.m, k0, t * THREADS + tid);
    if (g.b_fast)
#pragma unroll
        for (int t = 0; t < TB::TURNS; ++t) pb[t] = TB::address(g.b, g.b_ld, n0, g.n, k0, t * THREADS + tid);
    const int64_t da = (AC ? g.a_ld * TA::KE : TA::KE) * TA::S, db = (BC ? g.b_ld * TB::KE : TB::KE) * TB::S;

    auto stage = [&](int step, char* buf) {
        const int64_t k = k0 + (int64_t)step * TA::KE;
        const bool full = k + TA::KE <= k1;
        if (g.a_fast && full) {
#pragma unroll
            for (int t = 0; t < TA::TURNS; ++t) { to_lds(pa[t], buf + (t * THREADS + wave * 64) * 16); pa[t] += da; }
        } else {
            TA::slow(buf, g.a, g.a_ld, m0, g.m, k, k1);
        }
        buf += TA::BYTES;
        if (g.b_fast && full) {
#pragma unroll
            for (int t = 0; t < TB::TURNS; ++t) { to_lds(pb[t], buf + (t * THREADS + wave * 64) * 16); pb[t] += db; }
        } else {
            TB::slow(buf, g.b, g.b_ld, n0, g.n, k, k1);
        }
    };

    f32x4 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    if (steps > 0) stage(0, lds[0]);
    for (int s = 0; s < steps; ++s) {
        // this tile has landed, everywhere; nobody reads the other buffer any more
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (s + 1 < steps) stage(s + 1, lds[(s + 1) & 1]);
        const char *la = lds[s & 1], *lb = la + TA::BYTES;
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            u32x4 fa[TM], fb[TN];
#pragma unroll
            for (int j = 0; j < TN; ++j) fb[j] = TB::fragment(lb, (wn * TN + j) * 16, kk, lane);
#pragma unroll
            for (int i = 0; i < TM; ++i) fa[i] = TA::fragment(la, (wm * TM + i) * 16, kk, lane);
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j) acc[i][j] = mfma<E>(fb[j], fa[i], acc[i][j]);  // (transposed: a lane gets four n of one m)
        }
    }

    const int q = lane >> 4;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
        const int64_t m = m0 + (wm * TM + i) * 16 + (lane & 15);
        if (m >= g.m) continue;
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            const int64_t n = n0 + (wn * TN + j) * 16 + 4 * q;
            if (n >= g.n) continue;
            if (g.part) {
                float* p = g.part + ((int64_t)blockIdx.y * g.m + m) * g.n + n;
                if (g.n % 4 == 0) *(f32x4*)p = acc[i][j];
                else
#pragma unroll
                    for (int c = 0; c < 4; ++c)
                        if (n + c < g.n) p[c] = acc[i][j][c];
            } else {
                epilogue4<E>(g.e, m, n, g.n, acc[i][j]);
            }
        }
    }
}

// The partial sums of a split product, added in order, and the epilogue.
template <class E>
__global__ __launch_bounds__(256) void join_kernel(const float* __restrict__ part, int splits, int64_t m, int64_t n, Epilogue e) {
    const int64_t quads = (n + 3) / 4, all = m * quads;
    for (int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x; id < all; id += (int64_t)gridDim.x * 256) {
        const int64_t row = id / quads, col = (id - row * quads) * 4;
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
        const float* p = part + row * n + col;
        if (n % 4 == 0) {
#pragma unroll 4
            for (int s = 0; s < splits; ++s) v += *(const f32x4*)(p + (int64_t)s * m * n);
        } else {
            for (int s = 0; s < splits; ++s)
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (col + c < n) v[c] += p[(int64_t)s * m * n + c];
        }
        epilogue4<E>(e, row, col, n, v);
    }
}

// dz = dy act'(z) (rounded to the rows' type: the matrix pipe takes 16-bit operands) and the partial column sums of the unrounded dz.
// Threads of a workgroup: TX over vectors of columns, 256 / TX over rows; the rows of a workgroup are every gridDim.y-th group of them.
struct DzArgs {
    int64_t rows;
    int n, tx, act;
    float slope;
    const void *z, *dy;
    int64_t dy_ld;
    void* dz;     // [rows, n] or NULL
    float* part;  // [gridDim.y, n] or NULL
};

template <class E, int V>
__global__ __launch_bounds__(256) void dz_kernel(DzArgs a) {
    __shared__ float cols[256 * V];
    const int tx = threadIdx.x % a.tx, ty = threadIdx.x / a.tx, TY = 256 / a.tx;
    const int64_t c = ((int64_t)blockIdx.x * a.tx + tx) * V;
    const bool in = c < a.n;
    float sum[V];
#pragma unroll
    for (int j = 0; j < V; ++j) sum[j] = 0.f;
    if (in) {
#pragma unroll 4
        for (int64_t r = (int64_t)blockIdx.y * TY + ty; r < a.rows; r += (int64_t)gridDim.y * TY) {
            const Raw<E, V> dy = elem_load<E, V>(a.dy, r * a.dy_ld + c);
            float v[V];
            if (a.act != GCP_ACT_NONE) {
                const Raw<E, V> z = elem_load<E, V>(a.z, r * a.n + c);
#pragma unroll
                for (int j = 0; j < V; ++j) v[j] = (float)dy.x[j] * gcp_act_grad(a.act, (float)z.x[j], a.slope);
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j) v[j] = (float)dy.x[j];
            }
#pragma unroll
            for (int j = 0; j < V; ++j) sum[j] += v[j];
            if (a.dz) elem_store<E, V>(a.dz, r * a.n + c, v);
        }
    }
    if (!a.part) return;
#pragma unroll
    for (int j = 0; j < V; ++j) cols[threadIdx.x * V + j] = sum[j];
    __syncthreads();
    if (ty == 0 && in) {
        for (int y = 1; y < TY; ++y)
#pragma unroll
            for (int j = 0; j < V; ++j) sum[j] += cols[(y * a.tx + tx) * V + j];
#pragma unroll
        for (int j = 0; j < V; ++j) a.part[(int64_t)blockIdx.y * a.n + c + j] = sum[j];
    }
}

template <class F>
int by_type(int type, F f) {
    if (type == GCP_TYPE_F32) return f(ElemF32());
    if (type == GCP_TYPE_BF16) return f(ElemBf16());
    return f(ElemF16());
}

// ---- host -------------------------------------------------------------------------------------------------------------------------
struct Operand_ { const void* p; int64_t ld; bool across; };

bool pieces_ok(const Operand_& o, int64_t rows, int size) {
    const int pe = 16 / size;
    return aligned16(o.p) && o.ld % pe == 0 && (!o.across || rows % pe == 0);
}

template <class E, bool AC, bool BC>
int launch_tiles(const Gemm& g, int shape, hipStream_t stream) {
    const dim3 grid((unsigned)(g.tiles_m * g.tiles_n), (unsigned)g.splits);
    switch (shape) {
        case 0: hipLaunchKernelGGL(HIP_KERNEL_NAME(gemm_kernel<E, AC, BC, 64, 64, 2, 2>), grid, dim3(256), 0, stream, g); break;
        case 1: hipLaunchKernelGGL(HIP_KERNEL_NAME(gemm_kernel<E, AC, BC, 128, 128, 2, 2>), grid, dim3(256), 0, stream, g); break;
        default: hipLaunchKernelGGL(HIP_KERNEL_NAME(gemm_kernel<E, AC, BC, 256, 256, 2, 4>), grid, dim3(512), 0, stream, g); break;
    }
    GCP_HIP_CHECK_LAUNCH();
    return 0;
}

// C = A B^T with the epilogue.  ws: gcp_linear_plan(m, n, k, size).floats of workspace.
template <class E>
int product(int64_t m, int64_t n, int64_t k, Operand_ a, Operand_ b, const Epilogue& e, float* ws, hipStream_t stream) {
    const GcpLinearPlan plan = gcp_linear_plan(m, n, k, (int)sizeof(typename E::type));
    if (plan.tiles_m > INT32_MAX / plan.tiles_n) return GCPNET_E_UNSUPPORTED;
    if (plan.splits > 1 && !ws) return GCPNET_E_BADARG;
    Gemm g = {};
    g.m = m; g.n = n; g.k = k;
    g.a = a.p; g.a_ld = a.ld; g.b = b.p; g.b_ld = b.ld;
    g.a_fast = pieces_ok(a, m, (int)sizeof(typename E::type));
    g.b_fast = pieces_ok(b, n, (int)sizeof(typename E::type));
    g.tiles_m = (int)plan.tiles_m; g.tiles_n = (int)plan.tiles_n; g.splits = plan.splits; g.k_per = plan.k_per;
    g.part = plan.splits > 1 ? ws : nullptr;
    g.e = e;
    int rc;
    if (!a.across && !b.across) rc = launch_tiles<E, false, false>(g, plan.shape, stream);
    else if (!a.across) rc = launch_tiles<E, false, true>(g, plan.shape, stream);
    else rc = launch_tiles<E, true, true>(g, plan.shape, stream);
    if (rc || plan.splits == 1) return rc;
    const int64_t quads = m * ((n + 3) / 4), blocks = (quads + 255) / 256;
    hipLaunchKernelGGL(HIP_KERNEL_NAME(join_kernel<E>), dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(256), 0, stream, g.part, plan.splits, m, n, e);
    GCP_HIP_CHECK_LAUNCH();
    return 0;
}

bool quads_ok(const void* p, int64_t ld, int size) { return ((uintptr_t)p & (4 * size - 1)) == 0 && ld % 4 == 0; }

constexpr int DZ_GROUPS = 256;

int check_desc(const gcp_linear_t* l) {
    if (!l || l->rows < 0 || l->k < 1 || l->n < 1 || !elem_type_ok(l->type) || l->act < 0 || l->act > GCP_ACT_SIGMOID) return GCPNET_E_BADARG;
    if (l->bias_type != GCP_TYPE_F32 && l->bias_type != l->type) return GCPNET_E_BADARG;
    if (l->rows > 0 && (!l->x || l->x_ld < 0)) return GCPNET_E_BADARG;
    if (!l->w || l->w_ld < 0) return GCPNET_E_BADARG;
    if (l->rows > INT32_MAX) return GCPNET_E_UNSUPPORTED;
    return 0;
}

}  // namespace

extern "C" int64_t gcpnet_linear_act_workspace(int64_t rows, int k, int n, int type, int backward) {
    if (rows < 0 || k < 1 || n < 1 || !elem_type_ok(type)) return GCPNET_E_BADARG;
    const int size = elem_bytes(type);
    if (!backward) return gcp_linear_plan(rows, n, k, size).floats;
    const int64_t a = gcp_linear_plan(rows, k, n, size).floats, b = gcp_linear_plan(n, k, rows, size).floats, c = (int64_t)DZ_GROUPS * n;
    return a > b ? (a > c ? a : c) : (b > c ? b : c);
}

extern "C" int gcpnet_linear_act_forward(const gcp_linear_t* l, const void* residual, int64_t r_ld, void* y, void* z, float* workspace, void* stream) {
    if (int rc = check_desc(l)) return rc;
    if (l->rows == 0) return 0;
    if (!y || r_ld < 0) return GCPNET_E_BADARG;
    const int size = elem_bytes(l->type);
    Epilogue e = {};
    e.bias = l->bias; e.bias_f32 = l->bias_type == GCP_TYPE_F32;
    e.residual = residual; e.r_ld = r_ld;
    e.act = l->act; e.slope = l->slope;
    e.y = y; e.z = z;
    e.whole = l->n % 4 == 0 && quads_ok(y, l->n, size) && quads_ok(z, l->n, size) && quads_ok(residual, r_ld, size);
    return by_type(l->type, [&](auto t) {
        return product<decltype(t)>(l->rows, l->n, l->k, {l->x, l->x_ld, false}, {l->w, l->w_ld, false}, e, workspace, (hipStream_t)stream);
    });
}

extern "C" int gcpnet_linear_act_backward(const gcp_linear_t* l, const void* z, const void* dy, int64_t dy_ld, void* dz, void* dx, void* dw, void* db,
                                          float* workspace, void* stream) {
    if (int rc = check_desc(l)) return rc;
    const bool act = l->act != GCP_ACT_NONE;
    if (dy_ld < 0 || (l->rows > 0 && (!dy || (act && (!z || !dz))))) return GCPNET_E_BADARG;
    const int size = elem_bytes(l->type);
    const hipStream_t st = (hipStream_t)stream;
    const void* g = dy;  // the gradient of z
    int64_t g_ld = dy_ld;
    if (db || (act && l->rows > 0)) {
        if (db && !workspace) return GCPNET_E_BADARG;
        DzArgs a = {};
        a.rows = l->rows; a.n = l->n; a.act = l->act; a.slope = l->slope;
        a.z = z; a.dy = dy; a.dy_ld = dy_ld; a.dz = act ? dz : nullptr;
        a.part = db ? workspace : nullptr;
        const int v = 16 / size;
        const bool vec = l->n % v == 0 && dy_ld % v == 0 && aligned16(dy) && (!act || (aligned16(z) && aligned16(dz)));
        const int64_t across = vec ? l->n / v : l->n;
        a.tx = 8;
        while (a.tx < 256 && a.tx < across) a.tx *= 2;
        const int64_t bx = (across + a.tx - 1) / a.tx, ty = 256 / a.tx;
        // (two workgroups per CU in all; a thread takes eight rows or more before there are more groups of rows)
        int64_t by = (l->rows + 8 * ty - 1) / (8 * ty), most = (512 + bx - 1) / bx;
        by = by < most ? by : most;
        by = by < DZ_GROUPS ? by : DZ_GROUPS;
        if (by > 0) {
            const int rc = by_type(l->type, [&](auto t) {
                typedef decltype(t) E;
                if (vec) hipLaunchKernelGGL(HIP_KERNEL_NAME(dz_kernel<E, E::vec>), dim3((unsigned)bx, (unsigned)by), dim3(256), 0, st, a);
                else hipLaunchKernelGGL(HIP_KERNEL_NAME(dz_kernel<E, 1>), dim3((unsigned)bx, (unsigned)by), dim3(256), 0, st, a);
                GCP_HIP_CHECK_LAUNCH();
                return 0;
            });
            if (rc) return rc;
        }
        if (db)
            if (const int rc = gcp_column_sums(workspace, (int)by, 1, l->n, &db, &l->bias_type, st)) return rc;
        if (act) { g = dz; g_ld = l->n; }
    }
    return by_type(l->type, [&](auto t) {
        typedef decltype(t) E;
        Epilogue e = {};
        if (dx && l->rows > 0) {
            e.y = dx;
            e.whole = l->k % 4 == 0 && quads_ok(dx, l->k, size);
            if (int rc = product<E>(l->rows, l->k, l->n, {g, g_ld, false}, {l->w, l->w_ld, true}, e, workspace, st)) return rc;
        }
        if (dw) {
            e.y = dw;
            e.whole = l->k % 4 == 0 && quads_ok(dw, l->k, size);
            if (int rc = product<E>(l->n, l->k, l->rows, {g, g_ld, true}, {l->x, l->x_ld, true}, e, workspace, st)) return rc;
        }
        return 0;
    });
}
