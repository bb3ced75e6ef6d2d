// AdamW over many parameter tensors at once, moments in fp32 or in 8 bits, optional clipping by the global gradient norm.
//
//   g' = c g,  c = min(1, max_norm / (|g| + 1e-6));   m = b1 m + (1 - b1) g';   v = b2 v + (1 - b2) g'^2
//   p  = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// Bound: HBM.  Per element the step moves 28 B (fp32, fp32 moments), 16 B (fp32, 8-bit moments), 30 / 18 B (bf16 parameters: gradient
// and parameter 2 B each way, master copy 4 B each way): 10^8 elements take 532 us in the first form (5.26 TB/s) and, bf16 with 8-bit
// moments, 340 - 350 us (5.2 TB/s).  A wave owns 256 consecutive elements at a time, four per lane, so every
// load and store is one contiguous piece per wave and the scale of 256 8-bit moments is one wave reduction; a workgroup owns a chunk
// of 4096 elements, loads all of it before it computes, and finds its tensor by bisection in the launch arguments, so tensors of any
// mixture of sizes fill the chip.
#include <math.h>

#include <type_traits>

#include "common.h"

namespace {

typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x2v __attribute__((ext_vector_type(2)));

constexpr int CHUNK = 4096, QBLOCK = 256, ITER = CHUNK / (4 * QBLOCK);  // four waves x ITER blocks of 256
constexpr int NORM_CHUNK = 16384;
constexpr int64_t MAX_CHUNKS = (1 << 24) - 1;  // workgroups of 256 threads in a launch, which has less than 2^32 of them
constexpr int MAX_BEGIN = 448, MAX_NORM = 200;  // tensors per launch of the kernels before the update

// A tensor as the update takes it: no more than its kind needs, so that a launch takes as many as its arguments hold.
struct Plain { void *param; const void* grad; void *exp_avg, *exp_avg_sq; int64_t n_vec; };  // n_vec: 2 n + (16-byte accesses)
struct Master { float* master; };
struct Scales { float *exp_avg_scale, *exp_avg_sq_scale; uint32_t ordinal, unused; };
struct Nothing1 {};
struct Nothing2 {};
template <bool BF16, bool EIGHT>
struct Slot : Plain, std::conditional_t<BF16, Master, Nothing1>, std::conditional_t<EIGHT, Scales, Nothing2> {};

template <bool BF16, bool EIGHT>
struct StepArgs {
    static constexpr int MOST = (4096 - 64) / (int)(sizeof(Slot<BF16, EIGHT>) + sizeof(int));
    Slot<BF16, EIGHT> t[MOST];
    int first[MOST + 1];   // first chunk of each tensor
    const float* corr;     // {lr / (1 - b1^t), 1 / sqrt(1 - b2^t), t, -} of each tensor
    const float* clip;     // {norm, coefficient} or NULL
    int n;
    float b1, c1, b2, c2, eps, keep;  // c = 1 - b, keep = 1 - lr wd
    unsigned seed;
};
static_assert(sizeof(StepArgs<false, false>) <= 4096 && sizeof(StepArgs<true, true>) <= 4096, "kernel arguments");

// A bijection of 32 bits whose output bits depend evenly on the input bits: two rounds of xor-shift and multiply, with the constants that
// C. Wellons published for it (a search for the least bias, 2018).
__device__ __forceinline__ unsigned mix32(unsigned h) {
    h ^= h >> 16;
    h *= 0x7feb352du;
    h ^= h >> 15;
    h *= 0x846ca68bu;
    return h ^ (h >> 16);
}

// two values as bf16, nearest even (NaN stays NaN), the first in the low half
__device__ __forceinline__ unsigned bf16_pair(float a, float b) {
    typedef __bf16 pair __attribute__((ext_vector_type(2)));
    const pair p = {(__bf16)a, (__bf16)b};
    return __builtin_bit_cast(unsigned, p);
}

__device__ __forceinline__ bool finite_f(float x) { return (__float_as_uint(x) & 0x7fffffffu) < 0x7f800000u; }

// The power of two that takes `top` (>= 0, finite) into (224, 448], the end of e4m3's range: 2^(E - 8) for a mantissa up to 1.75,
// else 2^(E - 7); at least the smallest normal number, whose inverse is finite.  A power of two, so that a block whose largest
// element drifts keeps its grid of codes (and the scaling is exact).
__device__ __forceinline__ float block_scale(float top) {
    int e = (int)((__float_as_uint(top) + 0x1fffffu) >> 23) - 8;
    return __uint_as_float((unsigned)(e < 1 ? 1 : e) << 23);
}
__device__ __forceinline__ float pow2_inverse(float s) { return __uint_as_float(0x7f000000u - __float_as_uint(s)); }

// y in [0, 448] to a value of e4m3, rounded up with the probability of its place between the two neighbours (20 random bits r), never
// to 0 from above 0.  Rounding v to nearest would freeze it: a step changes v by at most 1 - b2 (0.1 %) of itself downwards, which
// never reaches half the distance of two codes (3 - 6 %); at random its expectation moves as it should.
__device__ __forceinline__ float e4m3_stochastic(float y, unsigned r) {
    const float whole = __uint_as_float((__float_as_uint(y) + r) & 0xfff00000u);
    float small = floorf(y * 512.f + (float)r * 0x1p-20f) * 0x1p-9f;
    if (y > 0.f && small == 0.f) small = 0x1p-9f;
    return y >= 0x1p-6f ? whole : small;
}

// The largest of the wave's values, in scalar registers: within rows of 16 lanes, then from row to row.
__device__ __forceinline__ unsigned wave_max(unsigned x) {
#define STEP(ctrl, rows) { const unsigned y = (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, ctrl, rows, 0xf, false); x = y > x ? y : x; }
    STEP(0x111, 0xf) STEP(0x112, 0xf) STEP(0x114, 0xf) STEP(0x118, 0xf)  // from 1, 2, 4, 8 lanes below
    STEP(0x142, 0xa) STEP(0x143, 0xc)                                    // row 0 to 1 and 2 to 3; rows 0 - 1 to 2 - 3
#undef STEP
    return (unsigned)__builtin_amdgcn_readlane((int)x, 63);
}

// sqrt and quotient of the parameter's update by the hardware's root and reciprocal, each good to a unit in the last place (the root takes
// no subnormal numbers: those are scaled).  With the full-precision forms an 8-bit step is bound by arithmetic, not by memory.
__device__ __forceinline__ float quick_sqrt(float v) {
    const bool low = v < 0x1p-96f;
    const float r = __builtin_amdgcn_sqrtf(low ? v * 0x1p64f : v);
    return low ? r * 0x1p-32f : r;
}

// four values of a wave's piece: whole vectors where the tensor's addresses allow them, else element by element, absent ones 0
template <bool VEC>
__device__ __forceinline__ f32x4 load_f32(const float* p, int64_t i, int64_t n) {
    if constexpr (VEC) return *(const f32x4*)(p + i);
    f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (i + j < n) x[j] = p[i + j];
    return x;
}
template <bool VEC>
__device__ __forceinline__ u32x2 load_u16x4(const unsigned short* p, int64_t i, int64_t n) {
    if constexpr (VEC) return *(const u32x2*)(p + i);
    u32x2 x = {0u, 0u};
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (i + j < n) x[j / 2] |= (unsigned)p[i + j] << (16 * (j & 1));
    return x;
}
__device__ __forceinline__ float bf16_of(u32x2 x, int j) { return __uint_as_float(j & 1 ? x[j / 2] & 0xffff0000u : x[j / 2] << 16); }
template <bool VEC>
__device__ __forceinline__ unsigned load_u8x4(const unsigned char* p, int64_t i, int64_t n) {
    if constexpr (VEC) return *(const unsigned*)(p + i);
    unsigned u = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (i + j < n) u |= (unsigned)p[i + j] << (8 * j);
    return u;
}
template <bool VEC>
__device__ __forceinline__ void store_f32(float* p, int64_t i, int64_t n, f32x4 x) {
    if constexpr (VEC) { *(f32x4*)(p + i) = x; return; }
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (i + j < n) p[i + j] = x[j];
}
template <bool VEC>
__device__ __forceinline__ void store_u16x4(unsigned short* p, int64_t i, int64_t n, u32x2 x) {
    if constexpr (VEC) { *(u32x2*)(p + i) = x; return; }
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (i + j < n) p[i + j] = (unsigned short)(x[j / 2] >> (16 * (j & 1)));
}
template <bool VEC>
__device__ __forceinline__ void store_u8x4(unsigned char* p, int64_t i, int64_t n, unsigned u) {
    if constexpr (VEC) { *(unsigned*)(p + i) = u; return; }
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (i + j < n) p[i + j] = (unsigned char)(u >> (8 * j));
}

__device__ __forceinline__ f32x4 e4m3_decode(unsigned u) {
    const f32x2v lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)u, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)u, true);
    return f32x4{lo[0], lo[1], hi[0], hi[1]};
}
__device__ __forceinline__ unsigned e4m3_encode(f32x4 x) {  // nearest even; |x| <= 448
    int u = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], u, true);
}
// codes of values that may be infinite or NaN: those become the code of NaN
__device__ __forceinline__ unsigned nan_codes(unsigned codes, f32x4 x) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (!finite_f(x[j])) codes |= 0x7fu << (8 * j);
    return codes;
}

struct Piece {  // one wave's 256 elements as loaded, four per lane
    f32x4 p, g, m, v;  // (p: the master copy of a bf16 parameter)
    u32x2 hp, hg;      // a bf16 parameter and its gradient
    unsigned mc, vc;
    float ms, vs;
};

template <bool BF16, bool EIGHT, bool VEC>
__device__ __forceinline__ void piece_load(const gcp_adamw_tensor_t& T, int64_t i, Piece& q) {
    if constexpr (BF16) {
        q.hp = load_u16x4<VEC>((const unsigned short*)T.param, i, T.n);
        q.hg = load_u16x4<VEC>((const unsigned short*)T.grad, i, T.n);
        q.p = load_f32<VEC>(T.master, i, T.n);
    } else {
        q.p = load_f32<VEC>((const float*)T.param, i, T.n);
        q.g = load_f32<VEC>((const float*)T.grad, i, T.n);
    }
    if constexpr (EIGHT) {
        q.mc = load_u8x4<VEC>((const unsigned char*)T.exp_avg, i, T.n);
        q.vc = load_u8x4<VEC>((const unsigned char*)T.exp_avg_sq, i, T.n);
        q.ms = T.exp_avg_scale[i / QBLOCK];
        q.vs = T.exp_avg_sq_scale[i / QBLOCK];
    } else {
        q.m = load_f32<VEC>((const float*)T.exp_avg, i, T.n);
        q.v = load_f32<VEC>((const float*)T.exp_avg_sq, i, T.n);
    }
}

template <bool BF16, bool EIGHT, bool VEC>
__device__ __forceinline__ void piece_update(const StepArgs<BF16, EIGHT>& a, const gcp_adamw_tensor_t& T, int64_t i, Piece& q, float clip, float lr1,
                                             float root2, unsigned key) {
    // (products and sums of the moments rounded one by one: the codes of 8-bit moments are then the same wherever they are computed)
#pragma clang fp contract(off)
    if constexpr (EIGHT) {
        q.m = e4m3_decode(q.mc);
        q.v = e4m3_decode(q.vc);
    }
    f32x4 p = q.p;
    if constexpr (BF16) {
        // a parameter that is not the rounding of its master copy was written by somebody else: it is taken as it is
        const u32x2 diff = {bf16_pair(p[0], p[1]) ^ q.hp[0], bf16_pair(p[2], p[3]) ^ q.hp[1]};
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if ((j & 1 ? diff[j / 2] >> 16 : diff[j / 2] & 0xffffu) != 0) p[j] = bf16_of(q.hp, j);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float g = (BF16 ? bf16_of(q.hg, j) : q.g[j]) * clip;
        if constexpr (EIGHT) {
            q.m[j] *= q.ms;
            q.v[j] *= q.vs;
        }
        q.m[j] = q.m[j] * a.b1 + g * a.c1;
        q.v[j] = q.v[j] * a.b2 + (g * a.c2) * g;
        p[j] = p[j] * a.keep - lr1 * (q.m[j] * __builtin_amdgcn_rcpf(quick_sqrt(q.v[j]) * root2 + a.eps));
    }
    if constexpr (BF16) {
        store_u16x4<VEC>((unsigned short*)T.param, i, T.n, u32x2{bf16_pair(p[0], p[1]), bf16_pair(p[2], p[3])});
        store_f32<VEC>(T.master, i, T.n, p);
    } else {
        store_f32<VEC>((float*)T.param, i, T.n, p);
    }
    if constexpr (EIGHT) {
        unsigned tm = 0, tv = 0;  // (magnitudes as whole numbers, which order like them; absent elements are 0)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const unsigned um = __float_as_uint(q.m[j]) & 0x7fffffffu, uv = __float_as_uint(q.v[j]) & 0x7fffffffu;
            tm = um > tm ? um : tm;
            tv = uv > tv ? uv : tv;
        }
        tm = wave_max(tm);
        tv = wave_max(tv);
        const bool all_finite = tm < 0x7f800000u && tv < 0x7f800000u;
        if (!all_finite) {  // infinities and NaN get the code of NaN and do not count for the scale
            unsigned fm = 0, fv = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const unsigned um = __float_as_uint(q.m[j]) & 0x7fffffffu, uv = __float_as_uint(q.v[j]) & 0x7fffffffu;
                if (um < 0x7f800000u && um > fm) fm = um;
                if (uv < 0x7f800000u && uv > fv) fv = uv;
            }
            tm = wave_max(fm);
            tv = wave_max(fv);
        }
        const float ms = block_scale(__uint_as_float(tm)), vs = block_scale(__uint_as_float(tv));
        const float mi = pow2_inverse(ms), vi = pow2_inverse(vs);
        f32x4 ym, yv;
        const unsigned k = i >> 32 ? mix32(key ^ mix32((unsigned)(i >> 32))) : key;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            ym[j] = q.m[j] * mi;
            yv[j] = e4m3_stochastic(q.v[j] * vi, mix32(k + (unsigned)i + j) & 0xfffffu);
        }
        unsigned cm, cv;
        if (all_finite) {
            cm = e4m3_encode(ym);
            cv = e4m3_encode(yv);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (!finite_f(q.m[j])) ym[j] = 0.f;
                if (!finite_f(q.v[j])) yv[j] = 0.f;
            }
            cm = nan_codes(e4m3_encode(ym), q.m);
            cv = nan_codes(e4m3_encode(yv), q.v);
        }
        store_u8x4<VEC>((unsigned char*)T.exp_avg, i, T.n, cm);
        store_u8x4<VEC>((unsigned char*)T.exp_avg_sq, i, T.n, cv);
        if ((threadIdx.x & 63) == 0) {
            T.exp_avg_scale[i / QBLOCK] = ms;
            T.exp_avg_sq_scale[i / QBLOCK] = vs;
        }
    } else {
        store_f32<VEC>((float*)T.exp_avg, i, T.n, q.m);
        store_f32<VEC>((float*)T.exp_avg_sq, i, T.n, q.v);
    }
}

template <bool BF16, bool EIGHT>
__global__ __launch_bounds__(256) void adamw_kernel(StepArgs<BF16, EIGHT> a) {
    int lo = 0, hi = a.n - 1;  // the tensor of this chunk
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (a.first[mid] <= (int)blockIdx.x) lo = mid; else hi = mid - 1;
    }
    const Slot<BF16, EIGHT>& slot = a.t[lo];
    gcp_adamw_tensor_t T;
    T.param = slot.param; T.grad = slot.grad; T.exp_avg = slot.exp_avg; T.exp_avg_sq = slot.exp_avg_sq;
    T.n = slot.n_vec >> 1;
    const bool vec = slot.n_vec & 1;
    if constexpr (BF16) T.master = slot.master;
    if constexpr (EIGHT) { T.exp_avg_scale = slot.exp_avg_scale; T.exp_avg_sq_scale = slot.exp_avg_sq_scale; }
    const int64_t at = (int64_t)((int)blockIdx.x - a.first[lo]) * CHUNK;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const float clip = a.clip ? a.clip[1] : 1.f, lr1 = a.corr[4 * lo], root2 = a.corr[4 * lo + 1];
    unsigned key = 0;
    if constexpr (EIGHT) key = mix32(mix32(a.seed + 0x9e3779b9u * slot.ordinal) ^ (unsigned)(int)a.corr[4 * lo + 2]);
    Piece q[ITER];
#pragma unroll
    for (int k = 0; k < ITER; ++k) {  // (uniform over a wave: a whole piece, the end of the tensor, or nothing)
        const int64_t b = at + (k * 4 + wave) * QBLOCK;
        if (vec && b + QBLOCK <= T.n) piece_load<BF16, EIGHT, true>(T, b + 4 * lane, q[k]);
        else if (b < T.n) piece_load<BF16, EIGHT, false>(T, b + 4 * lane, q[k]);
    }
#pragma unroll
    for (int k = 0; k < ITER; ++k) {
        const int64_t b = at + (k * 4 + wave) * QBLOCK;
        if (vec && b + QBLOCK <= T.n) piece_update<BF16, EIGHT, true>(a, T, b + 4 * lane, q[k], clip, lr1, root2, key);
        else if (b < T.n) piece_update<BF16, EIGHT, false>(a, T, b + 4 * lane, q[k], clip, lr1, root2, key);
    }
}

// Before the update: the step counts of up to MAX_BEGIN tensors advance in device memory (so that a captured step counts on),
// their bias corrections are formed in double, and the partial sums of the squared gradients become the norm and the coefficient.
struct BeginArgs {
    float* step[MAX_BEGIN];
    int n;
    float* corr;
    double lr, b1, b2;
    const float* part;
    int64_t n_part;
    float max_norm;
    float* clip;
};
static_assert(sizeof(BeginArgs) <= 4096, "kernel arguments");

__global__ __launch_bounds__(512) void adamw_begin_kernel(BeginArgs a) {
    for (int i = threadIdx.x; i < a.n; i += 512) {
        const float t = *a.step[i] + 1.f;
        *a.step[i] = t;
        a.corr[4 * i] = (float)(a.lr / (1.0 - pow(a.b1, (double)t)));
        a.corr[4 * i + 1] = (float)(1.0 / sqrt(1.0 - pow(a.b2, (double)t)));
        a.corr[4 * i + 2] = t;
    }
    if (!a.part) return;
    __shared__ double sums[512];
    double s = 0.0;
    for (int64_t i = threadIdx.x; i < a.n_part; i += 512) s += (double)a.part[i];
    sums[threadIdx.x] = s;
    __syncthreads();
    for (int d = 256; d; d >>= 1) {
        if ((int)threadIdx.x < d) sums[threadIdx.x] += sums[threadIdx.x + d];
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        const float norm = (float)sqrt(sums[0]);
        const float c = a.max_norm / (norm + 1e-6f);
        a.clip[0] = norm;
        a.clip[1] = c > 1.f ? 1.f : c;  // (NaN stays)
    }
}

// One partial sum of squares for every 16384 elements, in an order that does not depend on the launch.
struct NormArgs {
    const void* grad[MAX_NORM];
    int64_t n[MAX_NORM];
    int first[MAX_NORM + 1];
    int count, bf16;
    float* part;
};
static_assert(sizeof(NormArgs) <= 4096, "kernel arguments");

template <bool BF16, bool VEC>
__device__ __forceinline__ float square_sum(const void* g, int64_t at, int64_t n) {
    float s = 0.f;
#pragma unroll 8
    for (int k = 0; k < NORM_CHUNK / 1024; ++k) {
        const int64_t i = at + k * 1024 + 4 * (int)threadIdx.x;
        f32x4 x;
        if constexpr (BF16) {
            const u32x2 h = load_u16x4<VEC>((const unsigned short*)g, i, n);
            x = f32x4{bf16_of(h, 0), bf16_of(h, 1), bf16_of(h, 2), bf16_of(h, 3)};
        } else {
            x = load_f32<VEC>((const float*)g, i, n);
        }
        s += (x[0] * x[0] + x[1] * x[1]) + (x[2] * x[2] + x[3] * x[3]);
    }
    return s;
}

template <bool BF16>
__global__ __launch_bounds__(256) void grad_norm_kernel(NormArgs a) {
    int lo = 0, hi = a.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (a.first[mid] <= (int)blockIdx.x) lo = mid; else hi = mid - 1;
    }
    const int64_t at = (int64_t)((int)blockIdx.x - a.first[lo]) * NORM_CHUNK, n = a.n[lo];
    const bool vec = ((uintptr_t)a.grad[lo] & (BF16 ? 7 : 15)) == 0 && at + NORM_CHUNK <= n;
    float s = vec ? square_sum<BF16, true>(a.grad[lo], at, n) : square_sum<BF16, false>(a.grad[lo], at, n);
    __shared__ float sums[4];
#pragma unroll
    for (int d = 32; d; d >>= 1) s += __shfl_xor(s, d);
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) a.part[blockIdx.x] = (sums[0] + sums[1]) + (sums[2] + sums[3]);
}

bool aligned(const void* p, unsigned b) { return ((uintptr_t)p & (b - 1)) == 0; }

struct Options { double lr, beta1, beta2, eps, weight_decay; uint32_t seed; };

template <bool BF16, bool EIGHT>
int launch_steps(int n, const gcp_adamw_tensor_t* t, const Options& o, const float* corrections, const float* clip, hipStream_t stream) {
    for (int k = 0; k < n;) {
        StepArgs<BF16, EIGHT> a;
        a.n = 0;
        const int k0 = k;
        int64_t c = 0;
        for (; k < n && a.n < a.MOST; ++k) {
            const int64_t more = (t[k].n + CHUNK - 1) / CHUNK;
            if (more > MAX_CHUNKS) return GCPNET_E_UNSUPPORTED;
            if (c + more > MAX_CHUNKS) break;
            Slot<BF16, EIGHT>& s = a.t[a.n];
            s.param = t[k].param; s.grad = t[k].grad; s.exp_avg = t[k].exp_avg; s.exp_avg_sq = t[k].exp_avg_sq;
            const unsigned w = BF16 ? 8 : 16, q = EIGHT ? 4 : 16;
            const bool vec = aligned(t[k].param, w) && aligned(t[k].grad, w) && aligned(t[k].exp_avg, q) && aligned(t[k].exp_avg_sq, q) &&
                             (!BF16 || aligned(t[k].master, 16));
            s.n_vec = 2 * t[k].n + (vec ? 1 : 0);
            if constexpr (BF16) s.master = t[k].master;
            if constexpr (EIGHT) { s.exp_avg_scale = t[k].exp_avg_scale; s.exp_avg_sq_scale = t[k].exp_avg_sq_scale; s.ordinal = t[k].ordinal; s.unused = 0; }
            a.first[a.n++] = (int)c;
            c += more;
        }
        a.first[a.n] = (int)c;
        if (!c) continue;
        a.corr = corrections + 4 * (int64_t)k0;
        a.clip = clip;
        a.b1 = (float)o.beta1; a.c1 = (float)(1.0 - o.beta1);
        a.b2 = (float)o.beta2; a.c2 = (float)(1.0 - o.beta2);
        a.eps = (float)o.eps; a.keep = (float)(1.0 - o.lr * o.weight_decay);
        a.seed = o.seed;
        hipLaunchKernelGGL(HIP_KERNEL_NAME(adamw_kernel<BF16, EIGHT>), dim3((unsigned)c), dim3(256), 0, stream, a);
        GCP_HIP_CHECK_LAUNCH();
    }
    return 0;
}

}  // namespace

extern "C" int64_t gcpnet_grad_norm_partials(int n, const gcp_adamw_tensor_t* t) {
    if (n < 0 || (n > 0 && !t)) return GCPNET_E_BADARG;
    int64_t c = 0;
    for (int k = 0; k < n; ++k) {
        if (t[k].n < 0) return GCPNET_E_BADARG;
        c += (t[k].n + NORM_CHUNK - 1) / NORM_CHUNK;
    }
    return c;
}

extern "C" int gcpnet_grad_norm(int n, const gcp_adamw_tensor_t* t, int type, float* partials, void* stream) {
    if (n < 0 || (n > 0 && (!t || !partials)) || (type != GCP_TYPE_F32 && type != GCP_TYPE_BF16)) return GCPNET_E_BADARG;
    for (int k = 0; k < n; ++k)
        if (t[k].n < 0 || (t[k].n > 0 && !t[k].grad)) return GCPNET_E_BADARG;
    for (int k = 0; k < n;) {
        NormArgs a;
        int64_t c = 0;
        a.count = 0;
        for (; k < n && a.count < MAX_NORM; ++k) {
            if (t[k].n == 0) continue;
            const int64_t more = (t[k].n + NORM_CHUNK - 1) / NORM_CHUNK;
            if (more > MAX_CHUNKS) return GCPNET_E_UNSUPPORTED;
            if (c + more > MAX_CHUNKS) break;
            a.grad[a.count] = t[k].grad;
            a.n[a.count] = t[k].n;
            a.first[a.count++] = (int)c;
            c += more;
        }
        if (!c) continue;
        a.part = partials;
        if (type == GCP_TYPE_BF16) hipLaunchKernelGGL(grad_norm_kernel<true>, dim3((unsigned)c), dim3(256), 0, (hipStream_t)stream, a);
        else hipLaunchKernelGGL(grad_norm_kernel<false>, dim3((unsigned)c), dim3(256), 0, (hipStream_t)stream, a);
        GCP_HIP_CHECK_LAUNCH();
        partials += c;
    }
    return 0;
}

extern "C" int gcpnet_adamw_begin(int n, const gcp_adamw_tensor_t* t, double lr, double beta1, double beta2, float* corrections,
                                  const float* partials, int64_t n_partials, float max_norm, float* clip, void* stream) {
    if (n < 0 || (n > 0 && (!t || !corrections)) || (partials && !clip) || n_partials < 0) return GCPNET_E_BADARG;
    for (int k = 0; k < n; ++k)
        if (!t[k].step) return GCPNET_E_BADARG;
    for (int k = 0; k < n || (k == 0 && partials); k += MAX_BEGIN) {
        BeginArgs a = {};
        a.n = n - k < MAX_BEGIN ? n - k : MAX_BEGIN;
        for (int j = 0; j < a.n; ++j) a.step[j] = t[k + j].step;
        a.corr = corrections + 4 * (int64_t)k;
        a.lr = lr; a.b1 = beta1; a.b2 = beta2;
        a.part = k == 0 ? partials : nullptr;
        a.n_part = n_partials; a.max_norm = max_norm; a.clip = clip;
        hipLaunchKernelGGL(adamw_begin_kernel, dim3(1), dim3(512), 0, (hipStream_t)stream, a);
        GCP_HIP_CHECK_LAUNCH();
    }
    return 0;
}

extern "C" int gcpnet_adamw_step(int n, const gcp_adamw_tensor_t* t, int type, int state_bits, double lr, double beta1, double beta2,
                                 double eps, double weight_decay, const float* corrections, const float* clip, uint32_t seed, void* stream) {
    if (n < 0 || (n > 0 && (!t || !corrections)) || (type != GCP_TYPE_F32 && type != GCP_TYPE_BF16) || (state_bits != 8 && state_bits != 32))
        return GCPNET_E_BADARG;
    const bool half = type == GCP_TYPE_BF16, eight = state_bits == 8;
    for (int k = 0; k < n; ++k) {
        if (t[k].n < 0 || !t[k].step) return GCPNET_E_BADARG;
        if (t[k].n > 0 && (!t[k].param || !t[k].grad || !t[k].exp_avg || !t[k].exp_avg_sq || (half && !t[k].master) ||
                           (eight && (!t[k].exp_avg_scale || !t[k].exp_avg_sq_scale))))
            return GCPNET_E_BADARG;
    }
    const Options o = {lr, beta1, beta2, eps, weight_decay, seed};
    if (half) return eight ? launch_steps<true, true>(n, t, o, corrections, clip, (hipStream_t)stream) : launch_steps<true, false>(n, t, o, corrections, clip, (hipStream_t)stream);
    return eight ? launch_steps<false, true>(n, t, o, corrections, clip, (hipStream_t)stream) : launch_steps<false, false>(n, t, o, corrections, clip, (hipStream_t)stream);
}
