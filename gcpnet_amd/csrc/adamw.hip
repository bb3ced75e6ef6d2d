// AdamW over many parameter tensors at once, moments in fp32 or in 8 bits, optional clipping by the global gradient norm.
//
//   g' = c g,  c = min(1, max_norm / (|g| + 1e-6));   m = b1 m + (1 - b1) g';   v = b2 v + (1 - b2) g'^2
//   p  = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// Bound: HBM.  Per element the step moves 28 B (fp32, fp32 moments), 16 B (fp32, 8-bit moments), 30 / 18 B (bf16 parameters: gradient
// and parameter 2 B each way, master copy 4 B each way).  A wave owns 256 consecutive elements at a time, four per lane, so every
// load and store is one contiguous piece per wave and the scale of 256 8-bit moments is one wave reduction; a workgroup owns a chunk
// of 4096 elements, loads all of it before it computes, and finds its tensor by bisection in the launch arguments, so tensors of any
// mixture of sizes fill the chip.
#include <math.h>

#include "common.h"

namespace {

typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4v __attribute__((ext_vector_type(4)));
typedef float f32x2v __attribute__((ext_vector_type(2)));

constexpr int CHUNK = 4096, QBLOCK = 256, ITER = CHUNK / (4 * QBLOCK);  // four waves x ITER blocks of 256
constexpr int NORM_CHUNK = 16384;

struct StepArgs {
    gcp_adamw_tensor_t t[GCP_ADAMW_MAX_TENSORS];
    int first[GCP_ADAMW_MAX_TENSORS + 1];  // first chunk of each tensor
    const float* corr;                     // {lr / (1 - b1^t), sqrt(1 - b2^t)} of each tensor
    const float* clip;                     // {norm, coefficient} or NULL
    int n;
    float b1, c1, b2, c2, eps, keep;       // c = 1 - b, keep = 1 - lr wd
    unsigned seed;
};
static_assert(sizeof(StepArgs) <= 4096, "kernel arguments");

__device__ __forceinline__ unsigned mix32(unsigned h) {
    h ^= h >> 16;
    h *= 0x7feb352du;
    h ^= h >> 15;
    h *= 0x846ca68bu;
    return h ^ (h >> 16);
}

__device__ __forceinline__ float bf16_to_f(unsigned b) { return __uint_as_float(b << 16); }
__device__ __forceinline__ unsigned f_to_bf16(float x) {  // nearest even; NaN stays NaN
    const unsigned u = __float_as_uint(x);
    if ((u & 0x7fffffffu) > 0x7f800000u) return (u >> 16) | 0x40u;
    return (u + 0x7fffu + ((u >> 16) & 1u)) >> 16;
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

__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
    for (int d = 32; d; d >>= 1) x = fmaxf(x, __shfl_xor(x, d));
    return x;
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
__device__ __forceinline__ f32x4 load_bf16(const unsigned short* p, int64_t i, int64_t n) {
    f32x4 x = {0.f, 0.f, 0.f, 0.f};
    if constexpr (VEC) {
        const u32x2 u = *(const u32x2*)(p + i);
        x[0] = __uint_as_float(u[0] << 16); x[1] = __uint_as_float(u[0] & 0xffff0000u);
        x[2] = __uint_as_float(u[1] << 16); x[3] = __uint_as_float(u[1] & 0xffff0000u);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (i + j < n) x[j] = bf16_to_f(p[i + j]);
    }
    return x;
}
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
__device__ __forceinline__ void store_bf16(unsigned short* p, int64_t i, int64_t n, f32x4 x) {
    if constexpr (VEC) {
        u32x2 u;
        u[0] = f_to_bf16(x[0]) | f_to_bf16(x[1]) << 16;
        u[1] = f_to_bf16(x[2]) | f_to_bf16(x[3]) << 16;
        *(u32x2*)(p + i) = u;
        return;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (i + j < n) p[i + j] = (unsigned short)f_to_bf16(x[j]);
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
    f32x4 p, g, m, v, w;
    unsigned mc, vc;
    float ms, vs;
};

template <bool BF16, bool EIGHT, bool VEC>
__device__ __forceinline__ void piece_load(const gcp_adamw_tensor_t& T, int64_t i, Piece& q) {
    if constexpr (BF16) {
        q.p = load_bf16<VEC>((const unsigned short*)T.param, i, T.n);
        q.g = load_bf16<VEC>((const unsigned short*)T.grad, i, T.n);
        q.w = load_f32<VEC>(T.master, i, T.n);
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
__device__ __forceinline__ void piece_update(const StepArgs& a, const gcp_adamw_tensor_t& T, int64_t i, Piece& q, float clip, float lr1,
                                             float root2, unsigned key) {
    // (products and sums of the moments rounded one by one: the codes of 8-bit moments are then the same wherever they are computed)
#pragma clang fp contract(off)
    if constexpr (EIGHT) {
        q.m = e4m3_decode(q.mc);
        q.v = e4m3_decode(q.vc);
    }
    f32x4 p = q.p;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float g = q.g[j] * clip;
        if constexpr (EIGHT) {
            q.m[j] *= q.ms;
            q.v[j] *= q.vs;
        }
        // a parameter that is not the rounding of its master copy was written by somebody else: it is taken as it is
        if constexpr (BF16) p[j] = f_to_bf16(q.w[j]) == __float_as_uint(q.p[j]) >> 16 ? q.w[j] : q.p[j];
        q.m[j] = q.m[j] * a.b1 + g * a.c1;
        q.v[j] = q.v[j] * a.b2 + (g * a.c2) * g;
        p[j] = p[j] * a.keep - lr1 * (q.m[j] / (sqrtf(q.v[j]) / root2 + a.eps));
    }
    if constexpr (BF16) {
        store_bf16<VEC>((unsigned short*)T.param, i, T.n, p);
        store_f32<VEC>(T.master, i, T.n, p);
    } else {
        store_f32<VEC>((float*)T.param, i, T.n, p);
    }
    if constexpr (EIGHT) {
        float tm = 0.f, tv = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {  // (absent elements are 0)
            if (finite_f(q.m[j])) tm = fmaxf(tm, fabsf(q.m[j]));
            if (finite_f(q.v[j])) tv = fmaxf(tv, q.v[j]);
        }
        const float ms = block_scale(wave_max(tm)), vs = block_scale(wave_max(tv));
        const float mi = pow2_inverse(ms), vi = pow2_inverse(vs);
        f32x4 ym, yv;
        const unsigned k = i >> 32 ? mix32(key ^ mix32((unsigned)(i >> 32))) : key;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            ym[j] = finite_f(q.m[j]) ? q.m[j] * mi : 0.f;
            yv[j] = finite_f(q.v[j]) ? e4m3_stochastic(q.v[j] * vi, mix32(k + (unsigned)i + j) & 0xfffffu) : 0.f;
        }
        store_u8x4<VEC>((unsigned char*)T.exp_avg, i, T.n, nan_codes(e4m3_encode(ym), q.m));
        store_u8x4<VEC>((unsigned char*)T.exp_avg_sq, i, T.n, nan_codes(e4m3_encode(yv), q.v));
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
__global__ __launch_bounds__(256) void adamw_kernel(StepArgs a) {
    int lo = 0, hi = a.n - 1;  // the tensor of this chunk
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (a.first[mid] <= (int)blockIdx.x) lo = mid; else hi = mid - 1;
    }
    const gcp_adamw_tensor_t& T = a.t[lo];
    const int64_t at = (int64_t)((int)blockIdx.x - a.first[lo]) * CHUNK;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const float clip = a.clip ? a.clip[1] : 1.f, lr1 = a.corr[2 * lo], root2 = a.corr[2 * lo + 1];
    unsigned key = 0;
    if constexpr (EIGHT) key = mix32(mix32(a.seed + 0x9e3779b9u * T.ordinal) ^ (unsigned)(int)*T.step);
    if (T.vec && at + CHUNK <= T.n) {
        Piece q[ITER];
#pragma unroll
        for (int k = 0; k < ITER; ++k) piece_load<BF16, EIGHT, true>(T, at + (k * 4 + wave) * QBLOCK + 4 * lane, q[k]);
#pragma unroll
        for (int k = 0; k < ITER; ++k)
            piece_update<BF16, EIGHT, true>(a, T, at + (k * 4 + wave) * QBLOCK + 4 * lane, q[k], clip, lr1, root2, key);
    } else {
        for (int k = 0; k < ITER; ++k) {
            const int64_t b = at + (k * 4 + wave) * QBLOCK;
            if (b >= T.n) break;  // (wave-uniform)
            Piece q;
            piece_load<BF16, EIGHT, false>(T, b + 4 * lane, q);
            piece_update<BF16, EIGHT, false>(a, T, b + 4 * lane, q, clip, lr1, root2, key);
        }
    }
}

// Before the update: the step counts of up to GCP_ADAMW_MAX_BEGIN tensors advance in device memory (so that a captured step counts on),
// their bias corrections are formed in double, and the partial sums of the squared gradients become the norm and the coefficient.
struct BeginArgs {
    float* step[GCP_ADAMW_MAX_BEGIN];
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
        a.corr[2 * i] = (float)(a.lr / (1.0 - pow(a.b1, (double)t)));
        a.corr[2 * i + 1] = (float)sqrt(1.0 - pow(a.b2, (double)t));
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
    const void* grad[GCP_ADAMW_MAX_NORM];
    int64_t n[GCP_ADAMW_MAX_NORM];
    int first[GCP_ADAMW_MAX_NORM + 1];
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
        if constexpr (BF16) x = load_bf16<VEC>((const unsigned short*)g, i, n);
        else x = load_f32<VEC>((const float*)g, i, n);
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
        for (; k < n && a.count < GCP_ADAMW_MAX_NORM; ++k) {
            if (t[k].n == 0) continue;
            const int64_t more = (t[k].n + NORM_CHUNK - 1) / NORM_CHUNK;
            if (more > INT32_MAX / 2) return GCPNET_E_UNSUPPORTED;
            if (c + more > INT32_MAX / 2) break;
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
    for (int k = 0; k < n || (k == 0 && partials); k += GCP_ADAMW_MAX_BEGIN) {
        BeginArgs a = {};
        a.n = n - k < GCP_ADAMW_MAX_BEGIN ? n - k : GCP_ADAMW_MAX_BEGIN;
        for (int j = 0; j < a.n; ++j) a.step[j] = t[k + j].step;
        a.corr = corrections + 2 * (int64_t)k;
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
    for (int k = 0; k < n;) {
        StepArgs a;
        a.n = 0;
        const int k0 = k;
        int64_t c = 0;
        for (; k < n && a.n < GCP_ADAMW_MAX_TENSORS; ++k) {
            const int64_t more = (t[k].n + CHUNK - 1) / CHUNK;
            if (more > INT32_MAX / 2) return GCPNET_E_UNSUPPORTED;
            if (c + more > INT32_MAX / 2) break;
            a.t[a.n] = t[k];
            const unsigned w = half ? 8 : 16, s = eight ? 4 : 16;
            a.t[a.n].vec = aligned(t[k].param, w) && aligned(t[k].grad, w) && aligned(t[k].exp_avg, s) && aligned(t[k].exp_avg_sq, s) &&
                           (!half || aligned(t[k].master, 16));
            a.first[a.n++] = (int)c;
            c += more;
        }
        a.first[a.n] = (int)c;
        if (!c) continue;
        a.corr = corrections + 2 * (int64_t)k0;
        a.clip = clip;
        a.b1 = (float)beta1; a.c1 = (float)(1.0 - beta1);
        a.b2 = (float)beta2; a.c2 = (float)(1.0 - beta2);
        a.eps = (float)eps; a.keep = (float)(1.0 - lr * weight_decay);
        a.seed = seed;
#define ADAMW_LAUNCH(B, E) hipLaunchKernelGGL(HIP_KERNEL_NAME(adamw_kernel<B, E>), dim3((unsigned)c), dim3(256), 0, (hipStream_t)stream, a)
        if (half) { if (eight) ADAMW_LAUNCH(true, true); else ADAMW_LAUNCH(true, false); }
        else { if (eight) ADAMW_LAUNCH(false, true); else ADAMW_LAUNCH(false, false); }
#undef ADAMW_LAUNCH
        GCP_HIP_CHECK_LAUNCH();
    }
    return 0;
}
