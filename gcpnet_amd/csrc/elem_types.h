// Element types of the operators that take fp32, bf16 and fp16: vectors of V elements as they lie in memory, and their fp32 values.
#pragma once
#include "common.h"

struct ElemF32 { typedef float type; static constexpr int code = GCP_TYPE_F32, vec = 4; static constexpr float largest = 0x1.fffffep127f; };
struct ElemBf16 { typedef __bf16 type; static constexpr int code = GCP_TYPE_BF16, vec = 8; static constexpr float largest = 0x1.fep127f; };
struct ElemF16 { typedef _Float16 type; static constexpr int code = GCP_TYPE_F16, vec = 8; static constexpr float largest = 65504.f; };

template <class E, int V>
struct Raw {  // V elements as they lie in memory, 16 bytes in four registers
    unsigned u[4];
    __device__ __forceinline__ float operator[](int j) const {
        if constexpr (E::code == GCP_TYPE_F32) return __uint_as_float(u[j]);
        else if constexpr (E::code == GCP_TYPE_BF16) return __uint_as_float(j & 1 ? u[j / 2] & 0xffff0000u : u[j / 2] << 16);
        else return (float)__builtin_bit_cast(_Float16, (unsigned short)(j & 1 ? u[j / 2] >> 16 : u[j / 2]));
    }
};

// Loads and stores of V elements at any element's address: one 16-byte access (global memory takes it at any alignment), and element by
// element where only the first `count` of the V are there.
template <class E, int V>
__device__ __forceinline__ Raw<E, V> elem_load(const void* base, int64_t at) {
    static_assert(V * sizeof(typename E::type) == 16, "a vector is 16 bytes");
    Raw<E, V> r;
    __builtin_memcpy(r.u, (const typename E::type*)base + at, 16);
    return r;
}
template <class E, int V>
__device__ __forceinline__ Raw<E, V> elem_zero() {
    return Raw<E, V>{{0u, 0u, 0u, 0u}};
}
template <class E, int V>
__device__ __forceinline__ Raw<E, V> elem_load(const void* base, int64_t at, int count) {
    if (count == V) return elem_load<E, V>(base, at);
    Raw<E, V> r = elem_zero<E, V>();
    if (count > 0)
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (j < count) {
                if constexpr (E::code == GCP_TYPE_F32) r.u[j] = ((const unsigned*)base)[at + j];
                else r.u[j / 2] |= (unsigned)((const unsigned short*)base)[at + j] << (16 * (j & 1));
            }
    return r;
}
template <class E, int V>
__device__ __forceinline__ void elem_store(void* base, int64_t at, const float (&f)[V]) {
    typename E::type x[V];
#pragma unroll
    for (int j = 0; j < V; ++j) x[j] = (typename E::type)f[j];  // (nearest even)
    f32x4 q;
    __builtin_memcpy(&q, x, 16);
    __builtin_memcpy((typename E::type*)base + at, &q, 16);
}
template <class E, int V>
__device__ __forceinline__ void elem_store(void* base, int64_t at, const float (&f)[V], int count) {
    if (count == V) elem_store<E, V>(base, at, f);
    else if (count > 0)
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (j < count) ((typename E::type*)base)[at + j] = (typename E::type)f[j];
}

// A finite value held to the range of the rows' type, where the conversion would make it infinite; infinities and NaN stay.
template <class E>
__device__ __forceinline__ float elem_in_range(float x) {
    if constexpr (E::code == GCP_TYPE_F32) return x;
    const float in = __builtin_amdgcn_fmed3f(x, -E::largest, E::largest);
    return __builtin_isfinite(x) ? in : x;
}

// `count` of V values of a parameter vector of the rows' type, or fp32 (`f32`: uniform over the launch), as they lie in memory: requested
// early, unpacked where they are used.
template <class E, int V>
struct Param {
    unsigned u[V];
    __device__ __forceinline__ void unpack(bool f32, float (&f)[V]) const {
        if (E::code != GCP_TYPE_F32 && f32) {
#pragma unroll
            for (int j = 0; j < V; ++j) f[j] = __uint_as_float(u[j]);
        } else {
            const Raw<E, V> r = {{u[0], u[1], u[2], u[3]}};
#pragma unroll
            for (int j = 0; j < V; ++j) f[j] = r[j];
        }
    }
};
template <class E, int V>
__device__ __forceinline__ Param<E, V> param_load(const void* base, int64_t at, int count, bool f32) {
    Param<E, V> p;
    if (E::code != GCP_TYPE_F32 && f32) {
#pragma unroll
        for (int h = 0; h < V; h += 4) {
            const Raw<ElemF32, 4> r = elem_load<ElemF32, 4>(base, at + h, count - h < 4 ? count - h : 4);
#pragma unroll
            for (int j = 0; j < 4; ++j) p.u[h + j] = r.u[j];
        }
    } else {
        const Raw<E, V> r = elem_load<E, V>(base, at, count);
#pragma unroll
        for (int j = 0; j < V; ++j) p.u[j] = j < 4 ? r.u[j] : 0u;
    }
    return p;
}

// The sigmoid by the hardware's exponential and reciprocal.  The reciprocal is good to a unit in the last place; exp(-x) is off by about |x| + 2 half
// steps, relatively, since its argument is rounded, and below 0 so is the sigmoid: 4 units at x = -5, 8 at -20, 32 at -80.
__device__ __forceinline__ float elem_sigmoid(float x) { return __builtin_amdgcn_rcpf(1.f + __expf(-x)); }
__device__ __forceinline__ bool elem_by_sigmoid(int act) { return act == GCP_ACT_SILU || act == GCP_ACT_SIGMOID; }

// exp(x) - 1 for x <= 0, with e = exp(x): the difference itself from -1/2 down, where it is good to 5 half steps; above, where the difference would
// lose x in the rounding of 1 + x, x + x^2 p(x) with the polynomial that meets (exp(x) - 1 - x) / x^2 in the five Chebyshev points of [-1/2, 0]
// (0.2 half steps off, 1.3 with the roundings).
__device__ __forceinline__ float elem_expm1(float x, float e) {
    const float p = fmaf(fmaf(fmaf(fmaf(0x1.3135fap-10f, x, 0x1.0df336p-7f), x, 0x1.55323cp-5f), x, 0x1.5554cap-3f), x, 0.5f);
    return x > -0.5f ? fmaf(x * x, p, x) : e - 1.f;
}

// act(v), and with GRAD also act'(v), of V values; the choice is uniform and made once for all of them.  `s`: the sigmoids of v where the
// activation is made of them (else not looked at).
template <int V, bool GRAD>
__device__ __forceinline__ void elem_act_with(int act, float slope, const float (&v)[V], const float (&s)[V], float (&a)[V], float (&d)[V]) {
    if (elem_by_sigmoid(act)) {
        const bool silu = act == GCP_ACT_SILU;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float x = v[j], r = s[j] * (1.f - s[j]);
            a[j] = silu ? x * s[j] : s[j];
            if constexpr (GRAD) d[j] = silu ? fmaf(x, r, s[j]) : r;
        }
    } else if (act == GCP_ACT_SELU) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            // (both sides of 0, and one of them taken: no branches; a NaN is on the lower)
            const float x = v[j], e = __expf(x), em = elem_expm1(x, e);
            a[j] = (x > 0.f ? GCP_SELU_SCALE : GCP_SELU_SCALE * GCP_SELU_ALPHA) * (x > 0.f ? x : em);
            if constexpr (GRAD) d[j] = x > 0.f ? GCP_SELU_SCALE : GCP_SELU_SCALE * GCP_SELU_ALPHA * e;
        }
    } else {  // (none, relu, leakyrelu: a slope on each side)
        const float low = act == GCP_ACT_NONE ? 1.f : act == GCP_ACT_RELU ? 0.f : slope;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float x = v[j];
            a[j] = x < 0.f ? (low == 0.f ? 0.f : low * x) : x;  // (NaN stays)
            if constexpr (GRAD) d[j] = x > 0.f ? 1.f : low;
        }
    }
}
template <int V, bool GRAD>
__device__ __forceinline__ void elem_act(int act, float slope, const float (&v)[V], float (&a)[V], float (&d)[V]) {
    float s[V];
    if (elem_by_sigmoid(act))
#pragma unroll
        for (int j = 0; j < V; ++j) s[j] = elem_sigmoid(v[j]);
    elem_act_with<V, GRAD>(act, slope, v, s, a, d);
}

inline bool elem_type_ok(int t) { return t == GCP_TYPE_F32 || t == GCP_TYPE_BF16 || t == GCP_TYPE_F16; }
inline int elem_bytes(int t) { return t == GCP_TYPE_F32 ? 4 : 2; }
inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
