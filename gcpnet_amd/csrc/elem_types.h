// Element types of the operators that take fp32, bf16 and fp16: vectors of V elements as they lie in memory, and their fp32 values.
#pragma once
#include "common.h"

struct ElemF32 { typedef float type; static constexpr int code = GCP_TYPE_F32, vec = 4; };
struct ElemBf16 { typedef __bf16 type; static constexpr int code = GCP_TYPE_BF16, vec = 8; };
struct ElemF16 { typedef _Float16 type; static constexpr int code = GCP_TYPE_F16, vec = 8; };

template <class E, int V>
struct Raw {  // V elements, loaded and stored as one piece (V = 1 or 16 bytes' worth)
    typename E::type x[V];
    static constexpr int bytes = V * (int)sizeof(typename E::type);
};

template <class E, int V>
__device__ __forceinline__ Raw<E, V> elem_load(const void* base, int64_t at) {
    Raw<E, V> r;
    const typename E::type* p = (const typename E::type*)base + at;
    if constexpr (V == 1) {
        r.x[0] = *p;
    } else {
        static_assert(Raw<E, V>::bytes == 16, "a vector is 16 bytes");
        const f32x4 q = *(const f32x4*)p;
        __builtin_memcpy(r.x, &q, 16);
    }
    return r;
}
template <class E, int V>
__device__ __forceinline__ void elem_store(void* base, int64_t at, const float (&f)[V]) {
    typename E::type* p = (typename E::type*)base + at;
    if constexpr (V == 1) {
        *p = (typename E::type)f[0];
    } else {
        typename E::type x[V];
#pragma unroll
        for (int j = 0; j < V; ++j) x[j] = (typename E::type)f[j];  // (nearest even)
        f32x4 q;
        __builtin_memcpy(&q, x, 16);
        *(f32x4*)p = q;
    }
}
template <class E, int V>
__device__ __forceinline__ void elem_zero(Raw<E, V>& r) {
#pragma unroll
    for (int j = 0; j < V; ++j) r.x[j] = (typename E::type)0.f;
}

// V values of a parameter vector of the same type as the rows, or fp32 (`f32`: uniform over the launch)
template <class E, int V>
__device__ __forceinline__ void param_load(const void* base, int64_t at, bool f32, float (&f)[V]) {
    if (!base) return;
    if (E::code != GCP_TYPE_F32 && f32) {
#pragma unroll
        for (int j = 0; j < V; ++j) f[j] = ((const float*)base)[at + j];
    } else {
        const Raw<E, V> r = elem_load<E, V>(base, at);
#pragma unroll
        for (int j = 0; j < V; ++j) f[j] = (float)r.x[j];
    }
}

inline bool elem_type_ok(int t) { return t == GCP_TYPE_F32 || t == GCP_TYPE_BF16 || t == GCP_TYPE_F16; }
inline int elem_bytes(int t) { return t == GCP_TYPE_F32 ? 4 : 2; }
inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
