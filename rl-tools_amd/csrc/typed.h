// Tensors of either element type (rlt_type): vectors of 16 bytes, held as fp32 in registers.
#pragma once
#include "common.h"

typedef __bf16 rlt_bf16;
typedef __bf16 rlt_bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 rlt_bf16x8 __attribute__((ext_vector_type(8)));
typedef float rlt_f32x4 __attribute__((ext_vector_type(4)));

// `N` elements side by side: N = 1, or 16 bytes (aligned as such)
template <int N, typename T> __device__ __forceinline__ void rlt_load(const T* __restrict__ src, float* dst) {
    if constexpr (N == 1) dst[0] = (float)src[0];
    else {
        typedef T vector __attribute__((ext_vector_type(N)));
        const vector v = *reinterpret_cast<const vector*>(src);
#pragma unroll
        for (int i = 0; i < N; i++) dst[i] = (float)v[i];
    }
}
// rounds to nearest, ties to even
template <int N, typename T> __device__ __forceinline__ void rlt_store(T* __restrict__ dst, const float* src) {
    if constexpr (N == 1) dst[0] = (T)src[0];
    else {
        typedef T vector __attribute__((ext_vector_type(N)));
        vector v;
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = (T)src[i];
        *reinterpret_cast<vector*>(dst) = v;
    }
}

// whether rows of a tensor start on 16-byte boundaries
template <typename T> static inline bool rlt_vectors(const void* p, int64_t stride) { return (reinterpret_cast<uintptr_t>(p) % 16 == 0) && stride % (int64_t)(16 / sizeof(T)) == 0; }
