// What the convolution and the scan of selective blocks share: views as offsets, exponentials whose relative accuracy holds far from zero.
#pragma once
#include "typed.h"

struct rlt_part { void* data; int64_t step, row, head; };
static inline rlt_part rlt_part_of(const rlt_head_view* v) { return v ? rlt_part{v->data, v->step_stride, v->row_stride, v->head_stride} : rlt_part{}; }
static inline bool rlt_given(const rlt_head_view* v) { return v && v->data; }

// e^t for t <= 0. The power of two alone is off by about |t| units of 2^-24, as its exponent is rounded; what the rounding dropped goes in to first order. Below the smallest normal number it is 0; a NaN stays one.
__device__ __forceinline__ float rlt_exp_negative(float t) {
    const float at = t * 1.44269504088896341f, p = __builtin_amdgcn_exp2f(at);
    const float rest = fmaf(t, 1.44269504088896341f, -at) + t * 1.925963033500721e-8f;
    return at > -126.0f ? fmaf(p, rest * 0.6931471805599453f, p) : p;
}
// 1 / d for d in [1, 2^64): the instruction's result with one step of Newton's method
__device__ __forceinline__ float rlt_reciprocal(float d) {
    const float q = __builtin_amdgcn_rcpf(d);
    return fmaf(fmaf(-d, q, 1.0f), q, q);
}
// 1 / (1 + e^-x) and 1 / (1 + e^x), each with its relative accuracy
__device__ __forceinline__ void rlt_sigmoids(float x, float& s, float& other) {
    const float e = rlt_exp_negative(-fabsf(x)), large = rlt_reciprocal(1.0f + e), small = e * large;
    s = x >= 0.0f ? large : small;
    other = x >= 0.0f ? small : large;
}

// Sums over `parts` rows of a matrix of `columns` columns, in a fixed order, by a workgroup of 1,024 for sixteen columns: the sum of column `column` in the first sixteen threads. Sixty-four threads share a column, eight rows of each on their way
// at a time (777 parts of 804 columns: 4 us; 15 with sixteen threads to a column, which follow one row with the next).
constexpr int RLT_JOIN_COLUMNS = 16;
__device__ __forceinline__ float rlt_join_column(const float* __restrict__ from, int parts, size_t columns, size_t column, bool there) {
    __shared__ float sums[16][RLT_JOIN_COLUMNS];
    constexpr int AHEAD = 8, GROUPS = 1024 / RLT_JOIN_COLUMNS;
    const int group = threadIdx.x / RLT_JOIN_COLUMNS, lane = threadIdx.x & 63;
    float s = 0.0f;
    if (there) {
        int p = group;
        for (; p + (AHEAD - 1) * GROUPS < parts; p += AHEAD * GROUPS) {
            float v[AHEAD];
#pragma unroll
            for (int i = 0; i < AHEAD; i++) v[i] = from[(size_t)(p + i * GROUPS) * columns + column];
#pragma unroll
            for (int i = 0; i < AHEAD; i++) s += v[i];
        }
        float v[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; i++) v[i] = p + i * GROUPS < parts ? from[(size_t)(p + i * GROUPS) * columns + column] : 0.0f;
#pragma unroll
        for (int i = 0; i < AHEAD; i++) s += v[i];
    }
    s += __shfl_xor(s, 16, 64);
    s += __shfl_xor(s, 32, 64);
    if (lane < 16) sums[threadIdx.x >> 6][lane] = s;
    __syncthreads();
    if (threadIdx.x < 16) {
        s = 0.0f;
#pragma unroll
        for (int w = 0; w < 16; w++) s += sums[w][threadIdx.x];
    }
    return s;
}
