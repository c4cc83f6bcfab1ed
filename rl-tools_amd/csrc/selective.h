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
