// Scalar math of the state-space operators (ssm.hip, short_conv.hip): 32-bit throughout, rounded to the tensors' type by the
// caller, once, at a store.
#pragma once
#include "common.h"

#define LOG2E 1.4426950408889634f
#define LOG2E_LO 1.9259629911266175e-8f   // log2(e) - LOG2E
#define LN2 0.6931471805599453f

__device__ __forceinline__ float ld(const float* p) { return *p; }
__device__ __forceinline__ float ld(const bf16_t* p) { return bf2f(*p); }
__device__ __forceinline__ void st(float* p, float v) { *p = v; }
__device__ __forceinline__ void st(bf16_t* p, float v) { *p = f2bf(v); }

// exp(-|x|) by the hardware's 2^y: the part of x * log2(e) that its 24 bits lose comes back as a factor 1 + lost * ln 2
// (without it the relative error grows with |x|: 4e-7 at 7, where a step size of 0.001 sits). From 128 on the result is 0; the
// argument stops there (a NaN passes), as the product would leave the range with it and what it lost be no number: a step of
// size -inf or of the type's lowest value holds the state.
__device__ __forceinline__ float exp_neg_abs(float x) {
    const float ax = __builtin_elementwise_maximum(-fabsf(x), -128.f), hi = ax * LOG2E;
    const float lo = fmaf(ax, LOG2E, -hi) + ax * LOG2E_LO;
    const float p = __builtin_amdgcn_exp2f(hi);
    return fmaf(p, lo * LN2, p);
}
// softplus(x) = max(x, 0) + log(1 + e) and its slope 1 / (1 + exp(-x)), e = exp(-|x|). u = 1 + e keeps few of a small e's
// bits; what it lost, e - (u - 1), comes back over u: log(1 + e) = log u + (e - (u - 1)) / u (largest error measured over
// e = exp(-30) .. 1: 1.9e-7 of the value).
__device__ __forceinline__ float softplus(float x, float* slope = nullptr) {
    const float e = exp_neg_abs(x), u = 1.0f + e, r = __builtin_amdgcn_rcpf(u);
    if (slope) *slope = x >= 0.f ? r : e * r;
    return fmaxf(x, 0.f) + fmaf(e - (u - 1.0f), r, __builtin_amdgcn_logf(u) * LN2);
}
// A decay rate times c. It stops at the lowest finite value: a state of rate -inf (or whose product leaves the range) has no
// memory, but a step of size 0 - past a row's end, or one that is held - leaves it alone. A NaN passes.
__device__ __forceinline__ float rate(float a, float c) {
    return __builtin_elementwise_maximum(a * c, -3.402823466e38f);
}
// for gates: exp's error of |x| half steps stands next to 1, or where the gate is nearly shut
__device__ __forceinline__ float sigmoidf(float x) { return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * -LOG2E)); }

// Swapping rows of 16 lanes adds two values at a time.
__device__ __forceinline__ float add_swap16(float a, float b) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);     // rows a0+a1, b0+b1, a2+a3, b2+b3
}
__device__ __forceinline__ float add_swap32(float a, float b) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);     // rows a0+a2, a1+a3, b0+b2, b1+b3
}
template <int CTRL>
__device__ __forceinline__ float add_dpp(float v) {
    return v + __uint_as_float(__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), CTRL, 0xf, 0xf, true));
}
// sum over groups of L = 4, 8, 16, 32 or 64 neighbouring lanes, in every lane: adds across neighbours, then row swaps, no trip
// through LDS
template <int L>
__device__ __forceinline__ float lane_sum(float v) {
    v = add_dpp<0xB1>(v);                              // quad: lane ^ 1
    v = add_dpp<0x4E>(v);                              // quad: lane ^ 2
    if constexpr (L > 4) v = add_dpp<0x141>(v);        // row_half_mirror: the other quad of 8 lanes
    if constexpr (L > 8) v = add_dpp<0x140>(v);        // row_mirror: the other 8 lanes
    if constexpr (L > 16) v = add_swap16(v, v);
    if constexpr (L > 32) v = add_swap32(v, v);
    return v;
}
