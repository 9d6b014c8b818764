// Shared by the sequence operators (causal_conv.hip, scan.hip, block_norm.hip): gate functions and the final sum of per-block partials.
#pragma once
#include "common.h"

constexpr float SQ_LOG2E = 1.4426950408889634f, SQ_LN2 = 0.6931471805599453f;

// exp(x) for x <= 0 to about an ulp: x * log2(e) as a rounded product plus its rounding error (without the second term the relative error is
// |x| * 2^-24: 4e-7 at the softplus arguments of small step sizes)
__device__ __forceinline__ float sq_exp(float x) {
    const float t = x * SQ_LOG2E;
    const float lo = fmaf(x, SQ_LOG2E, -t) + x * 1.925963033500e-8f;  // log2(e) - fp32(log2(e))
    const float e = __builtin_amdgcn_exp2f(t);
    return x < -100.f ? e : fmaf(e, lo * SQ_LN2, e);
}
__device__ __forceinline__ float sq_sigmoid(float x) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-x * SQ_LOG2E)); }
__device__ __forceinline__ float sq_silu(float x) { return x * sq_sigmoid(x); }
// d silu(x) / dx
__device__ __forceinline__ float sq_silu_slope(float x) {
    const float s = sq_sigmoid(x);
    return s * fmaf(x, 1.f - s, 1.f);
}
// log(1 + exp(x)) = max(x, 0) + log1p(e), e = exp(-|x|); log1p(e) = log(w) + (e - (w - 1)) / w with w = fl(1 + e): the second term gives
// back what the sum lost, so that small results keep all their digits
__device__ __forceinline__ float sq_softplus(float x) {
    const float e = sq_exp(-fabsf(x)), w = 1.f + e;
    const float l = fmaf(__builtin_amdgcn_logf(w), SQ_LN2, (e - (w - 1.f)) * __builtin_amdgcn_rcpf(w));
    return (x > 0.f ? x : x != x ? x : 0.f) + l;
}

__device__ __forceinline__ int sq_len(const int* lengths, int b, int T) {
    if (!lengths) return T;
    const int n = lengths[b];
    return n < 0 ? 0 : n > T ? T : n;
}
