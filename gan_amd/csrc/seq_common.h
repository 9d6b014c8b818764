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

// Sums over the 64 lanes of many values at once: each step sends one half of the values each way across a lane bit, so that the work halves
// with it (V values cost 2V - 2 exchanges and adds and not 6V).  permlane swaps for the upper two lane bits, DPP for the others.
template <int CTRL>
__device__ __forceinline__ float sq_dpp(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float sq_fold32(float a, float b) {  // lanes 0-31: a over both halves, 32-63: b
    const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return __uint_as_float(x[0]) + __uint_as_float(x[1]);
}
__device__ __forceinline__ float sq_fold16(float a, float b) {
    const auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return __uint_as_float(x[0]) + __uint_as_float(x[1]);
}
template <int CTRL>
__device__ __forceinline__ float sq_fold(float a, float b, bool up) {
    return (up ? b : a) + sq_dpp<CTRL>(up ? a : b);
}
// n values (a power of two) in v; lane l leaves with v[0] = the sum of value (the top log2 n bits of l)
template <int V>
__device__ __forceinline__ float sq_lane_sums(float (&v)[V], int lane) {
    static_assert(V >= 1 && V <= 64 && (V & (V - 1)) == 0, "a power of two");
    int n = V;
#define SQ_FOLD(FN, ...)                                                              \
    if (n > 1) {                                                                      \
        n >>= 1;                                                                      \
        _Pragma("unroll") for (int i = 0; i < n; ++i) v[i] = FN(v[i], v[i + n] __VA_ARGS__); \
    } else
    SQ_FOLD(sq_fold32) v[0] = sq_fold32(v[0], v[0]);
    SQ_FOLD(sq_fold16) v[0] = sq_fold16(v[0], v[0]);
    SQ_FOLD(sq_fold<0x128>, , lane & 8) v[0] += sq_dpp<0x128>(v[0]);  // rotate by 8 within 16
    SQ_FOLD(sq_fold<0x141>, , lane & 4) v[0] += sq_dpp<0x141>(v[0]);  // mirror within 8
    SQ_FOLD(sq_fold<0x4E>, , lane & 2) v[0] += sq_dpp<0x4E>(v[0]);    // quads: 2 3 0 1
    SQ_FOLD(sq_fold<0xB1>, , lane & 1) v[0] += sq_dpp<0xB1>(v[0]);    // quads: 1 0 3 2
#undef SQ_FOLD
    return v[0];
}

// One column of a [rows][cols] matrix of partial sums, added up by `groups` threads of a block (thread group w of the column) in double: eight
// loads in flight, a fixed order.
__device__ __forceinline__ double sq_column(const float* p, size_t cols, int rows, int w, int groups) {
    double v = 0.0;
    int r = w;
    for (; r + 7 * groups < rows; r += 8 * groups) {
        float t[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) t[i] = p[(size_t)(r + i * groups) * cols];
#pragma unroll
        for (int i = 0; i < 8; ++i) v += (double)t[i];
    }
    for (; r < rows; r += groups) v += (double)p[(size_t)r * cols];
    return v;
}
// the 32 columns x 32 groups of a block of 1024: the column's sum, in its first group's threads
__device__ __forceinline__ double sq_groups32(double v, double (*acc)[32]) {
    const int c = threadIdx.x & 31, w = threadIdx.x >> 5;
    __syncthreads();
    acc[w][c] = v;
    __syncthreads();
    if (w == 0)
        for (int k = 1; k < 32; ++k) v += acc[k][c];
    return v;
}
