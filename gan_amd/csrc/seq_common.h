// Shared by the sequence operators (causal_conv.hip, scan.hip, block_norm.hip): gate functions and the final sum of per-block partials.
#pragma once
#include "common.h"

constexpr float SQ_LOG2E = 1.4426950408889634f, SQ_LN2 = 0.6931471805599453f;

__device__ __forceinline__ float sq_sigmoid(float x) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-x * SQ_LOG2E)); }
__device__ __forceinline__ float sq_silu(float x) { return x * sq_sigmoid(x); }
// d silu(x) / dx
__device__ __forceinline__ float sq_silu_slope(float x) {
    const float s = sq_sigmoid(x);
    return s * fmaf(x, 1.f - s, 1.f);
}
// log(1 + exp(x)) = max(x, 0) + log1p(e), e = exp(-|x|).  e: exp2 of the rounded product t = -|x| log2(e), times 1 + r with r = what t lacks
// (without it e is off by |x| 2^-24 of itself: 4e-7 at the arguments of small step sizes).  log1p(e) = log(w) + (e - (w - 1)) / w with
// w = fl(1 + e): the second term gives back what the sum lost, so that small results keep all their digits.  max(x, 0) as a choice that passes
// a NaN on and gives 0 at minus infinity.  `sigmoid`: the slope, 1 / (1 + exp(-x)), from the same e and w.
__device__ __forceinline__ float sq_softplus(float x, float& sigmoid) {
    const float ax = fminf(fabsf(x), 100.f), t = -ax * SQ_LOG2E;
    const float r = fmaf(-t, -1.9046542e-9f, fmaf(-t, SQ_LN2, -ax));  // ln 2 = fp32(ln 2) - 1.9046542e-9
    const float e2 = __builtin_amdgcn_exp2f(t), e = fmaf(e2, r, e2), w = 1.f + e, rw = __builtin_amdgcn_rcpf(w);
    sigmoid = (x < 0.f ? e : 1.f) * rw;
    return (x < 0.f ? 0.f : x) + fmaf(__builtin_amdgcn_logf(w), SQ_LN2, (e - (w - 1.f)) * rw);
}
__device__ __forceinline__ float sq_softplus(float x) {
    float s;
    return sq_softplus(x, s);
}

// A pointer that is the same in all lanes, as a scalar that is added to nowhere else: base plus a 32-bit offset per lane is then the address of a
// load (otherwise the compiler folds the offset into a 64-bit vector add, and two registers, for every row).
template <typename P>
__device__ __forceinline__ P* sq_scalar(P* p) {
    const uint64_t u = (uint64_t)p;
    const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)u), hi = __builtin_amdgcn_readfirstlane((unsigned)(u >> 32));
    return (P*)(((uint64_t)hi << 32) | lo);
}

__device__ __forceinline__ int sq_len(const int* lengths, int b, int T) {
    if (!lengths) return T;
    const int n = lengths[b];
    return n < 0 ? 0 : n > T ? T : n;
}

// A launch has at most 2^32 - 1 work-items along an axis.
inline bool sq_launch_fits(size_t blocks, size_t threads) { return blocks <= 0xffffffffUL / threads; }

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
// V values (a power of two) in v, folded over the lane bits TOP, TOP / 2, ... until one is left: a lane leaves with the sum, over the lanes that
// differ from it in these bits, of the value that they number
template <int V, int TOP>
__device__ __forceinline__ float sq_fold_down(float (&v)[V], int lane) {
    static_assert(V >= 1 && (V & (V - 1)) == 0 && V <= 2 * TOP, "a power of two, and a lane bit for each halving");
    int n = V;
    if (TOP >= 32 && n > 1) {
        n >>= 1;
#pragma unroll
        for (int i = 0; i < n; ++i) v[i] = sq_fold32(v[i], v[i + n]);
    }
    if (TOP >= 16 && n > 1) {
        n >>= 1;
#pragma unroll
        for (int i = 0; i < n; ++i) v[i] = sq_fold16(v[i], v[i + n]);
    }
    if (TOP >= 8 && n > 1) {
        n >>= 1;
#pragma unroll
        for (int i = 0; i < n; ++i) v[i] = sq_fold<0x128>(v[i], v[i + n], lane & 8);  // rotate by 8 within 16
    }
    if (TOP >= 4 && n > 1) {
        n >>= 1;
#pragma unroll
        for (int i = 0; i < n; ++i) v[i] = sq_fold<0x141>(v[i], v[i + n], lane & 4);  // mirror within 8
    }
    if (TOP >= 2 && n > 1) {
        n >>= 1;
#pragma unroll
        for (int i = 0; i < n; ++i) v[i] = sq_fold<0x4E>(v[i], v[i + n], lane & 2);  // quads: 2 3 0 1
    }
    if (TOP >= 1 && n > 1) v[0] = sq_fold<0xB1>(v[0], v[1], lane & 1);  // quads: 1 0 3 2
    return v[0];
}
// V values, each summed over all 64 lanes: lane l leaves with the sum of value (the top log2 V bits of l)
template <int V>
__device__ __forceinline__ float sq_lane_sums(float (&v)[V], int lane) {
    float s = sq_fold_down<V, 32>(v, lane);
    constexpr int REST = 64 / V;
    if (REST >= 64) s = sq_fold32(s, s);
    if (REST >= 32) s = sq_fold16(s, s);
    if (REST >= 16) s += sq_dpp<0x128>(s);
    if (REST >= 8) s += sq_dpp<0x141>(s);
    if (REST >= 4) s += sq_dpp<0x4E>(s);
    if (REST >= 2) s += sq_dpp<0xB1>(s);
    return s;
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
