// Short causal depthwise convolution along time (+ SiLU) with a carried window, on channels-last activations:
//   pre[b][t][c] = bias[c] + sum_k w[c][k] x[b][t - (K-1) + k][c],  y = act(pre),  rows before 0 from the window (or zero)
// forward, backward and the single-token step.  Bound by memory where the activations are large, else by vector issue.
//
// A thread owns V adjacent channels (one 8- or 16-byte access a row where alignment allows) and a run of rows, the last K of them in registers:
// slot (K-1 + r) mod K holds the run's row r, so that a turn of K rows moves nothing.  A row is read once by its run and K - 1 rows of every
// run again by the next one (from cache, mostly); the loads of the next K rows are in flight while K rows are worked on.
//
// Measured, bf16, four taps and SiLU: 16 x 2250 x 1024 forward 29 us (147 MB: 5.0 TB/s), backward 60 us (221 MB: 3.7 TB/s, the sums of dw and the
// activation's slope beside it); channel slices of wider rows 30 and 61 us; float32 52 and 100 us (5.7 and 4.4 TB/s).  64 x 375 x 512 14.6 and
// 28.6 us: 2.7 and 2.4 TB/s of memory traffic, the vector units busy 68 and 81 % of the time with 21 and 49 instructions an element; float32 18 and
// 42 us.  One row of 64 x 1024 2.7 us, of 256 x 2048 4.6 us.
#include "seq_common.h"

namespace {

constexpr int MAX_PARTS = 1024;  // blocks along time of the backward pass, each with a row of weight-gradient sums

template <typename T, int V> struct alignas(sizeof(T) * V) Pack { T v[V]; };

struct Map {
    int px, ry;      // channel pieces and runs of a block (px * ry = 256)
    int pieces, pb;  // pieces of a row, piece blocks
    int run, rpi;    // rows of a run, runs of an item
    long runs;       // of all items
};

// Runs as long as 1024 blocks (four a CU) allow, 16 to 128 rows: the K - 1 rows read twice are (K - 1) / 16 of them at the most, a fifth with four taps
// and 44 % with eight.  (16 x 2250 x 1024 bf16: 29 + 60 us; 32 + 57 with 512 blocks, 31 + 69 with 2048.  64 x 375 x 512: 14.6 + 28.6, 15.0 + 28.3,
// 14.6 + 29.1.)
Map make_map(int B, int T, int C, int vec) {
    Map m;
    m.pieces = (C + vec - 1) / vec;
    m.px = 64;
    while (m.px > 1 && m.px / 2 >= m.pieces) m.px >>= 1;
    m.ry = 256 / m.px;
    m.pb = (m.pieces + m.px - 1) / m.px;
    const long blocks_of_one_run = ((long)B * m.pb + m.ry - 1) / m.ry;
    long want = 1024 / (blocks_of_one_run < 1024 ? blocks_of_one_run : 1024);
    long run = (T + want - 1) / want;
    m.run = (int)(run < 16 ? 16 : run > 128 ? 128 : run);
    m.rpi = (T + m.run - 1) / m.run;
    m.runs = (long)B * m.rpi;
    return m;
}

template <typename T, int V>
__device__ __forceinline__ void load_row(float (&o)[V], const T* p, bool ok) {
    if (ok) {
        const Pack<T, V> r = *(const Pack<T, V>*)p;
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] = (float)r.v[e];
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] = 0.f;
    }
}
template <typename T, int V>
__device__ __forceinline__ void store_row(T* p, const float (&v)[V]) {
    Pack<T, V> r;
#pragma unroll
    for (int e = 0; e < V; ++e) r.v[e] = (T)v[e];
    *(Pack<T, V>*)p = r;
}

// row t of (window ; sequence), t = -(K-1) .. len - 1; zero where there is none
template <typename T, int V>
__device__ __forceinline__ void load_joined(float (&o)[V], const T* x, long x_ts, const T* state, int K, int C, int t, int len) {
    if (t >= 0) load_row<T, V>(o, x + (size_t)t * x_ts, t < len);
    else load_row<T, V>(o, state + (long)(t + K - 1) * C, state != nullptr);
}

template <typename T, int V, int K>
__global__ __launch_bounds__(256) void cconv_fwd_kernel(ga_causal_conv_params p, Map m) {
    const int px = threadIdx.x % m.px, piece = (blockIdx.x % m.pb) * m.px + px;
    const long run = (long)(blockIdx.x / m.pb) * m.ry + threadIdx.x / m.px;
    if (piece >= m.pieces || run >= m.runs) return;
    const int b = (int)(run / m.rpi), t0 = (int)(run % m.rpi) * m.run, c0 = piece * V;
    const int len = sq_len(p.lengths, b, p.T), rows = min(m.run, p.T - t0);
    const T* x = (const T*)p.x + (size_t)b * p.x_bs + c0;
    const T* st = p.state ? (const T*)p.state + (size_t)b * (K - 1) * p.C + c0 : nullptr;
    T* y = (T*)p.y + ((size_t)b * p.T + t0) * p.C + c0;
    Pack<T, V> next[K];
    auto load = [&](int r0) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < K; ++i) next[i] = *(const Pack<T, V>*)(x + (size_t)min(t0 + r0 + i, p.T - 1) * p.x_ts);
    };
    load(0);
    float w[K][V], bias[V], win[K][V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
        bias[e] = p.bias ? p.bias[c0 + e] : 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k) w[k][e] = p.w[(size_t)(c0 + e) * K + k];
    }
#pragma unroll
    for (int k = 0; k < K - 1; ++k) load_joined<T, V>(win[k], x, p.x_ts, st, K, p.C, t0 - (K - 1) + k, len);
    for (int r0 = 0; r0 < rows; r0 += K) {
        Pack<T, V> cur[K];
#pragma unroll
        for (int i = 0; i < K; ++i) cur[i] = next[i];
        if (r0 + K < rows) load(r0 + K);
#pragma unroll
        for (int i = 0; i < K; ++i) {
            const int r = r0 + i;
            const bool live = t0 + r < len;
            float o[V];
#pragma unroll
            for (int e = 0; e < V; ++e) {
                win[(K - 1 + i) % K][e] = live ? (float)cur[i].v[e] : 0.f;
                float v = bias[e];
#pragma unroll
                for (int k = 0; k < K; ++k) v = fmaf(w[k][e], win[(i + k) % K][e], v);
                if (p.act == GA_ACT_SILU) v = sq_silu(v);
                o[e] = live ? v : 0.f;
            }
            if (r < rows) store_row<T, V>(y + (size_t)r * p.C, o);
        }
    }
    if (p.last && t0 == 0) {
#pragma unroll
        for (int k = 0; k < K - 1; ++k) {
            float v[V];
            load_joined<T, V>(v, x, p.x_ts, st, K, p.C, len - (K - 1) + k, len);
            store_row<T, V>((T*)p.last + ((size_t)b * (K - 1) + k) * p.C + c0, v);
        }
    }
}

// dx[t] = sum_k w[k] g[t + K-1-k], g = dy act'(pre): a run goes K - 1 rows past its end; dw and dbias over its own rows, added up over the
// block's runs and left as one row of sums per block.
template <typename T, int V, int K>
__global__ __launch_bounds__(256) void cconv_bwd_kernel(ga_causal_conv_bwd_params p, Map m, int parts) {
    __shared__ float red[256][V];
    const int px = threadIdx.x % m.px, ry = threadIdx.x / m.px, piece = (blockIdx.x % m.pb) * m.px + px;
    const int part = blockIdx.x / m.pb;
    const bool in = piece < m.pieces;
    const int c0 = in ? piece * V : 0;
    float w[K][V], bias[V], dw[K][V], db[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
        bias[e] = p.bias ? p.bias[c0 + e] : 0.f;
        db[e] = 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            w[k][e] = p.w[(size_t)(c0 + e) * K + k];
            dw[k][e] = 0.f;
        }
    }
    if (in) {
        for (long run = (long)part * m.ry + ry; run < m.runs; run += (long)parts * m.ry) {
            const int b = (int)(run / m.rpi), t0 = (int)(run % m.rpi) * m.run;
            const int len = sq_len(p.lengths, b, p.T), rows = min(m.run, p.T - t0);
            const T* x = (const T*)p.x + (size_t)b * p.x_bs + c0;
            const T* st = p.state ? (const T*)p.state + (size_t)b * (K - 1) * p.C + c0 : nullptr;
            const T* gy = (const T*)p.dy + (size_t)b * p.T * p.C + c0;
            Pack<T, V> xn[K], gn[K];
            auto load = [&](int r0) __attribute__((always_inline)) {
#pragma unroll
                for (int i = 0; i < K; ++i) {
                    const int t = min(t0 + r0 + i, p.T - 1);
                    xn[i] = *(const Pack<T, V>*)(x + (size_t)t * p.x_ts);
                    gn[i] = *(const Pack<T, V>*)(gy + (size_t)t * p.C);
                }
            };
            load(0);
            float win[K][V], acc[K][V];  // the input's and its gradient's rows t - (K-1) .. t, in the same slots
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int e = 0; e < V; ++e) acc[k][e] = 0.f;
#pragma unroll
            for (int k = 0; k < K - 1; ++k) load_joined<T, V>(win[k], x, p.x_ts, st, K, p.C, t0 - (K - 1) + k, len);
            for (int r0 = 0; r0 < rows + K - 1; r0 += K) {
                Pack<T, V> xc[K], gc[K];
#pragma unroll
                for (int i = 0; i < K; ++i) { xc[i] = xn[i]; gc[i] = gn[i]; }
                if (r0 + K < rows + K - 1) load(r0 + K);
#pragma unroll
                for (int i = 0; i < K; ++i) {
                    const int r = r0 + i, t = t0 + r, ns = (K - 1 + i) % K;
                    const bool live = t < len, own = r < rows;
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        win[ns][e] = live ? (float)xc[i].v[e] : 0.f;
                        acc[ns][e] = 0.f;
                        float g = (float)gc[i].v[e];
                        if (p.act == GA_ACT_SILU) {
                            float v = bias[e];
#pragma unroll
                            for (int k = 0; k < K; ++k) v = fmaf(w[k][e], win[(i + k) % K][e], v);
                            g *= sq_silu_slope(v);
                        }
                        g = live ? g : 0.f;
                        const float go = own ? g : 0.f;
                        db[e] += go;
#pragma unroll
                        for (int k = 0; k < K; ++k) {
                            dw[k][e] = fmaf(go, win[(i + k) % K][e], dw[k][e]);
                            acc[(i + k) % K][e] = fmaf(w[k][e], g, acc[(i + k) % K][e]);
                        }
                    }
                    const int td = t - (K - 1);              // this row of dx is complete
                    const int from = td - (len - (K - 1));  // its place among the rows handed on as the window
                    float(&done)[V] = acc[i % K];
                    if (r < rows + K - 1 && (td >= t0 || t0 == 0)) {
                        if (p.dlast && from >= 0 && from < K - 1) {
                            float v[V];
                            load_row<T, V>(v, (const T*)p.dlast + ((size_t)b * (K - 1) + from) * p.C + c0, true);
#pragma unroll
                            for (int e = 0; e < V; ++e) done[e] += v[e];
                        }
                        if (td >= 0) {
                            float v[V];
#pragma unroll
                            for (int e = 0; e < V; ++e) v[e] = td < len ? done[e] : 0.f;
                            store_row<T, V>((T*)p.dx + ((size_t)b * p.T + td) * p.C + c0, v);
                        } else if (p.dstate) {
                            store_row<T, V>((T*)p.dstate + ((size_t)b * (K - 1) + td + K - 1) * p.C + c0, done);
                        }
                    }
                }
            }
        }
    }
#pragma unroll
    for (int k = 0; k <= K; ++k) {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < V; ++e) red[threadIdx.x][e] = k < K ? dw[k < K ? k : 0][e] : db[e];
        __syncthreads();
        if (ry == 0 && in) {
            float v[V];
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] = red[px][e];
            for (int j = 1; j < m.ry; ++j)
#pragma unroll
                for (int e = 0; e < V; ++e) v[e] += red[j * m.px + px][e];
            store_row<float, V>(p.ws + ((size_t)part * (K + 1) + k) * p.C + c0, v);
        }
    }
}

__global__ __launch_bounds__(1024) void cconv_dw_kernel(const float* __restrict__ ws, int parts, int K, int C, float* __restrict__ dw,
                                                        float* __restrict__ db) {
    __shared__ double acc[32][32];
    const long col = (long)blockIdx.x * 32 + (threadIdx.x & 31), cols = (long)(K + 1) * C;
    const double v = sq_groups32(col < cols ? sq_column(ws + col, cols, parts, threadIdx.x >> 5, 32) : 0.0, acc);
    if (threadIdx.x < 32 && col < cols) {
        const int k = (int)(col / C), c = (int)(col % C);
        if (k < K) dw[(size_t)c * K + k] = (float)v;
        else if (db) db[c] = (float)v;
    }
}

template <typename T>
__global__ __launch_bounds__(256) void cconv_step_kernel(ga_causal_conv_step_params p) {
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= (size_t)p.B * p.C) return;
    const int b = (int)(i / p.C), c = (int)(i % p.C);
    T* st = (T*)p.state + (size_t)b * p.state_bs + c;
    const T xn = ((const T*)p.x)[(size_t)b * p.x_bs + c];
    float v = p.bias ? p.bias[c] : 0.f;
    T row[GA_CCONV_MAX_TAPS];
#pragma unroll
    for (int k = 0; k < GA_CCONV_MAX_TAPS; ++k)
        if (k < p.K) {
            row[k] = k < p.K - 1 ? st[(size_t)k * p.C] : xn;
            v = fmaf(p.w[(size_t)c * p.K + k], (float)row[k], v);
        }
#pragma unroll
    for (int k = 0; k < GA_CCONV_MAX_TAPS - 1; ++k)
        if (k < p.K - 1) st[(size_t)k * p.C] = row[k + 1];
    if (p.act == GA_ACT_SILU) v = sq_silu(v);
    ((T*)p.y)[(size_t)b * p.C + c] = (T)v;
}

int bad(int B, int T, int C, int K, int act, int dtype) {
    if (B < 1 || T < 1 || T > 0x7fffffff - 256 || C < 1 || C > 0x7fffffff - 256 || K < 1 || K > GA_CCONV_MAX_TAPS || (act != GA_ACT_NONE && act != GA_ACT_SILU)) return GA_ERR_ARG;
    if (dtype != GA_DTYPE_F32 && dtype != GA_DTYPE_BF16) return GA_ERR_ARG;
    const Map m = make_map(B, T, C, 1);
    if ((m.runs + m.ry - 1) / m.ry * m.pb > 0x7fffffffL) return GA_ERR_ARG;
    return GA_OK;
}

int parts_of(const Map& m) {
    long want = (m.runs + m.ry - 1) / m.ry;
    const long cap = MAX_PARTS / m.pb > 0 ? MAX_PARTS / m.pb : 1;
    return (int)(want < cap ? want : cap);
}

template <typename T, int V, int K>
int fwd(const ga_causal_conv_params& p, hipStream_t s) {
    const Map m = make_map(p.B, p.T, p.C, V);
    const size_t blocks = (size_t)((m.runs + m.ry - 1) / m.ry) * m.pb;
    if (!sq_launch_fits(blocks, 256)) return GA_ERR_ARG;
    cconv_fwd_kernel<T, V, K><<<(unsigned)blocks, 256, 0, s>>>(p, m);
    GA_CHECK_LAUNCH();
    return GA_OK;
}
template <typename T, int V, int K>
int bwd(const ga_causal_conv_bwd_params& p, hipStream_t s) {
    const Map m = make_map(p.B, p.T, p.C, V);
    const int parts = parts_of(m);
    const size_t sums = ((size_t)(K + 1) * p.C + 31) / 32;
    if (!sq_launch_fits((size_t)parts * m.pb, 256) || !sq_launch_fits(sums, 1024)) return GA_ERR_ARG;
    cconv_bwd_kernel<T, V, K><<<(unsigned)(parts * m.pb), 256, 0, s>>>(p, m, parts);
    GA_CHECK_LAUNCH();
    cconv_dw_kernel<<<(unsigned)sums, 1024, 0, s>>>(p.ws, parts, K, p.C, p.dw, p.dbias);
    GA_CHECK_LAUNCH();
    return GA_OK;
}

template <typename T, int V, typename P, typename F> int by_taps(const P& p, F f) {
    // Window, gradients and weights of five taps and more for four channels do not fit the registers.  (K = 8: 16 + 40 us at 64 x 375 x 512 bf16, K = 4
    // 14.6 + 28.6.  Single channels, where widths or bases leave no wider access: K = 4 17.4 + 31.7, at 16 x 2250 x 1024 43 + 84 us against 29 + 60.)
    switch (p.K) {
        case 1: return f.template go<T, V, 1>(p);
        case 2: return f.template go<T, V, 2>(p);
        case 3: return f.template go<T, V, 3>(p);
        case 4: return f.template go<T, V, 4>(p);
        case 5: return f.template go<T, V == 4 ? 2 : V, 5>(p);
        case 6: return f.template go<T, V == 4 ? 2 : V, 6>(p);
        case 7: return f.template go<T, V == 4 ? 2 : V, 7>(p);
        case 8: return f.template go<T, V == 4 ? 2 : V, 8>(p);
        default: return GA_ERR_ARG;
    }
}
struct Fwd { hipStream_t s; template <typename T, int V, int K> int go(const ga_causal_conv_params& p) { return fwd<T, V, K>(p, s); } };
struct Bwd { hipStream_t s; template <typename T, int V, int K> int go(const ga_causal_conv_bwd_params& p) { return bwd<T, V, K>(p, s); } };

bool aligned(const void* p, size_t bytes) { return !((uintptr_t)p & (bytes - 1)); }

}  // namespace

extern "C" {

size_t ga_causal_conv_bwd_ws_elems(int B, int T, int C, int K) {
    if (bad(B, T, C, K, GA_ACT_NONE, GA_DTYPE_F32)) return 0;
    const int one = parts_of(make_map(B, T, C, 1)), vec = parts_of(make_map(B, T, C, K > 4 ? 2 : 4));
    return (size_t)(one > vec ? one : vec) * (K + 1) * C;
}

int ga_causal_conv_fwd(const ga_causal_conv_params* hp, int dtype, hipStream_t s) {
    if (!hp) return GA_ERR_ARG;
    const ga_causal_conv_params& p = *hp;
    const int rc = bad(p.B, p.T, p.C, p.K, p.act, dtype);
    if (rc) return rc;
    if (!p.x || !p.w || !p.y) return GA_ERR_ARG;
    const int v = 4;
    const size_t bytes = v * (dtype == GA_DTYPE_BF16 ? 2 : 4);
    const bool vec = p.C % v == 0 && p.x_bs % v == 0 && p.x_ts % v == 0 && aligned(p.x, bytes) && aligned(p.y, bytes) && aligned(p.state, bytes) &&
                     aligned(p.last, bytes);
    if (dtype == GA_DTYPE_BF16) return vec ? by_taps<bf16_t, 4>(p, Fwd{s}) : by_taps<bf16_t, 1>(p, Fwd{s});
    return vec ? by_taps<float, 4>(p, Fwd{s}) : by_taps<float, 1>(p, Fwd{s});
}

int ga_causal_conv_bwd(const ga_causal_conv_bwd_params* hp, int dtype, hipStream_t s) {
    if (!hp) return GA_ERR_ARG;
    const ga_causal_conv_bwd_params& p = *hp;
    const int rc = bad(p.B, p.T, p.C, p.K, p.act, dtype);
    if (rc) return rc;
    if (!p.x || !p.w || !p.dy || !p.dx || !p.dw || !p.ws) return GA_ERR_ARG;
    if ((uintptr_t)p.ws & 15) return GA_ERR_ALIGN;
    const int v = 4;
    const size_t bytes = v * (dtype == GA_DTYPE_BF16 ? 2 : 4);
    const bool vec = p.C % v == 0 && p.x_bs % v == 0 && p.x_ts % v == 0 && aligned(p.x, bytes) && aligned(p.dy, bytes) && aligned(p.dx, bytes) &&
                     aligned(p.state, bytes) && aligned(p.dstate, bytes) && aligned(p.dlast, bytes);
    if (dtype == GA_DTYPE_BF16) return vec ? by_taps<bf16_t, 4>(p, Bwd{s}) : by_taps<bf16_t, 1>(p, Bwd{s});
    return vec ? by_taps<float, 4>(p, Bwd{s}) : by_taps<float, 1>(p, Bwd{s});
}

int ga_causal_conv_step(const ga_causal_conv_step_params* hp, int dtype, hipStream_t s) {
    if (!hp) return GA_ERR_ARG;
    const ga_causal_conv_step_params& p = *hp;
    const int rc = bad(p.B, 1, p.C, p.K, p.act, dtype);
    if (rc) return rc;
    if (!p.x || !p.w || !p.y || (p.K > 1 && !p.state)) return GA_ERR_ARG;
    const size_t blocks = ((size_t)p.B * p.C + 255) / 256;
    if (!sq_launch_fits(blocks, 256)) return GA_ERR_ARG;
    if (dtype == GA_DTYPE_BF16) cconv_step_kernel<bf16_t><<<(unsigned)blocks, 256, 0, s>>>(p);
    else cconv_step_kernel<float><<<(unsigned)blocks, 256, 0, s>>>(p);
    GA_CHECK_LAUNCH();
    return GA_OK;
}

}  // extern "C"
