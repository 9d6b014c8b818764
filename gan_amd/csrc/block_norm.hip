// The two edges of a residual block in one pass over the rows:
//   n = norm(branch) wp + bp  (or the branch itself),  r = x + scale gate n,  y = (norm(r) w + b) (1 + a) + s
// norm: v / rms(v), or (v - mean) / std.  Statistics and all arithmetic in float32; r and y are rounded once each.  HBM-bound: the forward pass
// reads x, branch (and a gate per row), writes r and y; the backward pass recomputes r from them with the saved statistics, so that r itself
// is not read and its rounding does not enter the gradients.
//
// A row is held in the registers of 64 lanes (one wave) or of a whole block.  Column sums (the parameters' gradients) stay in registers over a
// block's rows and leave as one row of partial sums per block, added up in a fixed order: results do not depend on timing.
#include "seq_common.h"

namespace {

constexpr int MAX_PARTS = 1024;

template <typename T, int V> struct alignas(sizeof(T) * V) Pack { T v[V]; };

template <typename T, int V>
__device__ __forceinline__ void ldv(float* o, const T* p) {
    const Pack<T, V> r = *(const Pack<T, V>*)p;
#pragma unroll
    for (int e = 0; e < V; ++e) o[e] = (float)r.v[e];
}
template <typename T, int V>
__device__ __forceinline__ void stv(T* p, const float* v) {
    Pack<T, V> r;
#pragma unroll
    for (int e = 0; e < V; ++e) r.v[e] = (T)v[e];
    *(Pack<T, V>*)p = r;
}

// sums of two values over a row's threads, in every one of them
template <int G>
__device__ __forceinline__ float2 row_sum2(float2 v, float2 (*red)[4], int& slot) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) { v.x += __shfl_xor(v.x, o, 64); v.y += __shfl_xor(v.y, o, 64); }
    if (G == 64) return v;
    const int w = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) red[slot][w] = v;
    __syncthreads();
    const float2 a = red[slot][0], b = red[slot][1], c = red[slot][2], d = red[slot][3];
    slot ^= 1;  // the other one next: a wave that is ahead by one sum does not write what another still reads
    return make_float2((a.x + b.x) + (c.x + d.x), (a.y + b.y) + (c.y + d.y));
}

// (mean, 1 / sqrt(variance or mean square + eps)) of a row
template <int G, int P, int V>
__device__ __forceinline__ float2 row_stats(const float (&v)[P][V], const bool (&in)[P], int C, bool layer, float eps, float2 (*red)[4], int& slot) {
    float mean = 0.f;
    if (layer) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < P; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e) s += in[i] ? v[i][e] : 0.f;
        mean = row_sum2<G>(make_float2(s, 0.f), red, slot).x / (float)C;
    }
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < P; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float t = in[i] ? v[i][e] - mean : 0.f;
            s = fmaf(t, t, s);
        }
    const float ms = row_sum2<G>(make_float2(s, 0.f), red, slot).x / (float)C;
    return make_float2(mean, 1.f / sqrtf(ms + eps));
}

#define BN_COLUMNS()                                                                  \
    const int tid = G == 64 ? threadIdx.x & 63 : threadIdx.x;                         \
    const int w = G == 64 ? threadIdx.x >> 6 : 0;                                     \
    constexpr int RPB = 256 / G;                                                      \
    __shared__ float2 red[2][4];                                                      \
    int slot = 0;                                                                     \
    int col[P];                                                                       \
    bool in[P];                                                                       \
    _Pragma("unroll") for (int i = 0; i < P; ++i) {                                   \
        col[i] = (i * G + tid) * V;                                                   \
        in[i] = col[i] < p.C;                                                         \
    }

#define BN_EACH _Pragma("unroll") for (int i = 0; i < P; ++i) _Pragma("unroll") for (int e = 0; e < V; ++e)

template <int P, int V>
__device__ __forceinline__ void load_cols(float (&o)[P][V], const float* p, const int (&col)[P], const bool (&in)[P], float none) {
#pragma unroll
    for (int i = 0; i < P; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) o[i][e] = p && in[i] ? p[col[i] + e] : none;
}
template <typename T, int P, int V>
__device__ __forceinline__ void load_rows(float (&o)[P][V], const T* p, const int (&col)[P], const bool (&in)[P]) {
#pragma unroll
    for (int i = 0; i < P; ++i) {
        if (in[i]) ldv<T, V>(o[i], p + col[i]);
        else
#pragma unroll
            for (int e = 0; e < V; ++e) o[i][e] = 0.f;
    }
}

template <typename TX, typename TO, int G, int P, int V>
__global__ __launch_bounds__(256) void bnorm_fwd_kernel(ga_block_norm_params p, int items, long rows_per_item, int parts) {
    BN_COLUMNS();
    const int item = blockIdx.x / parts, part = blockIdx.x % parts;
    float wv[P][V], bv[P][V], wp[P][V], bp[P][V], sc[P][V], a1[P][V], sh[P][V];
    load_cols(wv, p.w, col, in, 1.f);
    load_cols(bv, p.b, col, in, 0.f);
    if (p.ab) {
        load_cols(a1, p.ab + (size_t)item * 2 * p.C, col, in, 0.f);
        load_cols(sh, p.ab + (size_t)item * 2 * p.C + p.C, col, in, 0.f);
        BN_EACH {
            const float a = 1.f + a1[i][e];
            wv[i][e] *= a;
            bv[i][e] = fmaf(bv[i][e], a, sh[i][e]);
        }
    }
    if (p.branch) {
        load_cols(wp, p.wp, col, in, 1.f);
        load_cols(bp, p.bp, col, in, 0.f);
        load_cols(sc, p.scale, col, in, 1.f);
        if (p.gate && !p.gate_rows) {
            load_cols(a1, (const float*)p.gate + (size_t)item * p.C, col, in, 0.f);
            BN_EACH sc[i][e] *= a1[i][e];
        }
    }
    for (long k = (long)part * RPB + w; k < rows_per_item + (G == 64 ? 0 : 0); k += (long)parts * RPB) {
        const size_t row = (size_t)item * rows_per_item + k, off = row * p.C;
        float r[P][V];
        load_rows<TX, P, V>(r, (const TX*)p.x + off, col, in);
        float4 st = make_float4(0.f, 1.f, 0.f, 1.f);
        if (p.branch) {
            float o[P][V], gt[P][V];
            load_rows<TO, P, V>(o, (const TO*)p.branch + off, col, in);
            if (p.gate_rows) load_rows<TO, P, V>(gt, (const TO*)p.gate + off, col, in);
            if (p.post) {
                const float2 s = row_stats<G, P, V>(o, in, p.C, p.layer, p.eps, red, slot);
                st.x = s.x;
                st.y = s.y;
            }
            BN_EACH {
                float n = fmaf((o[i][e] - st.x) * st.y, wp[i][e], bp[i][e]);
                if (p.gate_rows) n *= gt[i][e];
                r[i][e] = fmaf(sc[i][e], n, r[i][e]);
            }
#pragma unroll
            for (int i = 0; i < P; ++i)
                if (in[i]) stv<TX, V>((TX*)p.r + off + col[i], r[i]);
        }
        const float2 s = row_stats<G, P, V>(r, in, p.C, p.layer, p.eps, red, slot);
        st.z = s.x;
        st.w = s.y;
        BN_EACH r[i][e] = fmaf((r[i][e] - s.x) * s.y, wv[i][e], bv[i][e]);
#pragma unroll
        for (int i = 0; i < P; ++i)
            if (in[i]) stv<TO, V>((TO*)p.y + off + col[i], r[i]);
        if (p.stats && tid == 0) *(float4*)(p.stats + row * 4) = st;
    }
}

template <typename TX, typename TO, int G, int P, int V>
__global__ __launch_bounds__(256) void bnorm_bwd_kernel(ga_block_norm_bwd_params p, int items, long rows_per_item, int parts) {
    BN_COLUMNS();
    __shared__ float fold[G == 64 ? 4 : 1][G == 64 ? 64 * P * V : 1];
    const int item = blockIdx.x / parts, part = blockIdx.x % parts;
    const float inv = 1.f / (float)p.C;
    float wv[P][V], wp[P][V], bp[P][V], sc[P][V], tmp[P][V];
    load_cols(wv, p.w, col, in, 1.f);
    if (p.ab) {
        load_cols(tmp, p.ab + (size_t)item * 2 * p.C, col, in, 0.f);
        BN_EACH wv[i][e] *= 1.f + tmp[i][e];
    }
    if (p.branch) {
        load_cols(wp, p.wp, col, in, 1.f);
        load_cols(bp, p.bp, col, in, 0.f);
        load_cols(sc, p.scale, col, in, 1.f);
        if (p.gate && !p.gate_rows) {
            load_cols(tmp, (const float*)p.gate + (size_t)item * p.C, col, in, 0.f);
            BN_EACH sc[i][e] *= tmp[i][e];
        }
    }
    float s0[P][V], s1[P][V], s2[P][V], s3[P][V];
    BN_EACH s0[i][e] = s1[i][e] = s2[i][e] = s3[i][e] = 0.f;
    for (long k = (long)part * RPB + w; k < rows_per_item; k += (long)parts * RPB) {
        const size_t row = (size_t)item * rows_per_item + k, off = row * p.C;
        const float4 st = *(const float4*)(p.stats + row * 4);
        float r[P][V], o[P][V], gt[P][V], q[P][V];
        load_rows<TX, P, V>(r, (const TX*)p.x + off, col, in);
        if (p.branch) {
            load_rows<TO, P, V>(o, (const TO*)p.branch + off, col, in);
            if (p.gate_rows) load_rows<TO, P, V>(gt, (const TO*)p.gate + off, col, in);
            BN_EACH {
                o[i][e] = in[i] ? (o[i][e] - st.x) * st.y : 0.f;
                float n = fmaf(o[i][e], wp[i][e], bp[i][e]);
                if (p.gate_rows) n *= gt[i][e];
                r[i][e] = fmaf(sc[i][e], n, r[i][e]);
            }
        }
        BN_EACH q[i][e] = 0.f;
        if (p.dy) {
            load_rows<TO, P, V>(q, (const TO*)p.dy + off, col, in);
            float2 m = make_float2(0.f, 0.f);
            BN_EACH {
                const float dy = q[i][e];
                r[i][e] = in[i] ? (r[i][e] - st.z) * st.w : 0.f;
                s0[i][e] = fmaf(dy, r[i][e], s0[i][e]);
                s1[i][e] += dy;
                q[i][e] = dy * wv[i][e];
                m.x = fmaf(q[i][e], r[i][e], m.x);
                m.y += q[i][e];
            }
            m = row_sum2<G>(m, red, slot);
            m.x *= inv;
            m.y = p.layer ? m.y * inv : 0.f;
            BN_EACH q[i][e] = st.w * (fmaf(-r[i][e], m.x, q[i][e]) - m.y);
        }
        if (p.dr) {
            load_rows<TX, P, V>(r, (const TX*)p.dr + off, col, in);
            BN_EACH q[i][e] += r[i][e];
        }
#pragma unroll
        for (int i = 0; i < P; ++i)
            if (in[i]) stv<TX, V>((TX*)p.dx + off + col[i], q[i]);
        if (p.branch) {
            float2 m = make_float2(0.f, 0.f);
            if (p.gate_rows) {
                BN_EACH {
                    const float n = fmaf(o[i][e], wp[i][e], bp[i][e]);
                    r[i][e] = q[i][e] * sc[i][e] * n;  // the gate's gradient
                    q[i][e] *= gt[i][e];
                }
#pragma unroll
                for (int i = 0; i < P; ++i)
                    if (in[i]) stv<TO, V>((TO*)p.dgate + off + col[i], r[i]);
            }
            BN_EACH {
                s2[i][e] = fmaf(q[i][e], o[i][e], s2[i][e]);
                s3[i][e] += q[i][e];
                q[i][e] *= sc[i][e] * wp[i][e];
                m.x = fmaf(q[i][e], o[i][e], m.x);
                m.y += q[i][e];
            }
            if (p.post) {
                m = row_sum2<G>(m, red, slot);
                m.x *= inv;
                m.y = p.layer ? m.y * inv : 0.f;
                BN_EACH q[i][e] = st.y * (fmaf(-o[i][e], m.x, q[i][e]) - m.y);
            }
#pragma unroll
            for (int i = 0; i < P; ++i)
                if (in[i]) stv<TO, V>((TO*)p.dbranch + off + col[i], q[i]);
        }
    }
    float* out = p.ws + (size_t)blockIdx.x * 4 * p.C;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        float(&s)[P][V] = j == 0 ? s0 : j == 1 ? s1 : j == 2 ? s2 : s3;
        if (G == 64) {
            __syncthreads();
            BN_EACH fold[w][(i * V + e) * 64 + tid] = s[i][e];
            __syncthreads();
            if (w == 0) BN_EACH {
                const int f = (i * V + e) * 64 + tid;
                s[i][e] = (fold[0][f] + fold[1 % RPB][f]) + (fold[2 % RPB][f] + fold[3 % RPB][f]);
            }
        }
        if (w == 0) {
#pragma unroll
            for (int i = 0; i < P; ++i)
                if (in[i])
#pragma unroll
                    for (int e = 0; e < V; ++e) out[(size_t)j * p.C + col[i] + e] = s[i][e];
        }
    }
}

// one item's sums over its blocks, and the gradients of its own vectors
__global__ __launch_bounds__(256) void bnorm_items_kernel(ga_block_norm_bwd_params p, int parts, float* sums) {
    __shared__ double acc[4][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, item = blockIdx.y;
    const int c = blockIdx.x * 64 + lane;
    double v[4] = {0.0, 0.0, 0.0, 0.0};
    const float* s = p.ws + (size_t)item * parts * 4 * p.C;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (c < p.C)
            for (int k = w; k < parts; k += 4) v[j] += (double)s[((size_t)k * 4 + j) * p.C + c];
        __syncthreads();
        acc[w][lane] = v[j];
        __syncthreads();
        v[j] = (acc[0][lane] + acc[1][lane]) + (acc[2][lane] + acc[3][lane]);
    }
    if (w || c >= p.C) return;
#pragma unroll
    for (int j = 0; j < 4; ++j) sums[((size_t)item * 4 + j) * p.C + c] = (float)v[j];
    if (p.dab) {
        p.dab[(size_t)item * 2 * p.C + c] = (float)((p.w ? (double)p.w[c] : 1.0) * v[0] + (p.b ? (double)p.b[c] : 0.0) * v[1]);
        p.dab[(size_t)item * 2 * p.C + p.C + c] = (float)v[1];
    }
    if (p.gate && !p.gate_rows && p.dgate)
        ((float*)p.dgate)[(size_t)item * p.C + c] =
            (float)((p.scale ? (double)p.scale[c] : 1.0) * ((p.wp ? (double)p.wp[c] : 1.0) * v[2] + (p.bp ? (double)p.bp[c] : 0.0) * v[3]));
}

// the parameters' gradients from `rows` rows of sums (items when `by_item`, else blocks)
__global__ __launch_bounds__(1024) void bnorm_params_kernel(ga_block_norm_bwd_params p, const float* sums, int rows, int by_item) {
    __shared__ double acc[16][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, c = blockIdx.x * 64 + lane;
    double v[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (c < p.C)
            for (int k = w; k < rows; k += 16) {
                double f = 1.0;
                if (by_item && j < 2 && p.ab) f += (double)p.ab[(size_t)k * 2 * p.C + c];
                if (by_item && j >= 2 && p.gate && !p.gate_rows) f = (double)((const float*)p.gate)[(size_t)k * p.C + c];
                v[j] += f * (double)sums[((size_t)k * 4 + j) * p.C + c];
            }
        __syncthreads();
        acc[w][lane] = v[j];
        __syncthreads();
        double t = 0.0;
        for (int k = 0; k < 16; ++k) t += acc[k][lane];
        v[j] = t;
    }
    if (w || c >= p.C) return;
    const double s = p.scale ? (double)p.scale[c] : 1.0, wp = p.wp ? (double)p.wp[c] : 1.0, bp = p.bp ? (double)p.bp[c] : 0.0;
    if (p.dw) p.dw[c] = (float)v[0];
    if (p.db) p.db[c] = (float)v[1];
    if (p.dwp) p.dwp[c] = (float)(s * v[2]);
    if (p.dbp) p.dbp[c] = (float)(s * v[3]);
    if (p.dscale) p.dscale[c] = (float)(wp * v[2] + bp * v[3]);
}

struct Grid {
    int items, parts;
    long rows_per_item;
};
// without vectors of their own the items are one long item
Grid make_grid(int B, int T, bool by_item, int rows_per_block, int most) {
    Grid g;
    g.items = by_item ? B : 1;
    g.rows_per_item = by_item ? T : (long)B * T;
    long parts = (g.rows_per_item + rows_per_block - 1) / rows_per_block;
    const long cap = g.items < most ? most / g.items : 1;
    if (parts > cap) parts = cap;
    g.parts = (int)parts;
    return g;
}

bool aligned(const void* p, size_t bytes) { return !((uintptr_t)p & (bytes - 1)); }

int bad(int B, int T, int C, float eps, int xdt, int dt) {
    if (B < 1 || T < 1 || C < 1 || C > GA_BNORM_MAX_C || !(eps > 0.f)) return GA_ERR_ARG;
    if (dt != GA_DTYPE_F32 && dt != GA_DTYPE_BF16) return GA_ERR_ARG;
    if (xdt != dt && !(xdt == GA_DTYPE_F32 && dt == GA_DTYPE_BF16)) return GA_ERR_ARG;
    if ((long)B * T > 0x7fffffffL) return GA_ERR_ARG;
    return GA_OK;
}

struct Fwd {
    hipStream_t s;
    template <typename TX, typename TO, int G, int P, int V> int go(const ga_block_norm_params& p) {
        const Grid g = make_grid(p.B, p.T, p.ab || (p.gate && !p.gate_rows), 256 / G, 2048);
        bnorm_fwd_kernel<TX, TO, G, P, V><<<(unsigned)(g.items * g.parts), 256, 0, s>>>(p, g.items, g.rows_per_item, g.parts);
        GA_CHECK_LAUNCH();
        return GA_OK;
    }
};
struct Bwd {
    hipStream_t s;
    template <typename TX, typename TO, int G, int P, int V> int go(const ga_block_norm_bwd_params& p) {
        const bool by_item = p.ab || (p.gate && !p.gate_rows);
        const Grid g = make_grid(p.B, p.T, by_item, 256 / G, MAX_PARTS);
        const int blocks = g.items * g.parts;
        bnorm_bwd_kernel<TX, TO, G, P, V><<<(unsigned)blocks, 256, 0, s>>>(p, g.items, g.rows_per_item, g.parts);
        GA_CHECK_LAUNCH();
        const unsigned cb = (unsigned)((p.C + 63) / 64);
        const float* sums = p.ws;
        if (by_item) {
            float* items = p.ws + (size_t)blocks * 4 * p.C;
            for (int i0 = 0; i0 < g.items; i0 += 32768) {  // (a grid's second axis ends at 65535)
                ga_block_norm_bwd_params q = p;
                const int n = g.items - i0 < 32768 ? g.items - i0 : 32768;
                q.ws = p.ws + (size_t)i0 * g.parts * 4 * p.C;
                if (q.dab) q.dab += (size_t)i0 * 2 * p.C;
                if (q.dgate && !p.gate_rows) q.dgate = (float*)q.dgate + (size_t)i0 * p.C;
                bnorm_items_kernel<<<dim3(cb, (unsigned)n), 256, 0, s>>>(q, g.parts, items + (size_t)i0 * 4 * p.C);
                GA_CHECK_LAUNCH();
            }
            sums = items;
        }
        bnorm_params_kernel<<<cb, 1024, 0, s>>>(p, sums, by_item ? g.items : blocks, by_item);
        GA_CHECK_LAUNCH();
        return GA_OK;
    }
};

template <typename TX, typename TO, typename F, typename A>
int by_width(const A& p, bool vec, F f) {
    if (vec) {
        if (p.C <= 256) return f.template go<TX, TO, 64, 1, 4>(p);
        if (p.C <= 512) return f.template go<TX, TO, 64, 2, 4>(p);
        if (p.C <= 1024) return f.template go<TX, TO, 64, 4, 4>(p);
        if (p.C <= 2048) return f.template go<TX, TO, 256, 2, 4>(p);
        if (p.C <= 4096) return f.template go<TX, TO, 256, 4, 4>(p);
        return f.template go<TX, TO, 256, 8, 4>(p);
    }
    if (p.C <= 256) return f.template go<TX, TO, 64, 4, 1>(p);
    if (p.C <= 1024) return f.template go<TX, TO, 256, 4, 1>(p);
    return f.template go<TX, TO, 256, 32, 1>(p);
}
template <typename F, typename A>
int by_type(const A& p, int xdt, int dt, bool vec, F f) {
    if (dt == GA_DTYPE_F32) return by_width<float, float>(p, vec, f);
    return xdt == GA_DTYPE_F32 ? by_width<float, bf16_t>(p, vec, f) : by_width<bf16_t, bf16_t>(p, vec, f);
}

}  // namespace

extern "C" {

size_t ga_block_norm_bwd_ws_elems(int B, int T, int C, int by_item) {
    if (bad(B, T, C, 1.f, GA_DTYPE_F32, GA_DTYPE_F32)) return 0;
    const Grid g = make_grid(B, T, by_item != 0, 1, MAX_PARTS);  // one row a block: at least as many as any launch has
    return ((size_t)g.items * g.parts + (by_item ? (size_t)B : 0)) * 4 * C;
}

int ga_block_norm_fwd(const ga_block_norm_params* hp, int xdtype, int dtype, hipStream_t s) {
    if (!hp) return GA_ERR_ARG;
    const ga_block_norm_params& p = *hp;
    const int rc = bad(p.B, p.T, p.C, p.eps, xdtype, dtype);
    if (rc) return rc;
    if (!p.x || !p.y || (p.branch && !p.r) || (!p.branch && (p.gate || p.post)) || (p.gate_rows && !p.gate)) return GA_ERR_ARG;
    const size_t xb = xdtype == GA_DTYPE_BF16 ? 8 : 16, ob = dtype == GA_DTYPE_BF16 ? 8 : 16;
    const bool vec = p.C % 4 == 0 && aligned(p.x, xb) && aligned(p.r, xb) && aligned(p.branch, ob) && aligned(p.y, ob) && (!p.gate_rows || aligned(p.gate, ob));
    if (p.stats && !aligned(p.stats, 16)) return GA_ERR_ALIGN;
    return by_type(p, xdtype, dtype, vec, Fwd{s});
}

int ga_block_norm_bwd(const ga_block_norm_bwd_params* hp, int xdtype, int dtype, hipStream_t s) {
    if (!hp) return GA_ERR_ARG;
    const ga_block_norm_bwd_params& p = *hp;
    const int rc = bad(p.B, p.T, p.C, 1.f, xdtype, dtype);
    if (rc) return rc;
    if (!p.x || !p.stats || !p.dx || !p.ws || (!p.dy && !p.dr) || (p.branch && !p.dbranch) || (!p.branch && (p.gate || p.post)) ||
        (p.gate_rows && (!p.gate || !p.dgate)))
        return GA_ERR_ARG;
    const size_t xb = xdtype == GA_DTYPE_BF16 ? 8 : 16, ob = dtype == GA_DTYPE_BF16 ? 8 : 16;
    const bool vec = p.C % 4 == 0 && aligned(p.x, xb) && aligned(p.dr, xb) && aligned(p.dx, xb) && aligned(p.branch, ob) && aligned(p.dy, ob) &&
                     aligned(p.dbranch, ob) && (!p.gate_rows || (aligned(p.gate, ob) && aligned(p.dgate, ob)));
    if (!aligned(p.stats, 16)) return GA_ERR_ALIGN;
    return by_type(p, xdtype, dtype, vec, Bwd{s});
}

}  // extern "C"
