// The two edges of a residual block in one pass over the rows:
//   n = norm(branch) wp + bp  (or the branch itself),  r = x + scale gate n,  y = (norm(r) w + b) (1 + a) + s
// norm: v / rms(v), or (v - mean) / std.  Statistics and all arithmetic in float32; r and y are rounded once each.  HBM-bound: the forward pass
// reads x, branch (and a gate per row), writes r and y; the backward pass recomputes r from them with the saved statistics, so that r itself
// is not read and its rounding does not enter the gradients.
//
// A row is held in the registers of 64 lanes (one wave) or of a whole block.  Column sums (the parameters' gradients) stay in registers over a
// block's rows and leave as one row of partial sums per block, added up in a fixed order: results do not depend on timing.
//
// Measured at 16 x 2250 x 1024, residual float32, the rest bf16, a gate per row: forward 106 us (516 MB: 4.9 TB/s, what a large copy reaches),
// backward 159 us (811 MB: 5.1 TB/s) and 10 us for the parameter sums; all float32 148 us (737 MB: 5.0 TB/s) and 251 us with the sums (1180 MB:
// 4.7 TB/s).  64 x 375 x 512 bf16: 22 and 38 us, float32 34 and 61; one row of 64 items: 5 us.
#include "seq_common.h"

namespace {

constexpr int MAX_PARTS = 1024;  // blocks of a backward launch at the most, each with a row of sums

template <typename T, int V> struct alignas(sizeof(T) * V) Pack { T v[V]; };

template <typename T, int V>
__device__ __forceinline__ void stv(T* p, unsigned col, const float* v) {
    Pack<T, V> r;
#pragma unroll
    for (int e = 0; e < V; ++e) r.v[e] = (T)v[e];
    *(Pack<T, V>*)((char*)sq_scalar(p) + col * (unsigned)sizeof(T)) = r;
}

// sums of K values over the G threads of a row, in every one of them
template <int G, int K>
__device__ __forceinline__ void row_sums(float (&v)[K], float (*red)[8][16], int& slot) {
    const int lane = threadIdx.x & 63;
    const float s = sq_lane_sums<K>(v, lane);  // value k in the lanes from k * 64 / K on
    if (G == 64) {
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(s), k * (64 / K)));
        return;
    }
    if (lane % (64 / K) == 0) red[slot][lane / (64 / K)][threadIdx.x >> 6] = s;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
        v[k] = 0.f;
#pragma unroll
        for (int i = 0; i < G / 64; i += 4) {
            const float4 t = *(const float4*)(red[slot][k] + i);
            v[k] += (t.x + t.y) + (t.z + t.w);
        }
    }
    slot ^= 1;  // the other one next: a wave that is ahead by one sum does not write what another still reads
}

#define BN_COLUMNS()                                                                  \
    const int tid = G == 64 ? threadIdx.x & 63 : threadIdx.x;                         \
    const int w = G == 64 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;     \
    constexpr int RPB = G == 64 ? 4 : 1;                                              \
    __shared__ __attribute__((aligned(16))) float red[2][8][16];                      \
    int slot = 0;                                                                     \
    unsigned col[P];                                                                  \
    bool in[P];                                                                       \
    const float inv = 1.f / (float)p.C;                                               \
    _Pragma("unroll") for (int i = 0; i < P; ++i) {                                   \
        col[i] = (unsigned)(i * G + tid) * V;                                         \
        in[i] = col[i] < (unsigned)p.C;                                               \
        if (!in[i]) col[i] = 0; /* (read, never used or written) */                   \
    }

#define BN_EACH _Pragma("unroll") for (int i = 0; i < P; ++i) _Pragma("unroll") for (int e = 0; e < V; ++e)
#define BN_ROWS _Pragma("unroll") for (int j = 0; j < R; ++j)

template <int P, int V>
__device__ __forceinline__ void load_cols(float (&o)[P][V], const float* p, const unsigned (&col)[P], const bool (&in)[P], float none) {
#pragma unroll
    for (int i = 0; i < P; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float v = p ? sq_scalar(p)[col[i] + e] : none;
            o[i][e] = in[i] ? v : none;
        }
}
template <typename T, int P, int V>
__device__ __forceinline__ void load_raw(Pack<T, V> (&o)[P], const T* p, const unsigned (&col)[P]) {
#pragma unroll
    for (int i = 0; i < P; ++i) o[i] = *(const Pack<T, V>*)((const char*)sq_scalar(p) + col[i] * (unsigned)sizeof(T));
}
template <typename T, int P, int V>
__device__ __forceinline__ void convert(float (&o)[P][V], const Pack<T, V> (&r)[P]) {
    BN_EACH o[i][e] = (float)r[i].v[e];
}

// (mean, 1 / sqrt(variance or mean square + eps)) of R rows; the variance about the mean, in a second sum.  The squares are of v 2^-8 and their mean
// is multiplied by 2^16 again: 4096 squares of 1e18 add up to 4e39, beyond float32, where their mean is not.  (Both factors are exact, and the first
// comes with the subtraction: the same bits and the same instructions as without.  Squares that get below float32's normal numbers that way, 8e-34, are
// nothing beside an eps of 1e-30 to 24 bits, denormal as they are.)
constexpr float SQ_DOWN = 1.f / 256.f, SQ_UP = 65536.f;
template <int G, int P, int V, int R>
__device__ __forceinline__ void row_stats(const float (&v)[R][P][V], float (&mean)[R], float (&rstd)[R], const bool (&in)[P], float inv, bool layer,
                                          float eps, float (*red)[8][16], int& slot) {
    float s[R];
    BN_ROWS mean[j] = 0.f;
    if (layer) {
        BN_ROWS {
            s[j] = 0.f;
            BN_EACH s[j] += in[i] ? v[j][i][e] : 0.f;
        }
        row_sums<G, R>(s, red, slot);
        BN_ROWS mean[j] = s[j] * inv;
    }
    BN_ROWS {
        s[j] = 0.f;
        BN_EACH {
            const float t = in[i] ? fmaf(v[j][i][e], SQ_DOWN, -SQ_DOWN * mean[j]) : 0.f;
            s[j] = fmaf(t, t, s[j]);
        }
    }
    row_sums<G, R>(s, red, slot);
    BN_ROWS rstd[j] = 1.f / sqrtf(fmaf(s[j], inv * SQ_UP, eps));
}

// G threads a row, P pieces of V columns a thread, R rows at a time: their loads are in flight together and their sums share the exchanges.
// (One row at a time against this: 16 x 2250 x 1024 102 + 173 against 105 + 169 us, 64 x 375 x 256 13.5 + 26.8 against 12.4 + 28.0; one row an
// item 4.4 against 5.0.)
template <typename TX, typename TO, int G, int P, int V, int R>
__global__ __launch_bounds__(G == 64 ? 256 : G) void bnorm_fwd_kernel(ga_block_norm_params p, long rows_per_item, int parts) {
    BN_COLUMNS();
    const int item = blockIdx.x / parts, part = blockIdx.x % parts;
    float wv[P][V], bv[P][V], wp[P][V], bp[P][V], sc[P][V], tmp[P][V];
    load_cols(wv, p.w, col, in, 1.f);
    load_cols(bv, p.b, col, in, 0.f);
    if (p.ab) {
        load_cols(tmp, p.ab + (size_t)item * 2 * p.C, col, in, 0.f);
        BN_EACH { wv[i][e] = fmaf(wv[i][e], tmp[i][e], wv[i][e]); bv[i][e] = fmaf(bv[i][e], tmp[i][e], bv[i][e]); }
        load_cols(tmp, p.ab + (size_t)item * 2 * p.C + p.C, col, in, 0.f);
        BN_EACH bv[i][e] += tmp[i][e];
    }
    load_cols(wp, p.branch ? p.wp : nullptr, col, in, 1.f);
    load_cols(bp, p.branch ? p.bp : nullptr, col, in, 0.f);
    load_cols(sc, p.branch ? p.scale : nullptr, col, in, 1.f);
    if (p.gate && !p.gate_rows) {
        load_cols(tmp, (const float*)p.gate + (size_t)item * p.C, col, in, 0.f);
        BN_EACH sc[i][e] *= tmp[i][e];
    }
    const size_t row0 = (size_t)item * rows_per_item;
    for (long k = ((long)part * RPB + w) * R; k < rows_per_item; k += (long)parts * RPB * R) {
        size_t off[R];
        Pack<TX, V> xr[R][P];
        Pack<TO, V> orw[R][P], gr[R][P];
        BN_ROWS {
            off[j] = (row0 + min(k + j, rows_per_item - 1)) * p.C;
            load_raw<TX, P, V>(xr[j], (const TX*)p.x + off[j], col);
            if (p.branch) load_raw<TO, P, V>(orw[j], (const TO*)p.branch + off[j], col);
            if (p.gate_rows) load_raw<TO, P, V>(gr[j], (const TO*)p.gate + off[j], col);
        }
        float r[R][P][V], om[R], os[R], rm[R], rs[R];
        BN_ROWS { convert(r[j], xr[j]); om[j] = 0.f; os[j] = 1.f; }
        if (p.branch) {
            float o[R][P][V];
            BN_ROWS convert(o[j], orw[j]);
            if (p.post) row_stats<G, P, V, R>(o, om, os, in, inv, p.layer, p.eps, red, slot);
            BN_ROWS {
                BN_EACH {
                    float n = fmaf((o[j][i][e] - om[j]) * os[j], wp[i][e], bp[i][e]);
                    if (p.gate_rows) n *= (float)gr[j][i].v[e];
                    r[j][i][e] = fmaf(sc[i][e], n, r[j][i][e]);
                }
                if (k + j < rows_per_item) {
#pragma unroll
                    for (int i = 0; i < P; ++i)
                        if (in[i]) stv<TX, V>((TX*)p.r + off[j], col[i], r[j][i]);
                }
            }
        }
        row_stats<G, P, V, R>(r, rm, rs, in, inv, p.layer, p.eps, red, slot);
        BN_ROWS {
            if (k + j >= rows_per_item) break;
            BN_EACH r[j][i][e] = fmaf((r[j][i][e] - rm[j]) * rs[j], wv[i][e], bv[i][e]);
#pragma unroll
            for (int i = 0; i < P; ++i)
                if (in[i]) stv<TO, V>((TO*)p.y + off[j], col[i], r[j][i]);
            if (p.stats && tid == 0) *(float4*)(p.stats + (row0 + k + j) * 4) = make_float4(om[j], os[j], rm[j], rs[j]);
        }
    }
}

template <typename TX, typename TO, int G, int P, int V, int R>
__global__ __launch_bounds__(G == 64 ? 256 : G) void bnorm_bwd_kernel(ga_block_norm_bwd_params p, long rows_per_item, int parts) {
    BN_COLUMNS();
    __shared__ float fold[G == 64 ? 4 : 1][G == 64 ? 64 * P * V : 1];
    const int item = blockIdx.x / parts, part = blockIdx.x % parts;
    float wv[P][V], wp[P][V], bp[P][V], sc[P][V], tmp[P][V];
    load_cols(wv, p.w, col, in, 1.f);
    if (p.ab) {
        load_cols(tmp, p.ab + (size_t)item * 2 * p.C, col, in, 0.f);
        BN_EACH wv[i][e] = fmaf(wv[i][e], tmp[i][e], wv[i][e]);
    }
    load_cols(wp, p.branch ? p.wp : nullptr, col, in, 1.f);
    load_cols(bp, p.branch ? p.bp : nullptr, col, in, 0.f);
    load_cols(sc, p.branch ? p.scale : nullptr, col, in, 1.f);
    if (p.gate && !p.gate_rows) {
        load_cols(tmp, (const float*)p.gate + (size_t)item * p.C, col, in, 0.f);
        BN_EACH sc[i][e] *= tmp[i][e];
    }
    float s0[P][V], s1[P][V], s2[P][V], s3[P][V];
    BN_EACH s0[i][e] = s1[i][e] = s2[i][e] = s3[i][e] = 0.f;
    const size_t row0 = (size_t)item * rows_per_item;
    for (long k = ((long)part * RPB + w) * R; k < rows_per_item; k += (long)parts * RPB * R) {
        size_t off[R];
        bool live[R];
        Pack<TX, V> xr[R][P], dr[R][P];
        Pack<TO, V> orw[R][P], gr[R][P], dyr[R][P];
        float4 st[R];
        BN_ROWS {
            live[j] = k + j < rows_per_item;
            const size_t row = row0 + min(k + j, rows_per_item - 1);
            off[j] = row * p.C;
            st[j] = *(const float4*)(p.stats + row * 4);
            load_raw<TX, P, V>(xr[j], (const TX*)p.x + off[j], col);
            if (p.branch) load_raw<TO, P, V>(orw[j], (const TO*)p.branch + off[j], col);
            if (p.gate_rows) load_raw<TO, P, V>(gr[j], (const TO*)p.gate + off[j], col);
            if (p.dy) load_raw<TO, P, V>(dyr[j], (const TO*)p.dy + off[j], col);
            if (p.dr) load_raw<TX, P, V>(dr[j], (const TX*)p.dr + off[j], col);
        }
        float q[R][P][V], o[R][P][V], m[2 * R];
        BN_ROWS BN_EACH q[j][i][e] = o[j][i][e] = 0.f;
        if (p.branch) BN_ROWS BN_EACH o[j][i][e] = in[i] ? ((float)orw[j][i].v[e] - st[j].x) * st[j].y : 0.f;
        if (p.dy) {
            float r[R][P][V];
            BN_ROWS {
                m[j] = m[R + j] = 0.f;
                BN_EACH {
                    float v = (float)xr[j][i].v[e];
                    if (p.branch) {
                        float n = fmaf(o[j][i][e], wp[i][e], bp[i][e]);
                        if (p.gate_rows) n *= (float)gr[j][i].v[e];
                        v = fmaf(sc[i][e], n, v);
                    }
                    v = in[i] && live[j] ? (v - st[j].z) * st[j].w : 0.f;
                    const float dy = in[i] && live[j] ? (float)dyr[j][i].v[e] : 0.f;
                    s0[i][e] = fmaf(dy, v, s0[i][e]);
                    s1[i][e] += dy;
                    r[j][i][e] = v;
                    q[j][i][e] = dy * wv[i][e];
                    m[j] = fmaf(q[j][i][e], v, m[j]);
                    m[R + j] += q[j][i][e];
                }
            }
            row_sums<G, 2 * R>(m, red, slot);
            BN_ROWS {
                const float a = m[j] * inv, b = p.layer ? m[R + j] * inv : 0.f;
                BN_EACH q[j][i][e] = st[j].w * (fmaf(-r[j][i][e], a, q[j][i][e]) - b);
            }
        }
        BN_ROWS {
            if (p.dr) BN_EACH q[j][i][e] += in[i] && live[j] ? (float)dr[j][i].v[e] : 0.f;
#pragma unroll
            for (int i = 0; i < P; ++i)
                if (in[i] && live[j]) stv<TX, V>((TX*)p.dx + off[j], col[i], q[j][i]);
        }
        if (p.branch) {
            BN_ROWS {
                m[j] = m[R + j] = 0.f;
                if (p.gate_rows) {
                    float dg[P][V];
                    BN_EACH {
                        dg[i][e] = q[j][i][e] * sc[i][e] * fmaf(o[j][i][e], wp[i][e], bp[i][e]);
                        q[j][i][e] *= live[j] ? (float)gr[j][i].v[e] : 0.f;
                    }
#pragma unroll
                    for (int i = 0; i < P; ++i)
                        if (in[i] && live[j]) stv<TO, V>((TO*)p.dgate + off[j], col[i], dg[i]);
                }
                BN_EACH {
                    const float v = in[i] && live[j] ? q[j][i][e] : 0.f;
                    s2[i][e] = fmaf(v, o[j][i][e], s2[i][e]);
                    s3[i][e] += v;
                    q[j][i][e] = v * (sc[i][e] * wp[i][e]);
                    m[j] = fmaf(q[j][i][e], o[j][i][e], m[j]);
                    m[R + j] += q[j][i][e];
                }
            }
            if (p.post) row_sums<G, 2 * R>(m, red, slot);
            BN_ROWS {
                const float a = p.post ? m[j] * inv : 0.f, b = p.post && p.layer ? m[R + j] * inv : 0.f;
                BN_EACH q[j][i][e] = st[j].y * (fmaf(-o[j][i][e], a, q[j][i][e]) - b);
#pragma unroll
                for (int i = 0; i < P; ++i)
                    if (in[i] && live[j]) stv<TO, V>((TO*)p.dbranch + off[j], col[i], q[j][i]);
            }
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
                if (in[i]) stv<float, V>(out + (size_t)j * p.C, col[i], s[i]);
        }
    }
}

// one item's sums over its blocks, and the gradients of its own vectors; a block is 32 columns
__global__ __launch_bounds__(256) void bnorm_items_kernel(ga_block_norm_bwd_params p, int parts, float* sums) {
    __shared__ double acc[4][8][32];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, item = blockIdx.y, c = blockIdx.x * 32 + lane;
    const float* s = p.ws + (size_t)item * parts * 4 * p.C;
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[j][w][lane] = c < p.C ? sq_column(s + (size_t)j * p.C + c, (size_t)4 * p.C, parts, w, 8) : 0.0;
    __syncthreads();
    if (w || c >= p.C) return;
    double v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        v[j] = 0.0;
        for (int k = 0; k < 8; ++k) v[j] += acc[j][k][lane];
        sums[((size_t)item * 4 + j) * p.C + c] = (float)v[j];
    }
    if (p.dab) {
        p.dab[(size_t)item * 2 * p.C + c] = (float)((p.w ? (double)p.w[c] : 1.0) * v[0] + (p.b ? (double)p.b[c] : 0.0) * v[1]);
        p.dab[(size_t)item * 2 * p.C + p.C + c] = (float)v[1];
    }
    if (p.gate && !p.gate_rows && p.dgate)
        ((float*)p.dgate)[(size_t)item * p.C + c] =
            (float)((p.scale ? (double)p.scale[c] : 1.0) * ((p.wp ? (double)p.wp[c] : 1.0) * v[2] + (p.bp ? (double)p.bp[c] : 0.0) * v[3]));
}

// the parameters' gradients from `rows` rows of sums (items when `by_item`, else blocks); blockIdx.y: the norm in front / behind
__global__ __launch_bounds__(1024) void bnorm_params_kernel(ga_block_norm_bwd_params p, const float* sums, int rows, int by_item) {
    __shared__ double acc[32][32];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, c = blockIdx.x * 32 + lane, back = blockIdx.y;
    double v[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const float* s = sums + (size_t)(2 * back + j) * p.C + c;
        double t = 0.0;
        if (c < p.C) {
            if (by_item && (back ? p.gate && !p.gate_rows : p.ab != nullptr)) {
                for (int k = w; k < rows; k += 32) {
                    const double f = back ? (double)((const float*)p.gate)[(size_t)k * p.C + c] : 1.0 + (double)p.ab[(size_t)k * 2 * p.C + c];
                    t += f * (double)s[(size_t)k * 4 * p.C];
                }
            } else t = sq_column(s, (size_t)4 * p.C, rows, w, 32);
        }
        v[j] = sq_groups32(t, acc);
    }
    if (w || c >= p.C) return;
    if (!back) {
        if (p.dw) p.dw[c] = (float)v[0];
        if (p.db) p.db[c] = (float)v[1];
        return;
    }
    const double s = p.scale ? (double)p.scale[c] : 1.0, wp = p.wp ? (double)p.wp[c] : 1.0, bp = p.bp ? (double)p.bp[c] : 0.0;
    if (p.dwp) p.dwp[c] = (float)(s * v[0]);
    if (p.dbp) p.dbp[c] = (float)(s * v[1]);
    if (p.dscale) p.dscale[c] = (float)(wp * v[0] + bp * v[1]);
}

struct Grid {
    int items, parts;
    long rows_per_item;
};
// Without vectors of their own the items are one long item.  As many blocks as fit the card at once (`most`: more leave a last, partly filled
// round: 64 x 375 x 512 bf16 takes 21.7 + 38.4 us, 24.8 + 44.7 with four blocks a CU where fewer fit), and no more than the same number of turns
// over the rows needs.
Grid make_grid(int B, int T, bool by_item, int rows_per_turn, int most) {
    Grid g;
    g.items = by_item ? B : 1;
    g.rows_per_item = by_item ? T : (long)B * T;
    const long cap = g.items < most ? most / g.items : 1;
    const long turns = (g.rows_per_item + cap * rows_per_turn - 1) / (cap * rows_per_turn);
    g.parts = (int)((g.rows_per_item + turns * rows_per_turn - 1) / (turns * rows_per_turn));
    return g;
}
template <typename K>
int resident_blocks(K kernel, int threads) {
    int per_cu = 0;
    if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&per_cu, kernel, threads, 0) != hipSuccess || per_cu < 1) per_cu = 1;
    return 256 * (per_cu < 4 ? per_cu : 4);  // (the card's 256 CUs; MAX_PARTS at the most, which sizes the workspace)
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
    static constexpr int R(int fwd, int) { return fwd; }
    template <typename TX, typename TO, int G, int P, int V, int R> int go(const ga_block_norm_params& p) {
        constexpr int threads = G == 64 ? 256 : G;
        static const int most = resident_blocks(bnorm_fwd_kernel<TX, TO, G, P, V, R>, threads);
        const Grid g = make_grid(p.B, p.T, p.ab || (p.gate && !p.gate_rows), (G == 64 ? 4 : 1) * R, most);
        if (!sq_launch_fits((size_t)g.items * g.parts, threads)) return GA_ERR_ARG;
        bnorm_fwd_kernel<TX, TO, G, P, V, R><<<(unsigned)(g.items * g.parts), threads, 0, s>>>(p, g.rows_per_item, g.parts);
        GA_CHECK_LAUNCH();
        return GA_OK;
    }
};
struct Bwd {
    hipStream_t s;
    static constexpr int R(int, int bwd) { return bwd; }
    template <typename TX, typename TO, int G, int P, int V, int R> int go(const ga_block_norm_bwd_params& p) {
        const bool by_item = p.ab || (p.gate && !p.gate_rows);
        constexpr int threads = G == 64 ? 256 : G;
        static const int most = resident_blocks(bnorm_bwd_kernel<TX, TO, G, P, V, R>, threads);
        const Grid g = make_grid(p.B, p.T, by_item, (G == 64 ? 4 : 1) * R, most);
        if (!sq_launch_fits((size_t)g.items * g.parts, threads)) return GA_ERR_ARG;
        const int blocks = g.items * g.parts;
        bnorm_bwd_kernel<TX, TO, G, P, V, R><<<(unsigned)blocks, threads, 0, s>>>(p, g.rows_per_item, g.parts);
        GA_CHECK_LAUNCH();
        const unsigned cb = (unsigned)((p.C + 31) / 32);
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
        bnorm_params_kernel<<<dim3(cb, p.branch ? 2 : 1), 1024, 0, s>>>(p, sums, by_item ? g.items : blocks, by_item);
        GA_CHECK_LAUNCH();
        return GA_OK;
    }
};

// Quads of columns where the width and the bases allow (16 x 562 x 4096 bf16 58 + 121 us; single columns 62 + 126).  Up to 512 columns a row is a
// wave's: 64 x 375 x 512 takes 22 + 39 us, and 34 + 58 with 256 threads a row, half of them idle.  A wave with 1024 columns does not fit the
// registers (22 to 39 spilled in the backward kernel).
template <typename TX, typename TO, typename F, typename A>
int by_width(const A& p, bool vec, F f) {
    if (vec) {
        if (p.C <= 256) return f.template go<TX, TO, 64, 1, 4, F::R(4, 2)>(p);
        if (p.C <= 512) return f.template go<TX, TO, 64, 2, 4, F::R(2, 1)>(p);
        if (p.C <= 1024) return f.template go<TX, TO, 256, 1, 4, F::R(4, 2)>(p);
        if (p.C <= 2048) return f.template go<TX, TO, 256, 2, 4, F::R(2, 1)>(p);
        return f.template go<TX, TO, 512, 2, 4, 1>(p);
    }
    if (p.C <= 256) return f.template go<TX, TO, 64, 4, 1, F::R(2, 1)>(p);
    if (p.C <= 1024) return f.template go<TX, TO, 256, 4, 1, F::R(2, 1)>(p);
    return f.template go<TX, TO, 512, 8, 1, 1>(p);
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
    const size_t items = by_item ? (size_t)B : 1, rows = by_item ? (size_t)T : (size_t)B * T, cap = items < MAX_PARTS ? MAX_PARTS / items : 1;
    return (items * (rows < cap ? rows : cap) + (by_item ? items : 0)) * 4 * C;
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
    if (!aligned(p.stats, 16) || !aligned(p.ws, 16)) return GA_ERR_ALIGN;
    return by_type(p, xdtype, dtype, vec, Bwd{s});
}

}  // extern "C"
