// Selective state space scan:  h_t = exp(D_t A) h_{t-1} + D_t u_t B_t,  y_t = (<C_t, h_t> + D u_t) silu(z_t),  D_t = softplus(delta_t + bias)
// per channel d and state n, on channels-last activations; forward, backward and the single-token step.
//
// One block is 64 channels (one per lane) times all states (split over its four waves: a lane holds its wave's states in registers), walking
// along time in tiles of 16 rows.  What depends on a row and a channel alone (softplus, gates, the sums over states) is done once, four rows to
// a wave, and passes through LDS; B and C, which all channels of a group share, are first laid out in float32 in the order in which
// the waves read them (scan_maps_kernel) and come in as scalar loads, so that they cost no vector instruction and no LDS bandwidth.
#include "seq_common.h"
#include <stdlib.h>

namespace {

constexpr int TS = 16;          // rows of a tile
constexpr int RPW = TS / 4;     // rows that one wave prepares and finishes
constexpr int MAX_CHUNKS = 64;  // a block adds up the chunks before (behind) its own one by one

typedef const __attribute__((address_space(4))) float* uniform_ptr;

struct Plan {
    int NS, NP;               // states of a wave, of the four waves
    int Cg, cbg, nCb;         // channels of a group, 64-channel blocks of a group, of all groups
    int tiles;                // of a sequence
    int chunks, chunk_tiles;  // tiles of a chunk
};

Plan make_plan(int B, int T, int C, int N, int G) {
    Plan q;
    q.NS = N <= 4 ? 1 : N <= 8 ? 2 : N <= 16 ? 4 : N <= 32 ? 8 : 16;
    q.NP = 4 * q.NS;
    q.Cg = C / G;
    q.cbg = (q.Cg + 63) / 64;
    q.nCb = q.cbg * G;
    q.tiles = (T + TS - 1) / TS;
    const long blocks = (long)B * q.nCb;
    static const long target = getenv("SCAN_BLOCKS") ? atol(getenv("SCAN_BLOCKS")) : 1024;
    long want = (target + blocks - 1) / blocks;
    if (want > MAX_CHUNKS) want = MAX_CHUNKS;
    if (want > q.tiles) want = q.tiles;
    if (want < 1) want = 1;
    q.chunk_tiles = (int)((q.tiles + want - 1) / want);
    q.chunks = (q.tiles + q.chunk_tiles - 1) / q.chunk_tiles;
    return q;
}

struct Args {
    ga_scan_params p;
    Plan q;
};
struct BwdArgs {
    ga_scan_bwd_params p;
    Plan q;
};

// maps[b][group][tile][wave][row][B: NS | C: NS] in float32, wave w holding the states w NS .. w NS + NS - 1; zero rows behind an item's length and
// up to the whole tile, zero states behind N
template <typename T>
__global__ __launch_bounds__(256) void scan_maps_kernel(const T* __restrict__ Bm, const T* __restrict__ Cm, float* __restrict__ maps,
                                                        const int* __restrict__ lengths, Plan q, int B, int Tn, int N, int G, long b_bs,
                                                        long b_ts, long c_bs, long c_ts) {
    const size_t total = (size_t)B * G * q.tiles * TS * q.NP;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (size_t)gridDim.x * 256) {
        const int j = (int)(i % q.NS);
        const size_t row = i / q.NS;  // of a wave
        const int r = (int)(row % TS), w = (int)(row / TS % 4);
        const size_t bgt = row / (4 * TS);
        const int t = (int)(bgt % q.tiles) * TS + r, g = (int)(bgt / q.tiles % G), b = (int)(bgt / q.tiles / G), n = w * q.NS + j;
        const bool live = n < N && t < sq_len(lengths, b, Tn);
        const float vb = live ? (float)Bm[(size_t)b * b_bs + (size_t)t * b_ts + (size_t)g * N + n] : 0.f;
        const float vc = live ? (float)Cm[(size_t)b * c_bs + (size_t)t * c_ts + (size_t)g * N + n] : 0.f;
        maps[row * 2 * q.NS + j] = vb;
        maps[row * 2 * q.NS + q.NS + j] = vc;
    }
}

// where a block and a lane are
struct Place {
    int lane, w, chunk, b, g, d, len, tile0, tile1;
    bool ok;
    size_t item;  // first tile of the item's group in the maps
};
__device__ __forceinline__ Place place(const Plan& q, int nch, int first_chunk, int G, int T, const int* lengths) {
    Place x;
    x.lane = threadIdx.x & 63;
    x.w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int cb = blockIdx.x % q.nCb, rest = blockIdx.x / q.nCb;
    x.chunk = first_chunk + rest % nch;
    x.b = rest / nch;
    x.g = cb / q.cbg;
    const int din = (cb % q.cbg) * 64 + x.lane;
    x.ok = din < q.Cg;
    x.d = x.g * q.Cg + (x.ok ? din : q.Cg - 1);
    x.len = sq_len(lengths, x.b, T);
    x.tile0 = x.chunk * q.chunk_tiles;
    x.tile1 = min(x.tile0 + q.chunk_tiles, q.tiles);
    x.item = (size_t)(x.b * G + x.g) * q.tiles;
    return x;
}

// carry[s] <- exp(A sum of steps) carry[s] + end state, over the chunks from, from + dir, ... (count of them), eight loads in flight
template <int NS>
__device__ __forceinline__ void chain(float (&carry)[NS], const float (&A2)[NS], const float* ends, const float* ends_step, const Plan& q, int C, int b,
                                      int w, int d, int from, int dir, int count) {
    constexpr int U = NS <= 4 ? 8 : NS <= 8 ? 4 : 2;
    for (int k = 0; k < count; k += U) {
        float sum[U], end[U][NS];
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const size_t e = (size_t)b * q.chunks + (from + dir * min(k + i, count - 1));
            sum[i] = ends_step[e * C + d];
#pragma unroll
            for (int s = 0; s < NS; ++s) end[i][s] = ends[(e * q.NP + w * NS + s) * C + d];
        }
#pragma unroll
        for (int i = 0; i < U; ++i)
            if (k + i < count) {
#pragma unroll
                for (int s = 0; s < NS; ++s) carry[s] = fmaf(__builtin_amdgcn_exp2f(sum[i] * A2[s]), carry[s], end[i][s]);
            }
    }
}

// ENDS: only the state that each chunk but the last leaves behind when it starts from zero, and the sum of its steps
// (the chunk's decay is exp(A * that sum)).  Otherwise the outputs, each chunk from the states of the chunks before it.
template <typename T, int NS, bool ENDS>
__global__ __launch_bounds__(256) void scan_fwd_kernel(Args a) {
    const ga_scan_params& p = a.p;
    const Plan& q = a.q;
    // rows whose B and C are in scalar registers at a time, twice (one set on its way)
    constexpr int U = ENDS ? (NS <= 4 ? 4 : NS <= 8 ? 2 : 1) : (NS <= 4 ? 2 : 1);
    __shared__ float2 sd[TS][64];
    __shared__ float sy[ENDS ? 1 : 4][ENDS ? 1 : TS][64];
    const Place x = place(q, ENDS ? q.chunks - 1 : q.chunks, 0, p.G, p.T, p.lengths);
    const int lane = x.lane, w = x.w, d = x.d, len = x.len;
    const float bias = p.delta_bias ? p.delta_bias[d] : 0.f, Dd = p.D ? p.D[d] : 0.f;
    float A2[NS], h[NS];
#pragma unroll
    for (int s = 0; s < NS; ++s) {
        const int n = w * NS + s;
        A2[s] = n < p.N ? p.A[(size_t)d * p.N + n] * SQ_LOG2E : 0.f;
        h[s] = 0.f;
        if (!ENDS && p.state && n < p.N) h[s] = p.state[((size_t)x.b * p.C + d) * p.N + n];
    }
    const T* up = (const T*)p.u + (size_t)x.b * p.u_bs;
    const T* dp = (const T*)p.delta + (size_t)x.b * p.delta_bs;
    const T* zp = ENDS || !p.z ? nullptr : (const T*)p.z + (size_t)x.b * p.z_bs;
    T ru[RPW], rd[RPW], rz[RPW];
    float total = 0.f;
    auto load = [&](int tile) __attribute__((always_inline)) {  // (rows behind the last one read that one: no branch between the loads)
#pragma unroll
        for (int r = 0; r < RPW; ++r) {
            const int t = min(tile * TS + w * RPW + r, p.T - 1);
            ru[r] = (up + (size_t)t * p.u_ts)[d];
            rd[r] = (dp + (size_t)t * p.delta_ts)[d];
            if (zp) rz[r] = (zp + (size_t)t * p.z_ts)[d];
        }
    };
    load(x.tile0);
    if (!ENDS) chain<NS>(h, A2, p.ends, p.ends_step, q, p.C, x.b, w, d, 0, 1, x.chunk);
    uniform_ptr mp = (uniform_ptr)(uintptr_t)(p.maps + ((x.item + x.tile0) * 4 + w) * (TS * 2 * NS));
    float m[2][U][2 * NS];
    auto fetch = [&](float (&o)[U][2 * NS], uniform_ptr from) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < U; ++i)
#pragma unroll
            for (int j = 0; j < (ENDS ? NS : 2 * NS); ++j) o[i][j] = from[i * 2 * NS + j];
    };
    for (int tile = x.tile0; tile < x.tile1; ++tile) {
        float cu[RPW], cz[RPW];
#pragma unroll
        for (int r = 0; r < RPW; ++r) {
            const int row = w * RPW + r, t = tile * TS + row;
            const bool live = x.ok && t < len;
            const float raw = (float)rd[r] + bias;
            const float step = live ? p.softplus ? sq_softplus(raw) : raw : 0.f;
            cu[r] = live ? (float)ru[r] : 0.f;
            cz[r] = zp ? (float)rz[r] : 0.f;
            total += step;
            sd[row][lane] = make_float2(step, step * cu[r]);
        }
        fetch(m[0], mp);
        __syncthreads();
        if (tile + 1 < x.tile1) load(tile + 1);
        if (!ENDS && p.hs && x.ok) {
            float* hp = p.hs + (((size_t)x.b * q.tiles + tile) * q.NP + w * NS) * p.C;
#pragma unroll
            for (int s = 0; s < NS; ++s) (hp + (size_t)s * p.C)[d] = h[s];
        }
        float2 v[2][U];
        float y[TS];
#pragma unroll
        for (int i = 0; i < U; ++i) v[0][i] = sd[i][lane];
#pragma unroll
        for (int k = 0; k < TS / U; ++k) {
            if (k + 1 < TS / U) {
                fetch(m[(k + 1) & 1], mp + (k + 1) * U * 2 * NS);
#pragma unroll
                for (int i = 0; i < U; ++i) v[(k + 1) & 1][i] = sd[(k + 1) * U + i][lane];
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < U; ++i) {
                const float2 c = v[k & 1][i];
                const float* mm = m[k & 1][i];
                float o = 0.f;
#pragma unroll
                for (int s = 0; s < NS; ++s) {
                    h[s] = fmaf(__builtin_amdgcn_exp2f(c.x * A2[s]), h[s], c.y * mm[s]);
                    if (!ENDS) o = fmaf(mm[NS + s], h[s], o);
                }
                y[k * U + i] = o;
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        mp += 4 * TS * 2 * NS;
        if (!ENDS) {
#pragma unroll
            for (int t = 0; t < TS; ++t) sy[w][t][lane] = y[t];
        }
        __syncthreads();
        if (!ENDS) {
#pragma unroll
            for (int r = 0; r < RPW; ++r) {
                const int row = w * RPW + r, t = tile * TS + row;
                float o = fmaf(Dd, cu[r], (sy[0][row][lane] + sy[1][row][lane]) + (sy[2][row][lane] + sy[3][row][lane]));
                if (zp) o *= sq_silu(cz[r]);
                if (x.ok && t < p.T) ((T*)p.y + ((size_t)x.b * p.T + t) * p.C)[d] = (T)(t < len ? o : 0.f);
            }
        }
    }
    if (ENDS) {
        const size_t e = (size_t)x.b * q.chunks + x.chunk;
        if (x.ok) {
#pragma unroll
            for (int s = 0; s < NS; ++s) p.ends[(e * q.NP + w * NS + s) * p.C + d] = h[s];
        }
        sd[w][lane].x = total;
        __syncthreads();
        if (w == 0 && x.ok) p.ends_step[e * p.C + d] = (sd[0][lane].x + sd[1][lane].x) + (sd[2][lane].x + sd[3][lane].x);
    } else if (p.last && x.chunk == q.chunks - 1 && x.ok) {
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            const int n = w * NS + s;
            if (n < p.N) p.last[((size_t)x.b * p.C + d) * p.N + n] = h[s];
        }
    }
}

// The adjoint that each chunk but the first hands to the one before it when nothing comes in from behind:
//   g_t = carry + C_t dyg_t, carry = exp(D_t A) g_t, from the chunk's last row to its first
template <typename T, int NS>
__global__ __launch_bounds__(256) void scan_bwd_ends_kernel(BwdArgs a) {
    const ga_scan_bwd_params& p = a.p;
    const Plan& q = a.q;
    constexpr int U = NS <= 4 ? 4 : NS <= 8 ? 2 : 1;
    __shared__ float2 sd[TS][64];
    const Place x = place(q, q.chunks - 1, 1, p.G, p.T, p.lengths);
    const int lane = x.lane, w = x.w, d = x.d, len = x.len;
    const float bias = p.delta_bias ? p.delta_bias[d] : 0.f;
    float A2[NS], c[NS];
#pragma unroll
    for (int s = 0; s < NS; ++s) {
        const int n = w * NS + s;
        A2[s] = n < p.N ? p.A[(size_t)d * p.N + n] * SQ_LOG2E : 0.f;
        c[s] = 0.f;
    }
    const T* dp = (const T*)p.delta + (size_t)x.b * p.delta_bs;
    const T* zp = p.z ? (const T*)p.z + (size_t)x.b * p.z_bs : nullptr;
    const T* gp = (const T*)p.dy + (size_t)x.b * p.T * p.C;
    T rd[RPW], rz[RPW], rg[RPW];
    float total = 0.f;
    auto load = [&](int tile) __attribute__((always_inline)) {
#pragma unroll
        for (int r = 0; r < RPW; ++r) {
            const int t = min(tile * TS + w * RPW + r, p.T - 1);
            rd[r] = (dp + (size_t)t * p.delta_ts)[d];
            rg[r] = (gp + (size_t)t * p.C)[d];
            if (zp) rz[r] = (zp + (size_t)t * p.z_ts)[d];
        }
    };
    load(x.tile1 - 1);
    float m[2][U][NS];
    auto fetch = [&](float (&o)[U][NS], uniform_ptr from) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < U; ++i)
#pragma unroll
            for (int j = 0; j < NS; ++j) o[i][j] = from[i * 2 * NS + NS + j];
    };
    for (int tile = x.tile1 - 1; tile >= x.tile0; --tile) {
        uniform_ptr mp = (uniform_ptr)(uintptr_t)(p.maps + ((x.item + tile) * 4 + w) * (TS * 2 * NS));
#pragma unroll
        for (int r = 0; r < RPW; ++r) {
            const int row = w * RPW + r, t = tile * TS + row;
            const bool live = x.ok && t < len;
            const float raw = (float)rd[r] + bias;
            const float step = live ? p.softplus ? sq_softplus(raw) : raw : 0.f;
            float dy = (float)rg[r];
            if (zp) dy *= sq_silu((float)rz[r]);
            total += step;
            sd[row][lane] = make_float2(step, live ? dy : 0.f);
        }
        fetch(m[0], mp + (TS - U) * 2 * NS);
        __syncthreads();
        if (tile > x.tile0) load(tile - 1);
        float2 v[2][U];
#pragma unroll
        for (int i = 0; i < U; ++i) v[0][i] = sd[TS - U + i][lane];
#pragma unroll
        for (int k = 0; k < TS / U; ++k) {
            if (k + 1 < TS / U) {
                fetch(m[(k + 1) & 1], mp + (TS - (k + 2) * U) * 2 * NS);
#pragma unroll
                for (int i = 0; i < U; ++i) v[(k + 1) & 1][i] = sd[TS - (k + 2) * U + i][lane];
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = U - 1; i >= 0; --i) {
                const float2 o = v[k & 1][i];
#pragma unroll
                for (int s = 0; s < NS; ++s) c[s] = __builtin_amdgcn_exp2f(o.x * A2[s]) * fmaf(m[k & 1][i][s], o.y, c[s]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        __syncthreads();
    }
    const size_t e = (size_t)x.b * q.chunks + x.chunk;
    if (x.ok) {
#pragma unroll
        for (int s = 0; s < NS; ++s) p.ends[(e * q.NP + w * NS + s) * p.C + d] = c[s];
    }
    sd[w][lane].x = total;
    __syncthreads();
    if (w == 0 && x.ok) p.ends_step[e * p.C + d] = (sd[0][lane].x + sd[1][lane].x) + (sd[2][lane].x + sd[3][lane].x);
}

// Per tile, from the last to the first: the states again from the one saved at the tile's start (kept in registers, with the decays), then
// the adjoint backwards through them; NB states of a wave at a time.
template <typename T, int NS>
__global__ __launch_bounds__(256, NS <= 4 ? 2 : 1) void scan_bwd_kernel(BwdArgs a) {
    const ga_scan_bwd_params& p = a.p;
    const Plan& q = a.q;
    constexpr int NB = NS < 4 ? NS : 4, U = 2;
    __shared__ float2 sd[TS][64];     // step, step * u
    __shared__ float sg[TS][64];      // dy * gate
    __shared__ float sy[4][TS][64];   // <C, h> over a wave's states
    __shared__ float2 ss[4][TS][64];  // <g, B>, <g a h_prev, A>
    __shared__ float sm[4][TS][2 * NS];
    const Place x = place(q, q.chunks, 0, p.G, p.T, p.lengths);
    const int lane = x.lane, w = x.w, d = x.d, len = x.len;
    const float bias = p.delta_bias ? p.delta_bias[d] : 0.f, Dd = p.D ? p.D[d] : 0.f;
    float A2[NS], c[NS], dA[NS];
#pragma unroll
    for (int s = 0; s < NS; ++s) {
        const int n = w * NS + s;
        A2[s] = n < p.N ? p.A[(size_t)d * p.N + n] * SQ_LOG2E : 0.f;
        c[s] = p.dlast && n < p.N && x.ok ? p.dlast[((size_t)x.b * p.C + d) * p.N + n] : 0.f;
        dA[s] = 0.f;
    }
    const T* up = (const T*)p.u + (size_t)x.b * p.u_bs;
    const T* dp = (const T*)p.delta + (size_t)x.b * p.delta_bs;
    const T* zp = p.z ? (const T*)p.z + (size_t)x.b * p.z_bs : nullptr;
    const size_t orow = (size_t)x.b * p.T * p.C;
    const T* gp = (const T*)p.dy + orow;
    T ru[RPW], rd[RPW], rz[RPW], rg[RPW];
    auto load = [&](int tile) __attribute__((always_inline)) {
#pragma unroll
        for (int r = 0; r < RPW; ++r) {
            const int t = min(tile * TS + w * RPW + r, p.T - 1);
            ru[r] = (up + (size_t)t * p.u_ts)[d];
            rd[r] = (dp + (size_t)t * p.delta_ts)[d];
            rg[r] = (gp + (size_t)t * p.C)[d];
            if (zp) rz[r] = (zp + (size_t)t * p.z_ts)[d];
        }
    };
    load(x.tile1 - 1);
    chain<NS>(c, A2, p.ends, p.ends_step, q, p.C, x.b, w, d, q.chunks - 1, -1, q.chunks - 1 - x.chunk);
    float dD = 0.f, dbias = 0.f;
    for (int tile = x.tile1 - 1; tile >= x.tile0; --tile) {
        uniform_ptr mp = (uniform_ptr)(uintptr_t)(p.maps + ((x.item + tile) * 4 + w) * (TS * 2 * NS));
        const float* hp = p.hs + (((size_t)x.b * q.tiles + tile) * q.NP + w * NS) * p.C;
        float cu[RPW], craw[RPW], cz[RPW], cdy[RPW], cstep[RPW], cg[RPW], h0[NS];
#pragma unroll
        for (int s = 0; s < NS; ++s) h0[s] = (hp + (size_t)s * p.C)[d];
#pragma unroll
        for (int r = 0; r < RPW; ++r) {
            const int row = w * RPW + r, t = tile * TS + row;
            const bool live = x.ok && t < len;
            craw[r] = (float)rd[r] + bias;
            cstep[r] = live ? p.softplus ? sq_softplus(craw[r]) : craw[r] : 0.f;
            cu[r] = live ? (float)ru[r] : 0.f;
            cdy[r] = live ? (float)rg[r] : 0.f;
            cz[r] = zp && live ? (float)rz[r] : 0.f;
            cg[r] = zp ? cdy[r] * sq_silu(cz[r]) : cdy[r];
            sd[row][lane] = make_float2(cstep[r], cstep[r] * cu[r]);
            sg[row][lane] = cg[r];
        }
        __syncthreads();
        if (tile > x.tile0) load(tile - 1);
#pragma unroll
        for (int sb = 0; sb < NS / NB; ++sb) {
            float h[TS][NB], av[TS][NB];
            float m[2][U][2 * NB];
            float2 v[2][U];
            auto fetch = [&](int set, int t0) __attribute__((always_inline)) {
#pragma unroll
                for (int i = 0; i < U; ++i) {
#pragma unroll
                    for (int j = 0; j < NB; ++j) {
                        m[set][i][j] = mp[(t0 + i) * 2 * NS + sb * NB + j];
                        m[set][i][NB + j] = mp[(t0 + i) * 2 * NS + NS + sb * NB + j];
                    }
                    v[set][i] = sd[t0 + i][lane];
                }
            };
            fetch(0, 0);
#pragma unroll
            for (int k = 0; k < TS / U; ++k) {
                if (k + 1 < TS / U) fetch((k + 1) & 1, (k + 1) * U);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < U; ++i) {
                    const int t = k * U + i;
                    const float2 o = v[k & 1][i];
                    const float* mm = m[k & 1][i];
                    float y = sb && zp ? sy[w][t][lane] : 0.f;
#pragma unroll
                    for (int j = 0; j < NB; ++j) {
                        av[t][j] = __builtin_amdgcn_exp2f(o.x * A2[sb * NB + j]);
                        h[t][j] = fmaf(av[t][j], t ? h[t - 1][j] : h0[sb * NB + j], o.y * mm[j]);
                        y = fmaf(mm[NB + j], h[t][j], y);
                    }
                    if (zp) sy[w][t][lane] = y;
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            float gy[2][U];
            auto fetch_back = [&](int set, int t0) __attribute__((always_inline)) {
                fetch(set, t0);
#pragma unroll
                for (int i = 0; i < U; ++i) gy[set][i] = sg[t0 + i][lane];
            };
            fetch_back(0, TS - U);
            constexpr int PER = 64 / (2 * NB);  // lanes that share a value after the first folds
#pragma unroll
            for (int k = 0; k < TS / U; ++k) {
                if (k + 1 < TS / U) fetch_back((k + 1) & 1, TS - (k + 2) * U);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = U - 1; i >= 0; --i) {
                    const int t = TS - (k + 1) * U + i;
                    const float2 o = v[k & 1][i];
                    const float dy = gy[k & 1][i];
                    const float* mm = m[k & 1][i];
                    float2 s12 = sb ? ss[w][t][lane] : make_float2(0.f, 0.f);
                    float val[2 * NB];
#pragma unroll
                    for (int j = 0; j < NB; ++j) {
                        const int s = sb * NB + j;
                        const float gv = fmaf(mm[NB + j], dy, c[s]);
                        val[j] = gv * o.y;
                        val[NB + j] = dy * h[t][j];
                        s12.x = fmaf(gv, mm[j], s12.x);
                        c[s] = av[t][j] * gv;
                        const float qv = c[s] * (t ? h[t - 1][j] : h0[s]);
                        s12.y = fmaf(qv, A2[s], s12.y);
                        dA[s] = fmaf(qv, o.x, dA[s]);
                    }
                    ss[w][t][lane] = s12;
                    const float sum = sq_lane_sums<2 * NB>(val, lane);
                    if (lane % PER == 0) {
                        const int i2 = lane / PER;  // B's share in the first NB, C's in the others
                        sm[w][t][(i2 / NB) * NS + sb * NB + i2 % NB] = sum;
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < RPW; ++r) {
            const int row = w * RPW + r, t = tile * TS + row;
            const bool live = x.ok && t < len;
            const float2 x0 = ss[0][row][lane], x1 = ss[1][row][lane], x2 = ss[2][row][lane], x3 = ss[3][row][lane];
            const float s1 = (x0.x + x1.x) + (x2.x + x3.x), s2 = ((x0.y + x1.y) + (x2.y + x3.y)) * SQ_LN2;
            const float du = fmaf(cstep[r], s1, Dd * cg[r]);
            float dd = fmaf(cu[r], s1, s2);
            if (p.softplus) dd *= sq_sigmoid(craw[r]);
            dd = live ? dd : 0.f;
            dD = fmaf(cg[r], cu[r], dD);
            dbias += dd;
            if (x.ok && t < p.T) {
                const size_t o = orow + (size_t)t * p.C;
                ((T*)p.du + o)[d] = (T)(live ? du : 0.f);
                ((T*)p.ddelta + o)[d] = (T)dd;
                if (zp) {
                    const float y = fmaf(Dd, cu[r], (sy[0][row][lane] + sy[1][row][lane]) + (sy[2][row][lane] + sy[3][row][lane]));
                    ((T*)p.dz + o)[d] = (T)(live ? cdy[r] * y * sq_silu_slope(cz[r]) : 0.f);
                }
            }
        }
        // this block's share of dB and dC, in the layout of the maps
        const int slab = (blockIdx.x % q.nCb) % q.cbg;
        float* mo = p.dmaps + ((size_t)slab * p.B * p.G * q.tiles + x.item + tile) * (4 * TS * 2 * NS);
        for (int i = threadIdx.x; i < 4 * TS * 2 * NS; i += 256) mo[i] = (&sm[0][0][0])[i];
        __syncthreads();
    }
    const size_t e = (size_t)x.b * q.chunks + x.chunk;
    if (x.ok) {
#pragma unroll
        for (int s = 0; s < NS; ++s) p.dparams[(e * (q.NP + 2) + w * NS + s) * p.C + d] = dA[s];
        if (p.dstate && x.chunk == 0) {
#pragma unroll
            for (int s = 0; s < NS; ++s) {
                const int n = w * NS + s;
                if (n < p.N) p.dstate[((size_t)x.b * p.C + d) * p.N + n] = c[s];
            }
        }
    }
    sd[w][lane] = make_float2(dD, dbias);
    __syncthreads();
    if (w < 2 && x.ok) {
        const float v = w == 0 ? (sd[0][lane].x + sd[1][lane].x) + (sd[2][lane].x + sd[3][lane].x)
                               : (sd[0][lane].y + sd[1][lane].y) + (sd[2][lane].y + sd[3][lane].y);
        p.dparams[(e * (q.NP + 2) + q.NP + w) * p.C + d] = v;
    }
}

// dB, dC: the channel blocks' shares added up
template <typename T>
__global__ __launch_bounds__(256) void scan_dmaps_kernel(const float* __restrict__ dmaps, T* __restrict__ dB, T* __restrict__ dC, Plan q, int B,
                                                         int Tn, int N, int G) {
    const size_t total = (size_t)B * Tn * G * N, slab = (size_t)B * G * q.tiles * TS * 2 * q.NP;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (size_t)gridDim.x * 256) {
        const int n = (int)(i % N);
        const size_t row = i / N;
        const int g = (int)(row % G);
        const size_t bt = row / G;
        const int t = (int)(bt % Tn), b = (int)(bt / Tn);
        const float* s = dmaps + ((((size_t)b * G + g) * q.tiles + t / TS) * 4 + n / q.NS) * (TS * 2 * q.NS) + (t % TS) * 2 * q.NS + n % q.NS;
        float x = 0.f, y = 0.f;
        for (int k = 0; k < q.cbg; ++k, s += slab) { x += s[0]; y += s[q.NS]; }
        dB[i] = (T)x;
        dC[i] = (T)y;
    }
}

// dA [C][N], dD, ddelta_bias [C]: the items' and chunks' shares ([rows][NP + 2][C]) added up
__global__ __launch_bounds__(1024) void scan_dparams_kernel(const float* __restrict__ parts, int rows, int NP, int C, int N, float* __restrict__ dA,
                                                            float* __restrict__ dD, float* __restrict__ dbias) {
    __shared__ double acc[32][32];
    const long col = (long)blockIdx.x * 32 + (threadIdx.x & 31), cols = (long)(NP + 2) * C;
    const double v = sq_groups32(col < cols ? sq_column(parts + col, cols, rows, threadIdx.x >> 5, 32) : 0.0, acc);
    if (threadIdx.x < 32 && col < cols) {
        const int s = (int)(col / C), d = (int)(col % C);
        if (s < N) dA[(size_t)d * N + s] = (float)v;
        else if (s == NP && dD) dD[d] = (float)v;
        else if (s == NP + 1 && dbias) dbias[d] = (float)v;
    }
}

// One token: a thread holds four states of a channel, TPC threads (a power of two) a channel; the state is read and written once.
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void scan_step_kernel(ga_scan_step_params p, int tpc) {
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x, ch = i / tpc;
    const int part = (int)(i % tpc), n0 = part * 4;
    const bool ok = ch < (size_t)p.B * p.C;
    const int b = ok ? (int)(ch / p.C) : 0, d = ok ? (int)(ch % p.C) : 0, g = d / (p.C / p.G);
    const float u = (float)((const T*)p.u)[(size_t)b * p.u_bs + d];
    const float raw = (float)((const T*)p.delta)[(size_t)b * p.delta_bs + d] + (p.delta_bias ? p.delta_bias[d] : 0.f);
    const float step = p.softplus ? sq_softplus(raw) : raw;
    float* hp = p.state + (size_t)b * p.state_bs + (size_t)d * p.N + n0;
    const float* Ap = p.A + (size_t)d * p.N + n0;
    const T* Bp = (const T*)p.Bm + (size_t)b * p.b_bs + (size_t)g * p.N + n0;
    const T* Cp = (const T*)p.Cm + (size_t)b * p.c_bs + (size_t)g * p.N + n0;
    float y = 0.f;
    if (ok && n0 < p.N) {
        float h[4], A[4];
        if (VEC) {
            *(float4*)h = *(const float4*)hp;
            *(float4*)A = *(const float4*)Ap;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                h[j] = n0 + j < p.N ? hp[j] : 0.f;
                A[j] = n0 + j < p.N ? Ap[j] : 0.f;
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (!VEC && n0 + j >= p.N) break;
            h[j] = fmaf(__builtin_amdgcn_exp2f(step * (A[j] * SQ_LOG2E)), h[j], step * u * (float)Bp[j]);
            y = fmaf((float)Cp[j], h[j], y);
        }
        if (VEC) *(float4*)hp = *(float4*)h;
        else
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (n0 + j < p.N) hp[j] = h[j];
    }
    for (int o = tpc >> 1; o > 0; o >>= 1) y += __shfl_xor(y, o, 64);
    if (ok && part == 0) {
        if (p.D) y = fmaf(p.D[d], u, y);
        if (p.z) y *= sq_silu((float)((const T*)p.z)[(size_t)b * p.z_bs + d]);
        ((T*)p.y)[(size_t)b * p.C + d] = (T)y;
    }
}

int bad_sizes(int B, int T, int C, int N, int G, int dtype) {
    if (B < 1 || T < 1 || C < 1 || N < 1 || N > GA_SCAN_MAX_STATES || G < 1 || C % G) return GA_ERR_ARG;
    if (dtype != GA_DTYPE_F32 && dtype != GA_DTYPE_BF16) return GA_ERR_ARG;
    const Plan q = make_plan(B, T, C, N, G);
    if ((long)B * q.nCb * q.chunks > 0x7fffffffL || (long)B * G > 0x7fffffffL || (long)T + TS > 0x7fffffffL) return GA_ERR_ARG;
    return GA_OK;
}

int grid_for(size_t n) {
    const size_t g = (n + 255) / 256;
    return (int)(g < 4096 ? g : 4096);
}

template <typename T, int NS>
int launch_fwd(const Args& a, hipStream_t s) {
    const long blocks = (long)a.p.B * a.q.nCb;
    if (a.q.chunks > 1) {
        scan_fwd_kernel<T, NS, true><<<(unsigned)(blocks * (a.q.chunks - 1)), 256, 0, s>>>(a);
        GA_CHECK_LAUNCH();
    }
    scan_fwd_kernel<T, NS, false><<<(unsigned)(blocks * a.q.chunks), 256, 0, s>>>(a);
    GA_CHECK_LAUNCH();
    return GA_OK;
}

template <typename T, int NS>
int launch_bwd(const BwdArgs& a, hipStream_t s) {
    const long blocks = (long)a.p.B * a.q.nCb;
    if (a.q.chunks > 1) {
        scan_bwd_ends_kernel<T, NS><<<(unsigned)(blocks * (a.q.chunks - 1)), 256, 0, s>>>(a);
        GA_CHECK_LAUNCH();
    }
    scan_bwd_kernel<T, NS><<<(unsigned)(blocks * a.q.chunks), 256, 0, s>>>(a);
    GA_CHECK_LAUNCH();
    return GA_OK;
}

#define SCAN_DISPATCH(FN, T, ARGS)                 \
    (ARGS.q.NS == 16  ? FN<T, 16>(ARGS, s)         \
     : ARGS.q.NS == 8 ? FN<T, 8>(ARGS, s)          \
     : ARGS.q.NS == 4 ? FN<T, 4>(ARGS, s)          \
     : ARGS.q.NS == 2 ? FN<T, 2>(ARGS, s)          \
                      : FN<T, 1>(ARGS, s))

template <typename T>
int fwd(const Args& a, hipStream_t s) {
    const ga_scan_params& p = a.p;
    scan_maps_kernel<T><<<grid_for((size_t)p.B * p.G * a.q.tiles * TS * a.q.NP), 256, 0, s>>>((const T*)p.Bm, (const T*)p.Cm, p.maps, p.lengths, a.q, p.B, p.T,
                                                                                    p.N, p.G, p.b_bs, p.b_ts, p.c_bs, p.c_ts);
    GA_CHECK_LAUNCH();
    return SCAN_DISPATCH(launch_fwd, T, a);
}

template <typename T>
int bwd(const BwdArgs& a, hipStream_t s) {
    const ga_scan_bwd_params& p = a.p;
    const int rc = SCAN_DISPATCH(launch_bwd, T, a);
    if (rc) return rc;
    scan_dmaps_kernel<T><<<grid_for((size_t)p.B * p.T * p.G * p.N), 256, 0, s>>>(p.dmaps, (T*)p.dBm, (T*)p.dCm, a.q, p.B, p.T, p.N, p.G);
    GA_CHECK_LAUNCH();
    const long cols = (long)(a.q.NP + 2) * p.C;
    scan_dparams_kernel<<<(unsigned)((cols + 31) / 32), 1024, 0, s>>>(p.dparams, p.B * a.q.chunks, a.q.NP, p.C, p.N, p.dA, p.dD, p.ddelta_bias);
    GA_CHECK_LAUNCH();
    return GA_OK;
}

}  // namespace

extern "C" {

int ga_scan_sizes(int B, int T, int C, int N, int G, ga_scan_buffers* h_out) {
    if (!h_out || bad_sizes(B, T, C, N, G, GA_DTYPE_F32)) return GA_ERR_ARG;
    const Plan q = make_plan(B, T, C, N, G);
    h_out->maps = (size_t)B * G * q.tiles * TS * 2 * q.NP;
    h_out->hs = (size_t)B * q.tiles * q.NP * C;
    h_out->ends = q.chunks > 1 ? (size_t)B * q.chunks * q.NP * C : 0;
    h_out->ends_step = q.chunks > 1 ? (size_t)B * q.chunks * C : 0;
    h_out->dmaps = h_out->maps * q.cbg;
    h_out->dparams = (size_t)B * q.chunks * (q.NP + 2) * C;
    return GA_OK;
}

int ga_scan_fwd(const ga_scan_params* hp, int dtype, hipStream_t s) {
    if (!hp) return GA_ERR_ARG;
    const ga_scan_params& p = *hp;
    const int rc = bad_sizes(p.B, p.T, p.C, p.N, p.G, dtype);
    if (rc) return rc;
    const Args a{p, make_plan(p.B, p.T, p.C, p.N, p.G)};
    if (!p.u || !p.delta || !p.A || !p.Bm || !p.Cm || !p.y || !p.maps || (a.q.chunks > 1 && (!p.ends || !p.ends_step))) return GA_ERR_ARG;
    if ((uintptr_t)p.maps & 15) return GA_ERR_ALIGN;
    return dtype == GA_DTYPE_BF16 ? fwd<bf16_t>(a, s) : fwd<float>(a, s);
}

int ga_scan_bwd(const ga_scan_bwd_params* hp, int dtype, hipStream_t s) {
    if (!hp) return GA_ERR_ARG;
    const ga_scan_bwd_params& p = *hp;
    const int rc = bad_sizes(p.B, p.T, p.C, p.N, p.G, dtype);
    if (rc) return rc;
    const BwdArgs a{p, make_plan(p.B, p.T, p.C, p.N, p.G)};
    if (!p.u || !p.delta || !p.A || !p.dy || !p.maps || !p.hs || !p.du || !p.ddelta || !p.dA || !p.dBm || !p.dCm || !p.dmaps || !p.dparams ||
        (!p.z) != (!p.dz) || (a.q.chunks > 1 && (!p.ends || !p.ends_step)))
        return GA_ERR_ARG;
    if ((uintptr_t)p.maps & 15) return GA_ERR_ALIGN;
    return dtype == GA_DTYPE_BF16 ? bwd<bf16_t>(a, s) : bwd<float>(a, s);
}

int ga_scan_step(const ga_scan_step_params* hp, int dtype, hipStream_t s) {
    if (!hp) return GA_ERR_ARG;
    const ga_scan_step_params& p = *hp;
    const int rc = bad_sizes(p.B, 1, p.C, p.N, p.G, dtype);
    if (rc) return rc;
    if (!p.u || !p.delta || !p.A || !p.Bm || !p.Cm || !p.state || !p.y) return GA_ERR_ARG;
    int tpc = 1;
    while (tpc * 4 < p.N) tpc *= 2;
    const size_t blocks = ((size_t)p.B * p.C * tpc + 255) / 256;
    if (blocks > 0x7fffffffUL) return GA_ERR_ARG;
    const bool vec = p.N % 4 == 0 && p.state_bs % 4 == 0 && !(((uintptr_t)p.state | (uintptr_t)p.A) & 15);
    if (dtype == GA_DTYPE_BF16) {
        if (vec) scan_step_kernel<bf16_t, true><<<(unsigned)blocks, 256, 0, s>>>(p, tpc);
        else scan_step_kernel<bf16_t, false><<<(unsigned)blocks, 256, 0, s>>>(p, tpc);
    } else {
        if (vec) scan_step_kernel<float, true><<<(unsigned)blocks, 256, 0, s>>>(p, tpc);
        else scan_step_kernel<float, false><<<(unsigned)blocks, 256, 0, s>>>(p, tpc);
    }
    GA_CHECK_LAUNCH();
    return GA_OK;
}

}  // extern "C"
