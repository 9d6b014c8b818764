// Selective state space scan:  h_t = exp(D_t A) h_{t-1} + D_t u_t B_t,  y_t = (<C_t, h_t> + D u_t) silu(z_t),  D_t = softplus(delta_t + bias)
// per channel d and state n, on channels-last activations; forward, backward and the single-token step.
//
// One block is 64 channels (one per lane) times all states (split over its four waves: a lane holds its wave's states in registers), walking
// along time in tiles of 16 rows.  What depends on a row and a channel alone (softplus, gates, the sums over states) is done once, four rows to
// a wave, and passes through LDS; B and C, which all channels of a group share, are first laid out in float32 in the order in which
// the waves read them (scan_maps_kernel) and come in as scalar loads, so that they cost no vector instruction and no LDS bandwidth.
#include "seq_common.h"

namespace {

constexpr int TS = 16;          // rows of a tile
constexpr int RPW = TS / 4;     // rows that one wave prepares and finishes
constexpr int MAX_CHUNKS = 64;  // a block adds up the chunks before (behind) its own one by one

typedef const __attribute__((address_space(4))) float* uniform_ptr;

struct Plan {
    int NB, SB, NP;           // states per wave and state block, state blocks, 4 * NB * SB
    int Cg, cbg, nCb;         // channels of a group, 64-channel blocks of a group, of all groups
    int Tp, tiles;            // rows rounded up to a tile
    int chunks, chunk_tiles;  // tiles of a chunk
};

Plan make_plan(int B, int T, int C, int N, int G) {
    Plan q;
    q.NB = N <= 4 ? 1 : N <= 8 ? 2 : 4;
    q.SB = N <= 16 ? 1 : N <= 32 ? 2 : 4;
    q.NP = 4 * q.NB * q.SB;
    q.Cg = C / G;
    q.cbg = (q.Cg + 63) / 64;
    q.nCb = q.cbg * G;
    q.tiles = (T + TS - 1) / TS;
    q.Tp = q.tiles * TS;
    const long blocks = (long)B * q.nCb;
    long want = (1024 + blocks - 1) / blocks;
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

// state index of (wave, state block, j)
__device__ __forceinline__ int state_of(int w, int sb, int j, int NB) { return sb * 4 * NB + w * NB + j; }

// maps[b][row][group][wave][sb][B: NB | C: NB] in float32; zero rows behind an item's length and up to the whole tile, zero states behind N
template <typename T>
__global__ __launch_bounds__(256) void scan_maps_kernel(const T* __restrict__ Bm, const T* __restrict__ Cm, float* __restrict__ maps,
                                                        const int* __restrict__ lengths, Plan q, int B, int Tn, int N, int G, long b_bs,
                                                        long b_ts, long c_bs, long c_ts) {
    const size_t total = (size_t)B * q.Tp * G * q.NP;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (size_t)gridDim.x * 256) {
        const int s = (int)(i % q.NP);
        const size_t row = i / q.NP;
        const int g = (int)(row % G);
        const size_t bt = row / G;
        const int t = (int)(bt % q.Tp), b = (int)(bt / q.Tp);
        const int w = s / (q.NB * q.SB), sb = (s / q.NB) % q.SB, j = s % q.NB;
        const int n = sb * 4 * q.NB + w * q.NB + j;
        const bool live = n < N && t < sq_len(lengths, b, Tn);
        const float vb = live ? (float)Bm[(size_t)b * b_bs + (size_t)t * b_ts + (size_t)g * N + n] : 0.f;
        const float vc = live ? (float)Cm[(size_t)b * c_bs + (size_t)t * c_ts + (size_t)g * N + n] : 0.f;
        float* o = maps + row * (2 * q.NP) + (size_t)(w * q.SB + sb) * 2 * q.NB + j;
        o[0] = vb;
        o[q.NB] = vc;
    }
}

// ENDS: only the state that each chunk but the last leaves behind when it starts from zero, and the sum of its steps
// (the chunk's decay is exp(A * that sum)).  Otherwise the outputs, each chunk from the states of the chunks before it.
template <typename T, int NB, int SB, bool ENDS>
__global__ __launch_bounds__(256) void scan_fwd_kernel(Args a) {
    const ga_scan_params& p = a.p;
    const Plan& q = a.q;
    constexpr int NS = NB * SB;
    __shared__ float2 sd[TS][64];
    __shared__ float sy[ENDS ? 1 : 4][ENDS ? 1 : TS][64];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int cb = blockIdx.x % q.nCb, rest = blockIdx.x / q.nCb;
    const int nch = ENDS ? q.chunks - 1 : q.chunks;
    const int chunk = rest % nch, b = rest / nch;
    const int g = cb / q.cbg, din = (cb % q.cbg) * 64 + lane;
    const bool ok = din < q.Cg;
    const int d = g * q.Cg + (ok ? din : q.Cg - 1);
    const int len = sq_len(p.lengths, b, p.T);
    const float bias = p.delta_bias ? p.delta_bias[d] : 0.f, Dd = p.D ? p.D[d] : 0.f;
    float A2[NS], h[NS];
#pragma unroll
    for (int s = 0; s < NS; ++s) {
        const int n = state_of(w, s / NB, s % NB, NB);
        A2[s] = n < p.N ? p.A[(size_t)d * p.N + n] * SQ_LOG2E : 0.f;
        h[s] = 0.f;
        if (!ENDS && p.state && n < p.N) h[s] = p.state[((size_t)b * p.C + d) * p.N + n];
    }
    if (!ENDS) {
        for (int k = 0; k < chunk; ++k) {
            const size_t e = (size_t)b * q.chunks + k;
            const float sum = p.ends_step[e * p.C + d];
#pragma unroll
            for (int s = 0; s < NS; ++s) {
                const int n = state_of(w, s / NB, s % NB, NB);
                h[s] = fmaf(__builtin_amdgcn_exp2f(sum * A2[s]), h[s], p.ends[(e * q.NP + n) * p.C + d]);
            }
        }
    }
    const T* up = (const T*)p.u + (size_t)b * p.u_bs + d;
    const T* dp = (const T*)p.delta + (size_t)b * p.delta_bs + d;
    const T* zp = p.z ? (const T*)p.z + (size_t)b * p.z_bs + d : nullptr;
    T* yp = ENDS ? nullptr : (T*)p.y + (size_t)b * p.T * p.C + d;
    const int tile0 = chunk * q.chunk_tiles, tile1 = min(tile0 + q.chunk_tiles, q.tiles);
    const size_t mrow = (size_t)p.G * 2 * q.NP;
    uniform_ptr mp = (uniform_ptr)(uintptr_t)(p.maps + ((size_t)b * q.Tp + (size_t)tile0 * TS) * mrow + (size_t)g * 2 * q.NP + (size_t)w * SB * 2 * NB);
    float ru[RPW], rd[RPW], rz[RPW], total = 0.f;
    auto load = [&](int tile) __attribute__((always_inline)) {
#pragma unroll
        for (int r = 0; r < RPW; ++r) {
            const int t = tile * TS + w * RPW + r;
            const bool live = ok && t < len;
            ru[r] = live ? (float)up[(size_t)t * p.u_ts] : 0.f;
            rd[r] = live ? (float)dp[(size_t)t * p.delta_ts] : 0.f;
            rz[r] = !ENDS && zp && live ? (float)zp[(size_t)t * p.z_ts] : 0.f;
        }
    };
    load(tile0);
    for (int tile = tile0; tile < tile1; ++tile) {
        float cu[RPW], cz[RPW];
#pragma unroll
        for (int r = 0; r < RPW; ++r) {
            const int row = w * RPW + r, t = tile * TS + row;
            const float raw = rd[r] + bias;
            float step = p.softplus ? sq_softplus(raw) : raw;
            step = ok && t < len ? step : 0.f;
            cu[r] = ru[r];
            cz[r] = rz[r];
            total += step;
            sd[row][lane] = make_float2(step, step * ru[r]);
        }
        __syncthreads();
        if (tile + 1 < tile1) load(tile + 1);
        if (!ENDS && p.hs && ok) {
#pragma unroll
            for (int s = 0; s < NS; ++s) {
                const int n = state_of(w, s / NB, s % NB, NB);
                if (n < p.N) p.hs[(((size_t)b * q.tiles + tile) * p.N + n) * p.C + d] = h[s];
            }
        }
#pragma unroll
        for (int t = 0; t < TS; ++t) {
            const float2 v = sd[t][lane];
            float y = 0.f;
#pragma unroll
            for (int s = 0; s < NS; ++s) {
                const float bv = mp[t * mrow + (s / NB) * 2 * NB + s % NB];
                h[s] = fmaf(__builtin_amdgcn_exp2f(v.x * A2[s]), h[s], v.y * bv);
                if (!ENDS) y = fmaf(mp[t * mrow + (s / NB) * 2 * NB + NB + s % NB], h[s], y);
            }
            if (!ENDS) sy[w][t][lane] = y;
        }
        mp += TS * mrow;
        __syncthreads();
        if (!ENDS) {
#pragma unroll
            for (int r = 0; r < RPW; ++r) {
                const int row = w * RPW + r, t = tile * TS + row;
                float y = fmaf(Dd, cu[r], (sy[0][row][lane] + sy[1][row][lane]) + (sy[2][row][lane] + sy[3][row][lane]));
                if (zp) y *= sq_silu(cz[r]);
                if (ok && t < p.T) yp[(size_t)t * p.C] = (T)(t < len ? y : 0.f);
            }
        }
    }
    if (ENDS) {
        const size_t e = (size_t)b * q.chunks + chunk;
        if (ok) {
#pragma unroll
            for (int s = 0; s < NS; ++s) p.ends[(e * q.NP + state_of(w, s / NB, s % NB, NB)) * p.C + d] = h[s];
        }
        sd[w][lane].x = total;
        __syncthreads();
        if (w == 0 && ok) p.ends_step[e * p.C + d] = (sd[0][lane].x + sd[1][lane].x) + (sd[2][lane].x + sd[3][lane].x);
    } else if (p.last && chunk == q.chunks - 1 && ok) {
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            const int n = state_of(w, s / NB, s % NB, NB);
            if (n < p.N) p.last[((size_t)b * p.C + d) * p.N + n] = h[s];
        }
    }
}

// Sum of each of V values over the 64 lanes; lane l leaves with the sum of value (the top log2 V bits of l).  Each step sends one half of the
// values each way across a lane bit, so that the work halves with it: 2V - 2 adds and exchanges in place of 6V.
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
template <int V>
__device__ __forceinline__ float lane_sums(float (&v)[V], int lane) {
    static_assert(V >= 2 && V <= 64 && (V & (V - 1)) == 0, "a power of two");
    int n = V;
#define SQ_SWAP(BUILTIN)                                                                                            \
    if (n > 1) {                                                                                                    \
        n >>= 1;                                                                                                    \
        _Pragma("unroll") for (int i = 0; i < n; ++i) {                                                             \
            const auto x = BUILTIN(__float_as_uint(v[i]), __float_as_uint(v[i + n]), false, false);                 \
            v[i] = __uint_as_float(x[0]) + __uint_as_float(x[1]);                                                   \
        }                                                                                                           \
    } else {                                                                                                        \
        const auto x = BUILTIN(__float_as_uint(v[0]), __float_as_uint(v[0]), false, false);                         \
        v[0] = __uint_as_float(x[0]) + __uint_as_float(x[1]);                                                       \
    }
#define SQ_STEP(BIT, CTRL)                                                                                          \
    if (n > 1) {                                                                                                    \
        n >>= 1;                                                                                                    \
        const bool up = lane & BIT;                                                                                 \
        _Pragma("unroll") for (int i = 0; i < n; ++i) {                                                             \
            const float keep = up ? v[i + n] : v[i], give = up ? v[i] : v[i + n];                                   \
            v[i] = keep + dpp<CTRL>(give);                                                                          \
        }                                                                                                           \
    } else                                                                                                          \
        v[0] += dpp<CTRL>(v[0]);
    SQ_SWAP(__builtin_amdgcn_permlane32_swap)
    SQ_SWAP(__builtin_amdgcn_permlane16_swap)
    SQ_STEP(8, 0x128)  // rotate by 8 within 16
    SQ_STEP(4, 0x141)  // mirror within 8
    SQ_STEP(2, 0x4E)   // quads: 2 3 0 1
    SQ_STEP(1, 0xB1)   // quads: 1 0 3 2
#undef SQ_SWAP
#undef SQ_STEP
    return v[0];
}

// The adjoint that each chunk but the first hands to the one before it when nothing comes in from behind:
//   g_t = carry + C_t dyg_t, carry = exp(D_t A) g_t, from the chunk's last row to its first
template <typename T, int NB, int SB>
__global__ __launch_bounds__(256) void scan_bwd_ends_kernel(BwdArgs a) {
    const ga_scan_bwd_params& p = a.p;
    const Plan& q = a.q;
    constexpr int NS = NB * SB;
    __shared__ float2 sd[TS][64];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int cb = blockIdx.x % q.nCb, rest = blockIdx.x / q.nCb;
    const int chunk = 1 + rest % (q.chunks - 1), b = rest / (q.chunks - 1);
    const int g = cb / q.cbg, din = (cb % q.cbg) * 64 + lane;
    const bool ok = din < q.Cg;
    const int d = g * q.Cg + (ok ? din : q.Cg - 1);
    const int len = sq_len(p.lengths, b, p.T);
    const float bias = p.delta_bias ? p.delta_bias[d] : 0.f;
    float A2[NS], c[NS];
#pragma unroll
    for (int s = 0; s < NS; ++s) {
        const int n = state_of(w, s / NB, s % NB, NB);
        A2[s] = n < p.N ? p.A[(size_t)d * p.N + n] * SQ_LOG2E : 0.f;
        c[s] = 0.f;
    }
    const T* dp = (const T*)p.delta + (size_t)b * p.delta_bs + d;
    const T* zp = p.z ? (const T*)p.z + (size_t)b * p.z_bs + d : nullptr;
    const T* gp = (const T*)p.dy + (size_t)b * p.T * p.C + d;
    const int tile0 = chunk * q.chunk_tiles, tile1 = min(tile0 + q.chunk_tiles, q.tiles);
    const size_t mrow = (size_t)p.G * 2 * q.NP;
    float total = 0.f;
    for (int tile = tile1 - 1; tile >= tile0; --tile) {
        uniform_ptr mp = (uniform_ptr)(uintptr_t)(p.maps + ((size_t)b * q.Tp + (size_t)tile * TS) * mrow + (size_t)g * 2 * q.NP + (size_t)w * SB * 2 * NB);
#pragma unroll
        for (int r = 0; r < RPW; ++r) {
            const int row = w * RPW + r, t = tile * TS + row;
            const bool live = ok && t < len;
            const float raw = (live ? (float)dp[(size_t)t * p.delta_ts] : 0.f) + bias;
            float step = p.softplus ? sq_softplus(raw) : raw;
            step = live ? step : 0.f;
            float dy = live ? (float)gp[(size_t)t * p.C] : 0.f;
            if (zp) dy *= live ? sq_silu((float)zp[(size_t)t * p.z_ts]) : 0.f;
            total += step;
            sd[row][lane] = make_float2(step, dy);
        }
        __syncthreads();
#pragma unroll
        for (int t = TS - 1; t >= 0; --t) {
            const float2 v = sd[t][lane];
#pragma unroll
            for (int s = 0; s < NS; ++s)
                c[s] = __builtin_amdgcn_exp2f(v.x * A2[s]) * fmaf(mp[t * mrow + (s / NB) * 2 * NB + NB + s % NB], v.y, c[s]);
        }
        __syncthreads();
    }
    const size_t e = (size_t)b * q.chunks + chunk;
    if (ok) {
#pragma unroll
        for (int s = 0; s < NS; ++s) p.ends[(e * q.NP + state_of(w, s / NB, s % NB, NB)) * p.C + d] = c[s];
    }
    sd[w][lane].x = total;
    __syncthreads();
    if (w == 0 && ok) p.ends_step[e * p.C + d] = (sd[0][lane].x + sd[1][lane].x) + (sd[2][lane].x + sd[3][lane].x);
}

// Per tile, from the last to the first: the states again from the one saved at the tile's start (kept in registers, with the decays), then
// the adjoint backwards through them.
template <typename T, int NB, int SB>
__global__ __launch_bounds__(256) void scan_bwd_kernel(BwdArgs a) {
    const ga_scan_bwd_params& p = a.p;
    const Plan& q = a.q;
    constexpr int NS = NB * SB;
    __shared__ float2 sd[TS][64];      // step, step * u
    __shared__ float sg[TS][64];       // dy * gate
    __shared__ float sy[4][TS][64];    // <C, h> over a wave's states
    __shared__ float2 ss[4][TS][64];   // <g, B>, <g a h_prev, A>
    __shared__ float sm[TS][4 * SB * 2 * NB];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int cb = blockIdx.x % q.nCb, rest = blockIdx.x / q.nCb;
    const int chunk = rest % q.chunks, b = rest / q.chunks;
    const int g = cb / q.cbg, din = (cb % q.cbg) * 64 + lane;
    const bool ok = din < q.Cg;
    const int d = g * q.Cg + (ok ? din : q.Cg - 1);
    const int len = sq_len(p.lengths, b, p.T);
    const float bias = p.delta_bias ? p.delta_bias[d] : 0.f, Dd = p.D ? p.D[d] : 0.f;
    float A2[NS], c[NS], dA[NS];
#pragma unroll
    for (int s = 0; s < NS; ++s) {
        const int n = state_of(w, s / NB, s % NB, NB);
        A2[s] = n < p.N ? p.A[(size_t)d * p.N + n] * SQ_LOG2E : 0.f;
        c[s] = p.dlast && n < p.N && ok ? p.dlast[((size_t)b * p.C + d) * p.N + n] : 0.f;
        dA[s] = 0.f;
    }
    for (int k = q.chunks - 1; k > chunk; --k) {
        const size_t e = (size_t)b * q.chunks + k;
        const float sum = p.ends_step[e * p.C + d];
#pragma unroll
        for (int s = 0; s < NS; ++s)
            c[s] = fmaf(__builtin_amdgcn_exp2f(sum * A2[s]), c[s], p.ends[(e * q.NP + state_of(w, s / NB, s % NB, NB)) * p.C + d]);
    }
    const T* up = (const T*)p.u + (size_t)b * p.u_bs + d;
    const T* dp = (const T*)p.delta + (size_t)b * p.delta_bs + d;
    const T* zp = p.z ? (const T*)p.z + (size_t)b * p.z_bs + d : nullptr;
    const size_t orow = (size_t)b * p.T * p.C + d;
    const T* gp = (const T*)p.dy + orow;
    const int tile0 = chunk * q.chunk_tiles, tile1 = min(tile0 + q.chunk_tiles, q.tiles);
    const size_t mrow = (size_t)p.G * 2 * q.NP;
    float dD = 0.f, dbias = 0.f;
    for (int tile = tile1 - 1; tile >= tile0; --tile) {
        uniform_ptr mp = (uniform_ptr)(uintptr_t)(p.maps + ((size_t)b * q.Tp + (size_t)tile * TS) * mrow + (size_t)g * 2 * q.NP + (size_t)w * SB * 2 * NB);
        float cu[RPW], craw[RPW], cz[RPW], cdy[RPW], cstep[RPW], cg[RPW];
#pragma unroll
        for (int r = 0; r < RPW; ++r) {
            const int row = w * RPW + r, t = tile * TS + row;
            const bool live = ok && t < len;
            cu[r] = live ? (float)up[(size_t)t * p.u_ts] : 0.f;
            craw[r] = (live ? (float)dp[(size_t)t * p.delta_ts] : 0.f) + bias;
            cdy[r] = live ? (float)gp[(size_t)t * p.C] : 0.f;
            cz[r] = zp && live ? (float)zp[(size_t)t * p.z_ts] : 0.f;
            const float step = p.softplus ? sq_softplus(craw[r]) : craw[r];
            cstep[r] = live ? step : 0.f;
            cg[r] = zp ? cdy[r] * sq_silu(cz[r]) : cdy[r];
            sd[row][lane] = make_float2(cstep[r], cstep[r] * cu[r]);
            sg[row][lane] = cg[r];
        }
        __syncthreads();
#pragma unroll
        for (int sb = 0; sb < SB; ++sb) {
            float h0[NB], h[TS][NB], av[TS][NB];
#pragma unroll
            for (int j = 0; j < NB; ++j) {
                const int n = state_of(w, sb, j, NB);
                h0[j] = n < p.N ? p.hs[(((size_t)b * q.tiles + tile) * p.N + n) * p.C + d] : 0.f;
            }
#pragma unroll
            for (int t = 0; t < TS; ++t) {
                const float2 v = sd[t][lane];
                float y = sb && zp ? sy[w][t][lane] : 0.f;
#pragma unroll
                for (int j = 0; j < NB; ++j) {
                    av[t][j] = __builtin_amdgcn_exp2f(v.x * A2[sb * NB + j]);
                    h[t][j] = fmaf(av[t][j], t ? h[t - 1][j] : h0[j], v.y * mp[t * mrow + sb * 2 * NB + j]);
                    y = fmaf(mp[t * mrow + sb * 2 * NB + NB + j], h[t][j], y);
                }
                if (zp) sy[w][t][lane] = y;
            }
#pragma unroll
            for (int t = TS - 1; t >= 0; --t) {
                const float2 v = sd[t][lane];
                const float dy = sg[t][lane];
                float2 s12 = sb ? ss[w][t][lane] : make_float2(0.f, 0.f);
                float val[2 * NB];
#pragma unroll
                for (int j = 0; j < NB; ++j) {
                    const int s = sb * NB + j;
                    const float gv = fmaf(mp[t * mrow + sb * 2 * NB + NB + j], dy, c[s]);
                    val[j] = gv * v.y;
                    val[NB + j] = dy * h[t][j];
                    s12.x = fmaf(gv, mp[t * mrow + sb * 2 * NB + j], s12.x);
                    c[s] = av[t][j] * gv;
                    const float qv = c[s] * (t ? h[t - 1][j] : h0[j]);
                    s12.y = fmaf(qv, A2[s], s12.y);
                    dA[s] = fmaf(qv, v.x, dA[s]);
                }
                ss[w][t][lane] = s12;
                const float sum = lane_sums<2 * NB>(val, lane);
                constexpr int PER = 64 / (2 * NB);
                if (lane % PER == 0) sm[t][(w * SB + sb) * 2 * NB + lane / PER] = sum;
            }
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < RPW; ++r) {
            const int row = w * RPW + r, t = tile * TS + row;
            const bool live = ok && t < len;
            const float2 x0 = ss[0][row][lane], x1 = ss[1][row][lane], x2 = ss[2][row][lane], x3 = ss[3][row][lane];
            const float s1 = (x0.x + x1.x) + (x2.x + x3.x), s2 = ((x0.y + x1.y) + (x2.y + x3.y)) * SQ_LN2;
            const float du = fmaf(cstep[r], s1, Dd * cg[r]);
            float dd = fmaf(cu[r], s1, s2);
            if (p.softplus) dd *= sq_sigmoid(craw[r]);
            dd = live ? dd : 0.f;
            dD = fmaf(cg[r], cu[r], dD);
            dbias += dd;
            if (ok && t < p.T) {
                const size_t o = orow + (size_t)t * p.C;
                ((T*)p.du)[o] = (T)(live ? du : 0.f);
                ((T*)p.ddelta)[o] = (T)dd;
                if (zp) {
                    const float y = fmaf(Dd, cu[r], (sy[0][row][lane] + sy[1][row][lane]) + (sy[2][row][lane] + sy[3][row][lane]));
                    ((T*)p.dz)[o] = (T)(live ? cdy[r] * y * sq_silu_slope(cz[r]) : 0.f);
                }
            }
        }
        // this block's share of dB and dC, in the layout of the maps
        constexpr int MW = 4 * SB * 2 * NB;
        float* mo = p.dmaps + (size_t)(cb % q.cbg) * ((size_t)p.B * q.Tp * mrow) + ((size_t)b * q.Tp + (size_t)tile * TS) * mrow + (size_t)g * 2 * q.NP;
        for (int i = threadIdx.x; i < TS * MW; i += 256) mo[(size_t)(i / MW) * mrow + i % MW] = sm[i / MW][i % MW];
        __syncthreads();
    }
    const size_t e = (size_t)b * q.chunks + chunk;
    if (ok) {
#pragma unroll
        for (int s = 0; s < NS; ++s) p.dparams[(e * (q.NP + 2) + state_of(w, s / NB, s % NB, NB)) * p.C + d] = dA[s];
        if (p.dstate && chunk == 0) {
#pragma unroll
            for (int s = 0; s < NS; ++s) {
                const int n = state_of(w, s / NB, s % NB, NB);
                if (n < p.N) p.dstate[((size_t)b * p.C + d) * p.N + n] = c[s];
            }
        }
    }
    sd[w][lane] = make_float2(dD, dbias);
    __syncthreads();
    if (w < 2 && ok) {
        const float v = w == 0 ? (sd[0][lane].x + sd[1][lane].x) + (sd[2][lane].x + sd[3][lane].x)
                               : (sd[0][lane].y + sd[1][lane].y) + (sd[2][lane].y + sd[3][lane].y);
        p.dparams[(e * (q.NP + 2) + q.NP + w) * p.C + d] = v;
    }
}

// dB, dC: the channel blocks' shares added up
template <typename T>
__global__ __launch_bounds__(256) void scan_dmaps_kernel(const float* __restrict__ dmaps, T* __restrict__ dB, T* __restrict__ dC, Plan q, int B,
                                                         int Tn, int N, int G) {
    const size_t total = (size_t)B * Tn * G * N, slab = (size_t)B * q.Tp * G * 2 * q.NP;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (size_t)gridDim.x * 256) {
        const int n = (int)(i % N);
        const size_t row = i / N;
        const int g = (int)(row % G);
        const size_t bt = row / G;
        const int t = (int)(bt % Tn), b = (int)(bt / Tn);
        const int sb = n / (4 * q.NB), w = (n / q.NB) % 4, j = n % q.NB;
        const float* s = dmaps + (((size_t)b * q.Tp + t) * G + g) * 2 * q.NP + (size_t)(w * q.SB + sb) * 2 * q.NB + j;
        float x = 0.f, y = 0.f;
        for (int k = 0; k < q.cbg; ++k, s += slab) { x += s[0]; y += s[q.NB]; }
        dB[i] = (T)x;
        dC[i] = (T)y;
    }
}

// dA [C][N], dD, ddelta_bias [C]: the items' and chunks' shares ([rows][NP + 2][C]) added up
__global__ __launch_bounds__(1024) void scan_dparams_kernel(const float* __restrict__ parts, int rows, int NP, int C, int N, float* __restrict__ dA,
                                                            float* __restrict__ dD, float* __restrict__ dbias) {
    __shared__ double acc[16][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const long col = (long)blockIdx.x * 64 + lane, cols = (long)(NP + 2) * C;
    double v = 0.0;
    if (col < cols)
        for (int r = w; r < rows; r += 16) v += (double)parts[(size_t)r * cols + col];
    acc[w][lane] = v;
    __syncthreads();
    if (w == 0 && col < cols) {
        for (int k = 1; k < 16; ++k) v += acc[k][lane];
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
    if ((long)B * q.nCb * q.chunks > 0x7fffffffL || (long)T + TS > 0x7fffffffL) return GA_ERR_ARG;
    return GA_OK;
}

int grid_for(size_t n) {
    const size_t g = (n + 255) / 256;
    return (int)(g < 4096 ? g : 4096);
}

template <typename T, int NB, int SB>
int launch_fwd(const Args& a, hipStream_t s) {
    const long blocks = (long)a.p.B * a.q.nCb;
    if (a.q.chunks > 1) {
        scan_fwd_kernel<T, NB, SB, true><<<(unsigned)(blocks * (a.q.chunks - 1)), 256, 0, s>>>(a);
        GA_CHECK_LAUNCH();
    }
    scan_fwd_kernel<T, NB, SB, false><<<(unsigned)(blocks * a.q.chunks), 256, 0, s>>>(a);
    GA_CHECK_LAUNCH();
    return GA_OK;
}

template <typename T, int NB, int SB>
int launch_bwd(const BwdArgs& a, hipStream_t s) {
    const long blocks = (long)a.p.B * a.q.nCb;
    if (a.q.chunks > 1) {
        scan_bwd_ends_kernel<T, NB, SB><<<(unsigned)(blocks * (a.q.chunks - 1)), 256, 0, s>>>(a);
        GA_CHECK_LAUNCH();
    }
    scan_bwd_kernel<T, NB, SB><<<(unsigned)(blocks * a.q.chunks), 256, 0, s>>>(a);
    GA_CHECK_LAUNCH();
    return GA_OK;
}

#define SCAN_DISPATCH(FN, T, ARGS)                        \
    (ARGS.q.SB == 4   ? FN<T, 4, 4>(ARGS, s)              \
     : ARGS.q.SB == 2 ? FN<T, 4, 2>(ARGS, s)              \
     : ARGS.q.NB == 4 ? FN<T, 4, 1>(ARGS, s)              \
     : ARGS.q.NB == 2 ? FN<T, 2, 1>(ARGS, s)              \
                      : FN<T, 1, 1>(ARGS, s))

template <typename T>
int fwd(const Args& a, hipStream_t s) {
    const ga_scan_params& p = a.p;
    scan_maps_kernel<T><<<grid_for((size_t)p.B * a.q.Tp * p.G * a.q.NP), 256, 0, s>>>((const T*)p.Bm, (const T*)p.Cm, p.maps, p.lengths, a.q, p.B, p.T,
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
    scan_dparams_kernel<<<(unsigned)((cols + 63) / 64), 1024, 0, s>>>(p.dparams, p.B * a.q.chunks, a.q.NP, p.C, p.N, p.dA, p.dD, p.ddelta_bias);
    GA_CHECK_LAUNCH();
    return GA_OK;
}

}  // namespace

extern "C" {

int ga_scan_sizes(int B, int T, int C, int N, int G, ga_scan_buffers* h_out) {
    if (!h_out || bad_sizes(B, T, C, N, G, GA_DTYPE_F32)) return GA_ERR_ARG;
    const Plan q = make_plan(B, T, C, N, G);
    h_out->maps = (size_t)B * q.Tp * G * 2 * q.NP;
    h_out->hs = (size_t)B * q.tiles * N * C;
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
