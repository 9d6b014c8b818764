// Selective state space scan:  h_t = exp(D_t A) h_{t-1} + D_t u_t B_t,  y_t = (<C_t, h_t> + D u_t) silu(z_t),  D_t = softplus(delta_t + bias)
// per channel d and state n, on channels-last activations; forward, backward and the single-token step.
//
// One block is 64 channels (one per lane) times all states (split over its four waves: a lane holds its wave's states in registers), walking
// along time in tiles of 16 rows.  What depends on a row and a channel alone (softplus, gates, the sums over states) is done once, four rows to
// a wave, and passes through LDS; B and C, which all channels of a group share, are first laid out in float32 in the order in which
// the waves read them (scan_maps_kernel) and come in as scalar loads, so that they cost no vector instruction and no LDS bandwidth.
// Time is cut into chunks where channels and items alone do not fill the card: a first kernel walks every chunk from zero, a small one carries
// the states from chunk to chunk, the main one then walks each chunk from the state that comes in.
//
// Bound by vector issue.  Counted at 16 x 2250 x 1024 with 16 states, bf16, for a state and row: 7.8 vector instructions forward and 22.6 backward (the
// states walked again, the adjoint, sums over 64 channels for dB and dC), 5.1 and 5.4 more in the first kernels, all that is done once per row and
// channel included; an exp2 in each of the four takes the time of two others.  The vector units are busy 92 % of the forward main kernel's time, 83 %
// of the backward one's (two waves a SIMD: registers), 94 and 93 % of the first kernels'.
// Times of whole passes, replayed from a graph: at that size forward 269 us (227 MB, 46 us of memory time), 274 with the saved states, backward 616;
// a process's first passes take up to 8 % more.  Kernel by kernel, which adds up to more: forward maps 6, first 120, carry 6, main 184; backward
// first 126, carry 6, main 544, sums 28.  12 x 375 x 512: 39 and 66 us; one prompt of 2250 x 512: 32 us.  Float32 at 16 x 2250 x 1024: 281 and 706 us.
// 8 states 185 and 404 us; half the items with 32 states 247 and 928 us (a wave's 8 states take turns, the rest waits in LDS, one block a CU); a
// quarter with 64 states 241 and 831 us.  Numbers of states between these pay for the next one: 12 states 266 and 605 us, half the items with 17
// 242 and 899 us, a quarter with 33 234 and 800 us.
#include "seq_common.h"

namespace {

constexpr int TS = 16;          // rows of a tile
constexpr int RPW = TS / 4;     // rows that one wave prepares and finishes
constexpr int MAX_CHUNKS = 256;

typedef const __attribute__((address_space(4))) float* uniform_ptr;
// `p` as a value that the compiler cannot trace: loads through it are issued where they stand, and not all at once at the top (their results
// would be parked in vector registers, a move each way for every value)
__device__ __forceinline__ uniform_ptr here(uniform_ptr p) {
    asm volatile("" : "+s"(p));
    return p;
}

struct Plan {
    int NS, NP;               // states of a wave, of the four waves
    int Cg, cbg, nCb;         // channels of a group, 64-channel blocks of a group, of all groups
    int tiles;                // of a sequence
    int chunks, chunk_tiles;  // tiles of a chunk
};

Plan make_plan(int B, int T, int C, int N, int G) {
    Plan q;
    q.NS = N <= 8 ? 2 : N <= 16 ? 4 : N <= 32 ? 8 : 16;
    q.NP = 4 * q.NS;
    q.Cg = C / G;
    q.cbg = (q.Cg + 63) / 64;
    q.nCb = q.cbg * G;
    q.tiles = (T + TS - 1) / TS;
    const long blocks = (long)B * q.nCb;
    // Chunks for four blocks a CU, and for eight where a chunk is still long enough (16 tiles) not to notice its start: 16 x 2250 x 1024, as a
    // process's first work, takes 291 + 616 us with eight, 295 + 626 with four, 314 + 634 with two; 12 x 375 x 512 38 + 66 us with four, 43 + 73 with
    // eight.
    long want = (1024 + blocks - 1) / blocks;
    if (q.tiles / want >= 16) want = (2048 + blocks - 1) / blocks;
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
    int vec;  // quads of channels can be read and written at once
};
struct BwdArgs {
    ga_scan_bwd_params p;
    Plan q;
    int vec;
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

// The wave's part of a tile's B and C on its way from memory to this XCD's L2 while the rows come: the scalar loads of a tile follow one another, and
// each would wait for memory by itself.  (One word of every 128 bytes or less; `arrived` keeps the load.)
template <int NS>
__device__ __forceinline__ float warm(const float* wave_maps, int lane) { return wave_maps[lane * (TS * 2 * NS) / 64]; }
__device__ __forceinline__ void arrived(float v) { asm volatile("" ::"v"(v)); }

// Where a block and a lane are.  `d` counts channels, unsigned so that an address is a scalar base plus a 32-bit offset.
struct Place {
    int lane, w, chunk, b, g, len, tile0, tile1;
    int end;  // tile1, or the tile behind the item's last row where that comes first: nothing happens in the tiles from there on
    unsigned d;
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
    x.d = (unsigned)(x.g * q.Cg + (x.ok ? din : q.Cg - 1));
    x.len = sq_len(lengths, x.b, T);
    x.tile0 = x.chunk * q.chunk_tiles;
    x.tile1 = min(x.tile0 + q.chunk_tiles, q.tiles);
    x.end = max(x.tile0, min(x.tile1, (x.len + TS - 1) / TS));
    x.item = (size_t)(x.b * G + x.g) * q.tiles;
    return x;
}
template <typename T>
__device__ __forceinline__ T& at(void* base, unsigned d) { return *(T*)((char*)sq_scalar(base) + d * (unsigned)sizeof(T)); }
template <typename T>
__device__ __forceinline__ T at(const void* base, unsigned d) { return *(const T*)((const char*)sq_scalar(base) + d * (unsigned)sizeof(T)); }

template <typename T> struct alignas(4 * sizeof(T)) Quad { T v[4]; };

// The four elements of a tile that a lane prepares and finishes.  VEC: four adjacent channels of one row, one access for all four rows of a wave;
// otherwise (alignment, odd widths) one channel of each of the four rows.  (16 x 2250 x 1024 x 16 bf16: 269 + 616 us; one channel at a time 275 + 726.)
template <bool VEC>
struct Elems {
    int lane, w, g, first, Cg;  // first: the block's first channel in its group
    __device__ __forceinline__ Elems(const Place& x, const Plan& q)
        : lane(x.lane), w(x.w), g(x.g), first((int)(blockIdx.x % q.nCb) % q.cbg * 64), Cg(q.Cg) {}
    __device__ __forceinline__ int row(int e) const { return w * RPW + (VEC ? lane >> 4 : e); }
    __device__ __forceinline__ int ch(int e) const { return VEC ? (lane & 15) * 4 + e : lane; }
    __device__ __forceinline__ bool ok() const { return first + ch(0) < Cg; }  // (VEC: groups of whole quads only)
    __device__ __forceinline__ unsigned d(int e) const {
        const int c = first + ch(0);
        return (unsigned)(g * Cg + (ok() ? c : Cg - (VEC ? 4 : 1)) + (VEC ? e : 0));
    }
};

// A wave's rows of an activation: RPW rows of every tile
template <typename T, bool VEC>
struct Rows {
    const char* base;  // the wave's first row of the current tile
    unsigned step;     // bytes from row to row, less than 2^24
    __device__ __forceinline__ Rows(const void* p, long bs, long ts, int b, int row)
        : base((const char*)p + (b * bs + row * ts) * (long)sizeof(T)), step((unsigned)(ts * (long)sizeof(T))) {}
    __device__ __forceinline__ void move(int tiles) { base += (long)(tiles * TS) * (long)step; }
    // `row0`: the wave's first row; rows behind the last one, T - 1, read that one: no branch between the loads
    __device__ __forceinline__ void load(Quad<T>& o, const Elems<VEC>& el, unsigned d0, int row0, int T_) const {
        const int over = max(0, row0 - (T_ - 1)), most = T_ - 1 - (row0 - over);
        const char* b = base - (long)(over * (int)step);
        if (VEC) {
            const unsigned off = __umul24((unsigned)min(el.lane >> 4, most), step) + d0 * (unsigned)sizeof(T);
            o = *(const Quad<T>*)(sq_scalar(b) + off);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) o.v[e] = at<T>(b + (long)(min(e, most) * (int)step), d0);
        }
    }
};
// the outputs' rows, packed: `base` the wave's first row of the tile
template <typename T, bool VEC>
__device__ __forceinline__ void store_elems(char* base, unsigned step, const Elems<VEC>& el, unsigned d0, int row0, int T_, const float (&v)[4]) {
    if (VEC) {
        if (el.ok() && row0 + (el.lane >> 4) < T_) {
            Quad<T> o;
#pragma unroll
            for (int e = 0; e < 4; ++e) o.v[e] = (T)v[e];
            *(Quad<T>*)(sq_scalar(base) + (__umul24((unsigned)el.lane >> 4, step) + d0 * (unsigned)sizeof(T))) = o;
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (el.ok() && row0 + e < T_) at<T>((void*)(base + (long)(e * (int)step)), d0) = (T)v[e];
    }
}
// values of the four elements to / from a [TS][64] array in LDS
template <bool VEC>
__device__ __forceinline__ void put(float (*a)[64], const Elems<VEC>& el, const float (&v)[4]) {
    if (VEC) *(float4*)&a[el.row(0)][el.ch(0)] = make_float4(v[0], v[1], v[2], v[3]);
    else
#pragma unroll
        for (int e = 0; e < 4; ++e) a[el.row(e)][el.ch(e)] = v[e];
}
template <bool VEC>
__device__ __forceinline__ void put2(float2 (*a)[64], const Elems<VEC>& el, const float (&x)[4], const float (&y)[4]) {
    if (VEC) {
        float4* p = (float4*)&a[el.row(0)][el.ch(0)];
        p[0] = make_float4(x[0], y[0], x[1], y[1]);
        p[1] = make_float4(x[2], y[2], x[3], y[3]);
    } else
#pragma unroll
        for (int e = 0; e < 4; ++e) a[el.row(e)][el.ch(e)] = make_float2(x[e], y[e]);
}
// the four waves' values added up
template <bool VEC>
__device__ __forceinline__ void get_sum(float (&o)[4], float (*a)[TS][64], const Elems<VEC>& el) {
    if (VEC) {
        const int r = el.row(0), c = el.ch(0);
        const float4 p = *(const float4*)&a[0][r][c], q = *(const float4*)&a[1][r][c], s = *(const float4*)&a[2][r][c], t = *(const float4*)&a[3][r][c];
        o[0] = (p.x + q.x) + (s.x + t.x), o[1] = (p.y + q.y) + (s.y + t.y), o[2] = (p.z + q.z) + (s.z + t.z), o[3] = (p.w + q.w) + (s.w + t.w);
    } else
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int r = el.row(e), c = el.ch(e);
            o[e] = (a[0][r][c] + a[1][r][c]) + (a[2][r][c] + a[3][r][c]);
        }
}
template <bool VEC>
__device__ __forceinline__ void get_sum2(float (&x)[4], float (&y)[4], float2 (*a)[TS][64], const Elems<VEC>& el) {
    if (VEC) {
        const int r = el.row(0), c = el.ch(0);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float4 v[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = *(const float4*)&a[k][r][c + 2 * h];
            x[2 * h] = (v[0].x + v[1].x) + (v[2].x + v[3].x), y[2 * h] = (v[0].y + v[1].y) + (v[2].y + v[3].y);
            x[2 * h + 1] = (v[0].z + v[1].z) + (v[2].z + v[3].z), y[2 * h + 1] = (v[0].w + v[1].w) + (v[2].w + v[3].w);
        }
    } else
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int r = el.row(e), c = el.ch(e);
            const float2 p = a[0][r][c], q = a[1][r][c], s = a[2][r][c], t = a[3][r][c];
            x[e] = (p.x + q.x) + (s.x + t.x), y[e] = (p.y + q.y) + (s.y + t.y);
        }
}

// 2^s c + end for any s.  The steps of a chunk may grow a state (A > 0, or negative steps) by more than float32 holds although the state itself, small or
// exactly zero, stays inside: powers of two above 2^126 go into c's exponent, where zero stays zero.  (c < 2^128 is at least 2^-149: beyond s = 277 what
// is not zero is infinite.  Up to s = 126 the bits are those of exp2(s) c + end; a NaN passes on.)
__device__ __forceinline__ float grown(float s, float c, float end) {
    const float t = s > 400.f ? 400.f : s, over = fmaxf(ceilf(t) - 126.f, 0.f);
    return fmaf(__builtin_amdgcn_exp2f(t - over), __builtin_ldexpf(c, (int)over), end);
}

// What comes into each chunk, from what each one leaves behind by itself, in place: carry' = exp(A sum of steps) carry + end, over the chunks
// in order (forward) or against it (backward: dir < 0), from `first` [B][C][N] (or zero).  A wave takes 64 states and one of SEGS runs of up to U
// chunks, all their loads in flight at once (few threads, a long way to memory); with more runs than one each is first walked from zero, and the
// runs' ends meet in LDS.  (As a loop at the start of every block of the main kernel it cost 11 of the 23 us that a prompt of 2250 rows and 8
// blocks spent there; as a kernel that walks 71 chunks in one run, 11 us.)
template <int SEGS, int U>
__global__ __launch_bounds__(SEGS > 1 ? SEGS * 64 : 256) void scan_carry_kernel(const float* __restrict__ A, const float* __restrict__ first,
                                                                               float* __restrict__ ends, const float* __restrict__ ends_step, Plan q,
                                                                               int B, int C, int N, int dir) {
    __shared__ float se[SEGS][64], st[SEGS][64];
    const int lane = threadIdx.x & 63, seg = SEGS > 1 ? threadIdx.x >> 6 : 0;
    const size_t id = SEGS > 1 ? (size_t)blockIdx.x * 64 + lane : (size_t)blockIdx.x * 256 + threadIdx.x, all = (size_t)B * N * C;
    const size_t i = id < all ? id : all - 1;
    const int d = (int)(i % C), n = (int)(i / C % N), b = (int)(i / C / N);
    const int run = (q.chunks + SEGS - 1) / SEGS, k0 = seg * run, k1 = min(k0 + run, q.chunks);  // (run <= U)
    const float A2 = A[(size_t)d * N + n] * SQ_LOG2E;
    float c = first ? first[((size_t)b * C + d) * N + n] : 0.f;
    const float* sp = ends_step + (size_t)b * q.chunks * C + d;
    float* ep = ends + ((size_t)b * q.chunks * q.NP + n) * C + d;
    float sum[U], end[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int k = min(k0 + u, q.chunks - 1), chunk = dir < 0 ? q.chunks - 1 - k : k;
        sum[u] = sp[(size_t)chunk * C];
        end[u] = ep[(size_t)chunk * q.NP * C];
    }
    if (SEGS > 1) {
        float total = 0.f, e = 0.f;
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (k0 + u < k1) {
                e = grown(sum[u] * A2, e, end[u]);
                total += sum[u];
            }
        se[seg][lane] = e;
        st[seg][lane] = total;
        __syncthreads();
        for (int j = 0; j < seg; ++j) c = grown(st[j][lane] * A2, c, se[j][lane]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (k0 + u < k1 && id < all) {
            const int chunk = dir < 0 ? q.chunks - 1 - (k0 + u) : k0 + u;
            ep[(size_t)chunk * q.NP * C] = c;
            c = grown(sum[u] * A2, c, end[u]);  // (what the last chunk leaves is written by no block, and used here by nobody)
        }
}

// ENDS: only the state that each chunk but the last leaves behind when it starts from zero, and the sum of its steps
// (the chunk's decay is exp(A * that sum)).  Otherwise the outputs, each chunk from the states of the chunks before it.
template <typename T, int NS, bool ENDS, bool HASZ, bool VEC>
__global__ __launch_bounds__(256) void scan_fwd_kernel(Args a) {
    const ga_scan_params& p = a.p;
    const Plan& q = a.q;
    // rows whose B and C are in scalar registers at a time, twice (one set on its way)
    constexpr int U = ENDS ? (NS <= 4 ? 4 : NS <= 8 ? 2 : 1) : (NS <= 4 ? 2 : 1);
    __shared__ __attribute__((aligned(16))) float2 sd[TS][64];
    __shared__ __attribute__((aligned(16))) float sy[ENDS ? 1 : 4][ENDS ? 1 : TS][64];
    const Place x = place(q, ENDS ? q.chunks - 1 : q.chunks, 0, p.G, p.T, p.lengths);
    const int lane = x.lane, w = x.w, len = x.len;
    const unsigned d = x.d;
    const Elems<VEC> el(x, q);
    const unsigned d0 = el.d(0);
    float bias[4], Dd[4], total[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        bias[e] = p.delta_bias ? p.delta_bias[el.d(e)] : 0.f;
        Dd[e] = !ENDS && p.D ? p.D[el.d(e)] : 0.f;
        total[e] = 0.f;
    }
    float A2[NS], h[NS];
#pragma unroll
    for (int s = 0; s < NS; ++s) {
        const int n = w * NS + s;
        const float v = p.A[(size_t)d * p.N + min(n, p.N - 1)] * SQ_LOG2E;
        A2[s] = n < p.N ? v : 0.f;
        h[s] = 0.f;
    }
    if (!ENDS && q.chunks > 1) {
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            const int n = w * NS + s;
            const float v = p.ends[(((size_t)x.b * q.chunks + x.chunk) * q.NP + min(n, p.N - 1)) * p.C + d];
            h[s] = n < p.N ? v : 0.f;
        }
    } else if (!ENDS && p.state) {
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            const int n = w * NS + s;
            const float v = p.state[((size_t)x.b * p.C + d) * p.N + min(n, p.N - 1)];
            h[s] = n < p.N ? v : 0.f;
        }
    }
    const int row0 = x.tile0 * TS + w * RPW;
    Rows<T, VEC> us(p.u, p.u_bs, p.u_ts, x.b, row0), ds(p.delta, p.delta_bs, p.delta_ts, x.b, row0), zs(p.z, p.z_bs, p.z_ts, x.b, row0);
    const unsigned ystep = (unsigned)p.C * (unsigned)sizeof(T);
    char* yp = (char*)p.y + ((size_t)x.b * p.T + row0) * ystep;
    Quad<T> ru, rd, rz;
    float wm;
    auto load = [&](int tile) __attribute__((always_inline)) {
        wm = warm<NS>(p.maps + ((x.item + tile) * 4 + w) * (TS * 2 * NS), lane);
        us.load(ru, el, d0, tile * TS + w * RPW, p.T);
        ds.load(rd, el, d0, tile * TS + w * RPW, p.T);
        if (HASZ) zs.load(rz, el, d0, tile * TS + w * RPW, p.T);
    };
    load(x.tile0);
    uniform_ptr mp = (uniform_ptr)(uintptr_t)(p.maps + ((x.item + x.tile0) * 4 + w) * (TS * 2 * NS));
    float m[2][U][2 * NS];
    auto fetch = [&](float (&o)[U][2 * NS], uniform_ptr at) __attribute__((always_inline)) {
        uniform_ptr from = here(at);
#pragma unroll
        for (int i = 0; i < U; ++i)
#pragma unroll
            for (int j = 0; j < (ENDS ? NS : 2 * NS); ++j) o[i][j] = from[i * 2 * NS + j];
    };
    for (int tile = x.tile0; tile < x.end; ++tile) {
        float cu[4], cz[4], step[4], su[4];
        bool live[4];
        arrived(wm);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            live[e] = el.ok() && tile * TS + el.row(e) < len;
            const float raw = (float)rd.v[e] + bias[e], soft = sq_softplus(raw);
            step[e] = live[e] ? p.softplus ? soft : raw : 0.f;
            cu[e] = live[e] ? (float)ru.v[e] : 0.f;
            cz[e] = HASZ ? (float)rz.v[e] : 0.f;
            total[e] += step[e];
            su[e] = step[e] * cu[e];
        }
        put2(sd, el, step, su);
        fetch(m[0], mp);
        __syncthreads();
        if (tile + 1 < x.end) {
            us.move(1), ds.move(1), zs.move(1);
            load(tile + 1);
        }
        if (!ENDS && p.hs && x.ok) {
            float* hp = p.hs + (((size_t)x.b * q.tiles + tile) * q.NP + w * NS) * p.C;
#pragma unroll
            for (int s = 0; s < NS; ++s) at<float>(hp + (size_t)s * p.C, d) = h[s];
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
        if constexpr (!ENDS) {
            float o[4];
            get_sum(o, sy, el);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                o[e] = fmaf(Dd[e], cu[e], o[e]);
                if (HASZ) o[e] *= sq_silu(cz[e]);
                o[e] = live[e] ? o[e] : 0.f;
            }
            store_elems<T>(yp, ystep, el, d0, tile * TS + w * RPW, p.T, o);
            yp += (size_t)TS * ystep;
        }
    }
    if constexpr (!ENDS) {
        const float zero[4] = {0.f, 0.f, 0.f, 0.f};
        for (int tile = x.end; tile < x.tile1; ++tile, yp += (size_t)TS * ystep) store_elems<T>(yp, ystep, el, d0, tile * TS + w * RPW, p.T, zero);
    }
    if (ENDS) {
        const size_t e = (size_t)x.b * q.chunks + x.chunk;
        if (x.ok) {
#pragma unroll
            for (int s = 0; s < NS; ++s) p.ends[(e * q.NP + w * NS + s) * p.C + d] = h[s];
        }
        put2(sd, el, total, total);
        __syncthreads();
        if (w == 0 && x.ok) {
            float v = 0.f;
#pragma unroll
            for (int t = 0; t < TS; ++t) v += sd[t][lane].x;
            p.ends_step[e * p.C + d] = v;
        }
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
template <typename T, int NS, bool HASZ, bool VEC>
__global__ __launch_bounds__(256) void scan_bwd_ends_kernel(BwdArgs a) {
    const ga_scan_bwd_params& p = a.p;
    const Plan& q = a.q;
    constexpr int U = NS <= 4 ? 4 : NS <= 8 ? 2 : 1;
    __shared__ __attribute__((aligned(16))) float2 sd[TS][64];
    const Place x = place(q, q.chunks - 1, 1, p.G, p.T, p.lengths);
    const int lane = x.lane, w = x.w, len = x.len;
    const unsigned d = x.d;
    const Elems<VEC> el(x, q);
    const unsigned d0 = el.d(0);
    float bias[4], total[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        bias[e] = p.delta_bias ? p.delta_bias[el.d(e)] : 0.f;
        total[e] = 0.f;
    }
    float A2[NS], c[NS];
#pragma unroll
    for (int s = 0; s < NS; ++s) {
        const int n = w * NS + s;
        const float v = p.A[(size_t)d * p.N + min(n, p.N - 1)] * SQ_LOG2E;
        A2[s] = n < p.N ? v : 0.f;
        c[s] = 0.f;
    }
    const int row0 = max(x.end - 1, 0) * TS + w * RPW;
    Rows<T, VEC> ds(p.delta, p.delta_bs, p.delta_ts, x.b, row0), zs(p.z, p.z_bs, p.z_ts, x.b, row0), gs(p.dy, (long)p.T * p.C, p.C, x.b, row0);
    Quad<T> rd, rz, rg;
    float wm;
    auto load = [&](int tile) __attribute__((always_inline)) {
        wm = warm<NS>(p.maps + ((x.item + tile) * 4 + w) * (TS * 2 * NS), lane);
        ds.load(rd, el, d0, tile * TS + w * RPW, p.T);
        gs.load(rg, el, d0, tile * TS + w * RPW, p.T);
        if (HASZ) zs.load(rz, el, d0, tile * TS + w * RPW, p.T);
    };
    load(max(x.end - 1, 0));
    float m[2][U][NS];
    auto fetch = [&](float (&o)[U][NS], uniform_ptr at) __attribute__((always_inline)) {
        uniform_ptr from = here(at);
#pragma unroll
        for (int i = 0; i < U; ++i)
#pragma unroll
            for (int j = 0; j < NS; ++j) o[i][j] = from[i * 2 * NS + NS + j];
    };
    for (int tile = x.end - 1; tile >= x.tile0; --tile) {
        uniform_ptr mp = (uniform_ptr)(uintptr_t)(p.maps + ((x.item + tile) * 4 + w) * (TS * 2 * NS));
        float step[4], dy[4];
        arrived(wm);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const bool live = el.ok() && tile * TS + el.row(e) < len;
            const float raw = (float)rd.v[e] + bias[e], soft = sq_softplus(raw);
            step[e] = live ? p.softplus ? soft : raw : 0.f;
            dy[e] = (float)rg.v[e];
            if (HASZ) dy[e] *= sq_silu((float)rz.v[e]);
            dy[e] = live ? dy[e] : 0.f;
            total[e] += step[e];
        }
        put2(sd, el, step, dy);
        fetch(m[0], mp + (TS - U) * 2 * NS);
        __syncthreads();
        if (tile > x.tile0) {
            ds.move(-1), zs.move(-1), gs.move(-1);
            load(tile - 1);
        }
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
    put2(sd, el, total, total);
    __syncthreads();
    if (w == 0 && x.ok) {
        float v = 0.f;
#pragma unroll
        for (int t = 0; t < TS; ++t) v += sd[t][lane].x;
        p.ends_step[e * p.C + d] = v;
    }
}

// Per tile, from the last to the first: the states again from the one saved at the tile's start (kept in registers, with the decays), then
// the adjoint backwards through them; NB states of a wave at a time.  With more than NB the adjoint, dA and the rows' values wait in LDS for their turn: a
// vector register spilled here is not only slow (the compiler has been seen to place such copies under a branch's mask).
template <typename T, int NS, bool HASZ, bool VEC>
__global__ __launch_bounds__(256, NS <= 4 ? 2 : 1) void scan_bwd_kernel(BwdArgs a) {
    const ga_scan_bwd_params& p = a.p;
    const Plan& q = a.q;
    constexpr int NB = NS < 4 ? NS : 4, SB = NS / NB, U = 2;
    // the next tile's rows on their way (float32 rows, or ones of single channels, spill: they are loaded where they are used, and the pass of
    // 16 x 2250 x 1024 x 16 takes 706 and 726 us in place of 616)
    constexpr bool AHEAD = SB == 1 && VEC && sizeof(T) == 2;
    __shared__ __attribute__((aligned(16))) float2 sd[TS][64];     // step, step * u
    __shared__ __attribute__((aligned(16))) float sg[TS][64];      // dy * gate
    __shared__ __attribute__((aligned(16))) float sy[4][TS][64];   // <C, h> over a wave's states
    __shared__ __attribute__((aligned(16))) float2 ss[4][TS][64];  // <g, B>, <g a h_prev, A>
    __shared__ float sm[4][TS][2 * NS];
    __shared__ float wait[SB > 1 ? 2 * NS + 28 : 1][SB > 1 ? 256 : 1];
    const Place x = place(q, q.chunks, 0, p.G, p.T, p.lengths);
    const int lane = x.lane, w = x.w, len = x.len;
    const unsigned d = x.d;
    const Elems<VEC> el(x, q);
    const unsigned d0 = el.d(0);
    float bias[4], Dd[4], dD[4], dbias[4];
    auto load_params = [&](const float* pb, const float* pD) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (pb) bias[e] = pb[el.d(e)];
            if (pD) Dd[e] = pD[el.d(e)];
        }
    };
#pragma unroll
    for (int e = 0; e < 4; ++e) bias[e] = Dd[e] = dD[e] = dbias[e] = 0.f;
    if (SB == 1) load_params(p.delta_bias, p.D);
    const int row0 = max(x.end - 1, 0) * TS + w * RPW;
    Rows<T, VEC> us(p.u, p.u_bs, p.u_ts, x.b, row0), ds(p.delta, p.delta_bs, p.delta_ts, x.b, row0), zs(p.z, p.z_bs, p.z_ts, x.b, row0),
        gs(p.dy, (long)p.T * p.C, p.C, x.b, row0);
    const unsigned ostep = (unsigned)p.C * (unsigned)sizeof(T);
    size_t orow = ((size_t)x.b * p.T + row0) * ostep;  // of the outputs, in bytes
    Quad<T> ru, rd, rz, rg;
    float hn[NB];
    auto load_h = [&](int tile, int sb) __attribute__((always_inline)) {
        const float* hp = p.hs + (((size_t)x.b * q.tiles + tile) * q.NP + w * NS + sb * NB) * p.C;
#pragma unroll
        for (int j = 0; j < NB; ++j) hn[j] = at<float>(hp + (size_t)j * p.C, d);
    };
    float wm;
    auto load = [&](int tile) __attribute__((always_inline)) {
        if (AHEAD) wm = warm<NS>(p.maps + ((x.item + tile) * 4 + w) * (TS * 2 * NS), lane);
        load_h(tile, 0);
        const int first = tile * TS + w * RPW;
        us.load(ru, el, d0, first, p.T);
        ds.load(rd, el, d0, first, p.T);
        gs.load(rg, el, d0, first, p.T);
        if (HASZ) zs.load(rz, el, d0, first, p.T);
    };
    if (AHEAD) load(max(x.end - 1, 0));
    float A2[NB], c[NB], dA[NB];
    auto load_A = [&](int sb) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            const int n = w * NS + sb * NB + j;
            const float v = p.A[(size_t)d * p.N + min(n, p.N - 1)] * SQ_LOG2E;
            A2[j] = n < p.N ? v : 0.f;
        }
    };
#pragma unroll
    for (int sb = 0; sb < SB; ++sb) {
        load_A(sb);
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            const int n = w * NS + sb * NB + j;
            c[j] = dA[j] = 0.f;
            if (n < p.N && x.ok) {
                if (q.chunks > 1) c[j] = p.ends[(((size_t)x.b * q.chunks + x.chunk) * q.NP + n) * p.C + d];
                else if (p.dlast) c[j] = p.dlast[((size_t)x.b * p.C + d) * p.N + n];
            }
        }
        if (SB > 1) {
#pragma unroll
            for (int j = 0; j < NB; ++j) {
                wait[sb * NB + j][threadIdx.x] = c[j];
                wait[NS + sb * NB + j][threadIdx.x] = 0.f;
            }
        }
    }
    // what only a tile's end needs is read again from the kernel's arguments there: kept over the loop it costs the scalar registers of B and C
    const __attribute__((address_space(4))) BwdArgs* args = (const __attribute__((address_space(4))) BwdArgs*)__builtin_amdgcn_kernarg_segment_ptr();
    for (int tile = x.end - 1; tile >= x.tile0; --tile) {
        uniform_ptr mp = (uniform_ptr)(uintptr_t)(p.maps + ((x.item + tile) * 4 + w) * (TS * 2 * NS));
        float cu[4], cslope[4], cz[4], csig[4], cdy[4], cstep[4], cg[4], su[4], h0[NB];
        if (!AHEAD) load(tile);
        if (AHEAD) arrived(wm);
        if (SB > 1) {
            const float* pb = p.delta_bias;
            asm volatile("" : "+s"(pb));  // (loaded here and not kept over the loop)
            load_params(pb, nullptr);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const bool live = el.ok() && tile * TS + el.row(e) < len;
            const float raw = (float)rd.v[e] + bias[e];
            float slope;
            const float soft = sq_softplus(raw, slope), step = p.softplus ? soft : raw;
            cslope[e] = live ? p.softplus ? slope : 1.f : 0.f;
            cstep[e] = live ? step : 0.f;
            cu[e] = live ? (float)ru.v[e] : 0.f;
            cdy[e] = live ? (float)rg.v[e] : 0.f;
            cz[e] = HASZ && live ? (float)rz.v[e] : 0.f;
            csig[e] = HASZ ? sq_sigmoid(cz[e]) : 1.f;
            cg[e] = HASZ ? cdy[e] * (cz[e] * csig[e]) : cdy[e];
            su[e] = cstep[e] * cu[e];
        }
        put2(sd, el, cstep, su);
        put(sg, el, cg);
        if (SB == 1) {
#pragma unroll
            for (int j = 0; j < NB; ++j) h0[j] = hn[j];
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float* keep = &wait[2 * NS + 7 * e][threadIdx.x];
                keep[0] = cu[e], keep[256] = cslope[e], keep[512] = cz[e], keep[768] = csig[e], keep[1024] = cdy[e], keep[1280] = cstep[e], keep[1536] = cg[e];
            }
        }
        __syncthreads();
        if (tile > x.tile0) {
            us.move(-1), ds.move(-1), zs.move(-1), gs.move(-1);
            if (AHEAD) load(tile - 1);
        }
#pragma unroll
        for (int sb = 0; sb < SB; ++sb) {
            if (SB > 1) {
                load_A(sb);
#pragma unroll
                for (int j = 0; j < NB; ++j) {
                    h0[j] = hn[j];
                    c[j] = wait[sb * NB + j][threadIdx.x];
                    dA[j] = wait[NS + sb * NB + j][threadIdx.x];
                }
                if (sb + 1 < SB) load_h(tile, sb + 1);
            }
            float h[TS][NB], av[TS][NB];
            float m[2][U][2 * NB];
            float2 v[2][U];
            auto fetch = [&](int set, int t0) __attribute__((always_inline)) {
                uniform_ptr from = here(mp + t0 * 2 * NS + sb * NB);
#pragma unroll
                for (int i = 0; i < U; ++i) {
#pragma unroll
                    for (int j = 0; j < NB; ++j) {
                        m[set][i][j] = from[i * 2 * NS + j];
                        m[set][i][NB + j] = from[i * 2 * NS + NS + j];
                    }
                    v[set][i] = sd[t0 + i][lane];
                }
            };
            float gy[2][U];
            auto fetch_back = [&](int set, int t0) __attribute__((always_inline)) {
                fetch(set, t0);
#pragma unroll
                for (int i = 0; i < U; ++i) gy[set][i] = sg[t0 + i][lane];
            };
            fetch(0, 0);
#pragma unroll
            for (int k = 0; k < TS / U; ++k) {
                if (k + 1 < TS / U) fetch((k + 1) & 1, (k + 1) * U);
                else fetch_back(0, TS - U);  // the way back starts where this one ends
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < U; ++i) {
                    const int t = k * U + i;
                    const float2 o = v[k & 1][i];
                    const float* mm = m[k & 1][i];
                    float y = sb && HASZ ? sy[w][t][lane] : 0.f;
#pragma unroll
                    for (int j = 0; j < NB; ++j) {
                        av[t][j] = __builtin_amdgcn_exp2f(o.x * A2[j]);
                        h[t][j] = fmaf(av[t][j], t ? h[t - 1][j] : h0[j], o.y * mm[j]);
                        y = fmaf(mm[NB + j], h[t][j], y);
                    }
                    if (HASZ) sy[w][t][lane] = y;
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            static_assert(TS / U % 2 == 0, "the first set is free at the end");
            // a row's 2 NB products are folded until a lane has one, summed over 2 NB lanes; KEEP rows of these then over the other lanes
            constexpr int KEEP = TS < 64 / (2 * NB) ? TS : 64 / (2 * NB);
            float part[KEEP];
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
                        const float gv = fmaf(mm[NB + j], dy, c[j]);
                        val[j] = gv * o.y;
                        val[NB + j] = dy * h[t][j];
                        s12.x = fmaf(gv, mm[j], s12.x);
                        c[j] = av[t][j] * gv;
                        const float qv = c[j] * (t ? h[t - 1][j] : h0[j]);
                        s12.y = fmaf(qv, A2[j], s12.y);
                        dA[j] = fmaf(qv, o.x, dA[j]);
                    }
                    ss[w][t][lane] = s12;
                    part[t % KEEP] = sq_fold_down<2 * NB, 32>(val, lane);
                    if (t % KEEP == 0) {
                        constexpr int PER = 64 / (2 * NB), EXTRA = PER / KEEP;
                        static_assert(EXTRA <= 2, "at most one lane bit is left");
                        float sum = sq_fold_down<KEEP, PER / 2>(part, lane);
                        if (EXTRA == 2) sum += sq_dpp<0xB1>(sum);
                        const int i2 = lane / PER, row = t + lane % PER / EXTRA;  // B's share in the first NB, C's in the others
                        sm[w][row][(i2 / NB) * NS + sb * NB + i2 % NB] = sum;     // (EXTRA lanes write the same sum)
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            if (SB > 1) {
#pragma unroll
                for (int j = 0; j < NB; ++j) {
                    wait[sb * NB + j][threadIdx.x] = c[j];
                    wait[NS + sb * NB + j][threadIdx.x] = dA[j];
                }
            }
        }
        __syncthreads();
        asm volatile("" : "+s"(args));
        const auto& pc = args->p;
        if (SB > 1) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float* keep = &wait[2 * NS + 7 * e][threadIdx.x];
                cu[e] = keep[0], cslope[e] = keep[256], cz[e] = keep[512], csig[e] = keep[768], cdy[e] = keep[1024], cstep[e] = keep[1280], cg[e] = keep[1536];
            }
        }
        if (SB > 1) load_params(nullptr, pc.D);
        float s1[4], s2[4], y[4], du[4], dd[4], dz[4];
        get_sum2(s1, s2, ss, el);
        if (HASZ) get_sum(y, sy, el);
#pragma unroll
        for (int e = 0; e < 4; ++e) {  // (behind an item's end cstep, cg, cslope, cdy are zero, and with them what is stored)
            du[e] = fmaf(cstep[e], s1[e], Dd[e] * cg[e]);
            dd[e] = fmaf(cu[e], s1[e], s2[e] * SQ_LN2) * cslope[e];
            dD[e] = fmaf(cg[e], cu[e], dD[e]);
            dbias[e] += dd[e];
            dz[e] = HASZ ? cdy[e] * fmaf(Dd[e], cu[e], y[e]) * csig[e] * fmaf(cz[e], 1.f - csig[e], 1.f) : 0.f;
        }
        const int first = tile * TS + w * RPW;
        store_elems<T>((char*)pc.du + orow, ostep, el, d0, first, p.T, du);
        store_elems<T>((char*)pc.ddelta + orow, ostep, el, d0, first, p.T, dd);
        if (HASZ) store_elems<T>((char*)pc.dz + orow, ostep, el, d0, first, p.T, dz);
        orow -= (size_t)TS * ostep;
        // this block's share of dB and dC, in the layout of the maps
        const int slab = (blockIdx.x % q.nCb) % q.cbg;
        float* mo = pc.dmaps + ((size_t)slab * pc.B * pc.G * q.tiles + x.item + tile) * (4 * TS * 2 * NS);
#pragma unroll
        for (int i = 0; i < (4 * TS * 2 * NS + 255) / 256; ++i) {
            const int k = i * 256 + threadIdx.x;
            if (4 * TS * 2 * NS % 256 == 0 || k < 4 * TS * 2 * NS) at<float>(mo, (unsigned)k) = (&sm[0][0][0])[k];
        }
        // (no barrier: what the next tile writes before its first one is read here by nobody but its writer, or before the one above)
    }
    if (x.end < x.tile1) {  // tiles behind the item's end: no gradient
        const float zero[4] = {0.f, 0.f, 0.f, 0.f};
        const int slab = (blockIdx.x % q.nCb) % q.cbg;
        asm volatile("" : "+s"(args));
        const auto& pc = args->p;
        for (int tile = x.end; tile < x.tile1; ++tile) {
            const int first = tile * TS + w * RPW;
            const size_t o = ((size_t)x.b * pc.T + first) * ostep;
            store_elems<T>((char*)pc.du + o, ostep, el, d0, first, pc.T, zero);
            store_elems<T>((char*)pc.ddelta + o, ostep, el, d0, first, pc.T, zero);
            if (HASZ) store_elems<T>((char*)pc.dz + o, ostep, el, d0, first, pc.T, zero);
            float* mo = pc.dmaps + ((size_t)slab * pc.B * pc.G * q.tiles + x.item + tile) * (4 * TS * 2 * NS);
            for (int i = threadIdx.x; i < 4 * TS * 2 * NS; i += 256) mo[i] = 0.f;
        }
    }
    const size_t e = (size_t)x.b * q.chunks + x.chunk;
#pragma unroll
    for (int sb = 0; sb < SB; ++sb) {
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            const int s = sb * NB + j, n = w * NS + s;
            const float dAv = SB > 1 ? wait[NS + s][threadIdx.x] : dA[j], cv = SB > 1 ? wait[s][threadIdx.x] : c[j];
            if (x.ok) {
                p.dparams[(e * (q.NP + 2) + n) * p.C + d] = dAv;
                if (p.dstate && x.chunk == 0 && n < p.N) p.dstate[((size_t)x.b * p.C + d) * p.N + n] = cv;
            }
        }
    }
    __syncthreads();
    put2(sd, el, dD, dbias);
    __syncthreads();
    if (w < 2 && x.ok) {
        float v = 0.f;
#pragma unroll
        for (int t = 0; t < TS; ++t) v += w == 0 ? sd[t][lane].x : sd[t][lane].y;
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

// One token: a thread holds four states of a channel, 1 << shift threads a channel, a block channels of one item (nb blocks an item); the state is
// read and written once, and everything else is small: 256 x 1024 x 16 states, bf16, 7.8 us (35.7 MB: 4.6 TB/s), 17.3 with single elements of
// state, A, B and C (odd N or unaligned bases); 256 x 1024 x 64 28 us; one item of 512 x 16 2.5 us.
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void scan_step_kernel(ga_scan_step_params p, int shift, unsigned nb) {
    const unsigned b = blockIdx.x / nb, d = (blockIdx.x % nb) * (256u >> shift) + (threadIdx.x >> shift);
    const int n0 = (int)(threadIdx.x & ((1u << shift) - 1)) * 4;
    const unsigned dd = min(d, (unsigned)p.C - 1), g = p.G == 1 ? 0 : dd / (unsigned)(p.C / p.G);
    const bool ok = d < (unsigned)p.C, mine = ok && n0 < p.N;
    float* const state = p.state + (size_t)b * p.state_bs;
    const T* const Bp = (const T*)p.Bm + (size_t)b * p.b_bs;
    const T* const Cp = (const T*)p.Cm + (size_t)b * p.c_bs;
    float h[4], A[4];
    Quad<T> Bv, Cv;
    if (VEC) {
        const unsigned n = (unsigned)min(n0, p.N - 4);
        *(float4*)h = *(const float4*)(state + (size_t)dd * p.N + n);
        *(float4*)A = *(const float4*)(p.A + (size_t)dd * p.N + n);
        Bv = *(const Quad<T>*)(Bp + g * p.N + n);
        Cv = *(const Quad<T>*)(Cp + g * p.N + n);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const unsigned n = (unsigned)min(n0 + j, p.N - 1);
            h[j] = state[(size_t)dd * p.N + n];
            A[j] = p.A[(size_t)dd * p.N + n];
            Bv.v[j] = Bp[(size_t)g * p.N + n];
            Cv.v[j] = Cp[(size_t)g * p.N + n];
        }
    }
    const float u = (float)((const T*)p.u + (size_t)b * p.u_bs)[dd];
    const float z = p.z ? (float)((const T*)p.z + (size_t)b * p.z_bs)[dd] : 0.f, D = p.D ? p.D[dd] : 0.f;
    const float raw = (float)((const T*)p.delta + (size_t)b * p.delta_bs)[dd] + (p.delta_bias ? p.delta_bias[dd] : 0.f);
    const float step = p.softplus ? sq_softplus(raw) : raw, su = step * u;
    float y = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        h[j] = fmaf(__builtin_amdgcn_exp2f(step * (A[j] * SQ_LOG2E)), h[j], su * (float)Bv.v[j]);
        if (mine && (VEC || n0 + j < p.N)) y = fmaf((float)Cv.v[j], h[j], y);
    }
    if (mine) {
        if (VEC) *(float4*)(state + (size_t)d * p.N + n0) = *(float4*)h;
        else
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (n0 + j < p.N) state[(size_t)d * p.N + n0 + j] = h[j];
    }
    for (int o = 1 << shift >> 1; o > 0; o >>= 1) y += __shfl_xor(y, o, 64);
    if (mine && n0 == 0) {
        y = fmaf(D, u, y);
        if (p.z) y *= sq_silu(z);
        ((T*)p.y + (size_t)b * p.C)[d] = (T)y;
    }
}

int bad_sizes(int B, int T, int C, int N, int G, int dtype) {
    if (B < 1 || T < 1 || T > 0x7fffffff - TS || C < 1 || C > GA_SCAN_MAX_STRIDE || N < 1 || N > GA_SCAN_MAX_STATES || G < 1 || C % G) return GA_ERR_ARG;
    if (dtype != GA_DTYPE_F32 && dtype != GA_DTYPE_BF16) return GA_ERR_ARG;
    const Plan q = make_plan(B, T, C, N, G);
    if ((long)B * q.nCb * q.chunks > 0x7fffffffL || (long)B * G > 0x7fffffffL || ((size_t)B * N * C + 63) / 64 > 0x7fffffffUL)
        return GA_ERR_ARG;
    return GA_OK;
}

// whether rows of this tensor (absent: any) can be accessed in quads
bool quads(const void* p, long bs, long ts, size_t elem) { return !p || (!((uintptr_t)p & (4 * elem - 1)) && bs % 4 == 0 && ts % 4 == 0); }
bool bad_strides(long a, long b, long c) {
    return a < 0 || b < 0 || c < 0 || a > GA_SCAN_MAX_STRIDE || b > GA_SCAN_MAX_STRIDE || c > GA_SCAN_MAX_STRIDE;
}

int grid_for(size_t n) {
    const size_t g = (n + 255) / 256;
    return (int)(g < 4096 ? g : 4096);
}

int launch_carry(const float* A, const float* first, float* ends, const float* ends_step, const Plan& q, int B, int C, int N, int dir, hipStream_t s) {
    const size_t states = (size_t)B * N * C;  // (2^23 at the most: sequences are cut where there are fewer than 2048 blocks of 64 channels)
    static_assert(MAX_CHUNKS <= 16 * 16, "runs of the carry kernel");
    // (the whole forward pass, 8 chunks at 16 x 2250 x 1024: 291 us, 296 with loads for 32; 32 chunks at 4 x 2250 x 512: 63 us, 66 with 16 runs)
    if (q.chunks <= 8) scan_carry_kernel<1, 8><<<(unsigned)((states + 255) / 256), 256, 0, s>>>(A, first, ends, ends_step, q, B, C, N, dir);
    else if (q.chunks <= 32) scan_carry_kernel<1, 32><<<(unsigned)((states + 255) / 256), 256, 0, s>>>(A, first, ends, ends_step, q, B, C, N, dir);
    else scan_carry_kernel<16, 16><<<(unsigned)((states + 63) / 64), 1024, 0, s>>>(A, first, ends, ends_step, q, B, C, N, dir);
    GA_CHECK_LAUNCH();
    return GA_OK;
}

template <typename T, int NS, bool HASZ, bool VEC>
int launch_fwd_as(const Args& a, hipStream_t s) {
    const long blocks = (long)a.p.B * a.q.nCb;
    if (a.q.chunks > 1) {
        scan_fwd_kernel<T, NS, true, false, VEC><<<(unsigned)(blocks * (a.q.chunks - 1)), 256, 0, s>>>(a);
        GA_CHECK_LAUNCH();
        if (const int rc = launch_carry(a.p.A, a.p.state, a.p.ends, a.p.ends_step, a.q, a.p.B, a.p.C, a.p.N, 1, s)) return rc;
    }
    scan_fwd_kernel<T, NS, false, HASZ, VEC><<<(unsigned)(blocks * a.q.chunks), 256, 0, s>>>(a);
    GA_CHECK_LAUNCH();
    return GA_OK;
}
template <typename T, int NS>
int launch_fwd(const Args& a, hipStream_t s) {
    if (a.vec) return a.p.z ? launch_fwd_as<T, NS, true, true>(a, s) : launch_fwd_as<T, NS, false, true>(a, s);
    return a.p.z ? launch_fwd_as<T, NS, true, false>(a, s) : launch_fwd_as<T, NS, false, false>(a, s);
}

template <typename T, int NS, bool HASZ, bool VEC>
int launch_bwd_as(const BwdArgs& a, hipStream_t s) {
    const long blocks = (long)a.p.B * a.q.nCb;
    if (a.q.chunks > 1) {
        scan_bwd_ends_kernel<T, NS, HASZ, VEC><<<(unsigned)(blocks * (a.q.chunks - 1)), 256, 0, s>>>(a);
        GA_CHECK_LAUNCH();
        if (const int rc = launch_carry(a.p.A, a.p.dlast, a.p.ends, a.p.ends_step, a.q, a.p.B, a.p.C, a.p.N, -1, s)) return rc;
    }
    scan_bwd_kernel<T, NS, HASZ, VEC><<<(unsigned)(blocks * a.q.chunks), 256, 0, s>>>(a);
    GA_CHECK_LAUNCH();
    return GA_OK;
}
template <typename T, int NS>
int launch_bwd(const BwdArgs& a, hipStream_t s) {
    constexpr bool V = NS <= 8;  // (64 states: no registers for quads)
    if (V && a.vec) return a.p.z ? launch_bwd_as<T, NS, true, V>(a, s) : launch_bwd_as<T, NS, false, V>(a, s);
    return a.p.z ? launch_bwd_as<T, NS, true, false>(a, s) : launch_bwd_as<T, NS, false, false>(a, s);
}

#define SCAN_DISPATCH(FN, T, ARGS)                 \
    (ARGS.q.NS == 16  ? FN<T, 16>(ARGS, s)         \
     : ARGS.q.NS == 8 ? FN<T, 8>(ARGS, s)          \
     : ARGS.q.NS == 4 ? FN<T, 4>(ARGS, s)          \
                      : FN<T, 2>(ARGS, s))

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
    Args a{p, make_plan(p.B, p.T, p.C, p.N, p.G), 0};
    if (!p.u || !p.delta || !p.A || !p.Bm || !p.Cm || !p.y || !p.maps || (a.q.chunks > 1 && (!p.ends || !p.ends_step))) return GA_ERR_ARG;
    if (!sq_launch_fits((size_t)p.B * a.q.nCb * a.q.chunks, 256)) return GA_ERR_ARG;
    if (bad_strides(p.u_ts, p.delta_ts, p.z_ts)) return GA_ERR_ARG;
    if ((uintptr_t)p.maps & 15) return GA_ERR_ALIGN;
    const size_t el = dtype == GA_DTYPE_BF16 ? 2 : 4;
    a.vec = a.q.Cg % 4 == 0 && quads(p.u, p.u_bs, p.u_ts, el) && quads(p.delta, p.delta_bs, p.delta_ts, el) && quads(p.z, p.z_bs, p.z_ts, el) &&
            quads(p.y, 0, 0, el);
    return dtype == GA_DTYPE_BF16 ? fwd<bf16_t>(a, s) : fwd<float>(a, s);
}

int ga_scan_bwd(const ga_scan_bwd_params* hp, int dtype, hipStream_t s) {
    if (!hp) return GA_ERR_ARG;
    const ga_scan_bwd_params& p = *hp;
    const int rc = bad_sizes(p.B, p.T, p.C, p.N, p.G, dtype);
    if (rc) return rc;
    BwdArgs a{p, make_plan(p.B, p.T, p.C, p.N, p.G), 0};
    if (!p.u || !p.delta || !p.A || !p.dy || !p.maps || !p.hs || !p.du || !p.ddelta || !p.dA || !p.dBm || !p.dCm || !p.dmaps || !p.dparams ||
        (!p.z) != (!p.dz) || (a.q.chunks > 1 && (!p.ends || !p.ends_step)))
        return GA_ERR_ARG;
    if (!sq_launch_fits((size_t)p.B * a.q.nCb * a.q.chunks, 256) || !sq_launch_fits(((size_t)(a.q.NP + 2) * p.C + 31) / 32, 1024)) return GA_ERR_ARG;
    if (bad_strides(p.u_ts, p.delta_ts, p.z_ts)) return GA_ERR_ARG;
    if ((uintptr_t)p.maps & 15) return GA_ERR_ALIGN;
    const size_t el = dtype == GA_DTYPE_BF16 ? 2 : 4;
    a.vec = a.q.Cg % 4 == 0 && quads(p.u, p.u_bs, p.u_ts, el) && quads(p.delta, p.delta_bs, p.delta_ts, el) && quads(p.z, p.z_bs, p.z_ts, el) &&
            quads(p.dy, 0, 0, el) && quads(p.du, 0, 0, el) && quads(p.ddelta, 0, 0, el) && quads(p.dz, 0, 0, el);
    return dtype == GA_DTYPE_BF16 ? bwd<bf16_t>(a, s) : bwd<float>(a, s);
}

int ga_scan_step(const ga_scan_step_params* hp, int dtype, hipStream_t s) {
    if (!hp) return GA_ERR_ARG;
    const ga_scan_step_params& p = *hp;
    const int rc = bad_sizes(p.B, 1, p.C, p.N, p.G, dtype);
    if (rc) return rc;
    if (!p.u || !p.delta || !p.A || !p.Bm || !p.Cm || !p.state || !p.y) return GA_ERR_ARG;
    int shift = 0;
    while ((4 << shift) < p.N) ++shift;
    const size_t nb = ((size_t)p.C + (256 >> shift) - 1) / (256 >> shift), blocks = nb * p.B;
    if (!sq_launch_fits(blocks, 256)) return GA_ERR_ARG;
    const bool vec = p.N % 4 == 0 && p.state_bs % 4 == 0 && p.b_bs % 4 == 0 && p.c_bs % 4 == 0 && !(((uintptr_t)p.state | (uintptr_t)p.A) & 15) &&
                     !(((uintptr_t)p.Bm | (uintptr_t)p.Cm) & (dtype == GA_DTYPE_BF16 ? 7 : 15));
    if (dtype == GA_DTYPE_BF16) {
        if (vec) scan_step_kernel<bf16_t, true><<<(unsigned)blocks, 256, 0, s>>>(p, shift, (unsigned)nb);
        else scan_step_kernel<bf16_t, false><<<(unsigned)blocks, 256, 0, s>>>(p, shift, (unsigned)nb);
    } else {
        if (vec) scan_step_kernel<float, true><<<(unsigned)blocks, 256, 0, s>>>(p, shift, (unsigned)nb);
        else scan_step_kernel<float, false><<<(unsigned)blocks, 256, 0, s>>>(p, shift, (unsigned)nb);
    }
    GA_CHECK_LAUNCH();
    return GA_OK;
}

}  // extern "C"
