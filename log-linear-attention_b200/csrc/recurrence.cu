// Gated linear recurrence of independent channels,
//     h_t = exp(g_t) h_{t-1} + x_t,   o_t = h_t
// and its gradients: with e_t = exp(g_t) dh_t, what token t hands back to the state before it,
//     dh_t = do_t + e_{t+1},   dx_t = dh_t,   dg_t = e_t h_{t-1},   dh_0 = e_1.
//
// A run of tokens acts on a state as h -> A h + H, with A the product of its decays and H its own final state, and on e in the same form
// from its other end; runs compose.  LPR lanes of a warp take RUN tokens of LPR VEC neighbouring channels, the others the runs behind them; a CTA takes the runs of a
// tile of TILE tokens, a cluster of CTAs neighbouring tiles of a strip of channels, and the cluster walks the strip: one pass over the data, all sums in fp32, in an
// order that the sizes alone decide.
//
// It is bound by memory as long as little else is issued.  Tiles come to shared memory by asynchronous copies a round ahead, each warp its own rows, and are
// read, and their decays formed, once.  A cluster's barrier costs its CTAs about a microsecond a round, hence runs as long as registers and shared memory
// leave room for with two CTAs an SM (one in the forward of fp32 pairs of channels, whose two rounds take 131 KB), and clusters no larger than fill the chip.
// 2 x 16384 tokens of 2048 channels, bf16 with fp32 decays: forward 99 us, backward 189 us behind other calls (108 and 197 with cold caches), 5.4 and 5.0 TB/s of what they cannot do without.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "../../include/llattn.h"
#include "launch_count.h"
#include "pairs.cuh"

namespace llattn {
namespace rec {

typedef __nv_bfloat16 bf16;
namespace cg = cooperative_groups;
constexpr int WARPS = 8, SLOTS = 2, MAX_RANKS = 16;
constexpr int FWD_RUN = 16, BWD_RUN = 8;         // (three tensors: 16 tokens leave room for one CTA an SM)
constexpr int STATES = 64;                       // tokens from one state that the forward keeps to the next

struct Params {
    const void *x, *g, *d_o;
    const float* h0;          // (B,D) or null: zeros.  Backward: the gradient of the last state, or null
    void *o, *dx, *dg;
    float* h_last;            // (B,D) or null.  Backward: the gradient of the initial state, or null
    float* starts;            // (B, ceil(T / STATES), D) or null: the state before every STATES-th token
    int T, D, strips;         // strips of channels a sequence
};

// exp(g).  For bf16 callers 2^(g log2 e): ex2.approx is off by 2^-22 of the value at most and flushes what is below 2^-126; the rounding of its argument adds |g| 2^-24, and that of log2 e
// |g| 2^-26.  They round outputs to 2^-8, and expf has four times the instructions, which tiles that come from memory at full rate leave no room for.  fp32 callers get expf, 2^-22 of the
// value for all g and without the bias of ex2.approx (-1.9e-8 of the value on average where g is in (-1, 0)), which the states of tens of tokens add up: 3 x 1999
// tokens of 1001 channels, gates as logsigmoid(N(3, 1)), o 2.2e-7 off 64 bits with ex2.approx, 1.2e-7 with expf, 24 / 40 us with either.
template <bool EXACT>
__device__ __forceinline__ float decay(float g) {
    if constexpr (EXACT) return expf(g);
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(g * 1.4426950408889634f));
    return y;
}
template <bool EXACT>
__device__ __forceinline__ F2 decay(F2 g) {
    if constexpr (EXACT) {
        const float2 x = both(g);
        return pair(expf(x.x), expf(x.y));
    }
    const float2 t = both(mul(g, splat<F2>(1.4426950408889634f)));
    float2 y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y.x) : "f"(t.x));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y.y) : "f"(t.y));
    return pair(y.x, y.y);
}

// The VEC channels of a lane as a number: one value, or a pair.
template <int VEC>
struct Number {
    typedef F2 T;
};
template <>
struct Number<1> {
    typedef float T;
};
__device__ __forceinline__ void load(const bf16* p, float& v) { v = __bfloat162float(*p); }
__device__ __forceinline__ void load(const float* p, float& v) { v = *p; }
__device__ __forceinline__ void load(const bf16* p, F2& v) {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(p);
    v = pair(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ void load(const float* p, F2& v) { v.v = *reinterpret_cast<const unsigned long long*>(p); }
__device__ __forceinline__ void store(bf16* p, float v) { *p = __float2bfloat16(v); }
__device__ __forceinline__ void store(float* p, float v) { *p = v; }
__device__ __forceinline__ void store(bf16* p, F2 v) {
    const float2 f = both(v);
    uint32_t w;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(f.y), "f"(f.x));
    *reinterpret_cast<uint32_t*>(p) = w;
}
__device__ __forceinline__ void store(float* p, F2 v) { *reinterpret_cast<unsigned long long*>(p) = v.v; }
// (A, H): h -> A h + H
template <typename T>
struct Map {
    T A, H;
    __device__ __forceinline__ T operator()(T h) const { return fma2(A, h, H); }
};

// A warp's rows (tokens) of LPR VEC values of a tensor in shared memory, RUN of them for each of its 32 / LPR runs, brought there by asynchronous copies of CP bytes (0: by
// loads and stores); what lies behind the sequence or the channels is filled with zeros, which change nothing (a decay of 1, nothing added).  Runs are a row further
// apart than they are long, so that lanes of different runs read different banks.
template <int RUN, int LPR, typename E, int VEC, int CP>
struct Stage {
    static constexpr int SUB = 32 / LPR, ROWS = SUB * RUN, ROW = LPR * VEC * sizeof(E), PAD = SUB > 1 ? ROW : 0, BYTES = ROWS * ROW + SUB * PAD;
    // `src`: row 0, channel 0 of the strip (read where `left` > 0 alone); `cols` channels and `left` tokens are there
    static __device__ __forceinline__ void issue(unsigned char* dst, const E* src, long ld, int left, int cols, int lane) {
        if constexpr (CP == 0) {
            static_assert(VEC == 1, "a value a lane");
            const int first = lane / LPR * RUN, c = lane % LPR;
            E v[RUN];
#pragma unroll
            for (int i = 0; i < RUN; ++i) v[i] = first + i < left && c < cols ? src[(first + i) * ld + c] : E(0.f);
#pragma unroll
            for (int i = 0; i < RUN; ++i) reinterpret_cast<E*>(dst + (first + i) * ROW + lane / LPR * PAD)[c] = v[i];
        } else {
            constexpr int PER = CP / (int)sizeof(E), A_ROW = ROW / CP, N = ROWS * A_ROW / 32;              // values a copy, copies a row, copies a lane
            constexpr int STEP = 32 / A_ROW;                                                              // rows that a copy of the warp takes
            static_assert(32 % A_ROW == 0 && (RUN % STEP == 0 || STEP % RUN == 0), "whole rows, and whole runs of them or parts of one run");
            const int row = lane / A_ROW, at = lane % A_ROW * PER;
            const uint32_t to = (uint32_t)__cvta_generic_to_shared(dst + lane * CP) + (STEP > RUN ? row / RUN * PAD : 0);
            const E* from = src + row * ld + at;
            if (left >= ROWS && cols == LPR * VEC) {                                                      // most tiles: nothing to test
#pragma unroll
                for (int i = 0; i < N; ++i, from += STEP * ld) copy(to + i * 32 * CP + i * STEP / RUN * PAD, from, CP);
            } else {
#pragma unroll
                for (int i = 0; i < N; ++i, from += STEP * ld) {
                    const bool in = row + i * STEP < left && at < cols;                                   // (cols is a multiple of PER)
                    copy(to + i * 32 * CP + i * STEP / RUN * PAD, in ? from : src, in ? CP : 0);
                }
            }
        }
    }
    // `bytes` of CP bytes (a constant where nothing was tested); the rest are zeros
    static __device__ __forceinline__ void copy(uint32_t to, const E* from, int bytes) {
        if constexpr (CP == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(to), "l"(from), "r"(bytes) : "memory");
        else if constexpr (CP > 0) asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;\n" ::"r"(to), "l"(from), "n"(CP), "r"(bytes) : "memory");
    }
    // the lane's run
    static __device__ __forceinline__ void read(const unsigned char* at, int lane, typename Number<VEC>::T (&v)[RUN]) {
        at += lane / LPR * (RUN * ROW + PAD);
#pragma unroll
        for (int i = 0; i < RUN; ++i) load(reinterpret_cast<const E*>(at + i * ROW) + lane % LPR * VEC, v[i]);
    }
};
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_but() { asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory"); }
// Where a CTA is, and what forward and backward do alike.
template <int LPR, int VEC, int TILE>
struct Place {
    static constexpr int SUB = 32 / LPR;
    cg::cluster_group cluster;
    int ranks, rank, lane, sub, col, warp, b, c0, c, cols, NT, rounds;
    bool there;
    typedef typename Number<VEC>::T T;
    Map<T> (*all)[LPR];           // [2][ranks]: the cluster's tiles', of every other round
    __device__ Place(const Params& p, unsigned char* behind_slots) : cluster(cg::this_cluster()) {
        ranks = cluster.num_blocks();
        rank = cluster.block_rank();
        lane = threadIdx.x & 31;
        sub = lane / LPR;
        col = lane % LPR;
        warp = threadIdx.x >> 5;
        const int unit = blockIdx.x / ranks;
        b = unit / p.strips;
        c0 = unit % p.strips * LPR * VEC;
        c = c0 + col * VEC;
        cols = min(LPR * VEC, p.D - c0);
        there = c < p.D;
        NT = (p.T + TILE - 1) / TILE;
        rounds = (NT + ranks - 1) / ranks;
        all = reinterpret_cast<Map<T>(*)[LPR]>(behind_slots);
    }
    // Takes `carry` over the round's tiles, in the order of the ranks, given this CTA's; returns what reaches it.  Every run of a warp writes to other ranks.
    __device__ __forceinline__ T exchange(int round, const Map<T>& m, T& carry) {
        for (int x = warp * SUB + sub; x < ranks; x += WARPS * SUB) *cluster.map_shared_rank(&all[(round & 1) * ranks + rank][col], x) = m;
        __syncwarp();
        cluster.sync();
        T mine = carry;
        for (int x = 0; x < ranks; ++x) {
            if (x == rank) mine = carry;
            carry = all[(round & 1) * ranks + x][col](carry);
        }
        return mine;
    }
};

// A run's map -> that of the warp's runs up to it; returns that of those before it.  UP: tokens in order, else from the last run on.
template <bool UP, int LPR, typename T>
__device__ __forceinline__ Map<T> warp_scan(int sub, Map<T>& m) {
    constexpr int SUB = 32 / LPR;
    const int place = UP ? sub : SUB - 1 - sub;
    Map<T> before = {splat<T>(1.f), splat<T>(0.f)};
#pragma unroll
    for (int d = 1; d < SUB; d *= 2) {
        const T a = UP ? shfl_up(m.A, d * LPR) : shfl_down(m.A, d * LPR), h = UP ? shfl_up(m.H, d * LPR) : shfl_down(m.H, d * LPR);
        if (place >= d) {
            m.H = fma2(m.A, h, m.H);
            m.A = mul(m.A, a);
        }
    }
    if constexpr (SUB > 1) {
        const T a = UP ? shfl_up(m.A, LPR) : shfl_down(m.A, LPR), h = UP ? shfl_up(m.H, LPR) : shfl_down(m.H, LPR);
        if (place > 0) before = Map<T>{a, h};
    }
    return before;
}

template <typename X, typename G, int LPR, int VEC, int CPX, int CPG>
__global__ void __launch_bounds__(32 * WARPS, 2) recurrence_fwd_kernel(const __grid_constant__ Params p) {
    chain_wait();
    constexpr int RUN = FWD_RUN, SUB = 32 / LPR, TILE = WARPS * SUB * RUN;
    static_assert(STATES % RUN == 0, "states are kept at the starts of runs");
    using SX = Stage<RUN, LPR, X, VEC, CPX>;
    using SG = Stage<RUN, LPR, G, VEC, CPG>;
    constexpr int BYTES = SX::BYTES + SG::BYTES;
    extern __shared__ __align__(16) unsigned char staged[];           // [SLOTS][WARPS][BYTES], then Place::all
    typedef typename Number<VEC>::T T;
    __shared__ Map<T> agg[2][WARPS][LPR];                             // of the warps' runs, for every other round
    Place<LPR, VEC, TILE> at(p, staged + SLOTS * WARPS * BYTES);
    const int lane = at.lane, warp = at.warp;
    const long ld = p.D, base = (long)at.b * p.T * ld + at.c0;
    const auto slot = [&](int round) { return staged + (round % SLOTS * WARPS + warp) * BYTES; };
    const auto bring = [&](int round) {
        if (round < at.rounds) {
            const int t0 = (round * at.ranks + at.rank) * TILE + warp * SUB * RUN, left = p.T - t0;
            const long from = base + (left > 0 ? t0 * ld : 0);
            SX::issue(slot(round), static_cast<const X*>(p.x) + from, ld, left, at.cols, lane);
            SG::issue(slot(round) + SX::BYTES, static_cast<const G*>(p.g) + from, ld, left, at.cols, lane);
        }
        copies_commit();
    };
    bring(0);
    if (at.ranks > 1) at.cluster.sync();                              // every CTA is there to be written to
    T carry = splat<T>(0.f);
    if (p.h0 && at.there) load(p.h0 + (long)at.b * p.D + at.c, carry);
    for (int round = 0; round < at.rounds; ++round) {
        const int t0 = (round * at.ranks + at.rank) * TILE + (warp * SUB + at.sub) * RUN, left = p.T - t0;      // (a tile behind the last changes nothing)
        bring(round + 1);                                             // (into the slot of the round before, which all lanes have read)
        copies_but<1>();
        __syncwarp();
        T v[RUN], a[RUN], h;
        SX::read(slot(round), lane, v);
        SG::read(slot(round) + SX::BYTES, lane, a);
        Map<T> m = {splat<T>(1.f), splat<T>(0.f)};
#pragma unroll
        for (int i = 0; i < RUN; ++i) {
            a[i] = decay<sizeof(X) == 4>(a[i]);
            m.A = mul(m.A, a[i]);
            m.H = fma2(a[i], m.H, v[i]);
        }
        const Map<T> before = warp_scan<true, LPR>(at.sub, m);
        if (at.sub == SUB - 1) agg[round & 1][warp][at.col] = m;
        __syncthreads();
        if (at.ranks == 1) {
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                if (w == warp) h = carry;
                carry = agg[round & 1][w][at.col](carry);
            }
        } else {
            Map<T> all = {splat<T>(1.f), splat<T>(0.f)}, warps;       // of the tile; of the warps before this one
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                const Map<T> r = agg[round & 1][w][at.col];
                if (w == warp) warps = all;
                all.A = mul(all.A, r.A);
                all.H = r(all.H);
            }
            h = warps(at.exchange(round, all, carry));
        }
        if constexpr (SUB > 1) h = before(h);
        if (p.starts && t0 % STATES == 0 && at.there && left > 0) store(p.starts + ((long)at.b * ((p.T + STATES - 1) / STATES) + t0 / STATES) * p.D + at.c, h);
        if (at.there) {
            X* o = static_cast<X*>(p.o) + base + t0 * ld + at.col * VEC;
#pragma unroll
            for (int i = 0; i < RUN; ++i, o += ld) {
                if (i < left) {
                    h = fma2(a[i], h, v[i]);
                    store(o, h);
                }
            }
        }
        __syncwarp();
    }
    if (p.h_last && at.rank == 0 && threadIdx.x < LPR && at.there) store(p.h_last + (long)at.b * p.D + at.c, carry);
}

// The same from the other end: e takes the place of the state, the cluster's tiles are counted from the last one.  The states before a tile's tokens are
// made again from the one that the forward kept.
template <typename X, typename G, int LPR, int VEC, int CPX, int CPG>
__global__ void __launch_bounds__(32 * WARPS, 2) recurrence_bwd_kernel(const __grid_constant__ Params p) {
    chain_wait();
    constexpr int RUN = BWD_RUN, SUB = 32 / LPR, TILE = WARPS * SUB * RUN;
    static_assert(TILE % STATES == 0, "a tile starts where a state is kept");
    using SX = Stage<RUN, LPR, X, VEC, CPX>;
    using SG = Stage<RUN, LPR, G, VEC, CPG>;
    constexpr int BYTES = 2 * SX::BYTES + SG::BYTES;
    extern __shared__ __align__(16) unsigned char staged[];
    typedef typename Number<VEC>::T T;
    __shared__ Map<T> agg[2][WARPS][LPR];                             // of the warps' runs: A and E
    __shared__ T own[2][WARPS][LPR];                                  // H
    Place<LPR, VEC, TILE> at(p, staged + SLOTS * WARPS * BYTES);
    const int lane = at.lane, warp = at.warp, NS = (p.T + STATES - 1) / STATES;
    const long ld = p.D, base = (long)at.b * p.T * ld + at.c0;
    const auto tile_of = [&](int round) { return at.NT - 1 - round * at.ranks - at.rank; };        // (below 0: nothing there)
    const auto slot = [&](int round) { return staged + (round % SLOTS * WARPS + warp) * BYTES; };
    const auto bring = [&](int round) {
        if (round < at.rounds) {
            const int tile = tile_of(round), t0 = tile * TILE + warp * SUB * RUN, left = tile < 0 ? 0 : p.T - t0;
            const long from = base + (left > 0 ? t0 * ld : 0);
            SX::issue(slot(round), static_cast<const X*>(p.x) + from, ld, left, at.cols, lane);
            SX::issue(slot(round) + SX::BYTES, static_cast<const X*>(p.d_o) + from, ld, left, at.cols, lane);
            SG::issue(slot(round) + 2 * SX::BYTES, static_cast<const G*>(p.g) + from, ld, left, at.cols, lane);
        }
        copies_commit();
    };
    bring(0);
    if (at.ranks > 1) at.cluster.sync();
    T carry = splat<T>(0.f);
    if (p.h0 && at.there) load(p.h0 + (long)at.b * p.D + at.c, carry);
    for (int round = 0; round < at.rounds; ++round) {
        const int tile = tile_of(round), t0 = tile * TILE + (warp * SUB + at.sub) * RUN, left = tile < 0 ? 0 : p.T - t0, par = round & 1;
        bring(round + 1);
        T v[RUN], a[RUN], d[RUN], h = splat<T>(0.f), e;
        if (at.there && tile >= 0) load(p.starts + ((long)at.b * NS + tile * (TILE / STATES)) * p.D + at.c, h);
        copies_but<1>();
        __syncwarp();
        SX::read(slot(round), lane, v);
        SX::read(slot(round) + SX::BYTES, lane, d);
        SG::read(slot(round) + 2 * SX::BYTES, lane, a);
        Map<T> up = {splat<T>(1.f), splat<T>(0.f)}, down = up;
#pragma unroll
        for (int i = 0; i < RUN; ++i) {
            a[i] = decay<sizeof(X) == 4>(a[i]);
            up.A = mul(up.A, a[i]);
            up.H = fma2(a[i], up.H, v[i]);
        }
#pragma unroll
        for (int i = RUN - 1; i >= 0; --i) down.H = mul(a[i], add(d[i], down.H));
        down.A = up.A;
        const Map<T> before = warp_scan<true, LPR>(at.sub, up), behind = warp_scan<false, LPR>(at.sub, down);
        if (at.sub == SUB - 1) own[par][warp][at.col] = up.H;
        if (at.sub == 0) agg[par][warp][at.col] = down;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < WARPS; ++w)
            if (w < warp) h = fma2(agg[par][w][at.col].A, h, own[par][w][at.col]);
        if (at.ranks == 1) {
#pragma unroll
            for (int w = WARPS - 1; w >= 0; --w) {
                if (w == warp) e = carry;
                carry = agg[par][w][at.col](carry);
            }
        } else {
            Map<T> all = {splat<T>(1.f), splat<T>(0.f)}, warps;       // of the tile; of the warps behind this one
#pragma unroll
            for (int w = WARPS - 1; w >= 0; --w) {
                const Map<T> r = agg[par][w][at.col];
                if (w == warp) warps = all;
                all.A = mul(all.A, r.A);
                all.H = r(all.H);
            }
            e = warps(at.exchange(round, all, carry));
        }
        if constexpr (SUB > 1) {
            h = before(h);
            e = behind(e);
        }
        // the states before the run's tokens, in the place of x
#pragma unroll
        for (int i = 0; i < RUN; ++i) {
            const T next = fma2(a[i], h, v[i]);
            v[i] = h;
            h = next;
        }
        if (at.there && left > 0) {
            const long to = base + t0 * ld + at.col * VEC;
            X* dx = static_cast<X*>(p.dx) + to;
            G* dg = static_cast<G*>(p.dg) + to;
            if (left >= RUN) {                                        // (a test a token took 1 to 9 %)
                dx += (RUN - 1) * ld;
                dg += (RUN - 1) * ld;
#pragma unroll
                for (int i = RUN - 1; i >= 0; --i, dx -= ld, dg -= ld) {
                    const T dh = add(d[i], e);
                    e = mul(a[i], dh);
                    store(dx, dh);
                    store(dg, mul(e, v[i]));
                }
            } else {
#pragma unroll
                for (int i = RUN - 1; i >= 0; --i) {
                    if (i < left) {
                        const T dh = add(d[i], e);
                        e = mul(a[i], dh);
                        store(dx + i * ld, dh);
                        store(dg + i * ld, mul(e, v[i]));
                    }
                }
            }
        }
        __syncwarp();
    }
    if (p.h_last && at.rank == 0 && threadIdx.x < LPR && at.there) store(p.h_last + (long)at.b * p.D + at.c, carry);
}

template <typename X, typename G>
__global__ void __launch_bounds__(256) recurrence_step_kernel(float* h, const X* x, const G* g, X* o, long n) {
    chain_wait();
    const long i = (long)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    float v, a;
    load(x + i, v);
    load(g + i, a);
    v = fmaf(decay<sizeof(X) == 4>(a), h[i], v);
    h[i] = v;
    store(o + i, v);
}

// How wide a strip is and how many CTAs share it: what costs least, among clusters that run at once for all strips.
template <typename KernT>
struct Launch {
    KernT kern;
    long units;                       // sequences x strips
    int NT;
    size_t smem, summary;             // of a CTA, and more for each CTA of the cluster
    int LPR;
    float best;                       // cost
    cudaLaunchAttribute attr[2];
    cudaLaunchConfig_t cfg;
    int ranks;
    Launch(KernT kern, long units, int NT, size_t smem, size_t summary, int LPR)
        : kern(kern), units(units), NT(NT), smem(smem), summary(summary), LPR(LPR), best(INFINITY), attr{}, cfg{}, ranks(1) {
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[1].val.programmaticStreamSerializationAllowed = 1;
        cfg.blockDim = dim3(32 * WARPS);
    }
    void clusters_of(int n) {
        ranks = n;
        attr[0].val.clusterDim.x = n;
        cfg.gridDim = dim3((unsigned)(units * n));
        cfg.dynamicSmemBytes = smem + 2 * n * summary;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
    }
    cudaError_t choose() {
        struct Room {
            int dev;
            const void* kern;
            int clusters[MAX_RANKS + 1];          // of n CTAs that the device runs at once (0: not asked yet)
        };
        static thread_local Room table[128] = {};
        int dev;
        cudaError_t e = cudaGetDevice(&dev);
        if (e != cudaSuccess) return e;
        Room& room = table[((reinterpret_cast<uintptr_t>(kern) >> 4) + dev) & 127];
        if (room.dev != dev || room.kern != reinterpret_cast<const void*>(kern)) {
            e = allow_smem(kern, smem + 2 * MAX_RANKS * summary);
            if (e == cudaSuccess) e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
            if (e != cudaSuccess) return e;
            room = Room{dev, reinterpret_cast<const void*>(kern), {}};
        }
        if (units > 0x7fffffffl) return cudaSuccess;                   // (too narrow)
        int fastest = 1;
        best = cost(1);
        for (int n = 2; n <= NT && n <= MAX_RANKS && units * n <= AT_ONCE; ++n) {
            if (cost(n) >= best) continue;
            clusters_of(n);
            if (room.clusters[n] == 0) {
                e = cudaOccupancyMaxActiveClusters(&room.clusters[n], kern, &cfg);
                if (e != cudaSuccess) return e;
                if (room.clusters[n] == 0) room.clusters[n] = -1;
            }
            if (room.clusters[n] < units) continue;
            best = cost(n);
            fastest = n;
        }
        clusters_of(fastest);
        return cudaSuccess;
    }
    // Rounds, and two for the start, weighted with what one takes in this width and with what a cluster's CTAs wait for each other, for waves of two CTAs an SM, or one: a
    // bound on what runs at once that the forward of fp32 pairs, one CTA an SM, does not reach.  (Fitted to 18 shapes, 1 to 32 sequences of 100 to 32768 tokens, 64 to 4096 channels, with 1 to
    // 16 CTAs a strip of each width.  Forward and backward in us where few CTAs a strip, or many, are faster: 3 x 1999 tokens of 1001 channels, fp32, strips of 16 alone 24 / 40, of 32 in
    // clusters of two 26 / 51; 32768 tokens of 2048, bf16, strips of 32 in clusters of four 94 / 206, of 16 alone 103 / 290; 8192 tokens of 4096, fp32, strips of 16 alone 69 / 112, of 32 alone
    // 62 / 183: the forward is known to be off there.)
    static constexpr int AT_ONCE = 2 * 148;
    float cost(int n) const {
        const long ctas = units * n, rest = ctas % AT_ONCE;
        const float waves = (float)(ctas / AT_ONCE) + (rest == 0 ? 0.f : rest <= 148 ? 0.95f : 1.f);
        return (float)((NT + n - 1) / n + 2) * waves * (LPR == 32 ? 1.f : LPR == 16 ? 1.04f : 1.3f) * (n > 1 ? 1.5f + 0.15f * (float)(n - 2) : 1.f);
    }
    cudaError_t go(const Params& p, cudaStream_t st) {
        cfg.stream = st;
        cfg.attrs = attr;
        cfg.numAttrs = 2;
        const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p);
        if (e == cudaSuccess) LLATTN_LAUNCHED();
        return e;
    }
};
// LPR lanes of VEC channels a run; copies of CPX and CPG bytes (0: straight loads)
template <bool BACK, typename X, typename G, int LPR, int VEC, int CPX, int CPG>
auto launch_of(const Params& p, int B) {
    constexpr int RUN = BACK ? BWD_RUN : FWD_RUN, TILE = WARPS * (32 / LPR) * RUN;
    constexpr size_t SMEM = (size_t)SLOTS * WARPS * ((BACK ? 2 : 1) * Stage<RUN, LPR, X, VEC, CPX>::BYTES + Stage<RUN, LPR, G, VEC, CPG>::BYTES);
    const long units = (long)B * ((p.D + LPR * VEC - 1) / (LPR * VEC));
    if constexpr (BACK) return Launch<void (*)(Params)>(recurrence_bwd_kernel<X, G, LPR, VEC, CPX, CPG>, units, (p.T + TILE - 1) / TILE, SMEM, LPR * VEC * sizeof(float2), LPR);
    else return Launch<void (*)(Params)>(recurrence_fwd_kernel<X, G, LPR, VEC, CPX, CPG>, units, (p.T + TILE - 1) / TILE, SMEM, LPR * VEC * sizeof(float2), LPR);
}
// Strips as wide as a warp, or a half or a quarter of that with longer tiles: clusters of many CTAs wait longer for each other than narrow strips cost.
template <bool BACK, typename X, typename G, int VEC, int CPX, int CPG>
cudaError_t scan_with(Params p, int B, cudaStream_t st) {
    Launch<void (*)(Params)> l[3] = {launch_of<BACK, X, G, 32, VEC, CPX, CPG>(p, B), launch_of<BACK, X, G, 16, VEC, CPX, CPG>(p, B), launch_of<BACK, X, G, 8, VEC, CPX, CPG>(p, B)};
    int best = 0;
    for (int i = 0; i < 3; ++i) {
        const cudaError_t e = l[i].choose();
        if (e != cudaSuccess) return e;
        if (l[i].best < l[best].best) best = i;
    }
    p.strips = (p.D + (32 >> best) * VEC - 1) / ((32 >> best) * VEC);
    return l[best].go(p, st);
}
// Copies as wide as rows of D values start: 16 bytes where D fills whole words of them, else the pair or the value of a lane.
template <bool BACK, typename X, typename G>
cudaError_t scan(const Params& p, int B, cudaStream_t st) {
    if (p.D % (16 / (int)sizeof(X)) == 0) return scan_with<BACK, X, G, 2, 16, 16>(p, B, st);
    if (p.D % 2 == 0) return scan_with<BACK, X, G, 2, 2 * sizeof(X), 2 * sizeof(G)>(p, B, st);
    if constexpr (sizeof(X) == 4) return scan_with<BACK, X, G, 1, 4, 4>(p, B, st);
    else return scan_with<BACK, X, G, 1, 0, 0>(p, B, st);
}
template <bool BACK>
int scan_of(int x_f32, int g_f32, const Params& p, int B, void* stream) {
    cudaStream_t st = (cudaStream_t)stream;
    if (x_f32) return (int)scan<BACK, float, float>(p, B, st);
    return (int)(g_f32 ? scan<BACK, bf16, float>(p, B, st) : scan<BACK, bf16, bf16>(p, B, st));
}
int check(int x_f32, int g_f32, long B, long T, long D) {
    if (B < 1 || T < 1 || D < 1 || (x_f32 && !g_f32)) return LLATTN_ERR_UNSUPPORTED_SHAPE;
    if (T > (1 << 30) || B * ((D + 31) / 32) > 0x7fffffffl) return LLATTN_ERR_UNSUPPORTED_SHAPE;
    return 0;
}

}  // namespace rec
}  // namespace llattn

using namespace llattn;

extern "C" {

size_t llattn_recurrence_states_bytes(int B, int T, int D) {
    if (rec::check(0, 0, B, T, D) != 0) return 0;
    return (size_t)B * ((T + rec::STATES - 1) / rec::STATES) * D * sizeof(float);
}

int llattn_recurrence_fwd(const void* x, int x_is_f32, const void* g, int g_is_f32, const float* h0, void* o, float* h_last, float* states,
                          int B, int T, int D, void* stream) {
    const int rc = rec::check(x_is_f32, g_is_f32, B, T, D);
    if (rc != 0) return rc;
    if (!x || !g || !o) return LLATTN_ERR_NULL;
    if (misaligned(16, {x, g, h0, o, h_last, states})) return LLATTN_ERR_ALIGNMENT;
    rec::Params p = {};
    p.x = x;
    p.g = g;
    p.h0 = h0;
    p.o = o;
    p.h_last = h_last;
    p.starts = states;
    p.T = T;
    p.D = D;
    return rec::scan_of<false>(x_is_f32, g_is_f32, p, B, stream);
}

int llattn_recurrence_bwd(const void* x, int x_is_f32, const void* g, int g_is_f32, const float* states, const void* d_o, const float* dh_last,
                          void* dx, void* dg, float* dh0, int B, int T, int D, void* stream) {
    const int rc = rec::check(x_is_f32, g_is_f32, B, T, D);
    if (rc != 0) return rc;
    if (!x || !g || !states || !d_o || !dx || !dg) return LLATTN_ERR_NULL;
    if (misaligned(16, {x, g, states, d_o, dh_last, dx, dg, dh0})) return LLATTN_ERR_ALIGNMENT;
    rec::Params p = {};
    p.x = x;
    p.g = g;
    p.d_o = d_o;
    p.h0 = dh_last;
    p.dx = dx;
    p.dg = dg;
    p.h_last = dh0;
    p.starts = const_cast<float*>(states);
    p.T = T;
    p.D = D;
    return rec::scan_of<true>(x_is_f32, g_is_f32, p, B, stream);
}

int llattn_recurrence_step(float* h, const void* x, int x_is_f32, const void* g, int g_is_f32, void* o, int B, int D, void* stream) {
    const int rc = rec::check(x_is_f32, g_is_f32, B, 1, D);
    if (rc != 0) return rc;
    if (!h || !x || !g || !o) return LLATTN_ERR_NULL;
    if (misaligned(16, {h, x, g, o})) return LLATTN_ERR_ALIGNMENT;
    const long n = (long)B * D;
    if ((n + 255) / 256 > 0x7fffffffl) return LLATTN_ERR_UNSUPPORTED_SHAPE;
    const unsigned grid = (unsigned)((n + 255) / 256);
    cudaStream_t st = (cudaStream_t)stream;
    cudaError_t e;
    typedef rec::bf16 bf16;
    if (x_is_f32)
        e = launch_chained(rec::recurrence_step_kernel<float, float>, grid, 256, 0, st, h, (const float*)x, (const float*)g, (float*)o, n);
    else if (g_is_f32)
        e = launch_chained(rec::recurrence_step_kernel<bf16, float>, grid, 256, 0, st, h, (const bf16*)x, (const float*)g, (bf16*)o, n);
    else
        e = launch_chained(rec::recurrence_step_kernel<bf16, bf16>, grid, 256, 0, st, h, (const bf16*)x, (const bf16*)g, (bf16*)o, n);
    if (e == cudaSuccess) LLATTN_LAUNCHED();
    return (int)e;
}

}  // extern "C"
