// Sliding-window attention backward on the 5th-generation tensor cores: two kernels that make S and dP again from q, k, v, do and the statistics of the
// forward, so that every gradient is a sum in one CTA's tensor memory, in an order that the sizes alone decide.
//
// dQ: a CTA takes a tile of 128 queries of a head and walks the tiles of keys that they see,
//     S = Q K^T, dP = dO V^T,   dS = exp2(c S - lse) (dP - delta) as bf16 in the place of S,   dQ += dS K.
// dK, dV: a CTA takes a tile of 128 tokens of k and v and walks the tiles of queries that see it, of all heads that share it,
//     S^T = K Q^T, dP^T = V dO^T,   P^T = exp2(c S^T - lse), dV += P^T dO,   dS^T = P^T (dP^T - delta), dK += dS^T Q.
// P and dS are rounded to bf16 for those products: dq and dk are 1.40 to 1.47 times as far off 64 bits as their own rounding makes them, whatever the sizes (2.4e-3 in norm), but for
// sequences of few tokens, see there.
// In both, four or eight warps do the exponentials (64 columns a thread), one issues products, one brings tiles through two rings; the products of one
// half of a step run under the other half's exponentials.  (Summing dQ beside dK and dV would save two of the seven products a pair of tiles, for
// atomics on 64 KB of fp32 a pair.)
// T = 16384, 32 query heads on 8, K = 128, window 2048: 1.61 ms, 0.80 PFLOP/s counting five products (1.12 of the seven made).  The exponentials' side of a step is longer
// than its products: about 2100 cycles for 1536 of dQ, 2750 for 2048 of dK and dV; call after call the clocks give way to the power limit.  (Q and dO as operands in tensor memory, which
// halves what their products read from shared memory: 1.4 % less there, 2 to 3 % more for short sequences.)
#include "window.cuh"

namespace llattn {
namespace win {

namespace bwd {
// Two rings of tiles: those that two products of a step need, far apart (NA of them), and those of one (NB).  With K = 128 five tiles fit beside the two that stay, three
// and two: the next but one of either kind is on its way while a step runs; with K = 64 two and two, in each of two CTAs.  (One ring of four for both kinds: the dQ kernel waited for its keys, 527 us at T = 8192,
// 32 heads, window 2048.)
//
// A step is K columns of scores (keys in the dQ kernel, queries in the other) by 128 rows, 64 columns a thread: with K = 128 a whole tile, two threads a row, a CTA an SM; with
// K = 64 half a tile, a thread a row, and two CTAs an SM, whose waits and products run under each other's exponentials (whole tiles in one CTA there: 71 us for 62, 2 x 1999 tokens, 16 heads,
// window 512; 114 for 101, 8 x 2000 tokens, 8 heads on 2, window 300).  (With K = 128 the sums dV and dK alone fill half of tensor memory.)
template <int K>
struct Cta {
    static constexpr int HALVES = K / 64, STEPS = TILE / K;                          // threads a row; steps a tile
    static constexpr int WARPS = 4 * HALVES, MMA_WARP = WARPS, TMA_WARP = WARPS + 1, THREADS = 32 * WARPS + 128, PER_SM = K == 64 ? 2 : 1;
    static constexpr int TM = 4 * K;                                                 // columns of tensor memory: four blocks of K
    static constexpr int NA = K == 64 ? 2 : 3, NB = 2;
    static constexpr uint32_t TILE_BYTES = TILE * K * 2;
    static constexpr uint32_t stay_off = 0, a_off = 2 * TILE_BYTES, b_off = a_off + NA * TILE_BYTES;
    static constexpr uint32_t stat_off = b_off + NB * TILE_BYTES;                    // float [NA + NB][128]: lse beside A tiles of queries, delta beside B tiles
    static constexpr uint32_t bar_off = stat_off + (NA + NB) * TILE * 4, total = bar_off + 256;
    static_assert((total + 1024) * PER_SM <= 228 * 1024, "CTAs an SM");
    // registers: 384 threads are launched with 168 each, 256 (two CTAs an SM) with 128; 4 warps give theirs to the exponentials
    static __device__ __forceinline__ void regs_issue() {
        if constexpr (K == 128) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;\n");
        else asm volatile("setmaxnreg.dec.sync.aligned.u32 56;\n");
    }
    static __device__ __forceinline__ void regs_rows() {
        if constexpr (K == 128) asm volatile("setmaxnreg.inc.sync.aligned.u32 216;\n");
        else asm volatile("setmaxnreg.inc.sync.aligned.u32 200;\n");
    }
};
// The steps of a ring of N tiles: slot and phase of step n.
template <int N>
struct Ring {
    uint64_t *full, *empty;
    __device__ __forceinline__ uint64_t* filled(int n) const { return full + n % N; }
    __device__ __forceinline__ uint64_t* freed(int n) const { return empty + n % N; }
    static __device__ __forceinline__ uint32_t phase(int n) { return (n / N) & 1; }
    // the slot of step n is free
    __device__ __forceinline__ bool wait_free(int n, volatile int* abort) const { return n < N || umma::mbar_wait(freed(n), phase(n) ^ 1, abort); }
    __device__ __forceinline__ void init() const {
        for (int i = 0; i < N; ++i) {
            umma::mbar_init(full + i, 1);
            umma::mbar_init(empty + i, 1);
        }
    }
    // the copies in flight of `issued` tiles have ended
    __device__ __forceinline__ void drain(int issued) const {
        for (int i = issued > N ? issued - N : 0; i < issued; ++i) umma::mbar_wait(filled(i), phase(i));
    }
};

// exp2(c s - shift) of 64 scores; shift(u) gives the pair of values for keys u, u + 1.  Every fourth pair goes to the FMA pipes, as in the forward (2 x 1999 tokens, 16 heads of 64, window
// 512, us: none 73.1, every fourth 71.1; 8 x 2000 tokens, 8 heads on 2 of 64, window 300: 118.4, 113.8; T = 8192, 32 heads on 8 of 128, window 2048: none 761, every fourth 755,
// third 759, second 767).  Where long calls run on end power decides, and it makes no difference.
constexpr int POLY = 4;
template <typename ShiftT>
__device__ __forceinline__ void exponentials(float (&e)[64], float c, ShiftT minus_shift) {
    const F2 c2 = pair(c, c);
#pragma unroll
    for (int u = 0; u < 64; u += 2) {
        const F2 y = fma2(pair(e[u], e[u + 1]), c2, minus_shift(u));
        const float2 x = both(y), v = u / 2 % POLY == POLY - 1 ? exp2_poly(y) : make_float2(exp2_fast(x.x), exp2_fast(x.y));
        e[u] = v.x;
        e[u + 1] = v.y;
    }
}
// 64 values of a row as bf16 into the first half of the columns they came from
__device__ __forceinline__ void put_half(uint32_t taddr, const float (&v)[64]) {
#pragma unroll
    for (int i = 0; i < 64; i += 32) {
        uint32_t w[16];
#pragma unroll
        for (int u = 0; u < 16; ++u) w[u] = pack_bf16(v[i + 2 * u], v[i + 2 * u + 1]);
        umma::tmem_st16u(taddr + i / 2, w);
    }
    umma::tmem_wait_st();
    umma::fence_before_sync();
    __syncwarp();
}
// D += A B, A (128 x K) as put_half leaves it, B rows [0, K) of a tile stored [128][K]
template <int K>
__device__ __forceinline__ void gemm_step(uint32_t lead, uint32_t d, uint32_t a, uint32_t b_saddr, uint32_t idesc, bool accumulate) {
    umma::gemm_tm_lead<TILE, 64>(lead, d, a, b_saddr, idesc, accumulate);
    if constexpr (K == 128) umma::gemm_tm_lead<TILE, 64>(lead, d, a + 64, b_saddr + 64 * umma::ROW_BYTES, idesc, true);
}
// 32 rows of 64 fp32 columns times f, as bf16, rows [first, last) of them to `out`, `stride` bytes apart; buf: 4 KB of shared memory a warp
__device__ __forceinline__ void put_rows(uint32_t taddr, unsigned char* buf, int lane, bf16* out, long stride, float f, int first, int last) {
    const Rows<8> rows = {reinterpret_cast<uint4*>(buf), lane};
#pragma unroll
    for (int i = 0; i < 64; i += 32) {
        float o[32];
        umma::tmem_ld32(taddr + i, o);
#pragma unroll
        for (int u = 0; u < 32; u += 8)
            rows.put((i + u) / 8, pack_bf16(o[u] * f, o[u + 1] * f), pack_bf16(o[u + 2] * f, o[u + 3] * f), pack_bf16(o[u + 4] * f, o[u + 5] * f), pack_bf16(o[u + 6] * f, o[u + 7] * f));
    }
    rows.store(out, stride, first, last);
}
// the same unrounded; 8 KB
__device__ __forceinline__ void put_parts(uint32_t taddr, unsigned char* buf, int lane, float* out, long stride, int first, int last) {
    const Rows<16> rows = {reinterpret_cast<uint4*>(buf), lane};
#pragma unroll
    for (int i = 0; i < 64; i += 32) {
        float o[32];
        umma::tmem_ld32(taddr + i, o);
#pragma unroll
        for (int u = 0; u < 32; u += 4)
            rows.put((i + u) / 4, __float_as_uint(o[u]), __float_as_uint(o[u + 1]), __float_as_uint(o[u + 2]), __float_as_uint(o[u + 3]));
    }
    rows.store(out, stride, first, last);
}
__device__ __forceinline__ void load_stat(float* dst, const float* src, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n"
                 ::"r"(umma::smem_addr(dst)), "l"(src), "r"(TILE * 4), "r"(umma::smem_addr(bar)) : "memory");
}
}  // namespace bwd

template <int K, bool TWICE>
__global__ void __launch_bounds__(bwd::Cta<K>::THREADS, bwd::Cta<K>::PER_SM) window_dq_tc_kernel(const __grid_constant__ Params p) {
    chain_wait();
    clear_status(p);
    using namespace bwd;
    constexpr int twice = TWICE;
    using SM = Cta<K>;
    constexpr int STEPS = SM::STEPS, WARPS = SM::WARPS, MMA_WARP = SM::MMA_WARP, TMA_WARP = SM::TMA_WARP;
    constexpr int NA = SM::NA, NB = SM::NB, TM_S = 0, TM_DP = 2 * K, TM_DQ = 3 * K;         // S twice
    extern __shared__ __align__(1024) unsigned char smem[];
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + SM::bar_off);
    const Ring<NA> ringK = {bars, bars + NA};
    const Ring<NB> ringV = {bars + 2 * NA, bars + 2 * NA + NB};
    uint64_t *barQ = bars + 2 * (NA + NB), *barS = barQ + 1, *barDP = barS + 2, *barE = barDP + 1, *barDone = barE + 1;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(barDone + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    static_assert((2 * (NA + NB) + 6) * 8 + 8 <= 256, "barriers");
    float* sDelta = reinterpret_cast<float*>(smem + SM::stat_off);           // [128]

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    // heads first, later queries first: those see more tiles, and the last CTAs of a launch are its short ones.  (Sequences before tiles too, as in the other kernels: 92.3 us for
    // 89.0, both kernels, 4 x 1000 tokens.)
    const int h = blockIdx.x % p.H, q0 = (gridDim.x / p.H - 1 - blockIdx.x / p.H) * TILE, b = blockIdx.y, grp = h / (p.H / p.G);
    const Span span(q0, p.T, p.window, p.sinks);
    const int steps = span.count() << twice;
    const auto tile = [&](int n) { return span.tile(n >> twice); };
    if (tid == TMA_WARP * 32) {              // (the thread that brings the tiles need not wait for the others)
        ringK.init();
        ringV.init();
        umma::mbar_init(barQ, 1);
        umma::mbar_init(barS, 1);
        umma::mbar_init(barS + 1, 1);
        umma::mbar_init(barDP, 1);
        umma::mbar_init(barE, WARPS);
        umma::mbar_init(barDone, 1);
        umma::fence_mbar_init();
        *abort_flag = 0;
        tma::expect_tx(barQ, 2 * SM::TILE_BYTES);
        load_tile<K>(smem + SM::stay_off, &p.tq, h, q0, b, barQ);
        load_tile<K>(smem + SM::stay_off + SM::TILE_BYTES, &p.tdo, h, q0, b, barQ);
    }
    if (warp == MMA_WARP) umma::tmem_alloc(tmem_slot, SM::TM);
    umma::fence_before_sync();
    __syncthreads();
    umma::fence_after_sync();
    const uint32_t tmem = *tmem_slot;
    int nk = 0, nv = 0;                      // tiles brought (by the thread that does)

    if (warp >= WARPS) {
        SM::regs_issue();
        if (warp == TMA_WARP && lane == 0) {
            while (nv < steps) {
                if (!ringK.wait_free(nk, abort_flag)) break;
                tma::expect_tx(ringK.filled(nk), SM::TILE_BYTES);
                load_tile<K>(smem + SM::a_off + nk % NA * SM::TILE_BYTES, &p.tk, grp, tile(nk) * TILE, b, ringK.filled(nk));
                ++nk;
                if (!ringV.wait_free(nv, abort_flag)) break;
                tma::expect_tx(ringV.filled(nv), SM::TILE_BYTES);
                load_tile<K>(smem + SM::b_off + nv % NB * SM::TILE_BYTES, &p.tv, grp, tile(nv) * TILE, b, ringV.filled(nv));
                ++nv;
            }
        } else if (warp == MMA_WARP) {
            const uint32_t lead = umma::elect_one(), sQ = umma::smem_addr(smem + SM::stay_off), sDO = sQ + SM::TILE_BYTES;
            const uint32_t sK = umma::smem_addr(smem + SM::a_off), sV = umma::smem_addr(smem + SM::b_off);
            constexpr uint32_t idS = umma::idesc_bf16(128, K, false, false), idQ = umma::idesc_bf16(128, K, false, true);
            bool ok = umma::mbar_wait_warp(barQ, 0, abort_flag);
            // step m: part m % STEPS of tile m / STEPS
            const auto scores = [&](int m) {
                const int n = m / STEPS, u = m % STEPS;
                ok = ok && (u > 0 || umma::mbar_wait_warp(ringK.filled(n), ringK.phase(n), abort_flag));
                if (!ok) return;
                umma::gemm_kk_lead<TILE, TILE, K>(lead, tmem + TM_S + K * (m & 1), sQ, sK + n % NA * SM::TILE_BYTES + u * K * umma::ROW_BYTES, idS, false);
                umma::commit_lead(lead, barS + (m & 1));
            };
            const auto products = [&](int m) {
                const int n = m / STEPS, u = m % STEPS;
                ok = ok && (u > 0 || umma::mbar_wait_warp(ringV.filled(n), ringV.phase(n), abort_flag));
                if (!ok) return;
                umma::gemm_kk_lead<TILE, TILE, K>(lead, tmem + TM_DP, sDO, sV + n % NB * SM::TILE_BYTES + u * K * umma::ROW_BYTES, idS, false);
                umma::commit_lead(lead, barDP);
                if (u == STEPS - 1) umma::commit_lead(lead, ringV.freed(n));
            };
            scores(0);
            products(0);
            for (int m = 0; m < steps * STEPS && ok; ++m) {
                const int n = m / STEPS, u = m % STEPS;
                if (m + 1 < steps * STEPS) scores(m + 1);
                ok = ok && umma::mbar_wait_warp(barE, m & 1, abort_flag);
                umma::fence_after_sync();
                if (m + 1 < steps * STEPS) products(m + 1);
                if (!ok) break;
                gemm_step<K>(lead, tmem + TM_DQ, tmem + TM_S + K * (m & 1), sK + n % NA * SM::TILE_BYTES + u * K * umma::ROW_BYTES, idQ, m > 0);
                if (u == STEPS - 1) umma::commit_lead(lead, ringK.freed(n));
            }
            if (ok) umma::commit_lead(lead, barDone);
        }
    } else {
        SM::regs_rows();
        const int half = warp >> 2, row = (warp & 3) * 32 + lane, t = q0 + row;
        const long stat = ((long)b * p.H + h) * p.TP + t;
        const uint32_t tS = umma::tmem_addr(tmem, warp, TM_S + 64 * half), tDP = umma::tmem_addr(tmem, warp, TM_DP + 64 * half);
        const float c = p.scale * LOG2E, lse = p.lse[stat];
        // delta of the tile's rows, each warp its share of them, K / 8 lanes a row (a thread a row: 10 k cycles, for loads that touch a line a lane)
        constexpr int LANES = K / 8, ROWS = 32 / LANES, EACH = TILE / WARPS;
        uint4 xo[EACH / ROWS], xd[EACH / ROWS];
#pragma unroll
        for (int i = 0; i < EACH / ROWS; ++i) {
            const int r = q0 + warp * EACH + i * ROWS + lane / LANES;
            const long from = (((long)b * p.T + r) * p.H + h) * K + lane % LANES * 8;
            xo[i] = r < p.T ? *reinterpret_cast<const uint4*>(p.o + from) : make_uint4(0, 0, 0, 0);
            xd[i] = r < p.T ? *reinterpret_cast<const uint4*>(p.d_o + from) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < EACH / ROWS; ++i) {
            const uint32_t xs[4] = {xo[i].x, xo[i].y, xo[i].z, xo[i].w}, ys[4] = {xd[i].x, xd[i].y, xd[i].z, xd[i].w};
            float d = 0.f;
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                d = fmaf(__uint_as_float(xs[u] << 16), __uint_as_float(ys[u] << 16), d);
                d = fmaf(__uint_as_float(xs[u] & 0xffff0000u), __uint_as_float(ys[u] & 0xffff0000u), d);
            }
#pragma unroll
            for (int u = LANES / 2; u > 0; u >>= 1) d += __shfl_xor_sync(0xffffffffu, d, u);
            if (lane % LANES == 0) sDelta[warp * EACH + i * ROWS + lane / LANES] = d;
        }
        if (q0 < p.low_rows) {                             // with what the rounding of o took off
#pragma unroll
            for (int i = 0; i < EACH / ROWS; ++i) {
                const int r = q0 + warp * EACH + i * ROWS + lane / LANES;
                const uint4 xl = r < p.low_rows ? *reinterpret_cast<const uint4*>(p.low + (((long)b * p.low_rows + r) * p.H + h) * K + lane % LANES * 8) : make_uint4(0, 0, 0, 0);
                const uint32_t xs[4] = {xl.x, xl.y, xl.z, xl.w}, ys[4] = {xd[i].x, xd[i].y, xd[i].z, xd[i].w};
                float d = 0.f;
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    d = fmaf(__uint_as_float(xs[u] << 16), __uint_as_float(ys[u] << 16), d);
                    d = fmaf(__uint_as_float(xs[u] & 0xffff0000u), __uint_as_float(ys[u] & 0xffff0000u), d);
                }
#pragma unroll
                for (int u = LANES / 2; u > 0; u >>= 1) d += __shfl_xor_sync(0xffffffffu, d, u);
                if (lane % LANES == 0) sDelta[warp * EACH + i * ROWS + lane / LANES] += d;
            }
        }
        asm volatile("bar.sync 1, %0;\n" ::"n"(32 * WARPS) : "memory");
        const float delta = sDelta[row];
        if (half == 0) p.delta[stat] = delta;
        bool ok = true;
        for (int m = 0; m < steps * STEPS; ++m) {
            const int s0 = tile(m / STEPS) * TILE, from = s0 + m % STEPS * K + half * 64;
            ok = umma::mbar_wait_warp(barS + (m & 1), (m >> 1) & 1, abort_flag);
            if (!ok) break;
            umma::fence_after_sync();
            float e[64], d[64];
            tmem_ld64(tS + K * (m & 1), e);
            exponentials(e, c, [&](int) { return pair(-lse, -lse); });
            if (!all_seen(q0, s0, p.window, p.sinks)) {
#pragma unroll
                for (int i = 0; i < 64; i += 32) {
                    const uint32_t bits = seen_bits(t, from + i, p.window, p.sinks);
#pragma unroll
                    for (int u = 0; u < 32; ++u)
                        if (!(bits & (1u << u))) e[i + u] = 0.f;
                }
            }
            ok = umma::mbar_wait_warp(barDP, m & 1, abort_flag);
            if (!ok) break;
            umma::fence_after_sync();
            tmem_ld64(tDP, d);
#pragma unroll
            for (int i = 0; i < 64; i += 2) {
                const float2 v = both(mul(pair(e[i], e[i + 1]), add(pair(d[i], d[i + 1]), pair(-delta, -delta))));
                e[i] = v.x;
                e[i + 1] = v.y;
            }
            if (m / STEPS & twice) leave_rest(e);
            put_half(tS + K * (m & 1), e);
            if (lane == 0) arrive(barE);
        }
        if (ok) ok = umma::mbar_wait_warp(barDone, 0, abort_flag);
        if (ok) {
            umma::fence_after_sync();
            // (all products are done: the place of Q and dO is free)
            const int first = q0 + (warp & 3) * 32;
            put_rows(umma::tmem_addr(tmem, warp, TM_DQ + half * 64), smem + SM::stay_off + warp * 8192, lane, p.dq + (((long)b * p.T + first) * p.H + h) * K + half * 64,
                     (long)p.H * K * 2, p.scale, 0, min(p.T - first, 32));
        }
        umma::fence_before_sync();
    }
    __syncthreads();
    umma::fence_after_sync();
    // after a wait that gave up (none can from here on): copies and products that nobody waited for end before the CTA does
    if (*abort_flag) {
        if (tid == TMA_WARP * 32) {
            ringK.drain(nk);
            ringV.drain(nv);
        }
        if (warp == MMA_WARP) end_products(barQ, p.err, lane);
    }
    if (warp == MMA_WARP) umma::tmem_dealloc(tmem, SM::TM);
}

template <int K, bool TWICE>
__global__ void __launch_bounds__(bwd::Cta<K>::THREADS, bwd::Cta<K>::PER_SM) window_dkv_tc_kernel(const __grid_constant__ Params p, const __grid_constant__ Shares sh) {
    chain_wait();
    using namespace bwd;
    constexpr int twice = TWICE;
    using SM = Cta<K>;
    constexpr int STEPS = SM::STEPS, WARPS = SM::WARPS, MMA_WARP = SM::MMA_WARP, TMA_WARP = SM::TMA_WARP;
    constexpr int NA = SM::NA, NB = SM::NB, TM_S = 0, TM_DP = K, TM_DV = 2 * K, TM_DK = 3 * K;
    extern __shared__ __align__(1024) unsigned char smem[];
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + SM::bar_off);
    const Ring<NA> ringQ = {bars, bars + NA};
    const Ring<NB> ringDO = {bars + 2 * NA, bars + 2 * NA + NB};
    uint64_t *barKV = bars + 2 * (NA + NB), *barS = barKV + 1, *barDP = barS + 1, *barP = barDP + 1, *barDS = barP + 1, *barDone = barDS + 1;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(barDone + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    float* sStat = reinterpret_cast<float*>(smem + SM::stat_off);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    // groups and sequences first; tiles of sinks first, the last tiles, which few queries see, last  (sequences, then groups, outermost: 414 us for 394, both kernels, T = 4096, 32 heads
    // on 8, window 2048)
    const int units = p.B * p.G, x0 = blockIdx.x / units, grp = blockIdx.x % units % p.G, b = blockIdx.x % units / p.G, R = p.H / p.G, last = sh.tiles - 1;
    // far shares first, then the near ones; tile j of k and v, tiles [lo, hi] of queries, heads h0 on
    const bool far = x0 < sh.far_tiles * sh.chunks;
    const int x = far ? x0 : x0 - sh.far_tiles * sh.chunks, j = far ? x / sh.chunks : x / sh.splits, share = far ? x % sh.chunks : x % sh.splits;
    const int lo = far ? j + sh.near + share * sh.chunk : j, end = far ? lo + sh.chunk - 1 : j + sh.near - 1, hi = end < last ? end : last;
    const int each = far ? R : (R + sh.splits - 1) / sh.splits, h0 = grp * R + (far ? 0 : share * each), heads = min(each, grp * R + R - h0);
    if (lo > last || heads <= 0) return;                    // (a share that the last tiles do not reach; fewer heads than shares)
    const int s0 = j * TILE, per = hi - lo + 1, steps = heads * per << twice;
    if (tid == TMA_WARP * 32) {              // (the thread that brings the tiles need not wait for the others)
        ringQ.init();
        ringDO.init();
        umma::mbar_init(barKV, 1);
        umma::mbar_init(barS, 1);
        umma::mbar_init(barDP, 1);
        umma::mbar_init(barP, WARPS);
        umma::mbar_init(barDS, WARPS);
        umma::mbar_init(barDone, 1);
        umma::fence_mbar_init();
        *abort_flag = 0;
        tma::expect_tx(barKV, 2 * SM::TILE_BYTES);
        load_tile<K>(smem + SM::stay_off, &p.tk, grp, s0, b, barKV);
        load_tile<K>(smem + SM::stay_off + SM::TILE_BYTES, &p.tv, grp, s0, b, barKV);
    }
    if (warp == MMA_WARP) umma::tmem_alloc(tmem_slot, SM::TM);
    umma::fence_before_sync();
    __syncthreads();
    umma::fence_after_sync();
    const uint32_t tmem = *tmem_slot;
    int nq = 0, nd = 0;                      // tiles brought (by the thread that does)

    if (warp >= WARPS) {
        SM::regs_issue();
        if (warp == TMA_WARP && lane == 0) {
            int h = h0, i = lo;
            while (nd < steps) {
                const long stat = ((long)b * p.H + h) * p.TP + i * TILE;
                if (!ringQ.wait_free(nq, abort_flag)) break;
                tma::expect_tx(ringQ.filled(nq), SM::TILE_BYTES + TILE * 4);
                load_tile<K>(smem + SM::a_off + nq % NA * SM::TILE_BYTES, &p.tq, h, i * TILE, b, ringQ.filled(nq));
                load_stat(sStat + nq % NA * TILE, p.lse + stat, ringQ.filled(nq));
                ++nq;
                if (!ringDO.wait_free(nd, abort_flag)) break;
                tma::expect_tx(ringDO.filled(nd), SM::TILE_BYTES + TILE * 4);
                load_tile<K>(smem + SM::b_off + nd % NB * SM::TILE_BYTES, &p.tdo, h, i * TILE, b, ringDO.filled(nd));
                load_stat(sStat + (NA + nd % NB) * TILE, p.delta + stat, ringDO.filled(nd));
                ++nd;
                if ((nd & twice) == 0 && ++i > hi) {
                    i = lo;
                    ++h;
                }
            }
        } else if (warp == MMA_WARP) {
            const uint32_t lead = umma::elect_one(), sK = umma::smem_addr(smem + SM::stay_off), sV = sK + SM::TILE_BYTES;
            const uint32_t sQ = umma::smem_addr(smem + SM::a_off), sDO = umma::smem_addr(smem + SM::b_off);
            constexpr uint32_t idS = umma::idesc_bf16(128, K, false, false), idG = umma::idesc_bf16(128, K, false, true);
            bool ok = umma::mbar_wait_warp(barKV, 0, abort_flag);
            const auto scores = [&](int m) {
                const int n = m / STEPS, u = m % STEPS;
                ok = ok && (u > 0 || umma::mbar_wait_warp(ringQ.filled(n), ringQ.phase(n), abort_flag));
                if (!ok) return;
                umma::gemm_kk_lead<TILE, TILE, K>(lead, tmem + TM_S, sK, sQ + n % NA * SM::TILE_BYTES + u * K * umma::ROW_BYTES, idS, false);
                umma::commit_lead(lead, barS);
            };
            const auto products = [&](int m) {
                const int n = m / STEPS, u = m % STEPS;
                ok = ok && (u > 0 || umma::mbar_wait_warp(ringDO.filled(n), ringDO.phase(n), abort_flag));
                if (!ok) return;
                umma::gemm_kk_lead<TILE, TILE, K>(lead, tmem + TM_DP, sV, sDO + n % NB * SM::TILE_BYTES + u * K * umma::ROW_BYTES, idS, false);
                umma::commit_lead(lead, barDP);
            };
            scores(0);
            products(0);
            for (int m = 0; m < steps * STEPS && ok; ++m) {
                const int n = m / STEPS, u = m % STEPS;
                ok = umma::mbar_wait_warp(barP, m & 1, abort_flag);
                if (!ok) break;
                umma::fence_after_sync();
                gemm_step<K>(lead, tmem + TM_DV, tmem + TM_S, sDO + n % NB * SM::TILE_BYTES + u * K * umma::ROW_BYTES, idG, m > 0);
                if (m + 1 < steps * STEPS) scores(m + 1);
                ok = ok && umma::mbar_wait_warp(barDS, m & 1, abort_flag);
                if (!ok) break;
                umma::fence_after_sync();
                gemm_step<K>(lead, tmem + TM_DK, tmem + TM_DP, sQ + n % NA * SM::TILE_BYTES + u * K * umma::ROW_BYTES, idG, m > 0);
                // (delta, beside dO, is read until dS is there)
                if (u == STEPS - 1) {
                    umma::commit_lead(lead, ringDO.freed(n));
                    umma::commit_lead(lead, ringQ.freed(n));
                }
                if (m + 1 < steps * STEPS) products(m + 1);
            }
            if (ok) umma::commit_lead(lead, barDone);
        }
    } else {
        SM::regs_rows();
        const int half = warp >> 2, s = s0 + (warp & 3) * 32 + lane;
        const uint32_t tS = umma::tmem_addr(tmem, warp, TM_S + 64 * half), tDP = umma::tmem_addr(tmem, warp, TM_DP + 64 * half);
        const float c = p.scale * LOG2E;
        bool ok = true;
        int i = lo;
        for (int m = 0; m < steps * STEPS; ++m) {
            const int n = m / STEPS, u0 = m % STEPS * K + half * 64, t0 = i * TILE;
            if (((m + 1) & ((STEPS << twice) - 1)) == 0 && ++i > hi) i = lo;
            const bool rest = n & twice;
            const float *lse = sStat + n % NA * TILE + u0, *delta = sStat + (NA + n % NB) * TILE + u0;
            ok = umma::mbar_wait_warp(ringQ.filled(n), ringQ.phase(n), abort_flag) && umma::mbar_wait_warp(barS, m & 1, abort_flag);
            if (!ok) break;
            umma::fence_after_sync();
            float e[64], d[64];
            tmem_ld64(tS, e);
            exponentials(e, c, [&](int u) {
                const float2 m = *reinterpret_cast<const float2*>(lse + u);
                return pair(-m.x, -m.y);
            });
            if (!all_seen(t0, s0, p.window, p.sinks)) {
                // token s is seen by the queries from s on, as far as the window goes; a sink by all of them
#pragma unroll
                for (int k = 0; k < 64; k += 32) {
                    const uint32_t bits = seeing_bits(t0 + u0 + k, s, p.window, p.sinks);
#pragma unroll
                    for (int u = 0; u < 32; ++u)
                        if (!(bits & (1u << u))) e[k + u] = 0.f;
                }
            }
            if (rest) {                                        // (P stays for dS)
#pragma unroll
                for (int u = 0; u < 64; ++u) d[u] = e[u];
                leave_rest(d);
                put_half(tS, d);
            } else {
                put_half(tS, e);
            }
            if (lane == 0) arrive(barP);
            ok = umma::mbar_wait_warp(ringDO.filled(n), ringDO.phase(n), abort_flag) && umma::mbar_wait_warp(barDP, m & 1, abort_flag);
            if (!ok) break;
            umma::fence_after_sync();
            tmem_ld64(tDP, d);
#pragma unroll
            for (int u = 0; u < 64; u += 2) {
                const float2 m = *reinterpret_cast<const float2*>(delta + u);
                const float2 v = both(mul(pair(e[u], e[u + 1]), add(pair(d[u], d[u + 1]), pair(-m.x, -m.y))));
                e[u] = v.x;
                e[u + 1] = v.y;
            }
            if (rest) leave_rest(e);
            put_half(tDP, e);
            if (lane == 0) arrive(barDS);
        }
        if (ok) ok = umma::mbar_wait_warp(barDone, 0, abort_flag);
        if (ok) {
            umma::fence_after_sync();
            const int row0 = (warp & 3) * 32, first = s0 + row0, last = min(p.T - first, 32);
            const long at = (((long)b * p.T + first) * p.G + grp) * K + half * 64, unit = (long)b * p.G + grp;
            const uint32_t tDV = umma::tmem_addr(tmem, warp, TM_DV + half * 64), tDK = umma::tmem_addr(tmem, warp, TM_DK + half * 64);
            unsigned char* buf = smem + SM::stay_off + warp * 8192;              // (all products are done: the place of K and V is free)
            const int sink = j < sh.far_tiles ? max(min(p.sinks - first, 32), 0) : 0;        // tokens with parts from far
            if (far || sh.splits > 1 || j < sh.far_tiles) {
                float* part = far ? p.far_part + (((unit * sh.far_tiles + j) * sh.chunks + share) * sh.far_rows(p.sinks) + row0) * 2 * K
                                  : p.near_part + (((unit * sh.splits + share) * sh.near_tiles() + j) * TILE + row0) * 2 * K;
                const int parts = !far && sh.splits > 1 ? last : min(sink, last);
                put_parts(tDK, buf, lane, part + half * 64, 2 * K * sizeof(float), 0, parts);
                put_parts(tDV, buf, lane, part + K + half * 64, 2 * K * sizeof(float), 0, parts);
            }
            if (!far && sh.splits == 1) {
                put_rows(tDV, buf, lane, p.dv + at, (long)p.G * K * 2, 1.f, sink, last);
                put_rows(tDK, buf, lane, p.dk + at, (long)p.G * K * 2, p.scale, sink, last);
            }
        }
        umma::fence_before_sync();
    }
    __syncthreads();
    umma::fence_after_sync();
    if (*abort_flag) {
        if (tid == TMA_WARP * 32) {
            ringQ.drain(nq);
            ringDO.drain(nd);
        }
        if (warp == MMA_WARP) end_products(barKV, p.err, lane);
    }
    if (warp == MMA_WARP) umma::tmem_dealloc(tmem, SM::TM);
}

// Adds up the parts: a warp a token and group.  The tokens with parts are all of them, or the sinks among the first tiles.
template <int K>
__global__ void __launch_bounds__(256) window_join_kernel(const __grid_constant__ Params p, const __grid_constant__ Shares sh, int tokens) {
    chain_wait();
    const int lane = threadIdx.x & 31, R = p.H / p.G;
    const long row = (long)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (row >= (long)p.B * p.G * tokens) return;
    const int s = (int)(row % tokens), j = s / TILE;
    const long unit = row / tokens, b = unit / p.G, grp = unit % p.G;
    constexpr int N = K / 64;                             // pairs of columns a lane, of dk and of dv
    float2 sum[2 * N];
#pragma unroll
    for (int i = 0; i < 2 * N; ++i) sum[i] = make_float2(0.f, 0.f);
    const auto add = [&](const float* part) {
#pragma unroll
        for (int i = 0; i < 2 * N; ++i) {
            const float2 v = reinterpret_cast<const float2*>(part)[lane + 32 * i];
            sum[i].x += v.x;
            sum[i].y += v.y;
        }
    };
    // (four parts' loads in flight)
    const int each = (R + sh.splits - 1) / sh.splits, shares = (R + each - 1) / each;
#pragma unroll 4
    for (int x = 0; x < shares; ++x) add(p.near_part + (((unit * sh.splits + x) * sh.near_tiles() + j) * TILE + s % TILE) * 2 * K);
    if (j < sh.far_tiles && s < p.sinks) {
        const int chunks = (sh.tiles - j - sh.near + sh.chunk - 1) / sh.chunk;
#pragma unroll 4
        for (int x = 0; x < chunks; ++x) add(p.far_part + (((unit * sh.far_tiles + j) * sh.chunks + x) * sh.far_rows(p.sinks) + s % TILE) * 2 * K);
    }
    const long at = ((b * p.T + s) * p.G + grp) * K;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        reinterpret_cast<uint32_t*>(p.dk + at)[lane + 32 * i] = pack_bf16(sum[i].x * p.scale, sum[i].y * p.scale);
        reinterpret_cast<uint32_t*>(p.dv + at)[lane + 32 * i] = pack_bf16(sum[N + i].x, sum[N + i].y);
    }
}

template <int K, bool TWICE>
static cudaError_t launch(const Params& p, cudaStream_t st) {
    const size_t smem = bwd::Cta<K>::total;
    constexpr int THREADS = bwd::Cta<K>::THREADS;
    const Shares sh(p.B, p.T, p.H, p.G, K, p.window, p.sinks);
    const auto dq = window_dq_tc_kernel<K, TWICE>;
    const auto dkv = window_dkv_tc_kernel<K, TWICE>;
    cudaError_t e = allow_smem(dq, smem);
    if (e == cudaSuccess) e = allow_smem(dkv, smem);
    if (e != cudaSuccess) return e;
    e = launch_chained(dq, dim3((unsigned)sh.tiles * p.H, p.B), THREADS, smem, st, p);
    if (e != cudaSuccess) return e;
    LLATTN_LAUNCHED();
    e = launch_chained(dkv, (unsigned)(sh.far_tiles * sh.chunks + sh.tiles * sh.splits) * p.G * p.B, THREADS, smem, st, p, sh);
    if (e != cudaSuccess) return e;
    LLATTN_LAUNCHED();
    const int some = sh.far_tiles * TILE < p.sinks ? sh.far_tiles * TILE : p.sinks, tokens = sh.splits > 1 ? p.T : some;
    if (tokens == 0 || (sh.splits == 1 && sh.far_tiles == 0)) return e;
    e = launch_chained(window_join_kernel<K>, (unsigned)(((long)p.B * p.G * tokens + 7) / 8), 256, 0, st, p, sh, tokens);
    if (e == cudaSuccess) LLATTN_LAUNCHED();
    return e;
}
cudaError_t backward_tc(const Params& p, int K, cudaStream_t st) {
    if (few_tokens(p.T)) return K == 64 ? launch<64, true>(p, st) : launch<128, true>(p, st);
    return K == 64 ? launch<64, false>(p, st) : launch<128, false>(p, st);
}

}  // namespace win
}  // namespace llattn
