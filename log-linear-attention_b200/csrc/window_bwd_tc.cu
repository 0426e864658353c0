// Sliding-window attention backward on the 5th-generation tensor cores: two kernels that make S and dP again from q, k, v, do and the statistics of the
// forward, so that every gradient is a sum in one CTA's tensor memory, in an order that the sizes alone decide.
//
// dQ: a CTA takes a tile of 128 queries of a head and walks the tiles of keys that they see,
//     S = Q K^T, dP = dO V^T,   dS = exp2(c S - lse) (dP - delta) as bf16 in the place of S,   dQ += dS K.
// dK, dV: a CTA takes a tile of 128 tokens of k and v and walks the tiles of queries that see it, of all heads that share it,
//     S^T = K Q^T, dP^T = V dO^T,   P^T = exp2(c S^T - lse), dV += P^T dO,   dS^T = P^T (dP^T - delta), dK += dS^T Q.
// In both, eight warps do the exponentials (two threads a row, 64 columns each), one issues products, one brings tiles through a ring; the products of one
// half of a step run under the other half's exponentials.  (Summing dQ beside dK and dV would save two of the seven products a pair of tiles, for
// atomics on 64 KB of fp32 a pair.)
#include "window.cuh"

namespace llattn {
namespace win {

namespace bwd {
constexpr int NTHREADS = 384, MMA_WARP = 8, TMA_WARP = 9;
template <int K>
struct Smem {
    static constexpr int NST = K == 64 ? 8 : 4;
    static constexpr uint32_t TILE_BYTES = TILE * K * 2;
    static constexpr uint32_t a_off = 0, st_off = 2 * TILE_BYTES;                    // the two tiles that stay, the ring
    static constexpr uint32_t stat_off = st_off + NST * TILE_BYTES;                  // float [NST / 2][2][128]: lse, delta of a step's queries
    static constexpr uint32_t bar_off = stat_off + NST / 2 * 1024, total = bar_off + 256 + 1024;
};
// 128 x (168 - 72) registers go to the 256 threads of the exponentials
__device__ __forceinline__ void regs_issue() { asm volatile("setmaxnreg.dec.sync.aligned.u32 72;\n"); }
__device__ __forceinline__ void regs_rows() { asm volatile("setmaxnreg.inc.sync.aligned.u32 216;\n"); }

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
// D += A B, A (128 x 128) as put_half leaves it, B a tile stored [128][K]
template <int K>
__device__ __forceinline__ void gemm_halves(uint32_t lead, uint32_t d, uint32_t a, uint32_t b_saddr, uint32_t idesc, bool accumulate) {
    umma::gemm_tm_lead<TILE, 64>(lead, d, a, b_saddr, idesc, accumulate);
    umma::gemm_tm_lead<TILE, 64>(lead, d, a + 64, b_saddr + 64 * umma::ROW_BYTES, idesc, true);
}
// row of K / 2 fp32 columns times f, as bf16
template <int K>
__device__ __forceinline__ void put_row(uint32_t taddr, bf16* out, float f, bool there) {
#pragma unroll
    for (int i = 0; i < K / 2; i += 16) {
        float o[16];
        umma::tmem_ld16(taddr + i, o);
        uint32_t w[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) w[u] = pack_bf16(o[2 * u] * f, o[2 * u + 1] * f);
        if (there) store_32B(out + i, w);
    }
}
// the same unrounded
template <int K>
__device__ __forceinline__ void put_part(uint32_t taddr, float* out, bool there) {
#pragma unroll
    for (int i = 0; i < K / 2; i += 16) {
        float o[16];
        umma::tmem_ld16(taddr + i, o);
        if (there)
#pragma unroll
            for (int u = 0; u < 16; u += 4) *reinterpret_cast<float4*>(out + i + u) = make_float4(o[u], o[u + 1], o[u + 2], o[u + 3]);
    }
}
__device__ __forceinline__ void load_stat(float* dst, const float* src, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n"
                 ::"r"(umma::smem_addr(dst)), "l"(src), "r"(TILE * 4), "r"(umma::smem_addr(bar)) : "memory");
}
}  // namespace bwd

template <int K>
__global__ void __launch_bounds__(bwd::NTHREADS, 1) window_dq_tc_kernel(const __grid_constant__ Params p) {
    chain_wait();
    using namespace bwd;
    using SM = Smem<K>;
    constexpr int NST = SM::NST, TM_S = 0, TM_DP = 256, TM_DQ = 384;         // S twice
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = umma::align_1024(smem_raw);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + SM::bar_off);
    uint64_t *full = bars, *empty = bars + NST, *barQ = bars + 2 * NST, *barS = barQ + 1, *barDP = barS + 2, *barE = barDP + 1, *barDone = barE + 1;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(barDone + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    static_assert((2 * NST + 6) * 8 + 8 <= 256, "barriers");
    float* sDelta = reinterpret_cast<float*>(smem + SM::stat_off);           // [2][128]: the halves of the rows' sums

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int q0 = blockIdx.x * TILE, h = blockIdx.y, b = blockIdx.z, grp = h / (p.H / p.G);
    const Span span(q0, p.T, p.window, p.sinks);
    const int steps = span.count();
    const auto tile = [&](int n) { return span.tile(n); };
    if (tid == 0) {
        for (int i = 0; i < NST; ++i) {
            umma::mbar_init(full + i, 1);
            umma::mbar_init(empty + i, 1);
        }
        umma::mbar_init(barQ, 1);
        umma::mbar_init(barS, 1);
        umma::mbar_init(barS + 1, 1);
        umma::mbar_init(barDP, 1);
        umma::mbar_init(barE, 8);
        umma::mbar_init(barDone, 1);
        umma::fence_mbar_init();
        *abort_flag = 0;
    }
    if (warp == MMA_WARP) umma::tmem_alloc(tmem_slot, 512);
    umma::fence_before_sync();
    __syncthreads();
    umma::fence_after_sync();
    const uint32_t tmem = *tmem_slot;

    if (warp >= 8) {
        regs_issue();
        if (warp == TMA_WARP && lane == 0) {
            tma::expect_tx(barQ, 2 * SM::TILE_BYTES);
            load_tile<K>(smem + SM::a_off, &p.tq, h, q0, b, barQ);
            load_tile<K>(smem + SM::a_off + SM::TILE_BYTES, &p.tdo, h, q0, b, barQ);
            bool ok = true;
            int n = 0;
            for (; n < 2 * steps; ++n) {
                const int st = n % NST;
                if (n >= NST) ok = umma::mbar_wait(empty + st, (n / NST - 1) & 1, abort_flag);
                if (!ok) break;
                tma::expect_tx(full + st, SM::TILE_BYTES);
                load_tile<K>(smem + SM::st_off + st * SM::TILE_BYTES, n & 1 ? &p.tv : &p.tk, grp, tile(n >> 1) * TILE, b, full + st);
            }
            // after a wait that gave up: the copies in flight end before the CTA does
            if (*abort_flag) {
                umma::mbar_wait(barQ, 0);
                for (int i = n > NST ? n - NST : 0; i < n; ++i) umma::mbar_wait(full + i % NST, (i / NST) & 1);
            }
        } else if (warp == MMA_WARP) {
            const uint32_t lead = umma::elect_one(), sQ = umma::smem_addr(smem + SM::a_off), sDO = sQ + SM::TILE_BYTES, sT = umma::smem_addr(smem + SM::st_off);
            constexpr uint32_t idS = umma::idesc_bf16(128, 128, false, false), idQ = umma::idesc_bf16(128, K, false, true);
            bool ok = umma::mbar_wait_warp(barQ, 0, abort_flag);
            const auto wait_tile = [&](int n) {                  // position n of the ring's sequence; its address
                ok = ok && umma::mbar_wait_warp(full + n % NST, (n / NST) & 1, abort_flag);
                return sT + (n % NST) * SM::TILE_BYTES;
            };
            const auto scores = [&](int n) {
                const uint32_t at = wait_tile(2 * n);
                if (!ok) return;
                umma::gemm_kk_lead<TILE, TILE, K>(lead, tmem + TM_S + 128 * (n & 1), sQ, at, idS, false);
                umma::commit_lead(lead, barS + (n & 1));
            };
            const auto products = [&](int n) {
                const uint32_t at = wait_tile(2 * n + 1);
                if (!ok) return;
                umma::gemm_kk_lead<TILE, TILE, K>(lead, tmem + TM_DP, sDO, at, idS, false);
                umma::commit_lead(lead, barDP);
                umma::commit_lead(lead, empty + (2 * n + 1) % NST);
            };
            scores(0);
            products(0);
            for (int n = 0; n < steps && ok; ++n) {
                if (n + 1 < steps) scores(n + 1);
                ok = ok && umma::mbar_wait_warp(barE, n & 1, abort_flag);
                umma::fence_after_sync();
                if (n + 1 < steps) products(n + 1);
                if (!ok) break;
                gemm_halves<K>(lead, tmem + TM_DQ, tmem + TM_S + 128 * (n & 1), sT + (2 * n % NST) * SM::TILE_BYTES, idQ, n > 0);
                umma::commit_lead(lead, empty + 2 * n % NST);
            }
            if (ok) umma::commit_lead(lead, barDone);
        }
    } else {
        regs_rows();
        const int half = warp >> 2, row = (warp & 3) * 32 + lane, t = q0 + row;
        const bool there = t < p.T;
        const long at = (((long)b * p.T + t) * p.H + h) * K + half * (K / 2), stat = ((long)b * p.H + h) * p.TP + t;
        const uint32_t tS = umma::tmem_addr(tmem, warp, TM_S + 64 * half), tDP = umma::tmem_addr(tmem, warp, TM_DP + 64 * half);
        const float c = p.scale * LOG2E, lse = p.lse[stat];
        float delta = 0.f;
        if (there) {
#pragma unroll
            for (int i = 0; i < K / 2; i += 8) {
                const uint4 x = *reinterpret_cast<const uint4*>(p.o + at + i), y = *reinterpret_cast<const uint4*>(p.d_o + at + i);
                const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    delta = fmaf(__uint_as_float(xs[u] << 16), __uint_as_float(ys[u] << 16), delta);
                    delta = fmaf(__uint_as_float(xs[u] & 0xffff0000u), __uint_as_float(ys[u] & 0xffff0000u), delta);
                }
            }
        }
        sDelta[half * TILE + row] = delta;
        asm volatile("bar.sync 1, 256;\n" ::: "memory");
        delta = sDelta[row] + sDelta[TILE + row];
        if (half == 0) p.delta[stat] = delta;
        bool ok = true;
        for (int n = 0; n < steps; ++n) {
            const int s0 = tile(n) * TILE;
            ok = umma::mbar_wait_warp(barS + (n & 1), (n >> 1) & 1, abort_flag);
            if (!ok) break;
            umma::fence_after_sync();
            float e[64], d[64];
            tmem_ld64(tS + 128 * (n & 1), e);
#pragma unroll
            for (int i = 0; i < 64; ++i) e[i] = exp2_fast(fmaf(e[i], c, -lse));
            if (!all_seen(q0, s0, p.window, p.sinks)) {
#pragma unroll
                for (int i = 0; i < 64; ++i)
                    if (!sees(t, s0 + half * 64 + i, p.window, p.sinks)) e[i] = 0.f;
            }
            ok = umma::mbar_wait_warp(barDP, n & 1, abort_flag);
            if (!ok) break;
            umma::fence_after_sync();
            tmem_ld64(tDP, d);
#pragma unroll
            for (int i = 0; i < 64; ++i) e[i] *= d[i] - delta;
            put_half(tS + 128 * (n & 1), e);
            if (lane == 0) arrive(barE);
        }
        if (ok) ok = umma::mbar_wait_warp(barDone, 0, abort_flag);
        if (ok) {
            umma::fence_after_sync();
            put_row<K>(umma::tmem_addr(tmem, warp, TM_DQ + half * (K / 2)), p.dq + at, p.scale, there);
        }
        umma::fence_before_sync();
    }
    __syncthreads();
    umma::fence_after_sync();
    if (warp == MMA_WARP) {
        // products that nobody waited for, after a wait that gave up, end before their memory is handed back
        if (*abort_flag) {
            umma::commit_lead(umma::elect_one(), barQ);
            umma::mbar_wait(barQ, 1);
            if (lane == 0) atomicExch(p.err, 1);
        }
        umma::tmem_dealloc(tmem, 512);
    }
}

template <int K>
__global__ void __launch_bounds__(bwd::NTHREADS, 1) window_dkv_tc_kernel(const __grid_constant__ Params p, const __grid_constant__ Shares sh) {
    chain_wait();
    using namespace bwd;
    using SM = Smem<K>;
    constexpr int NST = SM::NST, TM_S = 0, TM_DP = 128, TM_DV = 256, TM_DK = 384;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = umma::align_1024(smem_raw);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + SM::bar_off);
    uint64_t *full = bars, *empty = bars + NST, *barKV = bars + 2 * NST, *barS = barKV + 1, *barDP = barS + 1, *barP = barDP + 1, *barDS = barP + 1, *barDone = barDS + 1;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(barDone + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    float* sStat = reinterpret_cast<float*>(smem + SM::stat_off);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int grp = blockIdx.y, b = blockIdx.z, R = p.H / p.G, last = sh.tiles - 1;
    // far shares first, then the near ones; tile j of k and v, tiles [lo, hi] of queries, heads h0 on
    const bool far = (int)blockIdx.x < sh.far_tiles * sh.chunks;
    const int x = far ? blockIdx.x : blockIdx.x - sh.far_tiles * sh.chunks, j = far ? x / sh.chunks : x / sh.splits, share = far ? x % sh.chunks : x % sh.splits;
    const int lo = far ? j + sh.near + share * sh.chunk : j, end = far ? lo + sh.chunk - 1 : j + sh.near - 1, hi = end < last ? end : last;
    const int each = far ? R : (R + sh.splits - 1) / sh.splits, h0 = grp * R + (far ? 0 : share * each), heads = min(each, grp * R + R - h0);
    if (lo > last || heads <= 0) return;                    // (a share that the last tiles do not reach; fewer heads than shares)
    const int s0 = j * TILE, per = hi - lo + 1, steps = heads * per;
    if (tid == 0) {
        for (int i = 0; i < NST; ++i) {
            umma::mbar_init(full + i, 1);
            umma::mbar_init(empty + i, 1);
        }
        umma::mbar_init(barKV, 1);
        umma::mbar_init(barS, 1);
        umma::mbar_init(barDP, 1);
        umma::mbar_init(barP, 8);
        umma::mbar_init(barDS, 8);
        umma::mbar_init(barDone, 1);
        umma::fence_mbar_init();
        *abort_flag = 0;
    }
    if (warp == MMA_WARP) umma::tmem_alloc(tmem_slot, 512);
    umma::fence_before_sync();
    __syncthreads();
    umma::fence_after_sync();
    const uint32_t tmem = *tmem_slot;

    if (warp >= 8) {
        regs_issue();
        if (warp == TMA_WARP && lane == 0) {
            tma::expect_tx(barKV, 2 * SM::TILE_BYTES);
            load_tile<K>(smem + SM::a_off, &p.tk, grp, s0, b, barKV);
            load_tile<K>(smem + SM::a_off + SM::TILE_BYTES, &p.tv, grp, s0, b, barKV);
            bool ok = true;
            int n = 0, h = h0, i = lo;
            for (; n < 2 * steps; ++n) {
                const int st = n % NST;
                if (n >= NST) ok = umma::mbar_wait(empty + st, (n / NST - 1) & 1, abort_flag);
                if (!ok) break;
                tma::expect_tx(full + st, SM::TILE_BYTES + TILE * 4);
                load_tile<K>(smem + SM::st_off + st * SM::TILE_BYTES, n & 1 ? &p.tdo : &p.tq, h, i * TILE, b, full + st);
                load_stat(sStat + st * TILE, (n & 1 ? p.delta : p.lse) + ((long)b * p.H + h) * p.TP + i * TILE, full + st);
                if ((n & 1) && ++i > hi) {
                    i = lo;
                    ++h;
                }
            }
            if (*abort_flag) {
                umma::mbar_wait(barKV, 0);
                for (int m = n > NST ? n - NST : 0; m < n; ++m) umma::mbar_wait(full + m % NST, (m / NST) & 1);
            }
        } else if (warp == MMA_WARP) {
            const uint32_t lead = umma::elect_one(), sK = umma::smem_addr(smem + SM::a_off), sV = sK + SM::TILE_BYTES, sT = umma::smem_addr(smem + SM::st_off);
            constexpr uint32_t idS = umma::idesc_bf16(128, 128, false, false), idG = umma::idesc_bf16(128, K, false, true);
            bool ok = umma::mbar_wait_warp(barKV, 0, abort_flag);
            const auto wait_tile = [&](int n) {
                ok = ok && umma::mbar_wait_warp(full + n % NST, (n / NST) & 1, abort_flag);
                return sT + (n % NST) * SM::TILE_BYTES;
            };
            const auto scores = [&](int n) {
                const uint32_t at = wait_tile(2 * n);
                if (!ok) return;
                umma::gemm_kk_lead<TILE, TILE, K>(lead, tmem + TM_S, sK, at, idS, false);
                umma::commit_lead(lead, barS);
            };
            const auto products = [&](int n) {
                const uint32_t at = wait_tile(2 * n + 1);
                if (!ok) return;
                umma::gemm_kk_lead<TILE, TILE, K>(lead, tmem + TM_DP, sV, at, idS, false);
                umma::commit_lead(lead, barDP);
            };
            scores(0);
            products(0);
            for (int n = 0; n < steps && ok; ++n) {
                ok = umma::mbar_wait_warp(barP, n & 1, abort_flag);
                if (!ok) break;
                umma::fence_after_sync();
                gemm_halves<K>(lead, tmem + TM_DV, tmem + TM_S, sT + (2 * n + 1) % NST * SM::TILE_BYTES, idG, n > 0);
                if (n + 1 < steps) scores(n + 1);
                ok = ok && umma::mbar_wait_warp(barDS, n & 1, abort_flag);
                if (!ok) break;
                umma::fence_after_sync();
                gemm_halves<K>(lead, tmem + TM_DK, tmem + TM_DP, sT + 2 * n % NST * SM::TILE_BYTES, idG, n > 0);
                // (delta, beside dO, is read until dS is there)
                umma::commit_lead(lead, empty + (2 * n + 1) % NST);
                umma::commit_lead(lead, empty + 2 * n % NST);
                if (n + 1 < steps) products(n + 1);
            }
            if (ok) umma::commit_lead(lead, barDone);
        }
    } else {
        regs_rows();
        const int half = warp >> 2, s = s0 + (warp & 3) * 32 + lane;
        const uint32_t tS = umma::tmem_addr(tmem, warp, TM_S + 64 * half), tDP = umma::tmem_addr(tmem, warp, TM_DP + 64 * half);
        const float c = p.scale * LOG2E;
        bool ok = true;
        int i = lo;
        for (int n = 0; n < steps; ++n) {
            const int t0 = i * TILE;
            if (++i > hi) i = lo;
            const float *lse = sStat + 2 * n % NST * TILE + half * 64, *delta = sStat + (2 * n + 1) % NST * TILE + half * 64;
            ok = umma::mbar_wait_warp(full + 2 * n % NST, (2 * n / NST) & 1, abort_flag) && umma::mbar_wait_warp(barS, n & 1, abort_flag);
            if (!ok) break;
            umma::fence_after_sync();
            float e[64], d[64];
            tmem_ld64(tS, e);
#pragma unroll
            for (int u = 0; u < 64; u += 4) {
                const float4 m = *reinterpret_cast<const float4*>(lse + u);
                e[u] = exp2_fast(fmaf(e[u], c, -m.x));
                e[u + 1] = exp2_fast(fmaf(e[u + 1], c, -m.y));
                e[u + 2] = exp2_fast(fmaf(e[u + 2], c, -m.z));
                e[u + 3] = exp2_fast(fmaf(e[u + 3], c, -m.w));
            }
            if (!all_seen(t0, s0, p.window, p.sinks)) {
#pragma unroll
                for (int u = 0; u < 64; ++u)
                    if (!sees(t0 + half * 64 + u, s, p.window, p.sinks)) e[u] = 0.f;
            }
            put_half(tS, e);
            if (lane == 0) arrive(barP);
            ok = umma::mbar_wait_warp(full + (2 * n + 1) % NST, ((2 * n + 1) / NST) & 1, abort_flag) && umma::mbar_wait_warp(barDP, n & 1, abort_flag);
            if (!ok) break;
            umma::fence_after_sync();
            tmem_ld64(tDP, d);
#pragma unroll
            for (int u = 0; u < 64; u += 4) {
                const float4 m = *reinterpret_cast<const float4*>(delta + u);
                e[u] *= d[u] - m.x;
                e[u + 1] *= d[u + 1] - m.y;
                e[u + 2] *= d[u + 2] - m.z;
                e[u + 3] *= d[u + 3] - m.w;
            }
            put_half(tDP, e);
            if (lane == 0) arrive(barDS);
        }
        if (ok) ok = umma::mbar_wait_warp(barDone, 0, abort_flag);
        if (ok) {
            umma::fence_after_sync();
            const long at = (((long)b * p.T + s) * p.G + grp) * K + half * (K / 2), unit = (long)b * p.G + grp;
            const uint32_t tDV = umma::tmem_addr(tmem, warp, TM_DV + half * (K / 2)), tDK = umma::tmem_addr(tmem, warp, TM_DK + half * (K / 2));
            const bool sink = j < sh.far_tiles && s < p.sinks;                     // a token with parts from far
            if (far || sh.splits > 1 || j < sh.far_tiles) {
                const int row = s - s0;
                float* part = far ? p.far_part + (((unit * sh.far_tiles + j) * sh.chunks + share) * sh.far_rows(p.sinks) + row) * 2 * K
                                  : p.near_part + (((unit * sh.splits + share) * sh.near_tiles() + j) * TILE + row) * 2 * K;
                const bool there = s < p.T && (sink || (!far && sh.splits > 1));
                put_part<K>(tDK, part + half * (K / 2), there);
                put_part<K>(tDV, part + K + half * (K / 2), there);
            }
            if (!far && sh.splits == 1) {
                put_row<K>(tDV, p.dv + at, 1.f, s < p.T && !sink);
                put_row<K>(tDK, p.dk + at, p.scale, s < p.T && !sink);
            }
        }
        umma::fence_before_sync();
    }
    __syncthreads();
    umma::fence_after_sync();
    if (warp == MMA_WARP) {
        if (*abort_flag) {
            umma::commit_lead(umma::elect_one(), barKV);
            umma::mbar_wait(barKV, 1);
            if (lane == 0) atomicExch(p.err, 1);
        }
        umma::tmem_dealloc(tmem, 512);
    }
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
    const int each = (R + sh.splits - 1) / sh.splits;
    for (int x = 0; x * each < R; ++x) add(p.near_part + (((unit * sh.splits + x) * sh.near_tiles() + j) * TILE + s % TILE) * 2 * K);
    if (j < sh.far_tiles && s < p.sinks)
        for (int x = 0; j + sh.near + x * sh.chunk < sh.tiles; ++x) add(p.far_part + (((unit * sh.far_tiles + j) * sh.chunks + x) * sh.far_rows(p.sinks) + s % TILE) * 2 * K);
    const long at = ((b * p.T + s) * p.G + grp) * K;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        reinterpret_cast<uint32_t*>(p.dk + at)[lane + 32 * i] = pack_bf16(sum[i].x * p.scale, sum[i].y * p.scale);
        reinterpret_cast<uint32_t*>(p.dv + at)[lane + 32 * i] = pack_bf16(sum[N + i].x, sum[N + i].y);
    }
}

template <int K>
static cudaError_t launch(const Params& p, cudaStream_t st) {
    const size_t smem = bwd::Smem<K>::total;
    const Shares sh(p.B, p.T, p.H, p.G, p.window, p.sinks);
    const auto dq = window_dq_tc_kernel<K>;
    const auto dkv = window_dkv_tc_kernel<K>;
    cudaError_t e = allow_smem(dq, smem);
    if (e == cudaSuccess) e = allow_smem(dkv, smem);
    if (e != cudaSuccess) return e;
    e = launch_chained(dq, dim3(sh.tiles, p.H, p.B), bwd::NTHREADS, smem, st, p);
    if (e != cudaSuccess) return e;
    LLATTN_LAUNCHED();
    e = launch_chained(dkv, dim3(sh.far_tiles * sh.chunks + sh.tiles * sh.splits, p.G, p.B), bwd::NTHREADS, smem, st, p, sh);
    if (e != cudaSuccess) return e;
    LLATTN_LAUNCHED();
    const int some = sh.far_tiles * TILE < p.sinks ? sh.far_tiles * TILE : p.sinks, tokens = sh.splits > 1 ? p.T : some;
    if (tokens == 0 || (sh.splits == 1 && sh.far_tiles == 0)) return e;
    e = launch_chained(window_join_kernel<K>, (unsigned)(((long)p.B * p.G * tokens + 7) / 8), 256, 0, st, p, sh, tokens);
    if (e == cudaSuccess) LLATTN_LAUNCHED();
    return e;
}
cudaError_t backward_tc(const Params& p, int K, cudaStream_t st) { return K == 64 ? launch<64>(p, st) : launch<128>(p, st); }

}  // namespace win
}  // namespace llattn
