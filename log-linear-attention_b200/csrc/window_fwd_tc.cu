// Sliding-window attention forward on the 5th-generation tensor cores.
//
// A CTA takes one or two tiles of 128 queries of a head and walks the tiles of keys that they see.  For each of them and each tile of queries
//     S = Q K^T            128 x 128 x K     into tensor memory
//     P = exp2(c S - m)    a warpgroup, a thread a row: running maximum m and sum, P as bf16 in the place of S
//     O += P V             128 x K x 128     P from tensor memory
// with the products of one tile of queries under the softmax of another: of the same CTA, or of the SM's other one.  The maximum that the exponents refer to moves only when
// a row's has grown by more than 2^8: O, in tensor memory, is rescaled then alone, and P never exceeds 2^8.
//     four warps a tile  softmax, rescaling and output
//     the next one       issues the products
//     the one after it   brings Q, then K and V tiles through a ring
// It is bound by the chain S, softmax, P V of a tile of queries, of which an SM has two in flight: about 3500 cycles a pair of tiles for 2048 of products (T = 16384, 32 query heads
// on 8, K = 128, window 2048: 514 us, 1.0 PFLOP/s of products that are not masked).  Two threads a row in the softmax were slower, 618 us for 572: the rows' maxima then
// go through shared memory.
// P is rounded to bf16, half a step 2^-8: outputs end 2.3e-3 off 64 bits, of which 1.7e-3 are their own rounding.  Two bf16 terms, the second in the other half of S's place, end at
// 1.7e-3, for a second product and eight more instructions a pair of scores (us, one term / two: T = 16384, window 2048, K = 128 507 / 691; 2 x 1999, window 512, K = 64 34 / 47; 4 x 1000,
// window 512, K = 128 39 / 51): TERMS, for sequences of at most FEW tokens alone.
// A wait that gives up sets the CTA's abort flag, after which every other wait ends at once, and the workspace's status word.
#include <type_traits>

#include "window.cuh"

namespace llattn {
namespace win {

namespace fwd {
constexpr float GROWTH = 8.f;

// X tiles of queries a CTA
template <int K, int X>
struct Cta {
    static constexpr int THREADS = 128 * X + 128, MMA_WARP = 4 * X, TMA_WARP = 4 * X + 1, PER_SM = X == 2 ? 1 : 2;
    static constexpr int TM_S = 0, TM_O = 128 * X, TM = 256 * X;              // S, then O, 128 columns a tile
    static constexpr int NST = K == 128 && X == 1 ? 2 : 4;                     // tiles in the ring (two CTAs an SM leave room for two of K = 128)
    static constexpr uint32_t TILE_BYTES = TILE * K * 2;
    static constexpr uint32_t q_off = 0, st_off = X * TILE_BYTES, bar_off = st_off + NST * TILE_BYTES, total = bar_off + 256 + 1024;
    // registers: 384 threads are launched with 168 each, 256 (two CTAs an SM) with 128; 4 warps give theirs to the softmax
    static __device__ __forceinline__ void regs_issue() {
        if constexpr (X == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;\n");
        else asm volatile("setmaxnreg.dec.sync.aligned.u32 56;\n");
    }
    static __device__ __forceinline__ void regs_rows() {
        if constexpr (X == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 216;\n");
        else asm volatile("setmaxnreg.inc.sync.aligned.u32 200;\n");
    }
};

// Of the pairs of exponentials of a tile every POLY-th goes to the FMA pipes, which are idle while the special-function units work (T = 16384, 32 heads, window 2048, us: none
// 590, every eighth 582, fourth 572, third 576, second 604).
constexpr int POLY = 4;

// The tiles of keys that A, or one of A and B, sees: A's list up to the end of the longer one.  (B's band starts no earlier, and where more of the sinks' tiles are in front of it than in
// front of A's, those are tiles of A's band.)
template <int X>
struct Seen {
    Span a, b;
    int count;
    __device__ Seen(const Params& p, int q0) : a(q0, p.T, p.window, p.sinks), b(X == 2 ? q0 + TILE : q0, p.T, p.window, p.sinks) {
        count = a.count() + (b.hi > a.hi ? b.hi - a.hi : 0);
    }
    __device__ int tile(int n) const { return a.tile(n); }
    __device__ bool in(int x, int j) const { return x == 0 ? a.has(j) : b.has(j); }
};
}  // namespace fwd

template <int K, int X, bool TERMS>
__global__ void __launch_bounds__(fwd::Cta<K, X>::THREADS, fwd::Cta<K, X>::PER_SM) window_fwd_tc_kernel(const __grid_constant__ Params p) {
    chain_wait();
    clear_status(p);
    using namespace fwd;
    using SM = Cta<K, X>;
    constexpr int NST = SM::NST, MMA_WARP = SM::MMA_WARP, TMA_WARP = SM::TMA_WARP, TM_S = SM::TM_S, TM_O = SM::TM_O;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = umma::align_1024(smem_raw);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + SM::bar_off);
    uint64_t *full = bars, *empty = bars + NST, *barQ = bars + 2 * NST, *barS = barQ + 2, *barP = barS + 2, *barO = barP + 4;
    constexpr int NBARS = 2 * NST + 10;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + SM::bar_off + NBARS * 8);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    // heads and sequences first, later queries first: those see more tiles, and the last CTAs of a launch are its short ones  (sequences outermost: 41.2 us for 37.4, 4 x 1000 tokens)
    const unsigned units = p.B * p.H, unit = blockIdx.x % units;
    const int h = unit % p.H, q0 = (gridDim.x / units - 1 - blockIdx.x / units) * X * TILE, b = unit / p.H, grp = h / (p.H / p.G);
    const Seen<X> w(p, q0);
    const int count = w.count;
    // position n of the ring's sequence: K, V of the first tile, K, V of the second, ...
    const auto bring = [&](int n) {
        tma::expect_tx(full + n % NST, SM::TILE_BYTES);
        load_tile<K>(smem + SM::st_off + n % NST * SM::TILE_BYTES, n & 1 ? &p.tv : &p.tk, grp, w.tile(n >> 1) * TILE, b, full + n % NST);
    };
    if (tid == TMA_WARP * 32) {              // (the thread that brings the tiles need not wait for the others)
        for (int i = 0; i < NST; ++i) {
            umma::mbar_init(full + i, 1);
            umma::mbar_init(empty + i, 1);
        }
        for (int x = 0; x < X; ++x) {
            umma::mbar_init(barQ + x, 1);
            umma::mbar_init(barS + x, 1);
            umma::mbar_init(barP + 2 * x, 4);
            umma::mbar_init(barP + 2 * x + 1, 4);
            umma::mbar_init(barO + x, 1);
        }
        umma::fence_mbar_init();
        *abort_flag = 0;
        // what the first product needs comes first
        tma::expect_tx(barQ, SM::TILE_BYTES);
        load_tile<K>(smem + SM::q_off, &p.tq, h, q0, b, barQ);
        bring(0);
        if (X == 2 && q0 + TILE < p.T) {
            tma::expect_tx(barQ + 1, SM::TILE_BYTES);
            load_tile<K>(smem + SM::q_off + SM::TILE_BYTES, &p.tq, h, q0 + TILE, b, barQ + 1);
        }
    }
    if (warp == MMA_WARP) umma::tmem_alloc(tmem_slot, SM::TM);
    umma::fence_before_sync();
    __syncthreads();
    umma::fence_after_sync();
    const uint32_t tmem = *tmem_slot;

    if (warp >= MMA_WARP) {
        SM::regs_issue();
        if (warp == TMA_WARP && lane == 0) {
            int n = 1;
            for (; n < 2 * count; ++n) {
                if (n >= NST && !umma::mbar_wait(empty + n % NST, (n / NST - 1) & 1, abort_flag)) break;
                bring(n);
            }
            abort_flag[1] = n;                          // (tiles brought; a register would cost the others 1 %)
        } else if (warp == MMA_WARP) {
            const uint32_t lead = umma::elect_one(), sQ = umma::smem_addr(smem + SM::q_off), sS = umma::smem_addr(smem + SM::st_off);
            constexpr uint32_t idS = umma::idesc_bf16(128, 128, false, false), idO = umma::idesc_bf16(128, K, false, true);
            bool ok = true;
            int done[2] = {0, 0};                       // products P V of A, B issued
            // step i: the products P V with tile i - 1, and S with tile i
            bool before[2] = {false, false};
            for (int i = 0; i <= count && ok; ++i) {
                bool haveK = false, haveV = false;
                const int nk = 2 * i, nv = 2 * i - 1;   // positions of K of this step and V of the one before in the ring's sequence
                for (int x = 0; x < X && ok; ++x) {
                    if (before[x]) {
                        if (!haveV) ok = umma::mbar_wait_warp(full + nv % NST, (nv / NST) & 1, abort_flag);
                        haveV = true;
                        // P comes in two halves, the first product under the exponentials of the second
                        for (int half = 0; half < 2; ++half) {
                            ok = ok && umma::mbar_wait_warp(barP + 2 * x + half, done[x] & 1, abort_flag);
                            if (!ok) break;
                            umma::fence_after_sync();
                            const uint32_t sV = sS + (nv % NST) * SM::TILE_BYTES + half * 64 * umma::ROW_BYTES;
                            umma::gemm_tm_lead<TILE, 64>(lead, tmem + TM_O + 128 * x, tmem + TM_S + 128 * x + 32 * half, sV, idO, done[x] > 0 || half > 0);
                            if (TERMS) umma::gemm_tm_lead<TILE, 64>(lead, tmem + TM_O + 128 * x, tmem + TM_S + 128 * x + 64 + 32 * half, sV, idO, true);
                        }
                        if (!ok) break;
                        umma::commit_lead(lead, barO + x);
                        ++done[x];
                    }
                    before[x] = i < count && w.in(x, w.tile(i));
                    if (before[x]) {
                        ok = umma::mbar_wait_warp(barQ + x, 0, abort_flag);
                        if (!ok) break;
                        if (!haveK) ok = umma::mbar_wait_warp(full + nk % NST, (nk / NST) & 1, abort_flag);
                        haveK = true;
                        if (!ok) break;
                        umma::gemm_kk_lead<TILE, TILE, K>(lead, tmem + TM_S + 128 * x, sQ + x * SM::TILE_BYTES, sS + (nk % NST) * SM::TILE_BYTES, idS, false);
                        umma::commit_lead(lead, barS + x);
                    }
                }
                if (!ok) break;
                // (not in the last round: the last commit is one that the rows wait for, so that none arrives at a CTA that is gone)
                if (i > 0 && i < count) umma::commit_lead(lead, empty + nv % NST);
                if (i < count) umma::commit_lead(lead, empty + nk % NST);
            }
        }
    } else {
        SM::regs_rows();
        const int x = warp >> 2, row = (warp & 3) * 32 + lane, t0 = q0 + x * TILE, t = t0 + row;
        const uint32_t tS = umma::tmem_addr(tmem, warp, TM_S + 128 * x), tO = umma::tmem_addr(tmem, warp, TM_O + 128 * x);
        const float c = p.scale * LOG2E;
        const F2 c2 = pair(c, c);
        const Span span(t0, p.T, p.window, p.sinks);
        const int n = span.count();
        float m = -INFINITY, sum = 0.f;
        bool ok = true;
        for (int i = 0; i < n; ++i) {
            const int s0 = span.tile(i) * TILE;
            const bool whole = all_seen(t0, s0, p.window, p.sinks);
            ok = umma::mbar_wait_warp(barS + x, i & 1, abort_flag);
            if (!ok) break;
            umma::fence_after_sync();
            float s[2][64];
            tmem_ld64(tS, s[0]);
            tmem_ld64(tS + 64, s[1]);
            if (!whole) {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const uint32_t bits = seen_bits(t, s0 + 32 * k, p.window, p.sinks);
#pragma unroll
                    for (int u = 0; u < 32; ++u)
                        if (!(bits & (1u << u))) s[k >> 1][(k & 1) * 32 + u] = -INFINITY;
                }
            }
            float top[4] = {s[0][0], s[0][1], s[0][2], s[0][3]};
#pragma unroll
            for (int k = 4; k < 128; k += 8)
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int e = k + u, f = k + 4 + u < 128 ? k + 4 + u : e;
                    top[u] = fmaxf(fmaxf(top[u], s[e >> 6][e & 63]), s[f >> 6][f & 63]);
                }
            const float now = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * c;
            const bool grown = now > m + GROWTH || (m == -INFINITY && now > m);
            if (i == 0) {
                m = now;
            } else if (__any_sync(0xffffffffu, grown)) {
                ok = umma::mbar_wait_warp(barO + x, (i - 1) & 1, abort_flag);
                if (!ok) break;
                umma::fence_after_sync();
                const float f = grown ? exp2_fast(m - now) : 1.f;
                if (grown) m = now;
                sum *= f;
#pragma unroll
                for (int k = 0; k < K; k += 16) {
                    float o[16];
                    umma::tmem_ld16(tO + k, o);
#pragma unroll
                    for (int u = 0; u < 16; ++u) o[u] *= f;
                    umma::tmem_st16(tO + k, o);
                }
            }
            const float ref = m == -INFINITY ? 0.f : m;        // a row that has seen nothing yet
            const F2 shift = pair(-ref, -ref);
            F2 part[2] = {pair(0.f, 0.f), pair(0.f, 0.f)};
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const auto exponentials = [&](auto mixed) {
#pragma unroll
                    for (int k = 0; k < 64; k += 32) {
                        uint32_t w[16], rest[16];
#pragma unroll
                        for (int u = 0; u < 16; ++u) {
                            const F2 y = fma2(pair(s[half][k + 2 * u], s[half][k + 2 * u + 1]), c2, shift);
                            float2 e;
                            if (decltype(mixed)::value && u % POLY == POLY - 1) {
                                e = exp2_poly(y);
                            } else {
                                const float2 v = both(y);
                                e = make_float2(exp2_fast(v.x), exp2_fast(v.y));
                            }
                            w[u] = TERMS ? cut_bf16(e.x, e.y) : pack_bf16(e.x, e.y);
                            if (TERMS) rest[u] = pack_bf16(cut_off(e.x), cut_off(e.y));
                            part[u & 1] = add(part[u & 1], pair(e.x, e.y));
                        }
                        umma::tmem_st16u(tS + 32 * half + k / 2, w);
                        if (TERMS) umma::tmem_st16u(tS + 64 + 32 * half + k / 2, rest);
                    }
                };
                // (hidden keys are exact zeros: the special-function unit's)
                if (whole) exponentials(std::true_type{});
                else exponentials(std::false_type{});
                umma::tmem_wait_st();
                umma::fence_before_sync();
                __syncwarp();
                if (lane == 0) arrive(barP + 2 * x + half);
            }
            const float2 a = both(add(part[0], part[1]));
            sum += a.x + a.y;
        }
        if (ok && n > 0) ok = umma::mbar_wait_warp(barO + x, (n - 1) & 1, abort_flag);
        if (ok && n > 0) {
            umma::fence_after_sync();
            const float f = 1.f / sum;
            // (all products with this tile's queries are done: their place is free)
            const int first = t0 + (warp & 3) * 32, last = min(p.T - first, 32), few = min(p.low_rows - first, 32);
            const Rows<K / 8> rows = {reinterpret_cast<uint4*>(smem + SM::q_off + warp * 32 * K * 2), lane};
            const auto take = [&](auto low) {
#pragma unroll
                for (int i = 0; i < K; i += 64) {
                    float o[64];
                    tmem_ld64(tO + i, o);
#pragma unroll
                    for (int u = 0; u < 64; u += 8) {
                        uint32_t w[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float a = o[u + 2 * e] * f, b = o[u + 2 * e + 1] * f;
                            w[e] = pack_bf16(a, b);
                            if (decltype(low)::value) w[e] = pack_bf16(a - __uint_as_float(w[e] << 16), b - __uint_as_float(w[e] & 0xffff0000u));
                        }
                        rows.put((i + u) / 8, w[0], w[1], w[2], w[3]);
                    }
                }
            };
            take(std::false_type{});
            rows.store(p.out + (((long)b * p.T + first) * p.H + h) * K, (long)p.H * K * 2, 0, last);
            if (few > 0) {                                 // (low_rows is 0 where no backward follows)
                take(std::true_type{});
                rows.store(p.low + (((long)b * p.low_rows + first) * p.H + h) * K, (long)p.H * K * 2, 0, few);
            }
            if (p.lse) p.lse[((long)b * p.H + h) * p.TP + t] = t < p.T ? m + log2f(sum) : INFINITY;
        }
        umma::fence_before_sync();
    }
    __syncthreads();
    umma::fence_after_sync();
    // after a wait that gave up (none can from here on): copies and products that nobody waited for end before the CTA does
    if (*abort_flag) {
        if (tid == TMA_WARP * 32) {
            if (X == 2 && q0 + TILE < p.T) umma::mbar_wait(barQ + 1, 0);
            const int brought = abort_flag[1];
            for (int i = brought > NST ? brought - NST : 0; i < brought; ++i) umma::mbar_wait(full + i % NST, (i / NST) & 1);
        }
        if (warp == MMA_WARP) end_products(barQ, p.err, lane);
    }
    if (warp == MMA_WARP) umma::tmem_dealloc(tmem, SM::TM);
}

template <int K, int X, bool TERMS>
static cudaError_t launch(const Params& p, cudaStream_t st) {
    using C = fwd::Cta<K, X>;
    const auto kern = window_fwd_tc_kernel<K, X, TERMS>;
    cudaError_t e = allow_smem(kern, C::total);
    if (e != cudaSuccess) return e;
    const unsigned grid = (unsigned)(p.T + X * TILE - 1) / (X * TILE) * p.H * p.B;
    e = launch_chained(kern, grid, C::THREADS, C::total, st, p);
    if (e == cudaSuccess) LLATTN_LAUNCHED();
    return e;
}
// One tile a CTA, two CTAs an SM, whose starts and ends run under each other's steps; or, where K = 128 and a query sees thousands of keys, two tiles that share what comes from memory (us,
// one tile / two: K = 128, 32 heads on 8, window 512, 8192 tokens 119 / 128; window 1024 164 / 169; window 2048, 4096 tokens 110 / 109, 8192 tokens 249 / 239; 8192 tokens, all that are
// before 482 / 439; K = 64, 16 heads, 2 x 1999 tokens, window 512 25.4 / 31.2; 8 heads on 2, 32768 tokens, window 4096 417 / 440; 32 heads on 8, 8192 tokens, all before 469 / 455).
cudaError_t forward_tc(const Params& p, int K, cudaStream_t st) {
    if (few_tokens(p.T)) return K == 64 ? launch<64, 1, true>(p, st) : launch<128, 1, true>(p, st);
    if (K == 64) return launch<64, 1, false>(p, st);
    return p.T >= 2048 && p.window >= 2048 ? launch<128, 2, false>(p, st) : launch<128, 1, false>(p, st);
}

}  // namespace win
}  // namespace llattn
