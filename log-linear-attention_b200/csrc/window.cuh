// What the kernels of the sliding-window attention share: parameters, which tokens a query sees, tiles.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "launch_count.h"
#include "pairs.cuh"
#include "tma.cuh"
#include "umma.cuh"

namespace llattn {
namespace win {

typedef __nv_bfloat16 bf16;
constexpr int TILE = 128;             // tokens of a tile of queries, and of keys
constexpr float LOG2E = 1.4426950408889634f;

struct Params {
    CUtensorMap tq, tk, tv, tdo;      // (B,T,heads,K), boxes of 128 tokens x 64 columns of one head
    const bf16 *o, *d_o;
    bf16 *out, *dq, *dk, *dv;
    float *lse, *delta;               // (B,H,TP), TP the length up to whole tiles; lse = log2 of the sum, infinity behind the sequence
    bf16* low;                        // (B,low_rows,H,K): what rounding took off the first rows of o
    int low_rows;
    int* err;                         // status word of the workspace
    int B, T, TP, H, G, window, sinks;
    float scale;
    // backward of k and v, see Shares: fp32 parts of dK and dV
    float *near_part, *far_part;
};

// How the sums of dK and dV are shared out.  A tile of 128 tokens is seen by the queries of its own tile and of the `near - 1` behind it; its CTA takes their heads, or
// one of `splits` shares of them where there are too few tiles to fill the chip; twice as many as SMs where two fit on one (K = 64), or
// where the window reaches back to the start, so that the first tiles have several times the steps of the last, if 16 steps and more are left to a share (us, fewer / more: 2048 tokens, all
// before, 16 heads on 2 of 64 100 / 73, of 128 91 / 74, 32 on 4 169 / 128; but 4096 tokens, 8 heads on 2 of 64, window 512 72 / 76, 16 on 2 of 128, window 1024 129 / 137).  The first `far_tiles` tiles, of sinks, are seen by all later queries too: those come in
// `chunks` shares of `chunk` tiles, about as many steps as a share of the others (one CTA for all of them would run on alone: T = 16384, window 2048, 4 sinks, 8 groups 2.7 ms
// in the place of 1.9 for the whole backward; chunks of `near` tiles where the others are split by heads: 1024 tokens, 4 heads on one, window 256 37 us for 24).  What is shared is left as fp32 parts, and added up in a fixed order.
struct Shares {
    int tiles, near, splits, far_tiles, chunks, chunk;
    Shares(int B, int T, int H, int G, int K, int window, int sinks) {
        const long units = (long)B * G;
        const int R = H / G;
        tiles = (T + TILE - 1) / TILE;
        near = (TILE - 1 + window - 1) / TILE + 1;
        const auto shares = [&](int ctas) { return (int)(ctas / (units * tiles) < R ? ctas / (units * tiles) : R); };
        splits = shares(148);
        const int more = shares(2 * 148), reach = near < tiles ? near : tiles;
        if ((K == 64 || near >= tiles) && more > splits && (long)((R + more - 1) / more) * reach >= 16) splits = more;
        if (splits < 1) splits = 1;
        const int sink_tiles = ((sinks < T ? sinks : T) + TILE - 1) / TILE;
        far_tiles = sink_tiles < tiles - near ? sink_tiles : tiles - near > 0 ? tiles - near : 0;
        chunks = chunk = 0;
        if (far_tiles > 0) {
            const int length = tiles - near;
            long n = 2 * 148 / (units * far_tiles);
            if (n > 32) n = 32;
            const long most = ((long)length * splits + near - 1) / near;       // (all heads of chunk tiles: as many steps as a share of near ones)
            if (n > most) n = most;
            chunk = (int)((length + (n < 1 ? 1 : n) - 1) / (n < 1 ? 1 : n));
            chunks = (length + chunk - 1) / chunk;
        }
    }
    __host__ __device__ int near_tiles() const { return splits > 1 ? tiles : far_tiles; }          // tiles with parts of their own queries
    __host__ __device__ int far_rows(int sinks) const { return sinks < TILE ? sinks : TILE; }      // rows of a far part
    size_t near_floats(int B, int G, int K) const { return (size_t)B * G * splits * near_tiles() * TILE * 2 * K; }
    size_t far_floats(int B, int G, int K, int sinks) const { return (size_t)B * G * far_tiles * chunks * far_rows(sinks) * 2 * K; }
};

// delta = do . o is subtracted from do . v.  For a row that sees n tokens the rounding of o to bf16 leaves an error in dS of sqrt(e / n) of the rounding of dS itself (the output is a mean
// of about n / e values); where n is small it is the larger of the two (n = 2: dq and dk 3.1e-3 off in the place of 2.4e-3).  So the forward keeps what the rounding took off for
// such rows: all of them where the window is short, else those of the first tile.
constexpr int FEW = 64;
inline int low_rows(int T, int window, int sinks) { return window + sinks < FEW || T < TILE ? T : TILE; }

// The tiles of keys that the queries [q0, q0 + 128) see are the first `sink` ones and [lo, hi].
struct Span {
    int lo, hi, sink;
    __host__ __device__ Span(int q0, int T, int window, int sinks) {
        const int first = q0 - window + 1;                 // (window <= 2^29)
        lo = first > 0 ? first / TILE : 0;
        hi = q0 < T ? q0 / TILE : -1;
        const int n = (min_(sinks, T) + TILE - 1) / TILE;
        sink = n < lo ? n : lo;
    }
    static __host__ __device__ int min_(int a, int b) { return a < b ? a : b; }
    __host__ __device__ bool has(int j) const { return j <= hi && (j >= lo || j < sink); }
    // the same as a list
    __host__ __device__ int count() const { return hi < 0 ? 0 : sink + hi - lo + 1; }
    __host__ __device__ int tile(int n) const { return n < sink ? n : lo + n - sink; }
};
// whether every query of the tile from q0 on sees every key of the tile from s0 on
__device__ __forceinline__ bool all_seen(int q0, int s0, int window, int sinks) {
    return s0 + TILE - 1 <= q0 && (q0 + TILE - 1 - s0 < window || s0 + TILE - 1 < sinks);
}
// Which of 32 keys from s0 on query t sees, and which of 32 queries from t0 on see key s: a bit each.
__device__ __forceinline__ uint32_t below(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; }
__device__ __forceinline__ uint32_t seen_bits(int t, int s0, int window, int sinks) {
    return below(t - s0 + 1) & (~below(t - window + 1 - s0) | below(sinks - s0));
}
__device__ __forceinline__ uint32_t seeing_bits(int t0, int s, int window, int sinks) {
    return ~below(s - t0) & (s < sinks ? 0xffffffffu : below(s + window - t0));
}

// 2^x of a pair on the FMA pipes, for a share of the exponentials where the special-function unit (four lanes a cycle and scheduler) is the bottleneck.  x = n + f with n the
// nearest integer, which adding 1.5 2^23 leaves in the low bits; 2^f, f in [-1/2, 1/2], by the minimax polynomial of degree 4 in the relative error (Remez exchange:
// 2.6e-6), times 2^n (a product, not an addition to the exponent, so that NaN stays NaN).  Below -126 the result is 2^-126.
__device__ __forceinline__ float at_least(float x, float low) {                // NaN if x is
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(x), "f"(low));
    return y;
}
__device__ __forceinline__ float2 exp2_poly(F2 x) {
    const float2 v = both(x);
    x = pair(at_least(v.x, -126.f), at_least(v.y, -126.f));
    const F2 magic = pair(12582912.f, 12582912.f), back = pair(-12582912.f, -12582912.f);
    const F2 r = add(x, magic), n = add(r, back), f = fma2(n, pair(-1.f, -1.f), x);
    F2 y = pair(0.009570102207362652f, 0.009570102207362652f);
    y = fma2(y, f, pair(0.05591785907745361f, 0.05591785907745361f));
    y = fma2(y, f, pair(0.240247443318367f, 0.240247443318367f));
    y = fma2(y, f, pair(0.6931217908859253f, 0.6931217908859253f));
    y = fma2(y, f, pair(0.9999992847442627f, 0.9999992847442627f));
    const float2 k = both(r);
    return both(mul(y, pair(__int_as_float(0x3f800000 + (__float_as_int(k.x) << 23)), __int_as_float(0x3f800000 + (__float_as_int(k.y) << 23)))));
}

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// A value >= 0 as two bf16 terms: its upper half, and what that cuts off, which is rounded.  The lowest bit of the latter is set: it is never 0 where the value is not, so that infinity times
// the value is infinity in both terms (and rounds to 0 where it is).
__device__ __forceinline__ uint32_t cut_bf16(float lo, float hi) { return __byte_perm(__float_as_uint(lo), __float_as_uint(hi), 0x7632); }
__device__ __forceinline__ float cut_off(float x) {
    const uint32_t w = __float_as_uint(x);
    return __uint_as_float(w | 1u) - __uint_as_float(w & 0xffff0000u);
}
// A sequence of at most FEW tokens is computed without the rounding of P and dS: an output or a gradient that is a sum of two or three products has no other roundings for theirs to average with
// (2 to 5 tokens, one head: dq and dk 2.2e-3 to 3.3e-3 off in the place of 1.7e-3), and such calls are the host's time in any case.  The forward multiplies P in two terms; the backward
// visits each tile twice, the second time with what rounding took off.  (Kernels of their own: the tests cost the others 1 to 3 %.)  Steps are shifted by `twice`, and those of the second visits
// have the bit.  (By the tokens alone: a sequence has the same gradients in any batch.  All others, from 65 tokens of two heads to 3000, are 1.40 to 1.47 times as far off 64 bits as rounding
// dq and dk makes them, the square root of two roundings.)
inline bool few_tokens(int T) { return T <= FEW; }
template <int N>
__device__ __forceinline__ void leave_rest(float (&e)[N]) {
#pragma unroll
    for (int u = 0; u < N; ++u) e[u] -= __bfloat162float(__float2bfloat16(e[u]));
}
// 64 consecutive fp32 columns of this thread's lane, both loads in flight before the wait
__device__ __forceinline__ void tmem_ld64(uint32_t taddr, float (&v)[64]) {
    uint32_t r[64];
#pragma unroll
    for (int i = 0; i < 2; ++i)
        asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
            "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
            : "=r"(r[32 * i + 0]), "=r"(r[32 * i + 1]), "=r"(r[32 * i + 2]), "=r"(r[32 * i + 3]), "=r"(r[32 * i + 4]), "=r"(r[32 * i + 5]), "=r"(r[32 * i + 6]),
              "=r"(r[32 * i + 7]), "=r"(r[32 * i + 8]), "=r"(r[32 * i + 9]), "=r"(r[32 * i + 10]), "=r"(r[32 * i + 11]), "=r"(r[32 * i + 12]), "=r"(r[32 * i + 13]),
              "=r"(r[32 * i + 14]), "=r"(r[32 * i + 15]), "=r"(r[32 * i + 16]), "=r"(r[32 * i + 17]), "=r"(r[32 * i + 18]), "=r"(r[32 * i + 19]), "=r"(r[32 * i + 20]),
              "=r"(r[32 * i + 21]), "=r"(r[32 * i + 22]), "=r"(r[32 * i + 23]), "=r"(r[32 * i + 24]), "=r"(r[32 * i + 25]), "=r"(r[32 * i + 26]), "=r"(r[32 * i + 27]),
              "=r"(r[32 * i + 28]), "=r"(r[32 * i + 29]), "=r"(r[32 * i + 30]), "=r"(r[32 * i + 31])
            : "r"(taddr + 32 * i)
            : "memory");
    asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
    // every destination register passes through here, so that no use of it can be scheduled above the wait
#pragma unroll
    for (int i = 0; i < 64; i += 16)
        asm volatile(""
                     : "+r"(r[i]), "+r"(r[i + 1]), "+r"(r[i + 2]), "+r"(r[i + 3]), "+r"(r[i + 4]), "+r"(r[i + 5]), "+r"(r[i + 6]), "+r"(r[i + 7]), "+r"(r[i + 8]),
                       "+r"(r[i + 9]), "+r"(r[i + 10]), "+r"(r[i + 11]), "+r"(r[i + 12]), "+r"(r[i + 13]), "+r"(r[i + 14]), "+r"(r[i + 15]));
#pragma unroll
    for (int i = 0; i < 64; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(umma::smem_addr(bar)) : "memory");
}
// The first CTA of a call's first kernel clears the status word: a wait of another sets it when it gives up, 2^20 polls later.  (A memset in front of the
// kernel costs every call 4 us.)
__device__ __forceinline__ void clear_status(const Params& p) {
    if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *p.err = 0;
}
// The issuing warp, after a wait that gave up: the first tiles' copy, whose barrier `bar` is, and all products have ended; the status word says so.
__device__ __forceinline__ void end_products(uint64_t* bar, int* err, int lane) {
    umma::mbar_wait(bar, 0);
    __syncwarp();
    umma::commit_lead(umma::elect_one(), bar);
    umma::mbar_wait(bar, 1);
    if (lane == 0) atomicExch(err, 1);
    __syncwarp();
}
// The way of a warp's 32 rows, a thread a row, to global memory: through 32 WORDS 16-byte words of shared memory, so that neighbouring lanes store neighbouring words of a row.  (Straight
// from the threads, 32 bytes of a row each: 159 us for 156 in the forward of 4 x 4096 tokens, 36.9 for 35.7 in the backward of 8 x 256.)
template <int WORDS>
struct Rows {
    uint4* buf;
    int lane;
    static_assert(WORDS == 8 || WORDS == 16, "rows of 128 or 256 bytes");
    // eight lanes that store together, and eight that load together, meet eight different words of a line
    __device__ __forceinline__ uint4* word(int row, int w) const { return buf + row * WORDS + (w ^ (row & 7)); }
    __device__ __forceinline__ void put(int w, uint32_t a, uint32_t b, uint32_t c, uint32_t d) const { *word(lane, w) = make_uint4(a, b, c, d); }
    // rows [first, last) to `out` + row * stride bytes
    __device__ __forceinline__ void store(void* out, long stride, int first, int last) const {
        __syncwarp();
#pragma unroll
        for (int i = 0; i < WORDS; ++i) {
            const int row = i * (32 / WORDS) + lane / WORDS, w = lane % WORDS;
            const uint4 v = *word(row, w);
            if (row >= first && row < last) *reinterpret_cast<uint4*>(static_cast<char*>(out) + row * stride + w * 16) = v;
        }
        __syncwarp();
    }
};
// one tile of a map into a shared-memory operand tile of K / 64 panels
template <int K>
__device__ __forceinline__ void load_tile(unsigned char* dst, const CUtensorMap* map, int head, int tok0, int batch, uint64_t* bar) {
#pragma unroll
    for (int p = 0; p < K / 64; ++p) tma::load_seq_panel(dst + p * TILE * umma::ROW_BYTES, map, p * 64, head, tok0, batch, bar);
}

cudaError_t forward_tc(const Params& p, int K, cudaStream_t st);
cudaError_t backward_tc(const Params& p, int K, cudaStream_t st);
cudaError_t decode_step(const bf16* q, const bf16* k, const bf16* v, bf16* kc, bf16* vc, long long* counts, bf16* o, int B, int H, int G, int K, int window,
                        int sinks, float scale, cudaStream_t st);

}  // namespace win
}  // namespace llattn
