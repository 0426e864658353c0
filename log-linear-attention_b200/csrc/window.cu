// Attention over a sliding window with sinks: query t sees the tokens s <= t with t - s < window or s < sinks,
//     o_t = sum_s P_ts v_s,   P_ts = exp(scale q_t . k_s - lse_t),   lse_t = log sum_s exp(scale q_t . k_s)
// and the gradients, with delta_t = do_t . o_t,
//     dV_s = sum_t P_ts do_t,   dS_ts = P_ts (do_t . v_s - delta_t),   dQ_t = scale sum_s dS_ts k_s,   dK_s = scale sum_t dS_ts q_t.
// H query heads share G heads of k and v: dK and dV are sums over the H / G heads too.
//
// Here: the C entries and the cache of a decoding sequence.  Forward: window_fwd_tc.cu, backward: window_bwd_tc.cu, steps: window_step.cu.
#include "../../include/llattn.h"
#include "window.cuh"

namespace llattn {
namespace win {

// Slot c of a sequence of n tokens holds token c if c < sinks, else the last token that is c modulo the window, counted from the end of the sinks; zeros where there is none.
__global__ void __launch_bounds__(256) window_fill_kernel(const bf16* k, const bf16* v, const long long* lengths, bf16* kc, bf16* vc, long long* counts, int T,
                                                          int G, int K, int window, int sinks) {
    chain_wait();
    const int slots = sinks + window, b = blockIdx.y;
    const long words = (long)G * K / 8;                                    // of 16 bytes, a token
    long long n = lengths ? lengths[b] : T;
    n = n < 0 ? 0 : n > T ? T : n;
    const long i = (long)blockIdx.x * 256 + threadIdx.x;
    if (i < G) counts[(long)b * G + i] = n;
    if (i >= slots * words) return;
    const int c = (int)(i / words);
    const long w = i % words;
    uint4 kw = make_uint4(0, 0, 0, 0), vw = kw;
    if (c < n) {
        const long t = c < sinks ? c : c + (n - 1 - c) / window * window, at = ((long)b * T + t) * words + w;
        kw = reinterpret_cast<const uint4*>(k)[at];
        vw = reinterpret_cast<const uint4*>(v)[at];
    }
    reinterpret_cast<uint4*>(kc)[(long)b * slots * words + i] = kw;
    reinterpret_cast<uint4*>(vc)[(long)b * slots * words + i] = vw;
}

int check(long B, long T, long H, long G, int K, long window, long sinks, float scale) {
    if (B < 1 || T < 1 || G < 1 || H < 1 || (K != 64 && K != 128) || window < 1 || sinks < 0 || !(scale > 0.f) || !(scale < INFINITY)) return LLATTN_ERR_UNSUPPORTED_SHAPE;
    if (H % G != 0) return LLATTN_ERR_BAD_GROUPS;
    if (T > (1 << 24) || window > (1 << 29) || sinks > (1 << 29) || B > 65535 || H > 65535 || (T + 127) / 128 * H * B > 0x3fffffffl) return LLATTN_ERR_UNSUPPORTED_SHAPE;
    return 0;
}
int padded(int T) { return (T + TILE - 1) / TILE * TILE; }
size_t lse_bytes(int B, int T, int H) { return (size_t)B * H * padded(T) * sizeof(float); }
void statistics(Params& p, void* stats) {
    if (!stats) return;
    p.lse = static_cast<float*>(stats);
    p.low = reinterpret_cast<bf16*>(static_cast<char*>(stats) + lse_bytes(p.B, p.T, p.H));
    p.low_rows = low_rows(p.T, p.window, p.sinks);
}
void shape(Params& p, void* workspace, int B, int T, int H, int G, int window, int sinks, float scale) {
    p.err = static_cast<int*>(workspace);
    p.B = B;
    p.T = T;
    p.TP = padded(T);
    p.H = H;
    p.G = G;
    p.window = window;
    p.sinks = sinks;
    p.scale = scale;
}
// Tensor maps are made by the driver, for the calling thread's context: a thread that has made no runtime call yet gets it here.
cudaError_t current_context() {
    int device;
    const cudaError_t e = cudaGetDevice(&device);
    return e == cudaSuccess ? cudaSetDevice(device) : e;
}
bool maps(Params& p, const void* q, const void* k, const void* v, int K) {
    return tma::make_seq_map(&p.tq, q, p.B, p.T, p.H, K, TILE, 2) == 0 && tma::make_seq_map(&p.tk, k, p.B, p.T, p.G, K, TILE, 2) == 0 &&
           tma::make_seq_map(&p.tv, v, p.B, p.T, p.G, K, TILE, 2) == 0;
}

}  // namespace win
}  // namespace llattn

using namespace llattn;

extern "C" {

size_t llattn_window_stats_bytes(int B, int T, int H, int K, int window, int sinks) {
    if (win::check(B, T, H, 1, K, window, sinks, 1.f) != 0) return 0;
    return win::lse_bytes(B, T, H) + (size_t)B * win::low_rows(T, window, sinks) * H * K * sizeof(win::bf16);
}
size_t llattn_window_workspace_bytes(int B, int T, int H, int G, int K, int window, int sinks) {
    if (win::check(B, T, H, G, K, window, sinks, 1.f) != 0) return 0;
    const win::Shares sh(B, T, H, G, K, window, sinks);
    return 256 + win::lse_bytes(B, T, H) + (sh.near_floats(B, G, K) + sh.far_floats(B, G, K, sinks)) * sizeof(float);
}

int llattn_window_fwd(const void* q, const void* k, const void* v, void* o, void* stats, void* workspace, size_t workspace_bytes, int B, int T, int H, int G, int K,
                      int window, int sinks, float scale, void* stream) {
    const int rc = win::check(B, T, H, G, K, window, sinks, scale);
    if (rc != 0) return rc;
    if (!q || !k || !v || !o) return LLATTN_ERR_NULL;
    if (misaligned(16, {q, k, v, o, stats})) return LLATTN_ERR_ALIGNMENT;
    if (!workspace || misaligned(256, {workspace}) || workspace_bytes < 256) return LLATTN_ERR_WORKSPACE;
    win::Params p = {};
    p.out = (win::bf16*)o;
    win::shape(p, workspace, B, T, H, G, window, sinks, scale);
    win::statistics(p, stats);
    cudaStream_t st = (cudaStream_t)stream;
    const cudaError_t e = win::current_context();
    if (e != cudaSuccess) return (int)e;
    if (!win::maps(p, q, k, v, K)) return LLATTN_ERR_TENSOR_MAP;
    return (int)win::forward_tc(p, K, st);
}

int llattn_window_bwd(const void* q, const void* k, const void* v, const void* o, const void* stats, const void* d_o, void* dq, void* dk, void* dv, void* workspace,
                      size_t workspace_bytes, int B, int T, int H, int G, int K, int window, int sinks, float scale, void* stream) {
    const int rc = win::check(B, T, H, G, K, window, sinks, scale);
    if (rc != 0) return rc;
    if (!q || !k || !v || !o || !stats || !d_o || !dq || !dk || !dv) return LLATTN_ERR_NULL;
    if (misaligned(16, {q, k, v, o, stats, d_o, dq, dk, dv})) return LLATTN_ERR_ALIGNMENT;
    if (!workspace || misaligned(256, {workspace}) || workspace_bytes < llattn_window_workspace_bytes(B, T, H, G, K, window, sinks)) return LLATTN_ERR_WORKSPACE;
    win::Params p = {};
    p.o = (const win::bf16*)o;
    p.d_o = (const win::bf16*)d_o;
    p.dq = (win::bf16*)dq;
    p.dk = (win::bf16*)dk;
    p.dv = (win::bf16*)dv;
    p.delta = reinterpret_cast<float*>(static_cast<char*>(workspace) + 256);
    p.near_part = p.delta + (long)B * H * win::padded(T);
    p.far_part = p.near_part + win::Shares(B, T, H, G, K, window, sinks).near_floats(B, G, K);
    win::shape(p, workspace, B, T, H, G, window, sinks, scale);
    win::statistics(p, const_cast<void*>(stats));
    cudaStream_t st = (cudaStream_t)stream;
    const cudaError_t e = win::current_context();
    if (e != cudaSuccess) return (int)e;
    if (!win::maps(p, q, k, v, K) || tma::make_seq_map(&p.tdo, d_o, B, T, H, K, win::TILE, 2) != 0) return LLATTN_ERR_TENSOR_MAP;
    return (int)win::backward_tc(p, K, st);
}

int llattn_window_fill(const void* k, const void* v, const long long* lengths, void* k_cache, void* v_cache, long long* counts, int B, int T, int G, int K,
                       int window, int sinks, void* stream) {
    const int rc = win::check(B, T, G, G, K, window, sinks, 1.f);
    if (rc != 0) return rc;
    if (!k || !v || !k_cache || !v_cache || !counts) return LLATTN_ERR_NULL;
    if (misaligned(16, {k, v, lengths, k_cache, v_cache, counts})) return LLATTN_ERR_ALIGNMENT;
    const long n = (long)(window + sinks) * G * K / 8, blocks = ((n > G ? n : G) + 255) / 256;
    if (B > 65535 || blocks > 0x7fffffffl) return LLATTN_ERR_UNSUPPORTED_SHAPE;
    cudaStream_t st = (cudaStream_t)stream;
    const dim3 grid((unsigned)blocks, B);
    const auto *kk = (const win::bf16*)k, *vv = (const win::bf16*)v;
    const cudaError_t e = launch_chained(win::window_fill_kernel, grid, 256, 0, st, kk, vv, lengths, (win::bf16*)k_cache, (win::bf16*)v_cache, counts, T, G, K, window, sinks);
    if (e == cudaSuccess) LLATTN_LAUNCHED();
    return (int)e;
}

int llattn_window_step(const void* q, const void* k, const void* v, void* k_cache, void* v_cache, long long* counts, void* o, int B, int H, int G, int K, int window,
                       int sinks, float scale, void* stream) {
    const int rc = win::check(B, 1, H, G, K, window, sinks, scale);
    if (rc != 0) return rc;
    if (!q || !k || !v || !k_cache || !v_cache || !counts || !o) return LLATTN_ERR_NULL;
    if (misaligned(16, {q, k, v, k_cache, v_cache, counts, o})) return LLATTN_ERR_ALIGNMENT;
    cudaStream_t st = (cudaStream_t)stream;
    return (int)win::decode_step((const win::bf16*)q, (const win::bf16*)k, (const win::bf16*)v, (win::bf16*)k_cache, (win::bf16*)v_cache, counts, (win::bf16*)o, B, H, G, K,
                                 window, sinks, scale, st);
}

}  // extern "C"
