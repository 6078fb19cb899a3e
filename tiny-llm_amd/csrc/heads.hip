// heads.hip -- the query, key and value heads of a batch of tokens between their projections and the
// attention: biases, RMSNorm of each head, rotation by the token's position, in one pass
// (qk_norm_rope), and the same with keys and values going to a paged cache (kv_append).
//
// With x' = x + bias, y = x' * w / sqrt(mean(x'^2) + eps), and for i < r/2 the pair (y_i, y_{i+r/2})
// turned by the angle pos * theta^(-2i/r).
//
// Every element is read and written once, so a long batch is bound by HBM and a short one by latency.
// A head lies in D / (2 V) lanes of a wave, each holding V elements at u V and the V partners at
// r/2 + u V in 16-byte loads, so norm and rotation stay in registers: the norm is a butterfly over
// the head's lanes. A wave takes several heads of one token side by side and goes on to the token's
// next heads with the same cosines and sines. All of its loads go out before anything waits for one (a
// load behind a store waits for that store: loads between the rounds' stores took 96 us where this takes 69).
//
// 8191 tokens of 32 + 8 heads of 128 in fp32, 335 MB read and written: 69 us, 4.85 TB/s, which is what a copy of such a
// size reaches here (4.8 to 5.3). One token: 3.5 us, a launch and two dependent loads. 12520 tokens of 14 + 2 + 2
// heads of 64 into bf16 pages, 109 MB: 26 us, 4.2 TB/s.
//
// Angles: turns = pos * freq / 2 pi in fp64, reduced to the nearest whole turn there (exact to 2^-53 of
// the turns, so positions in the millions keep 30 bits of angle), then an fp32 sine of the remainder.
// fp32 angles are off by pos * 2^-25 radians, 4e-3 at position 120000.
#include <algorithm>
#include <cmath>

#include "heads.h"

namespace tqhip {
namespace {

template <typename T, typename C, int V, int LPH, bool APPEND>
__global__ __launch_bounds__(kHeadThreads) void heads_kernel(HeadArgs a) {
    finish_heads<T, C, V, LPH, APPEND>(a, blockIdx.x);
}

template <typename T, typename C, bool APPEND>
int launch_heads(HeadArgs a, bool wide, hipStream_t s) {
    constexpr int V = 16 / sizeof(T);
    const int lph = wide ? a.D / (2 * V) : 64;
    const int64_t groups = plan_heads(a, lph);
    if (groups > INT32_MAX / kHeadThreads) return kTooLarge;
    const dim3 grid(static_cast<unsigned>(groups));
    switch (wide ? lph : 0) {
        case 0: heads_kernel<T, C, 1, 64, APPEND><<<grid, kHeadThreads, 0, s>>>(a); break;
        case 4: heads_kernel<T, C, V, 4, APPEND><<<grid, kHeadThreads, 0, s>>>(a); break;
        case 8: heads_kernel<T, C, V, 8, APPEND><<<grid, kHeadThreads, 0, s>>>(a); break;
        case 16: heads_kernel<T, C, V, 16, APPEND><<<grid, kHeadThreads, 0, s>>>(a); break;
        default: heads_kernel<T, C, V, 32, APPEND><<<grid, kHeadThreads, 0, s>>>(a); break;
    }
    return hipGetLastError() == hipSuccess ? kOk : kLaunchFailed;
}

int run_heads(const tqhip_head_proj &p, const tqhip_kv_cache *cache, const tqhip_seqs *seqs, hipStream_t s) {
    const int ok = check_heads(p);
    if (ok != kOk) return ok;
    const bool q = p.q && p.q_out, k = cache || (p.k && p.k_out);
    if ((!p.q) != (!p.q_out) || (!cache && (!p.k) != (!p.k_out))) return kBadShape;
    if ((!q && !k) || (q && p.n_heads < 1) || (k && p.n_kv_heads < 1)) return kBadShape;
    if (!cache && !p.positions && p.rotary_dim) return kBadShape;
    if (std::max(p.n_heads, p.n_kv_heads) > kMostHeads) return kTooLarge;
    HeadArgs a{{p.q, p.k, p.v}, {}, {p.q_bias, p.k_bias, p.v_bias}, {p.q_norm, p.k_norm}, {p.q_out, p.k_out}, {},
               {nullptr, nullptr}, {q ? p.n_heads : 0, k ? p.n_kv_heads : 0, cache ? p.n_kv_heads : 0}, p.n_tokens,
               p.head_dim, p.rotary_dim, p.eps, p.rotary_dim && !p.inv_freq ? std::log2(p.theta) : 0.0, p.inv_freq,
               p.positions, 1, nullptr, nullptr, 0, {nullptr, 0, 0, FastDiv(1), 0, 0, 0}};
    const int64_t in[3] = {p.q_stride, p.k_stride, p.v_stride}, out[2] = {p.q_out_stride, p.k_out_stride};
    for (int i = 0; i < 3; ++i) {
        const int64_t row = static_cast<int64_t>(i == 0 ? p.n_heads : p.n_kv_heads) * p.head_dim;
        a.in_stride[i] = in[i] ? in[i] : row;
        if (i < 2) a.out_stride[i] = out[i] ? out[i] : row;
        if (a.heads[i] && p.n_tokens > 1 && (a.in_stride[i] < row || (i < 2 && a.out_stride[i] < row))) return kBadShape;
    }
    const int bytes = type_bytes(p.dtype);
    bool wide = wide_lanes(p) > 0;
    for (int i = 0; i < 3; ++i)
        if (a.heads[i]) wide = wide && aligned(a.in[i], a.in_stride[i], bytes);
    for (const float *f : {p.q_bias, p.k_bias, p.v_bias, p.q_norm, p.k_norm}) wide = wide && aligned(f, 0, 4);
    if (q) wide = wide && aligned(p.q_out, a.out_stride[0], bytes);
    if (!cache) {
        if (k) wide = wide && aligned(p.k_out, a.out_stride[1], bytes);
        switch (p.dtype) {
            case TQHIP_F32: return launch_heads<float, float, false>(a, wide, s);
            case TQHIP_F16: return launch_heads<f16, f16, false>(a, wide, s);
            default: return launch_heads<bf16, bf16, false>(a, wide, s);
        }
    }
    const int st = check_cache(*cache, *seqs);
    if (st != kOk) return st;
    if (!p.k || !p.v || cache->n_kv_heads != p.n_kv_heads || cache->head_dim != p.head_dim ||
        seqs->n_tokens != p.n_tokens || !rows_apart(*cache))
        return kBadShape;
    // f16 / bf16 activations go into a cache of their own type, f32 into any
    if (p.dtype != TQHIP_F32 && cache->dtype != p.dtype) return kBadShape;
    a.pages = make_pages(*cache, *seqs);
    a.cache[0] = cache->k;
    a.cache[1] = cache->v;
    a.q_start = seqs->q_start;
    a.kv_len = seqs->kv_len;
    a.n_seqs = seqs->n_seqs;
    const int cb = type_bytes(cache->dtype);
    for (const void *c : {cache->k, cache->v}) wide = wide && aligned(c, a.pages.page_stride, cb);
    wide = wide && a.pages.token_stride * cb % 16 == 0 && a.pages.head_stride * cb % 16 == 0;
    if (p.dtype == TQHIP_F16) return launch_heads<f16, f16, true>(a, wide, s);
    if (p.dtype == TQHIP_BF16) return launch_heads<bf16, bf16, true>(a, wide, s);
    switch (cache->dtype) {
        case TQHIP_F32: return launch_heads<float, float, true>(a, wide, s);
        case TQHIP_F16: return launch_heads<float, f16, true>(a, wide, s);
        default: return launch_heads<float, bf16, true>(a, wide, s);
    }
}

}  // namespace

int check_heads(const tqhip_head_proj &p) {
    if (!type_known(p.dtype) || p.n_tokens < 1 || p.head_dim < 2 || p.head_dim > 512 || p.head_dim % 2 ||
        p.rotary_dim < 0 || p.rotary_dim > p.head_dim || p.rotary_dim % 2 || p.n_heads < 0 || p.n_kv_heads < 0)
        return kBadShape;
    if (p.rotary_dim && !p.inv_freq && !(p.theta > 0.0 && std::isfinite(p.theta))) return kBadShape;
    return p.eps >= 0.0f ? kOk : kBadShape;
}

int finish_queries(const tqhip_head_proj &p, const tqhip_kv_cache &rows, const tqhip_seqs &seqs, hipStream_t s) {
    const HeadArgs a = query_args(p, rows, seqs);
    const bool wide = wide_queries(p, a);
    switch (p.dtype) {
        case TQHIP_F32: return launch_heads<float, float, true>(a, wide, s);
        case TQHIP_F16: return launch_heads<f16, f16, true>(a, wide, s);
        default: return launch_heads<bf16, bf16, true>(a, wide, s);
    }
}

}  // namespace tqhip

extern "C" {

int tqhip_qk_norm_rope_dev(const tqhip_head_proj *proj, void *stream) {
    if (!proj) return tqhip::kBadShape;
    return tqhip::run_heads(*proj, nullptr, nullptr, static_cast<hipStream_t>(stream));
}

int tqhip_kv_append_dev(const tqhip_head_proj *proj, const tqhip_kv_cache *cache, const tqhip_seqs *seqs,
                        void *stream) {
    if (!proj || !cache || !seqs) return tqhip::kBadShape;
    return tqhip::run_heads(*proj, cache, seqs, static_cast<hipStream_t>(stream));
}

}  // extern "C"
