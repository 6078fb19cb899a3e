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

#include "batch.h"
#include "tq_common.h"

namespace tqhip {
namespace {

constexpr int kHeadThreads = 256;
constexpr int kHeadWaves = kHeadThreads / 64;
constexpr int kHeadRounds = 4;

struct HeadArgs {
    const void *in[3];       // q, k, v
    int64_t in_stride[3];
    const float *bias[3];
    const float *norm[2];    // q, k
    void *out[2];            // q_out, k_out
    int64_t out_stride[2];
    void *cache[2];
    int heads[3];            // 0: the call has none of these
    int n_tokens, D, rot;
    float eps;
    double log2_theta;
    const float *inv_freq;
    const int *positions;
    int split;               // waves that share a token's heads
    const int *q_start, *kv_len;
    int n_seqs;
    Pages pages;
};

// V: elements per load; LPH: lanes per head (V > 1: D = 2 V LPH). V = 1 takes every even D up to 512,
// one wave per head, up to four pairs per lane.
template <typename T, typename C, int V, int LPH, bool APPEND>
__global__ __launch_bounds__(kHeadThreads) void heads_kernel(HeadArgs a) {
    constexpr int NU = V == 1 ? 4 : 1;
    constexpr int HPI = 64 / LPH;
    const int lane = threadIdx.x & 63;
    const int wave = blockIdx.x * kHeadWaves + (threadIdx.x >> 6);
    const int t = wave / a.split, part = wave - t * a.split;
    if (t >= a.n_tokens) return;
    const int n_heads = a.heads[0] + a.heads[1] + a.heads[2];
    const int iters = (n_heads + HPI - 1) / HPI;
    const int it0 = iters * part / a.split, it1 = iters * (part + 1) / a.split;  // at most kHeadRounds
    const int half = a.rot / 2;
    const int sub = lane / LPH;

    int at0[NU], at1[NU];
    bool has[NU], turned[NU];
#pragma unroll
    for (int j = 0; j < NU; ++j) {
        const int u = V == 1 ? lane + 64 * j : lane % LPH;
        const int rot_units = half / V;
        has[j] = V > 1 || u < a.D / 2;
        turned[j] = has[j] && u < rot_units;
        at0[j] = !has[j] ? 0 : turned[j] ? u * V : a.rot + 2 * V * (u - rot_units);
        at1[j] = !has[j] ? 0 : turned[j] ? half + u * V : at0[j] + V;
    }
    const auto kind_of = [&](int &h) {
        const int kind = h < a.heads[0] ? 0 : h < a.heads[0] + a.heads[1] ? 1 : 2;
        if (kind > 0) h -= a.heads[0];
        if (kind > 1) h -= a.heads[1];
        return kind;
    };
    // All of the wave's elements are requested at once, before anything waits, and without branches (heads past the last are the
    // last again): a load after a store would wait for the store too, since both count on one in-order counter.
    vec<T, V> raw0[kHeadRounds][NU], raw1[kHeadRounds][NU];
#pragma unroll
    for (int i = 0; i < kHeadRounds; ++i) {
        int h = min(min(it0 + i, it1 - 1) * HPI + sub, n_heads - 1);
        const int kind = kind_of(h);
        const T *src = static_cast<const T *>(a.in[kind]) + t * a.in_stride[kind] + h * a.D;
#pragma unroll
        for (int j = 0; j < NU; ++j) {
            raw0[i][j] = *reinterpret_cast<const vec<T, V> *>(src + at0[j]);
            raw1[i][j] = *reinterpret_cast<const vec<T, V> *>(src + at1[j]);
        }
    }

    int pos = 0;
    int64_t row = -1;
    if constexpr (APPEND) {
        int b;
        if (!find_token(a.q_start, a.kv_len, a.n_seqs, t, b, pos) || pos < 0) return;
        row = row_offset(a.pages, b, pos);
    }
    if (!APPEND || a.positions) pos = a.positions ? a.positions[t] : 0;

    // The token's cosines and sines are formed one pair per lane and go to the lanes of all heads through LDS of the wave's own
    // (formed where they are used, each is formed 64 V / half times over).
    __shared__ __attribute__((aligned(16))) float turn[kHeadWaves][2][256];
    float *cosines = turn[threadIdx.x >> 6][0], *sines = turn[threadIdx.x >> 6][1];
    float c[NU][V], s[NU][V];
    for (int i = lane; i < half; i += 64) {
        constexpr double kInvTwoPi = 0.15915494309189535;
        const double freq = a.inv_freq ? static_cast<double>(a.inv_freq[i]) : exp2(-a.log2_theta * i / half);
        const double w = pos * (freq * kInvTwoPi);
        sincospif(static_cast<float>(2.0 * (w - rint(w))), &sines[i], &cosines[i]);
    }
    wave_lds_order();
#pragma unroll
    for (int j = 0; j < NU; ++j)
        if (turned[j]) {
            load_as_float<float, V>(cosines + at0[j], c[j]);
            load_as_float<float, V>(sines + at0[j], s[j]);
        }

#pragma unroll
    for (int i = 0; i < kHeadRounds; ++i) {
        if (it0 + i >= it1) break;
        int h = (it0 + i) * HPI + sub;
        const bool live = h < n_heads;
        const int kind = kind_of(h);
        const float *bias = a.bias[kind];
        float x0[NU][V], x1[NU][V];
        float sq = 0.0f;
#pragma unroll
        for (int j = 0; j < NU; ++j) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                x0[j][e] = has[j] ? static_cast<float>(raw0[i][j][e]) : 0.0f;
                x1[j][e] = has[j] ? static_cast<float>(raw1[i][j][e]) : 0.0f;
            }
            if (bias && live && has[j]) {
                float b0[V], b1[V];
                load_as_float<float, V>(bias + h * a.D + at0[j], b0);
                load_as_float<float, V>(bias + h * a.D + at1[j], b1);
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    x0[j][e] += b0[e];
                    x1[j][e] += b1[e];
                }
            }
#pragma unroll
            for (int e = 0; e < V; ++e) sq += x0[j][e] * x0[j][e] + x1[j][e] * x1[j][e];
        }
        if (a.norm[0] || a.norm[1]) {
#pragma unroll
            for (int d = 1; d < LPH; d *= 2) sq += __shfl_xor(sq, d);
            const float *w = kind < 2 ? a.norm[kind] : nullptr;
            if (w) {
                const float r = 1.0f / sqrtf(sq / static_cast<float>(a.D) + a.eps);
#pragma unroll
                for (int j = 0; j < NU; ++j) {
                    float w0[V], w1[V];
                    load_as_float<float, V>(w + at0[j], w0);
                    load_as_float<float, V>(w + at1[j], w1);
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        x0[j][e] = x0[j][e] * r * w0[e];
                        x1[j][e] = x1[j][e] * r * w1[e];
                    }
                }
            }
        }
        if (!live) continue;
#pragma unroll
        for (int j = 0; j < NU; ++j) {
            if (!has[j]) continue;
            if (turned[j] && kind < 2) {
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float y0 = x0[j][e], y1 = x1[j][e];
                    x0[j][e] = y0 * c[j][e] - y1 * s[j][e];
                    x1[j][e] = y1 * c[j][e] + y0 * s[j][e];
                }
            }
            if (APPEND && kind > 0) {
                if (row >= 0) {
                    C *dst = static_cast<C *>(a.cache[kind - 1]) + row + h * a.pages.head_stride;
                    store_rounded<C, V>(dst + at0[j], x0[j]);
                    store_rounded<C, V>(dst + at1[j], x1[j]);
                }
            } else {
                T *dst = static_cast<T *>(a.out[kind]) + t * a.out_stride[kind] + h * a.D;
                store_rounded<T, V>(dst + at0[j], x0[j]);
                store_rounded<T, V>(dst + at1[j], x1[j]);
            }
        }
    }
}

template <typename T, typename C, bool APPEND>
int launch_heads(HeadArgs a, bool wide, hipStream_t s) {
    constexpr int V = 16 / sizeof(T);
    const int lph = wide ? a.D / (2 * V) : 64;
    const int iters = (a.heads[0] + a.heads[1] + a.heads[2] + 64 / lph - 1) / (64 / lph);
    // A wave takes up to kHeadRounds rounds of heads, fewer where that gives every CU eight waves.
    const int64_t want = int64_t{8} * device_cu_count() / a.n_tokens;
    a.split = static_cast<int>(std::max<int64_t>((iters + kHeadRounds - 1) / kHeadRounds, std::min<int64_t>(iters, want)));
    const int64_t groups = (static_cast<int64_t>(a.n_tokens) * a.split + kHeadWaves - 1) / kHeadWaves;
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

bool aligned(const void *p, int64_t stride, int bytes) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride * bytes % 16 == 0;
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
    const int bytes = type_bytes(p.dtype), v = 16 / bytes, lanes = p.head_dim / (2 * v);
    bool wide = p.head_dim % (2 * v) == 0 && p.rotary_dim % (2 * v) == 0 && lanes >= 4 && lanes <= 32 &&
                (lanes & (lanes - 1)) == 0;
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

// The queries of a call whose keys and values are another kernel's: a call without them, whose positions are those in the cache.
int finish_queries(const tqhip_head_proj &p, const tqhip_kv_cache &rows, const tqhip_seqs &seqs, hipStream_t s) {
    HeadArgs a{{p.q, nullptr, nullptr}, {p.q_stride, 0, 0}, {p.q_bias, nullptr, nullptr}, {p.q_norm, nullptr}, {p.q_out, nullptr}, {p.q_out_stride, 0},
               {nullptr, nullptr}, {p.n_heads, 0, 0}, p.n_tokens, p.head_dim, p.rotary_dim, p.eps,
               p.rotary_dim && !p.inv_freq ? std::log2(p.theta) : 0.0, p.inv_freq, p.positions, 1, seqs.q_start, seqs.kv_len, seqs.n_seqs,
               make_pages(rows, seqs)};
    const int64_t row = static_cast<int64_t>(p.n_heads) * p.head_dim;
    if (!a.in_stride[0]) a.in_stride[0] = row;
    if (!a.out_stride[0]) a.out_stride[0] = row;
    if (p.n_tokens > 1 && (a.in_stride[0] < row || a.out_stride[0] < row)) return kBadShape;
    const int bytes = type_bytes(p.dtype), v = 16 / bytes, lanes = p.head_dim / (2 * v);
    const bool wide = p.head_dim % (2 * v) == 0 && p.rotary_dim % (2 * v) == 0 && lanes >= 4 && lanes <= 32 && (lanes & (lanes - 1)) == 0 &&
                      aligned(p.q, a.in_stride[0], bytes) && aligned(p.q_out, a.out_stride[0], bytes) && aligned(p.q_bias, 0, 4) &&
                      aligned(p.q_norm, 0, 4);
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
