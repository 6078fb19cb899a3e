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
// next heads with the same cosines and sines, and to its next token with the same frequencies.
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
    const int waves = gridDim.x * kHeadWaves;
    const int n_heads = a.heads[0] + a.heads[1] + a.heads[2];
    const int iters = (n_heads + HPI - 1) / HPI;
    const int per = (iters + a.split - 1) / a.split;
    const int part = wave % a.split;
    const int it0 = part * per, it1 = min(it0 + per, iters);
    const int half = a.rot / 2;
    const int sub = lane / LPH;

    int at0[NU], at1[NU];
    bool has[NU], turned[NU];
    double turns[NU][V];  // per position
#pragma unroll
    for (int j = 0; j < NU; ++j) {
        const int u = V == 1 ? lane + 64 * j : lane % LPH;
        const int rot_units = half / V;
        has[j] = V > 1 || u < a.D / 2;
        turned[j] = has[j] && u < rot_units;
        at0[j] = turned[j] ? u * V : a.rot + 2 * V * (u - rot_units);
        at1[j] = turned[j] ? half + u * V : at0[j] + V;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            constexpr double kInvTwoPi = 0.15915494309189535;
            const int i = u * V + e;
            turns[j][e] = !turned[j] ? 0.0
                          : a.inv_freq ? static_cast<double>(a.inv_freq[i]) * kInvTwoPi
                                       : exp2(-a.log2_theta * i / half) * kInvTwoPi;
        }
    }

    for (int t = wave / a.split; t < a.n_tokens; t += waves / a.split) {
        int pos = 0;
        int64_t row = -1;
        if constexpr (APPEND) {
            const int b = last_start_at_or_before(a.q_start, a.n_seqs, t);
            if (b < 0) continue;
            const int end = a.q_start[b + 1];
            if (t >= end) continue;
            pos = a.kv_len[b] - (end - t);
            if (pos < 0) continue;
            row = row_offset(a.pages, b, pos);
        }
        if (!APPEND || a.positions) pos = a.positions ? a.positions[t] : 0;
        float c[NU][V], s[NU][V];
#pragma unroll
        for (int j = 0; j < NU; ++j)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const double w = pos * turns[j][e];
                sincospif(static_cast<float>(2.0 * (w - rint(w))), &s[j][e], &c[j][e]);
            }
        for (int it = it0; it < it1; ++it) {
            int h = it * HPI + sub;
            const bool live = h < n_heads;
            const int kind = h < a.heads[0] ? 0 : h < a.heads[0] + a.heads[1] ? 1 : 2;
            if (kind > 0) h -= a.heads[0];
            if (kind > 1) h -= a.heads[1];
            const T *src = static_cast<const T *>(a.in[kind]) + t * a.in_stride[kind] + h * a.D;
            const float *bias = a.bias[kind];
            float x0[NU][V], x1[NU][V];
            float sq = 0.0f;
#pragma unroll
            for (int j = 0; j < NU; ++j) {
#pragma unroll
                for (int e = 0; e < V; ++e) x0[j][e] = x1[j][e] = 0.0f;
                if (live && has[j]) {
                    load_as_float<T, V>(src + at0[j], x0[j]);
                    load_as_float<T, V>(src + at1[j], x1[j]);
                    if (bias) {
#pragma unroll
                        for (int e = 0; e < V; ++e) {
                            x0[j][e] += bias[h * a.D + at0[j] + e];
                            x1[j][e] += bias[h * a.D + at1[j] + e];
                        }
                    }
                }
#pragma unroll
                for (int e = 0; e < V; ++e) sq += x0[j][e] * x0[j][e] + x1[j][e] * x1[j][e];
            }
            if (a.norm[0] || a.norm[1]) {
#pragma unroll
                for (int d = 1; d < LPH; d *= 2) sq += __shfl_xor(sq, d);
                const float *w = kind == 0 ? a.norm[0] : kind == 1 ? a.norm[1] : nullptr;
                if (w) {
                    const float r = 1.0f / sqrtf(sq / static_cast<float>(a.D) + a.eps);
#pragma unroll
                    for (int j = 0; j < NU; ++j)
                        if (has[j]) {
#pragma unroll
                            for (int e = 0; e < V; ++e) {
                                x0[j][e] = x0[j][e] * r * w[at0[j] + e];
                                x1[j][e] = x1[j][e] * r * w[at1[j] + e];
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
}

template <typename T, typename C, bool APPEND>
void launch_heads(HeadArgs a, bool wide, hipStream_t s) {
    constexpr int V = 16 / sizeof(T);
    const int lph = wide ? a.D / (2 * V) : 64;
    const int iters = (a.heads[0] + a.heads[1] + a.heads[2] + 64 / lph - 1) / (64 / lph);
    // A token's heads are shared by as many waves as it takes to give every CU eight of them.
    const int64_t want = int64_t{8} * device_cu_count();
    a.split = static_cast<int>(std::min<int64_t>(iters, std::max<int64_t>(1, want / a.n_tokens)));
    const int64_t waves = static_cast<int64_t>(a.n_tokens) * a.split;
    int64_t blocks = std::min<int64_t>((waves + kHeadWaves - 1) / kHeadWaves, int64_t{8} * device_cu_count());
    // (the token loop steps by waves / split, so the waves have to be a multiple of split)
    const int64_t step = a.split;
    blocks = (blocks + step - 1) / step * step;
    const dim3 grid(static_cast<unsigned>(blocks));
    if (!wide) {
        heads_kernel<T, C, 1, 64, APPEND><<<grid, kHeadThreads, 0, s>>>(a);
        return;
    }
    switch (lph) {
        case 4: heads_kernel<T, C, V, 4, APPEND><<<grid, kHeadThreads, 0, s>>>(a); break;
        case 8: heads_kernel<T, C, V, 8, APPEND><<<grid, kHeadThreads, 0, s>>>(a); break;
        case 16: heads_kernel<T, C, V, 16, APPEND><<<grid, kHeadThreads, 0, s>>>(a); break;
        default: heads_kernel<T, C, V, 32, APPEND><<<grid, kHeadThreads, 0, s>>>(a); break;
    }
}

bool aligned(const void *p, int64_t stride, int bytes) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride * bytes % 16 == 0;
}

int run_heads(const tqhip_head_proj &p, const tqhip_kv_cache *cache, const tqhip_seqs *seqs, hipStream_t s) {
    if (!type_known(p.dtype) || p.n_tokens < 1 || p.head_dim < 2 || p.head_dim > 512 || p.head_dim % 2 ||
        p.rotary_dim < 0 || p.rotary_dim > p.head_dim || p.rotary_dim % 2 || p.n_heads < 0 || p.n_kv_heads < 0)
        return kBadShape;
    const bool q = p.q && p.q_out, k = cache || (p.k && p.k_out);
    if ((!p.q) != (!p.q_out) || (!cache && (!p.k) != (!p.k_out))) return kBadShape;
    if ((!q && !k) || (q && p.n_heads < 1) || (k && p.n_kv_heads < 1)) return kBadShape;
    if (!cache && !p.positions && p.rotary_dim) return kBadShape;
    if (p.rotary_dim && !p.inv_freq && !(p.theta > 0.0 && std::isfinite(p.theta))) return kBadShape;
    if (!(p.eps >= 0.0f)) return kBadShape;
    if (static_cast<int64_t>(std::max(p.n_heads, p.n_kv_heads)) * p.head_dim > INT32_MAX / 4) return kTooLarge;
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
    if (q) wide = wide && aligned(p.q_out, a.out_stride[0], bytes);
    if (!cache) {
        if (k) wide = wide && aligned(p.k_out, a.out_stride[1], bytes);
        switch (p.dtype) {
            case TQHIP_F32: launch_heads<float, float, false>(a, wide, s); break;
            case TQHIP_F16: launch_heads<f16, f16, false>(a, wide, s); break;
            default: launch_heads<bf16, bf16, false>(a, wide, s); break;
        }
        return hipGetLastError() == hipSuccess ? kOk : kLaunchFailed;
    }
    const int st = check_cache(*cache, *seqs);
    if (st != kOk) return st;
    if (!p.k || !p.v || cache->n_kv_heads != p.n_kv_heads || cache->head_dim != p.head_dim ||
        seqs->n_tokens != p.n_tokens)
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
    if (p.dtype == TQHIP_F16) {
        launch_heads<f16, f16, true>(a, wide, s);
    } else if (p.dtype == TQHIP_BF16) {
        launch_heads<bf16, bf16, true>(a, wide, s);
    } else {
        switch (cache->dtype) {
            case TQHIP_F32: launch_heads<float, float, true>(a, wide, s); break;
            case TQHIP_F16: launch_heads<float, f16, true>(a, wide, s); break;
            default: launch_heads<float, bf16, true>(a, wide, s); break;
        }
    }
    return hipGetLastError() == hipSuccess ? kOk : kLaunchFailed;
}

}  // namespace
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
