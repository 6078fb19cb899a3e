// heads.h -- the heads of a batch of tokens finished (biases, norm, rotation), as heads.hip describes it, for its kernels and for the queries that
// ride along with append8.hip's.
#pragma once

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
// one wave per head, up to four pairs per lane. group: of kHeadThreads threads, of those that plan_heads counts.
template <typename T, typename C, int V, int LPH, bool APPEND>
__device__ inline void finish_heads(const HeadArgs &a, int group) {
    constexpr int NU = V == 1 ? 4 : 1;
    constexpr int HPI = 64 / LPH;
    const int lane = threadIdx.x & 63;
    const int wave = group * kHeadWaves + (threadIdx.x >> 6);
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

// A wave takes up to kHeadRounds rounds of heads, fewer where that gives every CU eight waves. lph: lanes a head.
inline int64_t plan_heads(HeadArgs &a, int lph) {
    const int iters = (a.heads[0] + a.heads[1] + a.heads[2] + 64 / lph - 1) / (64 / lph);
    const int64_t want = int64_t{8} * device_cu_count() / a.n_tokens;
    a.split = static_cast<int>(std::max<int64_t>((iters + kHeadRounds - 1) / kHeadRounds, std::min<int64_t>(iters, want)));
    return (static_cast<int64_t>(a.n_tokens) * a.split + kHeadWaves - 1) / kHeadWaves;
}

inline bool aligned(const void *p, int64_t stride, int bytes) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride * bytes % 16 == 0;
}
// Lanes a head on the vector path for what is loaded V elements at a time, 0 where it has none.
inline int wide_lanes(const tqhip_head_proj &p) {
    const int v = 16 / type_bytes(p.dtype), lanes = p.head_dim / (2 * v);
    return p.head_dim % (2 * v) == 0 && p.rotary_dim % (2 * v) == 0 && lanes >= 4 && lanes <= 32 && (lanes & (lanes - 1)) == 0 ? lanes : 0;
}

// The queries of a call whose keys and values are another kernel's: a call without them, whose positions are those in the cache.
inline HeadArgs query_args(const tqhip_head_proj &p, const tqhip_kv_cache &rows, const tqhip_seqs &seqs) {
    const int64_t row = static_cast<int64_t>(p.n_heads) * p.head_dim;
    return {{p.q, nullptr, nullptr}, {p.q_stride ? p.q_stride : row, 0, 0}, {p.q_bias, nullptr, nullptr}, {p.q_norm, nullptr}, {p.q_out, nullptr},
            {p.q_out_stride ? p.q_out_stride : row, 0}, {nullptr, nullptr}, {p.n_heads, 0, 0}, p.n_tokens, p.head_dim, p.rotary_dim, p.eps,
            p.rotary_dim && !p.inv_freq ? std::log2(p.theta) : 0.0, p.inv_freq, p.positions, 1, seqs.q_start, seqs.kv_len, seqs.n_seqs,
            make_pages(rows, seqs)};
}
inline bool wide_queries(const tqhip_head_proj &p, const HeadArgs &a) {
    const int bytes = type_bytes(p.dtype);
    return wide_lanes(p) && aligned(p.q, a.in_stride[0], bytes) && aligned(p.q_out, a.out_stride[0], bytes) && aligned(p.q_bias, 0, 4) &&
           aligned(p.q_norm, 0, 4);
}

}  // namespace
}  // namespace tqhip
