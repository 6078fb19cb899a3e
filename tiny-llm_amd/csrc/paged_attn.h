// paged_attn.h -- what the attention kernels over a paged cache share (paged_attn.hip: f32, f16 and bf16 caches; paged_attn8.hip: codes of
// 8 bits): arguments, operands as terms of 16 bits, the rows and keys of a tile, a row by the formula, the join of the parts
// and how a call is cut.
#pragma once

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <optional>
#include <type_traits>

#include "batch.h"
#include "lane_sum.h"
#include "tq_common.h"

namespace tqhip {
namespace {

struct AttnArgs {
    const void *q, *k, *v;
    void *out;
    int64_t q_stride, out_stride;
    const int *q_start, *kv_len;
    int n_seqs, n_tokens, n_heads, group;  // group: query heads per key/value head
    float scale;                           // |scale| * log2 e; the sign goes into q
    float sign;
    int causal, window;
    int parts, span;                       // parts of `span` keys, the last one to the end
    float *part_o;                         // [n_tokens * n_heads][parts][head_dim], unnormalised
    float2 *part_ml;                       // [n_tokens * n_heads][parts]: exponent bias, sum of weights
    Pages pages;
    const float2 *scales;                  // of codes of 8 bits: [n_pages][key/value heads][blocks of a page], of the keys and of the values
    FastDiv block{1};                      // tokens that share them
    int blocks;
};

// ---- codes of 8 bits ------------------------------------------------------------------------------

struct i8 {};    // integers from -127 to 127
struct e4m3 {};  // numbers of 4 bits of exponent and 3 of fraction, up to 448, NaN at all ones
template <typename C>
constexpr bool kCodes = std::is_same_v<C, i8> || std::is_same_v<C, e4m3>;
template <typename C>
using Stored = std::conditional_t<kCodes<C>, unsigned char, C>;

// The four codes of a word as floats.
template <typename C>
__device__ inline vec<float, 4> four_codes(unsigned u) {
    if constexpr (std::is_same_v<C, i8>) {
        return vec<float, 4>{static_cast<float>(static_cast<int>(u << 24) >> 24), static_cast<float>(static_cast<int>(u << 16) >> 24),
                             static_cast<float>(static_cast<int>(u << 8) >> 24), static_cast<float>(static_cast<int>(u) >> 24)};
    } else {
        return vec<float, 4>{__builtin_amdgcn_cvt_f32_fp8(u, 0), __builtin_amdgcn_cvt_f32_fp8(u, 1), __builtin_amdgcn_cvt_f32_fp8(u, 2),
                             __builtin_amdgcn_cvt_f32_fp8(u, 3)};
    }
}

// N stored elements as floats (codes without their scale).
template <typename C, int N>
__device__ inline void load_stored(const Stored<C> *p, float *out) {
    if constexpr (!kCodes<C>) {
        load_as_float<C, N>(p, out);
    } else if constexpr (N >= 4) {
        const vec<unsigned, N / 4> u = *reinterpret_cast<const vec<unsigned, N / 4> *>(p);
#pragma unroll
        for (int i = 0; i < N; ++i) out[i] = four_codes<C>(u[i / 4])[i % 4];
    } else {
        unsigned u = p[0];
        if constexpr (N == 2) u = *reinterpret_cast<const unsigned short *>(p);
#pragma unroll
        for (int i = 0; i < N; ++i) out[i] = four_codes<C>(u)[i];
    }
}

// The scales of the row of position p in a page that exists.
__device__ inline float2 row_scales(const AttnArgs &a, int page, int kvh, int p) {
    const int row = p - a.pages.page_size.quot(p) * static_cast<int>(a.pages.page_size.d), heads = a.n_heads / a.group;
    return a.scales[(static_cast<int64_t>(page) * heads + kvh) * a.blocks + a.block.quot(row)];
}

// ---- numbers as terms of 16 bits ----------------------------------------------------------------

// How a product's operands are held: E the type of the matrix instruction, QT terms of a query element
// or a weight, KT of a cache element. 16-bit activations meet a cache of their own type as they are.
// fp32 activations keep their precision: against an fp16 cache two fp16 terms (22 bits), against
// a bf16 one three bf16 terms (24 bits), and an fp32 cache is three bf16 terms itself. Codes of 8 bits are fp16 numbers without
// rounding, and queries of 16 bits meet them as one fp16 term: bf16's 8 bits fit, and a row's power of two keeps its range. (One term
// rounds the weights too, once more than the result: bf16 prompts over a bf16 cache are 2.1e-3 from 64 bits, where the result's
// rounding alone is 1.6e-3. A second term would be half as many products again, for bits that the result does not keep.)
// Over codes a bf16 row's weights are one fp16 term as well: 1.67e-3 from 64 bits in all, 1.66e-3 with the result's rounding alone. An f16
// result does show it: 2.3e-4 to 2.7e-4, 2.0e-4 to 2.1e-4 without. So f16 rows get a second term of their weights, and are off by their result's
// rounding. It costs 1 % of a step of single tokens (64 over up to 16000 keys 214 us, 212 with one term), 4 % of drafted ones (94.5, 91), 16 % of
// chunks (201, 173), 23 % of prompts (two of up to 8192: 1281, 1041).
template <typename T, typename C>
struct Terms {
    using E = std::conditional_t<std::is_same_v<C, f16> || kCodes<C>, f16, bf16>;
    static constexpr int KT = std::is_same_v<C, float> ? 3 : 1;
    static constexpr int QT = !std::is_same_v<T, float> ? 1 : std::is_same_v<E, f16> ? 2 : 3;
    // terms of a weight times its value's scale, over codes
    static constexpr int WT = std::is_same_v<T, f16> ? 2 : QT;
    // products of term i and term j are kept while i + j < max(QT, KT): the next ones are below 2^-24
    static constexpr int kMost = QT > KT ? QT : KT;
};

// x as N terms of 16 bits, the largest first: the last one rounded to nearest even, those before it so
// that the rest is exact. bf16 terms before the last are cut off, which cannot overflow.
template <typename E, int N>
__device__ inline void split(const float *x, vec<E, 8> *out) {
    float r[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = x[i];
#pragma unroll
    for (int n = 0; n < N; ++n) {
        if (n == N - 1) {
#pragma unroll
            for (int i = 0; i < 8; ++i) out[n][i] = static_cast<E>(r[i]);
        } else if constexpr (std::is_same_v<E, bf16>) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const unsigned u = __float_as_uint(r[i]);
                out[n][i] = __builtin_bit_cast(bf16, static_cast<unsigned short>(u >> 16));
                const float cut = __uint_as_float(u & 0xffff0000u);
                r[i] = r[i] == cut ? 0.0f : r[i] - cut;  // (an infinity is its first term)
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                out[n][i] = static_cast<E>(r[i]);
                r[i] -= static_cast<float>(out[n][i]);
            }
        }
    }
}

using f32x4 = vec<float, 4>;
using f32x16 = vec<float, 16>;
__device__ inline f32x4 mfma16(vec<f16, 8> a, vec<f16, 8> b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ inline f32x4 mfma16(vec<bf16, 8> a, vec<bf16, 8> b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ inline f32x16 mfma32(vec<f16, 8> a, vec<f16, 8> b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ inline f32x16 mfma32(vec<bf16, 8> a, vec<bf16, 8> b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// l plus the eight elements, two at a time.
__device__ inline float add_all(vec<f16, 8> p, float l) {
    const vec<f16, 2> ones{static_cast<f16>(1.0f), static_cast<f16>(1.0f)};
#pragma unroll
    for (int i = 0; i < 8; i += 2) l = __builtin_amdgcn_fdot2(vec<f16, 2>{p[i], p[i + 1]}, ones, l, false);
    return l;
}
__device__ inline float add_all(vec<bf16, 8> p, float l) {
    const vec<bf16, 2> ones{static_cast<bf16>(1.0f), static_cast<bf16>(1.0f)};
#pragma unroll
    for (int i = 0; i < 8; i += 2) l = __builtin_amdgcn_fdot2_f32_bf16(vec<bf16, 2>{p[i], p[i + 1]}, ones, l, false);
    return l;
}

// Four rows of 16 elements each, held 4 elements a lane by 16 lanes, as columns: lane i gets column i's four.
template <typename E>
__device__ inline vec<E, 4> lds_columns(const E *p) {
    using raw = vec<short, 4>;
    return __builtin_bit_cast(vec<E, 4>, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) raw *)p));
}

template <typename C>
__device__ inline bool is_finite(C x) {
    if constexpr (std::is_same_v<C, float>)
        return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u;
    constexpr unsigned short kExp = std::is_same_v<C, f16> ? 0x7c00 : 0x7f80;
    return (__builtin_bit_cast(vec<unsigned short, sizeof(C) / 2>, x)[0] & kExp) != kExp;
}

// A value that all lanes of the wave hold.
__device__ inline unsigned long long scalar(unsigned long long v) {
    const unsigned lo = __builtin_amdgcn_readfirstlane(static_cast<unsigned>(v));
    const unsigned hi = __builtin_amdgcn_readfirstlane(static_cast<unsigned>(v >> 32));
    return static_cast<unsigned long long>(hi) << 32 | lo;
}

// Bits below n (none for n <= 0, all from 32 on).
__device__ inline unsigned below(int n) { return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1u; }

// A chunk of 8 cache elements as its terms.
template <typename C, typename E, int KT>
__device__ inline void as_terms(const vec<C, 8> &x, vec<E, 8> *out) {
    if constexpr (KT == 1) {
        out[0] = x;
    } else {
        float f[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = x[e];
        split<E, KT>(f, out);
    }
}

// Infinities and NaN replaced by zeros; false if there were any.
template <typename C>
__device__ inline bool make_finite(vec<C, 8> &x) {
    bool finite = true;
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (!is_finite<C>(x[e])) {
            finite = false;
            x[e] = static_cast<C>(0.0f);
        }
    return finite;
}

// 16 bytes per lane from global memory to LDS, lane after lane from `to` (the same in all lanes), without passing through
// registers; wait_loads waits for all that the wave has under way.
// STREAM: rows that are read once, past the caches' other contents.
template <bool STREAM, typename T, typename E>
__device__ inline void global_to_lds(const T *from, E *to) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)from,
                                     (__attribute__((address_space(3))) void *)to, 16, 0, STREAM ? 2 : 0);
}
__device__ inline void wait_loads() {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt((7 << 4) | (15 << 8));  // vmcnt(0)
    __builtin_amdgcn_sched_barrier(0);
}

// A row's sums are brought down to a new maximum only once it exceeds the one they stand at by that power of two: the weights stay
// within fp16's range, and what their sums lose by it is nothing, since a factor of a power of two is common to all of them.
// (With fp32 results 2^1: an exponent of up to 7 has three bits less behind its point than one near 0.)
template <int QT>
constexpr float kHeadroom = QT == 1 ? 7.0f : 1.0f;

// Weights are 2^(s c + bias), held as large as fp16's range lets them be, 2^15 with the headroom: below 2^-14 they are subnormal, off by up
// to 2^-25, and weights small beside the largest count where its value is small. (Two terms at 2^8 lost half of the bits of weights
// 2^-20 of the largest.) bf16 has the range.
template <typename E, int QT>
constexpr float kWeightShift = std::is_same_v<E, f16> ? 15.0f - kHeadroom<QT> : 0.0f;

// A bias is a rounded number: the key that it stands at has a weight of 2^kWeightShift times 2^(up to half a step of the bias) either way,
// and with scores of many millions that leaves fp16's range, and then fp32's. A row whose bias is past the last power of two at which it
// does not (half a step of 1/2 on top of 2^15, of 8 in bf16, which would bear more) gets a sum of NaN, so formula_row takes it: by
// size, not by whether it overflowed, so the parts of a row are treated alike.
template <typename E>
__device__ inline float checked_sum(float bias, float l) {
    return fabsf(bias) > (std::is_same_v<E, f16> ? 0x1p24f : 0x1p28f) ? NAN : l;
}

// ---- the sequence and the rows of a tile -----------------------------------------------------------

// A tile of (token, head of the group) rows.
struct TileRows : Run {
    int pos0, len;  // position of the sequence's first new token, its cached length
};
template <int BM>
__device__ inline bool find_tile(const AttnArgs &a, int tile, TileRows &t) {
    if (!find_run<BM>(a.q_start, a.n_seqs, a.n_tokens, a.group, tile, t)) return false;
    const int kv = max(a.kv_len[t.b], 0);
    t.pos0 = kv - t.n;
    t.len = min(kv, a.pages.table_stride * static_cast<int>(a.pages.page_size.d));
    return true;
}

// Keys [lo, hi) of the row's token at position p (p < 0 where a sequence has more new tokens than positions: a window of up to
// INT_MAX is taken from 0 then, so that the difference fits).
__device__ inline int key_lo(const AttnArgs &a, int p) { return a.causal && a.window > 0 ? max(0, max(p + 1, 0) - a.window) : 0; }
__device__ inline int key_hi(const AttnArgs &a, int p, int len) { return a.causal ? min(p + 1, len) : len; }

// The factor that takes a score to a power of two's exponent is at least this: a masked score is minus infinity, and 0 times that is
// no number. (What it adds to an exponent is nothing for scores below 1e30.)
constexpr float kLeastScale = 1e-37f;

// A row's query as the operand of the score products: N chunks of 8 elements, at(i) the place of chunk i, in each of the lanes that hold
// the row (wide(x): the largest x over them). Returns the factor that takes a product to a power of two's exponent. fp32 rows
// against fp16 keys are scaled by a power of two, which that factor takes back, so that their largest element is below 2^15: at the upper
// end of fp16's range, because an element's second term is off by up to 2^-25 where it is subnormal, which is to be little for small
// elements beside a large one too: 2^-39 of the largest. (With the largest below 1, elements 1000 times smaller kept 15 bits.)
template <typename T, typename E, int QT, int N, typename At, typename Wide>
__device__ inline float load_query(const AttnArgs &a, const T *qp, vec<E, 8> (*q)[N], At at, Wide wide) {
    float c = a.scale;
    if constexpr (std::is_same_v<T, E>) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            q[0][i] = *reinterpret_cast<const vec<E, 8> *>(qp + at(i));
            if (a.sign < 0.0f) q[0][i] = -q[0][i];
        }
    } else {
        int ex = 0;
        if constexpr (std::is_same_v<E, f16>) {
            float mx = 0.0f;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                float x[8];
                load_as_float<T, 8>(qp + at(i), x);
#pragma unroll
                for (int e = 0; e < 8; ++e) mx = fmaxf(mx, fabsf(x[e]));
            }
            mx = wide(mx);
            if (mx > 0.0f && mx < INFINITY) (void)frexpf(mx, &ex), ex -= 15;
            c = fmaxf(ldexpf(c, ex), kLeastScale);
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float x[8];
            load_as_float<T, 8>(qp + at(i), x);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = ldexpf(x[e], -ex) * a.sign;
            vec<E, 8> terms[QT];
            split<E, QT>(x, terms);
#pragma unroll
            for (int n = 0; n < QT; ++n) q[n][i] = terms[n];
        }
    }
    return c;
}

// ---- a row by the formula ------------------------------------------------------------------------

// One row's keys [k0, k1) by one wave, in 64 bits, a key a lane for the scores and dimensions a lane for the values. The tiles take
// numbers: in their terms an infinity is itself, then a zero or an infinity of the other sign, and a weight that rounds to zero
// makes no number of an infinite value. So a row whose result there is not finite is done again here (nothing is
// added to the tiles' loops for it), and what a row gives does not depend on where tiles and parts end: a key of weight zero (a
// score of minus infinity) does not count whatever its value, a score of plus infinity or NaN makes the row NaN, an infinite value
// its dimension's sum. A row of NaN ends at its first 64 keys. Writes the row's output, or its part's sums.
template <typename T, typename C, int D>
__device__ inline void formula_row(const AttnArgs &a, int b, int row, int token0, int kvh, int k0, int k1) {
    constexpr int V = D / 64;
    const int lane = threadIdx.x & 63, token = token0 + row / a.group, head = kvh * a.group + row % a.group;
    const T *q = static_cast<const T *>(a.q) + token * a.q_stride + head * D;
    const Stored<C> *kc = static_cast<const Stored<C> *>(a.k) + kvh * a.pages.head_stride;
    const Stored<C> *vc = static_cast<const Stored<C> *>(a.v) + kvh * a.pages.head_stride + lane * V;
    const double c = static_cast<double>(a.scale) * a.sign;
    const auto offset = [&](int key, float2 &by) {
        const int page = key < k1 ? page_number(a.pages, b, key) : -1;
        const int64_t o = row_in_page(a.pages, page, key);
        by = make_float2(1.0f, 1.0f);
        if constexpr (kCodes<C>)
            if (o >= 0) by = row_scales(a, page, kvh, key);
        return o;
    };
    const auto score = [&](int64_t o, float by) {
        double s = 0.0;
#pragma unroll 1
        for (int d = 0; d < D; d += 8) {  // (unrolled, it would take more registers than the tiles)
            float x[8], y[8];
            load_as_float<T, 8>(q + d, x);
            load_stored<C, 8>(kc + max(o, int64_t{0}) + d, y);
#pragma unroll
            for (int e = 0; e < 8; ++e) s += static_cast<double>(x[e]) * (kCodes<C> ? static_cast<double>(y[e]) * by : static_cast<double>(y[e]));
        }
        return o < 0 ? static_cast<double>(-INFINITY) : s * c;
    };
    float2 by;
    double m = -INFINITY;
    bool number = true;
    for (int k = k0; k < k1 && number; k += 64) {
        const int64_t o = offset(k + lane, by);
        const double s = score(o, by.x);
        number = __ballot(!(s < INFINITY)) == 0;
        m = fmax(m, s);
    }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) m = fmax(m, __shfl_xor(m, d));
    double l = 0.0, acc[V] = {};
    for (int k = k0; k < k1 && number && m > -INFINITY; k += 64) {
        const int64_t o = offset(k + lane, by);
        const float w = exp2f(static_cast<float>(score(o, by.x) - m));
        l += w;
        for (int j = 0; j < min(64, k1 - k); ++j) {
            const float wj = __shfl(w, j);
            if (wj == 0.0f) continue;
            float x[V];
            load_stored<C, V>(vc + __shfl(static_cast<long long>(o), j), x);
            const double g = kCodes<C> ? static_cast<double>(wj) * __shfl(by.y, j) : static_cast<double>(wj);
#pragma unroll
            for (int i = 0; i < V; ++i) acc[i] += g * x[i];
        }
    }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) l += __shfl_xor(l, d);
    if (!number) l = NAN;
    float o[V];
    if (a.parts > 1) {
        const int64_t at = (static_cast<int64_t>(token) * a.n_heads + head) * a.parts + blockIdx.y;
        // (as everywhere, weights are 2^(score + bias): what the bias loses by its rounding goes into the sums, as far as fp32 holds it)
        const float bias = l > 0.0 ? static_cast<float>(fmin(fmax(-m, -FLT_MAX), FLT_MAX)) : 0.0f;
        const double g = l > 0.0 ? exp2(fmin(fmax(m + bias, -64.0), 64.0)) : 1.0;
        if (lane == 0) a.part_ml[at] = make_float2(bias, static_cast<float>(l * g));
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] = static_cast<float>(acc[i] * g);
        store_rounded<float, V>(a.part_o + at * D + lane * V, o);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] = l == 0.0 ? 0.0f : static_cast<float>(acc[i] / l);
        store_rounded<T, V>(static_cast<T *>(a.out) + token * a.out_stride + head * D + lane * V, o);
    }
}

// 0 where all numbers are finite, NaN where one is not.
template <int N>
__device__ inline float not_finite(const vec<float, N> &x, float z) {
#pragma unroll
    for (int i = 0; i < N; ++i) z = fmaf(x[i], 0.0f, z);
    return z;
}

// ---- tiles ----------------------------------------------------------------------------------------

constexpr int kFewRows = 16;
constexpr int kFewKeys = 32;   // per wave and step
constexpr int kFewStep = 4 * kFewKeys;
constexpr int kTileRows = 128;

// ---- the join of the parts ----------------------------------------------------------------------

// out = sum over parts of 2^(least bias - bias) o, over the same sum of l. A lane of each wave holds a part's bias and sum (64 at a
// time) and its factor. W waves share a token's head: with many parts (few rows) their outputs are dealt to four waves, whose
// loads do not wait for one another and which meet in LDS; with few parts (many rows) one wave takes them all. (One wave with
// a loop over the parts, a load at a time, took 0.4 us a part; four waves for two parts cost a 2048-token prompt 20 us.)
template <typename T, int D, int W>
__global__ __launch_bounds__(256) void attn_join(AttnArgs a) {
    constexpr int V = D / 64;
    __shared__ float meet[W][64][V];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) % W;
    const int row = blockIdx.x * (4 / W) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) / W;
    const int token = row / a.n_heads, head = row - token * a.n_heads;
    if (token >= a.n_tokens) return;
    const int64_t at = (static_cast<int64_t>(token) * a.n_heads + head) * a.parts;
    int b, pos;
    if (!find_token(a.q_start, a.kv_len, a.n_seqs, token, b, pos)) return;
    const int len = min(max(a.kv_len[b], 0), a.pages.table_stride * static_cast<int>(a.pages.page_size.d));
    const int lo = key_lo(a, pos), hi = key_hi(a, pos, len);
    const int z0 = min(lo / a.span, a.parts - 1), z1 = hi > lo ? min((hi - 1) / a.span + 1, a.parts) : z0;
    float acc[V] = {}, l = 0.0f, bias = INFINITY;  // of the parts so far: their least bias
    for (int z = z0; z < z1; z += 64) {
        const float2 ml = z + lane < z1 ? a.part_ml[at + z + lane] : make_float2(INFINITY, 0.0f);
        const float mine = ml.y != 0.0f ? ml.x : INFINITY;
        const float least = fminf(bias, -xor_max_wave(-mine));
        const float f = ml.y != 0.0f ? exp2f(least - mine) : 0.0f;
        const float old = bias == INFINITY ? 0.0f : exp2f(least - bias);
        bias = least;
        l = l * old + sum_wave(ml.y * f);
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] *= old;
        const int n = min(64, z1 - z);
        for (int j = wave; j < n; j += 4 * W) {  // four parts' loads at a time
            float o[4][V];
#pragma unroll
            for (int y = 0; y < 4; ++y)
                load_as_float<float, V>(a.part_o + (at + z + min(j + y * W, n - 1)) * D + lane * V, o[y]);
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                const float fj = j + y * W < n ? __shfl(f, min(j + y * W, n - 1)) : 0.0f;
#pragma unroll
                for (int i = 0; i < V; ++i) acc[i] += fj != 0.0f ? o[y][i] * fj : 0.0f;
            }
        }
    }
    if constexpr (W > 1) {
#pragma unroll
        for (int i = 0; i < V; ++i) meet[wave][lane][i] = acc[i];
        __syncthreads();
        if (wave != 0) return;
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] = (meet[0][lane][i] + meet[1][lane][i]) + (meet[2][lane][i] + meet[3][lane][i]);
    }
    float o[V];
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = l == 0.0f ? 0.0f : acc[i] / l;
    store_rounded<T, V>(static_cast<T *>(a.out) + token * a.out_stride + head * D + lane * V, o);
}

// ---- host ----------------------------------------------------------------------------------------

// How the work is cut, from the host's numbers alone.
constexpr int64_t kMostPartBytes = int64_t{128} << 20;  // of attn_few's parts, where there are several
constexpr int kMaxParts = 512;  // (a short window in a long cache asks for many, most of them empty)

inline int64_t part_row_bytes(const tqhip_kv_cache &c) { return c.head_dim * sizeof(float) + sizeof(float2); }

struct Plan {
    bool few;
    int rows, tiles, parts, span;  // rows of a tile: 16 or (over codes of 8 bits) 32, or 128
};

inline Plan plan(const tqhip_attn &p, const tqhip_kv_cache &c, const tqhip_seqs &s, bool codes) {
    const int group = p.n_heads / c.n_kv_heads;
    const int64_t rows = static_cast<int64_t>(s.n_tokens) * group;
    Plan n{};
    // Tiles of 16 rows read the cache once for each; they win up to 32 rows a sequence (64 sequences of up to 4000 keys, 32 heads of
    // 128: 16 rows 140 us, against 182 with tiles of 128; 32 rows 195 and 189; 64 rows 294 and 223), and, whatever the rows, as long
    // as there are few of them in all, because there they come in shorter parts (one sequence of 64 rows on 8 K/V heads 22 us and 32,
    // 128 rows 34 and 34; 448 rows on 2 heads of 64 30 and 41, 1792 rows 79 and 47; 1024 on one of 256 52 and 81).
    // Codes of 8 bits win there for twice the rows, of a sequence (32 sequences of up to 9000 keys, 32 heads of 128 over 8: 45 rows of
    // bf16 154 us, against 180 with tiles of 128; 35 of fp32 170 and 237; but 87 of fp32 342 and 268), and for twice as many tiles in all.
    // There the two cross at 256 to 384 rows on each of 8 heads of 128 (over 4000 keys; 224 rows bf16 32 us and 32, fp32 37 and 41; 256 rows 32 and 33, 39
    // and 41; 384 rows 44 and 34, 53 and 43), past the rule on two of 64 (896 rows 23 and 28, 25 and 33; 1792 rows 29 and 33, 32 and 38; 3584 rows
    // 46 and 44, 52 and 52), and on one of 256 before it in bf16 and past it in fp32 (1200 rows 59 and 53, 50 and 79; 1792 rows 68 and 56, 59 and 81;
    // 2400 rows 75 and 58, 69 and 84).
    const int more = codes ? 2 : 1;
    n.few = rows <= int64_t{2 * more} * kFewRows * s.n_seqs || (rows + kFewRows - 1) / kFewRows * c.n_kv_heads <= 56 * more;
    // Over codes, 32 rows a tile where sequences have more than 16, so that their keys are read once: five tokens each of 32 sequences of
    // up to 9000 keys, 20 rows a head: 101 us, against 118 with tiles of 16. (Heads of 256 with fp32 terms do not fit the registers twice.)
    const bool pairs = codes && !(c.head_dim == 256 && p.dtype == TQHIP_F32);
    n.rows = !n.few ? kTileRows : pairs && rows > int64_t{kFewRows} * s.n_seqs ? 2 * kFewRows : kFewRows;
    n.tiles = static_cast<int>(rows / n.rows) + s.n_seqs;
    const int64_t most = static_cast<int64_t>(s.table_stride) * c.page_size;
    const int64_t kv = s.max_kv > 0 ? std::min<int64_t>(s.max_kv, most) : most;
    // keys that one tile reads
    const int64_t seen = p.causal && p.window > 0 ? std::min<int64_t>(kv, int64_t{p.window} + n.rows) : kv;
    const int64_t blocks = static_cast<int64_t>(n.tiles) * c.n_kv_heads, cus = device_cu_count();
    const auto up = [](int64_t x, int64_t to) { return (x + to - 1) / to * to; };
    if (n.few) {
        // A workgroup's start and end cost as much as some 500 keys, so parts are as long as two workgroups per CU make them, up to
        // 1024 keys, which evens out ragged lengths. One token of 32 heads over 30000 keys: 35 us in parts of 512, 61 of
        // 128; of 14 heads over 3000: 14 of 128, 31 of 1024; 64 sequences of up to 16000: 423 of 1024, 455 of 512, 428 of 4096; over codes of
        // 8 bits, half the bytes a key, 269 of 1024, 245 of 2048, 242 of 4096.
        const int64_t full = std::max<int64_t>(s.n_seqs, (rows + n.rows - 1) / n.rows) * c.n_kv_heads;  // tiles that there are
        n.span = static_cast<int>(std::clamp<int64_t>(up(seen * full / (2 * cus), kFewStep), kFewStep, codes ? 2048 : 1024));
        // Every row has room for every part up to the longest sequence's, and a workgroup too, most of them empty where one sequence of
        // many is long: parts grow with the rows. 256 tokens of 32 heads of 128, one over 131072 keys, the rest over 2000: 740 us
        // and 126 MB (64 MB at most: 711; 256: 887; parts of 1024: 1278 and 520 MB); 8 tokens each: 1369 (1845; 1172; 2587 and 4160 MB).
        const int64_t most_parts = std::max<int64_t>(1, kMostPartBytes / (rows * c.n_kv_heads * part_row_bytes(c)));
        if (kv > most_parts * n.span) n.span = static_cast<int>(up((kv + most_parts - 1) / most_parts, kFewStep));
    } else {
        // Two workgroups are resident per CU. With fewer tiles than 1.5 rounds of them, parts give three rounds, which evens out
        // ragged lengths too; of 512 keys at least, for a part's output is written and read again. Chunks of 257 over up
        // to 8000 (28 tiles of 8 heads): 206 us in parts of 1536, 243 of 4096, 334 whole; 512 over 16000: 302, 281, 612;
        // a prompt of 5000 of 14 heads (514 tiles of 2 heads): 130 whole, 159 of 4096.
        const int64_t slots = 2 * cus;
        const int64_t parts = 2 * blocks >= 3 * slots ? 1 : (3 * slots + blocks - 1) / blocks;
        n.span = static_cast<int>(parts == 1 ? kv : std::min(kv, std::max<int64_t>(512, up((seen + parts - 1) / parts, 64))));
    }
    if (kv > int64_t{kMaxParts} * n.span) n.span = static_cast<int>(up(kv, int64_t{kMaxParts} * 128) / kMaxParts);
    n.parts = static_cast<int>((kv + n.span - 1) / n.span);
    return n;
}

inline size_t plan_bytes(const Plan &n, const tqhip_attn &p, const tqhip_kv_cache &c, const tqhip_seqs &s) {
    if (n.parts == 1) return 0;
    return static_cast<size_t>(s.n_tokens) * p.n_heads * n.parts * part_row_bytes(c);
}
template <typename T, int D>
void launch_join(const AttnArgs &a, const Plan &n, hipStream_t s) {
    if (n.parts == 1) return;
    const int rows = a.n_tokens * a.n_heads;
    if (n.parts > 8 && rows <= INT32_MAX / 256)  // (a launch has less than 2^32 threads along x)
        attn_join<T, D, 4><<<rows, 256, 0, s>>>(a);
    else
        attn_join<T, D, 1><<<(rows + 3) / 4, 256, 0, s>>>(a);
}

// Checks of the queries and of alignments (cb: bytes of a cache element) beyond check_cache's.
inline int check_attn(const tqhip_attn &p, const tqhip_kv_cache &c, const tqhip_seqs &s, int cb) {
    if (!p.q || !p.out || !type_known(p.dtype) || p.n_heads < 1 || p.n_heads % c.n_kv_heads || p.window < 0 ||
        !std::isfinite(p.scale * 1.4426950408889634f))
        return kBadShape;
    if (c.head_dim != 64 && c.head_dim != 128 && c.head_dim != 256) return kBadShape;
    const int qb = type_bytes(p.dtype);
    int64_t page, token, head;
    (void)cache_strides(c, &page, &token, &head);
    const uintptr_t bases = reinterpret_cast<uintptr_t>(p.q) | reinterpret_cast<uintptr_t>(p.out) |
                            reinterpret_cast<uintptr_t>(c.k) | reinterpret_cast<uintptr_t>(c.v);
    if (bases % 16 || p.q_stride * qb % 16 || p.out_stride * qb % 16 || page * cb % 16 || token * cb % 16 || head * cb % 16)
        return kBadShape;
    const int64_t row = static_cast<int64_t>(p.n_heads) * c.head_dim;
    if (s.n_tokens > 1 && ((p.q_stride && p.q_stride < row) || (p.out_stride && p.out_stride < row))) return kBadShape;
    // workgroups along x, of 256 threads: a sixteenth of the rows and one a sequence and key/value head, then a quarter of the rows
    if (static_cast<int64_t>(s.n_tokens) * p.n_heads > INT32_MAX / 32 || static_cast<int64_t>(s.n_seqs) * p.n_heads > INT32_MAX / 256)
        return kTooLarge;
    return kOk;
}

// A checked call with the workspace that its plan needs: launch(arguments, plan).
template <typename Launch>
int run_attn(const tqhip_attn &p, const tqhip_kv_cache &c, const tqhip_seqs &b, const Plan &n, hipStream_t s, Launch launch) {
    int st = kOk;
    const size_t bytes = plan_bytes(n, p, c, b);
    void *ws = p.workspace;
    if (reinterpret_cast<uintptr_t>(ws) % 256) return kBadShape;
    if (ws && p.workspace_bytes < bytes) return kNoScratch;
    std::optional<ScratchCall> call;
    if (bytes && !ws) {
        call.emplace(s);
        if ((st = call->workspace(bytes, &ws)) != kOk) return st;
    }
    const int64_t row = static_cast<int64_t>(p.n_heads) * c.head_dim;
    const float c2 = std::max(std::fabs(p.scale) * 1.4426950408889634f, kLeastScale);
    const int64_t parts = static_cast<int64_t>(b.n_tokens) * p.n_heads * n.parts;
    float *po = static_cast<float *>(ws);
    const AttnArgs a{p.q, c.k, c.v, p.out, p.q_stride ? p.q_stride : row, p.out_stride ? p.out_stride : row, b.q_start,
                     b.kv_len, b.n_seqs, b.n_tokens, p.n_heads, p.n_heads / c.n_kv_heads, c2, p.scale < 0 ? -1.0f : 1.0f,
                     p.causal, p.window, n.parts, n.span, po, bytes ? reinterpret_cast<float2 *>(po + parts * c.head_dim) : nullptr,
                     make_pages(c, b)};
    launch(a, n);
    return hipGetLastError() == hipSuccess ? kOk : kLaunchFailed;
}

}  // namespace
}  // namespace tqhip
