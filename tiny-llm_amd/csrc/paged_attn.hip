// paged_attn.hip -- attention of the new tokens of a batch of sequences over their paged cache.
//
// For query head h of a token at position p, k and v of key/value head h / group:
//   out = sum_j w_j v_j / sum_j w_j,  w_j = 2^(c q.k_j + bias),  c = scale log2 e,
// over the positions j that p may attend to. `bias` is minus the row's largest c q.k_j so far, up to a headroom, so the keys are
// read once: when a larger score comes, the sums so far are multiplied by 2^(new bias - old bias). The keys of a row may be cut
// into parts, whose sums are joined the same way by a second launch.
//
// The rows of a tile are the tokens of one sequence times the query heads that share a key/value head, so its keys are read once
// for all of them. Both products run on the matrix cores, transposed: S^T = K Q^T puts the scores of a row into the lanes
// that hold that row, so maximum and sum are formed within two or four lanes, and the weights are where the second
// product, V^T W^T, wants them. V's columns come from LDS through transposing reads. 16-bit operands go in as they are; fp32
// ones as two or three 16-bit terms (see Terms), which keeps 22 to 24 bits at 2 to 6 matrix instructions a product.
//
// Two kernels: attn_few (tiles of 16 rows, up to 32 rows a sequence or few in all) is bound by reading the cache, attn_tiles (128
// rows) by the products and what surrounds them. One workgroup in eight goes to each XCD, in turn, and its number mod the
// key/value heads is its head: with 8 of them an XCD reads one head's keys and keeps them in its L2.
// (Every XCD taking all heads: 878 us instead of 789 for the prompts below.)
//   64 tokens of 32 heads on 8 of 128, up to 16000 fp16 keys each (2.06 GB):        395 us, 5.2 TB/s
//   two prompts of up to 8192, the same heads, all in bf16 (706 GFLOP):             735 to 807 us, 0.87 to 0.96 PFLOP/s
//   four chunks of up to 257 fp32 tokens over up to 8000 fp16 keys, the same heads:  191 to 206 us (72 GFLOP of two terms each), 17 of them the join
//   three prompts of up to 5001 fp32 tokens, a window of 1000 bf16 keys, 14 heads on 2 of 64: 130 to 138 us (33.5 GFLOP of three terms each)
//   one fp32 token of 14 heads on 2 of 64 over 3000 fp32 keys:                        9.5 us and 4.0 for the join
// (from card to card; one of them took 880, 217 and 144 us for the three that the products bound)
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
};

// ---- numbers as terms of 16 bits ----------------------------------------------------------------

// How a product's operands are held: E the type of the matrix instruction, QT terms of a query element
// or a weight, KT of a cache element. 16-bit activations meet a cache of their own type as they are.
// fp32 activations keep their precision: against an fp16 cache two fp16 terms (22 bits), against
// a bf16 one three bf16 terms (24 bits), and an fp32 cache is three bf16 terms itself.
// (One term rounds the weights too, once more than the result: bf16 prompts are 2.1e-3 from 64 bits, where the result's
// rounding alone is 1.6e-3. A second term would be half as many products again, for bits that the result does not keep.)
template <typename T, typename C>
struct Terms {
    using E = std::conditional_t<std::is_same_v<C, f16>, f16, bf16>;
    static constexpr int KT = std::is_same_v<C, float> ? 3 : 1;
    static constexpr int QT = std::is_same_v<T, C> && !std::is_same_v<C, float> ? 1 : std::is_same_v<C, f16> ? 2 : 3;
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

// A row's query as the operand of the score products: N chunks of 8 elements, STEP apart, in each of the lanes that hold the
// row (wide(x): the largest x over them). Returns the factor that takes a product to a power of two's exponent. fp32 rows
// against fp16 keys are scaled by a power of two, which that factor takes back, so that their largest element is below 2^15: at the upper
// end of fp16's range, because an element's second term is off by up to 2^-25 where it is subnormal, which is to be little for small
// elements beside a large one too: 2^-39 of the largest. (With the largest below 1, elements 1000 times smaller kept 15 bits.)
template <typename T, typename E, int QT, int N, int STEP, typename Wide>
__device__ inline float load_query(const AttnArgs &a, const T *qp, vec<E, 8> (*q)[N], Wide wide) {
    float c = a.scale;
    if constexpr (QT == 1) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            q[0][i] = *reinterpret_cast<const vec<E, 8> *>(qp + STEP * i);
            if (a.sign < 0.0f) q[0][i] = -q[0][i];
        }
    } else {
        int ex = 0;
        if constexpr (std::is_same_v<E, f16>) {
            float mx = 0.0f;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                float x[8];
                load_as_float<T, 8>(qp + STEP * i, x);
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
            load_as_float<T, 8>(qp + STEP * i, x);
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
    const C *kc = static_cast<const C *>(a.k) + kvh * a.pages.head_stride;
    const C *vc = static_cast<const C *>(a.v) + kvh * a.pages.head_stride + lane * V;
    const double c = static_cast<double>(a.scale) * a.sign;
    const auto offset = [&](int key) { return key < k1 ? row_offset(a.pages, b, key) : int64_t{-1}; };
    const auto score = [&](int64_t o) {
        double s = 0.0;
#pragma unroll 1
        for (int d = 0; d < D; d += 8) {  // (unrolled, it would take more registers than the tiles)
            float x[8], y[8];
            load_as_float<T, 8>(q + d, x);
            load_as_float<C, 8>(kc + max(o, int64_t{0}) + d, y);
#pragma unroll
            for (int e = 0; e < 8; ++e) s += static_cast<double>(x[e]) * y[e];
        }
        return o < 0 ? static_cast<double>(-INFINITY) : s * c;
    };
    double m = -INFINITY;
    bool number = true;
    for (int k = k0; k < k1 && number; k += 64) {
        const double s = score(offset(k + lane));
        number = __ballot(!(s < INFINITY)) == 0;
        m = fmax(m, s);
    }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) m = fmax(m, __shfl_xor(m, d));
    double l = 0.0, acc[V] = {};
    for (int k = k0; k < k1 && number && m > -INFINITY; k += 64) {
        const int64_t o = offset(k + lane);
        const float w = exp2f(static_cast<float>(score(o) - m));
        l += w;
        for (int j = 0; j < min(64, k1 - k); ++j) {
            const float wj = __shfl(w, j);
            if (wj == 0.0f) continue;
            float x[V];
            load_as_float<C, V>(vc + __shfl(static_cast<long long>(o), j), x);
#pragma unroll
            for (int i = 0; i < V; ++i) acc[i] += static_cast<double>(wj) * x[i];
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

// ---- few rows: tiles of 16 rows ------------------------------------------------------------------

// A tile's keys are dealt to the four waves 32 at a time; each wave keeps a softmax of its own, and the four meet at the end, so no
// wave waits for another. K goes from the cache straight into operand registers, V into LDS of the wave's own, whose
// transposing reads turn its rows into columns. Reading the cache is the work (a query row takes 2 to 4 flops a byte), so the loads of
// the next step are issued as soon as this step's have arrived, before anything is computed on them.
constexpr int kFewRows = 16;
constexpr int kFewKeys = 32;   // per wave and step
constexpr int kFewStep = 4 * kFewKeys;

template <typename T, typename C, int D>
__global__ __launch_bounds__(256, (D == 256 || (D == 128 && sizeof(C) == 4) ? 1 : 2)) void attn_few(AttnArgs a) {
    using Tm = Terms<T, C>;
    using E = typename Tm::E;
    constexpr int QT = Tm::QT, KT = Tm::KT;
    // V of a step: as it is in two buffers (chunks of 16 bytes permuted as in attn_tiles) when the cache holds the instruction's
    // type; else one of its terms after the other in one buffer.
    constexpr bool kDirect = KT == 1;
    constexpr int VS = kDirect ? D : D + 16, ND = D / 16, NS = D / 32, CH = D / 8, NV = kFewKeys * CH / 64;
    __shared__ struct {
        union {
            __attribute__((aligned(16))) E v[4][kDirect ? 2 : 1][kFewKeys][VS];
            float o[4][kFewRows][D];
        };
        float meet[2][4][kFewRows];
    } sh;

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, col = lane & 15;
    const int kv_heads = a.n_heads / a.group;
    const int kvh = blockIdx.x % kv_heads;
    TileRows t;
    if (!find_tile<kFewRows>(a, blockIdx.x / kv_heads, t)) return;
    const int rows = t.n * a.group;
    const int last = min(t.r0 + kFewRows, rows) - 1;
    const int p_first = t.pos0 + t.r0 / a.group, p_last = t.pos0 + last / a.group;
    int ke = key_hi(a, p_last, t.len), kb = max(min(key_lo(a, p_first), ke), 0);  // (a window past the table is empty)
    if (a.parts > 1) {
        kb = max(kb, static_cast<int>(blockIdx.y) * a.span);
        if (static_cast<int>(blockIdx.y) < a.parts - 1) ke = min(ke, (static_cast<int>(blockIdx.y) + 1) * a.span);
        if (kb >= ke) return;
    }
    const int full_lo = key_lo(a, p_last), full_hi = key_hi(a, p_first, t.len);
    const int r = min(t.r0 + col, rows - 1);
    const int token = t.first + r / a.group, head = kvh * a.group + r % a.group;
    const int pos = t.pos0 + r / a.group;
    const int lo = key_lo(a, pos), hi = key_hi(a, pos, t.len);

    const C *kc = static_cast<const C *>(a.k) + kvh * a.pages.head_stride + 8 * g;
    const C *vc = static_cast<const C *>(a.v) + kvh * a.pages.head_stride + 8 * g;
    const auto swap = [](int row) { return (D == 64 ? row >> 1 & 3 : row & 7) << 1; };  // of a value row's chunks
    vec<C, 8> kr[2][2][NS], vr[kDirect ? 1 : 2][NS];
    // The lane's keys of a step are k0 + col and k0 + 16 + col. All loads of the loop are unconditional (a page past the table is its
    // last entry, a row that does not exist is row 0 of page 0): the compiler counts the loads that may stay under way at
    // a wait, and a load under a branch counts as none, so every wait would be for all of them.
    const auto pages_of = [&](int k0, int *page) {
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
            const int i = min(a.pages.page_size.quot(k0 + 16 * kt + col), a.pages.table_stride - 1);
            page[kt] = a.pages.table[static_cast<int64_t>(t.b) * a.pages.table_stride + i];
        }
    };
    const auto offsets = [&](int k0, const int *page, int64_t *o) {
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
            const int key = k0 + 16 * kt + col;
            o[kt] = key < ke ? row_in_page(a.pages, page[kt], key) : -1;
        }
    };
    const auto load_rows = [&](const C *base, const int64_t *o, vec<C, 8> (*x)[NS]) {
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
            const C *row = base + max(o[kt], int64_t{0});
#pragma unroll
            for (int i = 0; i < NS; ++i) x[kt][i] = *reinterpret_cast<const vec<C, 8> *>(row + 32 * i);
        }
    };

    const auto load_values = [&](const int64_t *o, E *__restrict__ to) __attribute__((always_inline)) {
        if constexpr (kDirect) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {  // 64 chunks in order; the row's offset is held by lane `row % 16`
                const int first = 64 * i / CH, row = first + lane / CH;
                const int64_t ro = __shfl(static_cast<long long>(max(o[first / 16], int64_t{0})), row & 15);
                // (streamed: a decode step of 64 requests takes 397 us so, 420 without. K's lines are read in two halves, which
                // streaming fetches twice: 451 us.)
                global_to_lds<true>(vc - 8 * g + ro + ((lane % CH) ^ swap(row)) * 8, to + 64 * i * 8);
            }
        } else {
            load_rows(vc, o, vr);
        }
    };

    int64_t off[2];
    int next[2];
    int k0 = kb + wave * kFewKeys;
    pages_of(k0, next);
    offsets(k0, next, off);
    pages_of(k0 + kFewStep, next);
    load_rows(kc, off, kr[0]);
    load_values(off, &sh.v[wave][0][0][0]);
    vec<E, 8> q[QT][NS];
    const float c = load_query<T, E, QT, NS, 32>(a, static_cast<const T *>(a.q) + token * a.q_stride + head * D + 8 * g, q,
                                                 [&](float x) {
                                                     x = fmaxf(x, lane_xor<16>(x, lane));
                                                     return fmaxf(x, lane_xor<32>(x, lane));
                                                 });
    f32x4 acc[ND];
#pragma unroll
    for (int i = 0; i < ND; ++i) acc[i] = f32x4{};
    float m = -INFINITY, bias = 0.0f, l = 0.0f;

    // (The restrict pointers tell the compiler that the next step's transfers do not touch the values that are read meanwhile.)
    const auto step = [&](const vec<C, 8> (*k_now)[NS], vec<C, 8> (*k_next)[NS], const E *__restrict__ v_now, E *__restrict__ v_next)
                          __attribute__((always_inline)) {
        const unsigned exist = static_cast<unsigned>(__ballot(off[0] >= 0) & 0xffff) |
                               static_cast<unsigned>(__ballot(off[1] >= 0) & 0xffff) << 16;
        const bool partial = k0 < full_lo || k0 + kFewKeys > full_hi || exist != ~0u;
        wait_loads();
        offsets(k0 + kFewStep, next, off);
        pages_of(k0 + 2 * kFewStep, next);
        load_rows(kc, off, k_next);
        if constexpr (kDirect) load_values(off, v_next);
        // S^T: the lane holds its row's scores of keys 16 kt + 4 g + i
        f32x4 s[2];
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
            s[kt] = f32x4{};
#pragma unroll
            for (int i = 0; i < NS; ++i) {
                vec<E, 8> kf[KT];
                as_terms<C, E, KT>(k_now[kt][i], kf);
#pragma unroll
                for (int kj = 0; kj < KT; ++kj)
#pragma unroll
                    for (int qi = 0; qi < QT; ++qi)
                        if (qi + kj < Tm::kMost) s[kt] = mfma16(kf[kj], q[qi][i], s[kt]);
            }
        }
        if (partial) {
            const int k1 = k0 + 4 * g;
            const unsigned may = (exist >> (4 * g)) & below(hi - k1) & ~below(lo - k1);
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (!(may & (1u << (16 * kt + i)))) s[kt][i] = -INFINITY;
        }
        float mx = m;
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[kt][i]);
        mx = fmaxf(mx, lane_xor<16>(mx, lane));
        mx = fmaxf(mx, lane_xor<32>(mx, lane));
        if (__ballot((mx - m) * c > kHeadroom<QT>)) {
            const float nb = mx == -INFINITY ? 0.0f : fmaf(-mx, c, kWeightShift<E, QT>);
            const float f = m == -INFINITY ? 0.0f : exp2f(nb - bias);
            m = mx;
            bias = nb;
            l *= f;
#pragma unroll
            for (int i = 0; i < ND; ++i) acc[i] *= f;
        }
        float w[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            w[e] = __builtin_amdgcn_exp2f(fmaf(s[e / 4][e % 4], c, bias));
            l += w[e];
        }
        vec<E, 8> p[QT];
        split<E, QT>(w, p);
        if (partial) {  // infinite and NaN values as in attn_tiles
            unsigned wild = 0;
            if constexpr (kDirect) {
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    vec<C, 8> *at = reinterpret_cast<vec<C, 8> *>(const_cast<E *>(v_now)) + 64 * i + lane;
                    vec<C, 8> x = *at;
                    const bool finite = make_finite<C>(x);
                    if (!finite) *at = x;
                    unsigned long long bad = __ballot(!finite);  // by chunk: CH of them a row
                    for (int row = 64 * i / CH; bad; ++row, bad >>= CH)
                        if (bad & ((1ull << CH) - 1)) wild |= 1u << row;
                }
                wave_lds_order();
            } else {
#pragma unroll
                for (int kt = 0; kt < 2; ++kt) {
                    bool finite = true;
#pragma unroll
                    for (int i = 0; i < NS; ++i) finite = make_finite<C>(vr[kt][i]) && finite;
                    const unsigned long long bad = __ballot(!finite);
                    wild |= static_cast<unsigned>((bad | bad >> 16 | bad >> 32 | bad >> 48) & 0xffff) << (16 * kt);
                }
            }
            if (wild & exist & below(hi - k0) & ~below(lo - k0)) l = NAN;  // (formula_row takes the row)
        }
#pragma unroll
        for (int kj = 0; kj < KT; ++kj) {
            if constexpr (!kDirect) {
#pragma unroll
                for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                    for (int i = 0; i < NS; ++i) {
                        vec<E, 8> vf[KT];
                        as_terms<C, E, KT>(vr[kt][i], vf);
                        *reinterpret_cast<vec<E, 8> *>(&sh.v[wave][0][16 * kt + col][32 * i + 8 * g]) = vf[kj];
                    }
                wave_lds_order();
                if (kj == KT - 1) load_values(off, v_next);
            }
#pragma unroll
            for (int d = 0; d < ND; ++d) {
                const int i = lane & 15, row = 4 * g + i / 4;
                const int ch = (2 * d + (i & 3) / 2) ^ (kDirect ? swap(row) : 0);
                const E *v0 = (kDirect ? v_now : &sh.v[wave][0][0][0]) + row * VS + ch * 8 + 4 * (i & 1);
                const vec<E, 4> a0 = lds_columns(v0), a1 = lds_columns(v0 + 16 * VS);
                const vec<E, 8> vf = __builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
                for (int qi = 0; qi < QT; ++qi)
                    if (qi + kj < Tm::kMost) acc[d] = mfma16(vf, p[qi], acc[d]);
            }
            if constexpr (!kDirect) wave_lds_order();
        }
        k0 += kFewStep;
    };
    E *v0 = &sh.v[wave][0][0][0], *v1 = &sh.v[wave][kDirect ? 1 : 0][0][0];
    while (k0 < ke) {
        step(kr[0], kr[1], v0, v1);
        if (k0 >= ke) break;
        step(kr[1], kr[0], v1, v0);
    }
    wait_loads();  // (the loads past the last step: into LDS that is used for other things below)
    l += lane_xor<16>(l, lane);
    l += lane_xor<32>(l, lane);
    l = checked_sum<E>(bias, l);
    // the four waves' sums, brought to the least exponent bias among those that have any
    if (g == 0) {
        sh.meet[0][wave][col] = bias;
        sh.meet[1][wave][col] = l;
    }
    __syncthreads();  // (and every wave is done with V)
    float least = INFINITY, total = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w)
        if (sh.meet[1][w][col] != 0.0f) least = fminf(least, sh.meet[0][w][col]);
#pragma unroll
    for (int w = 0; w < 4; ++w)
        if (sh.meet[1][w][col] != 0.0f) total += sh.meet[1][w][col] * exp2f(least - sh.meet[0][w][col]);
    const float f = l != 0.0f ? exp2f(least - bias) : 0.0f;
    if (l != 0.0f) {
#pragma unroll
        for (int d = 0; d < ND; ++d) acc[d] *= f;
    }
#pragma unroll
    for (int d = 0; d < ND; ++d) *reinterpret_cast<f32x4 *>(&sh.o[wave][col][16 * d + 4 * g]) = acc[d];
    __syncthreads();
    // thread: row tid / 16, every 16th group of four dimensions
    const int row = tid >> 4;
    const int r2 = t.r0 + row, token2 = t.first + r2 / a.group, head2 = kvh * a.group + r2 % a.group;
    const float total2 = __shfl(total, row), least2 = __shfl(least, row);
    f32x4 o[D / 64];
    float z = total2 * 0.0f;
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
        const int d = 4 * (tid & 15) + 64 * i;
        o[i] = *reinterpret_cast<f32x4 *>(&sh.o[0][row][d]);
#pragma unroll
        for (int w = 1; w < 4; ++w) o[i] += *reinterpret_cast<f32x4 *>(&sh.o[w][row][d]);
        z = not_finite<4>(o[i], z);
    }
    const unsigned long long odd = __ballot(r2 < rows && z != 0.0f);  // 16 lanes a row
    if (r2 < rows && !(odd >> (lane & 48) & 0xffff)) {
        const int64_t at = (static_cast<int64_t>(token2) * a.n_heads + head2) * a.parts + blockIdx.y;
        if (a.parts > 1 && (tid & 15) == 0) a.part_ml[at] = make_float2(least2, total2);
        const float inv = total2 == 0.0f ? 0.0f : 1.0f / total2;
#pragma unroll
        for (int i = 0; i < D / 64; ++i) {
            const int d = 4 * (tid & 15) + 64 * i;
            if (a.parts > 1) {
                *reinterpret_cast<f32x4 *>(a.part_o + at * D + d) = o[i];
            } else {
                float x[4] = {o[i][0] * inv, o[i][1] * inv, o[i][2] * inv, o[i][3] * inv};
                store_rounded<T, 4>(static_cast<T *>(a.out) + token2 * a.out_stride + head2 * D + d, x);
            }
        }
    }
    if (__builtin_expect(odd == 0, 1)) return;
#pragma unroll 1
    for (int i = 0; i < 4; ++i)
        if (odd >> (16 * i) & 0xffff) {
            const int ro = t.r0 + 4 * wave + i, p = t.pos0 + ro / a.group;
            formula_row<T, C, D>(a, t.b, ro, t.first, kvh, max(kb, key_lo(a, p)), min(ke, key_hi(a, p, t.len)));
        }
}

// ---- many rows: tiles of 128 rows ---------------------------------------------------------------

// A wave takes 32 of the rows, all four the same keys: 64 at a time (32 where registers are short), K and V in LDS, the next tile's
// on the way there while this one's are used. Two workgroups a CU, so a wave that waits for LDS or for its workgroup leaves
// the SIMD to one of the other's. Of the time of the bf16 prompts at the top the matrix cores are busy 42 %, the vector
// units 42 %, LDS 24 %; of 789 us, without the exponentials they would take 760, without the next tile's loads 670, without the second
// product's instructions 694, and the loads and barriers alone 451: it is no single unit but the waits between them.
template <typename T, typename C, int D>
struct TileShape {
    using Tm = Terms<T, C>;
    static constexpr int BN = (D == 256 && Tm::QT > 1) || (D == 128 && Tm::QT == 3 && Tm::KT == 1) ? 32 : 64;
    static constexpr int kWavesPerSimd = D == 256 || (D == 128 && Tm::KT == 3) ? 1 : 2;
};

constexpr int kTileRows = 128;

template <typename T, typename C, int D>
__global__ __launch_bounds__(256, (TileShape<T, C, D>::kWavesPerSimd)) void attn_tiles(AttnArgs a) {
    using Tm = Terms<T, C>;
    using E = typename Tm::E;
    constexpr int QT = Tm::QT, KT = Tm::KT, BN = TileShape<T, C, D>::BN;
    constexpr int NCH = BN * (D / 8) / 256;  // chunks of 8 elements per thread
    constexpr int NK = BN / 32, ND = D / 32, CH = D / 8, kTiles = 256 / BN;
    // The tile's rows as they are, two buffers, when the cache holds the instruction's type; else one buffer of terms. A row's chunks
    // of 16 bytes are permuted by an exclusive or (key_swap, value_swap) so that the reads below meet every bank once.
    constexpr bool kDirect = KT == 1;
    constexpr int kPlanes = kDirect ? 2 : KT;
    // (One object: with several, the compiler holds the transfers to one of them against the reads of the others, and waits for the
    // next tile before it reads this one. What has to be waited for is waited for below.)
    __shared__ struct {
        __attribute__((aligned(16))) E k[kPlanes][BN][D];
        __attribute__((aligned(16))) E v[kPlanes][BN][D];
        int64_t offs[2][256];           // element offsets of the rows of 256 keys, several tiles, and of the next 256
        unsigned long long here[2][4];  // which of those keys exist
        unsigned long long wild[2];     // keys of a partly masked tile whose values are not all finite
    } sh;

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5, col = lane & 31;
    const int kv_heads = a.n_heads / a.group;
    const int kvh = blockIdx.x % kv_heads;
    const int tile = gridDim.x / kv_heads - 1 - static_cast<int>(blockIdx.x) / kv_heads;  // the longest first
    TileRows t;
    if (!find_tile<kTileRows>(a, tile, t)) return;
    const int rows = t.n * a.group;
    const int last = min(t.r0 + kTileRows, rows) - 1;
    const int p_first = t.pos0 + t.r0 / a.group, p_last = t.pos0 + last / a.group;
    int ke = key_hi(a, p_last, t.len), kb = max(min(key_lo(a, p_first), ke), 0);  // (a window past the table is empty)
    if (a.parts > 1) {
        kb = max(kb, static_cast<int>(blockIdx.y) * a.span);
        if (static_cast<int>(blockIdx.y) < a.parts - 1) ke = min(ke, (static_cast<int>(blockIdx.y) + 1) * a.span);
        // (a row without keys gets its zeros from the join; the first part writes nothing for it)
        if (kb >= ke) return;
    }
    // keys that every row may attend to
    const int full_lo = key_lo(a, p_last), full_hi = key_hi(a, p_first, t.len);

    // this lane's row
    const int wr0 = t.r0 + wave * 32;
    const int r = min(wr0 + col, rows - 1);
    const int token = t.first + r / a.group, head = kvh * a.group + r % a.group;
    const int pos = t.pos0 + r / a.group;
    const int lo = key_lo(a, pos), hi = key_hi(a, pos, t.len);
    const bool wave_live = wr0 < rows;
    const int wp_first = t.pos0 + min(wr0, rows - 1) / a.group, wp_last = t.pos0 + min(wr0 + 31, rows - 1) / a.group;
    const int w_lo = key_lo(a, wp_first), w_hi = key_hi(a, wp_last, t.len);

    vec<E, 8> q[QT][D / 16];
    const float c = load_query<T, E, QT, D / 16, 16>(a, static_cast<const T *>(a.q) + token * a.q_stride + head * D + 8 * h, q,
                                                     [&](float x) { return fmaxf(x, lane_xor<32>(x, lane)); });
    const C *kc = static_cast<const C *>(a.k) + kvh * a.pages.head_stride;
    const C *vc = static_cast<const C *>(a.v) + kvh * a.pages.head_stride;
    const auto key_swap = [](int row) { return (D == 64 ? row >> 1 : row) & (D == 64 ? 7 : 15); };
    const auto value_swap = [](int row) { return (row & 3) << (D == 64 ? 1 : 2); };
    vec<C, 8> kr[kDirect ? 1 : NCH], vr[kDirect ? 1 : NCH];
    // A tile's rows on their way: straight into LDS, 64 chunks in order per instruction, the lane choosing the global chunk that belongs
    // at its place, or into registers. For a key that does not exist row 0 of page 0 is loaded.
    const auto load_tile = [&](int n, E *__restrict__ k_to, E *__restrict__ v_to) __attribute__((always_inline)) {
        const int64_t *from = sh.offs[n / kTiles & 1] + n % kTiles * BN;
        int64_t o[NCH];
#pragma unroll
        for (int i = 0; i < NCH; ++i) o[i] = from[(tid + 256 * i) / CH];
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            const int ch = tid + 256 * i, row = ch / CH, at = ch % CH;
            if constexpr (kDirect) {
                const int first = (wave * 64 + 256 * i) * 8;  // element of the wave's first chunk
                global_to_lds<false>(kc + o[i] + (at ^ key_swap(row)) * 8, k_to + first);
                global_to_lds<false>(vc + o[i] + (at ^ value_swap(row)) * 8, v_to + first);
            } else {
                kr[i] = *reinterpret_cast<const vec<C, 8> *>(kc + o[i] + at * 8);
                vr[i] = *reinterpret_cast<const vec<C, 8> *>(vc + o[i] + at * 8);
            }
        }
    };
    // 256 keys' pages are looked up while the tiles of the 256 before run, and their offsets put into LDS before the last of those.
    const auto key_page = [&](int n) {
        const int key = kb + n * 256 + tid;
        return key < ke ? page_number(a.pages, t.b, key) : -1;
    };
    const auto put_offsets = [&](int n, int page) {
        const int64_t o = row_in_page(a.pages, page, kb + n * 256 + tid);
        const unsigned long long m = __ballot(o >= 0);
        sh.offs[n & 1][tid] = max(o, int64_t{0});
        if (lane == 0) sh.here[n & 1][wave] = m;
    };

    f32x16 acc[ND];
#pragma unroll
    for (int i = 0; i < ND; ++i) acc[i] = f32x16{};
    float m = -INFINITY, bias = 0.0f, l = 0.0f;

    put_offsets(0, key_page(0));
    if (tid < 2) sh.wild[tid] = 0;
    __syncthreads();
    if (kb < ke) load_tile(0, &sh.k[0][0][0], &sh.v[0][0][0]);
    int next_page = key_page(1);
    // (The restrict pointers tell the compiler that the next tile's transfers do not touch the values that are read meanwhile.)
    const auto step = [&](int n, int k0, bool partial, unsigned long long exist, const E *__restrict__ v_now, E *__restrict__ k_next,
                          E *__restrict__ v_next) __attribute__((always_inline)) {
        const int buf = n & 1;
        if (k0 + BN < ke) load_tile(n + 1, k_next, v_next);
        if (!wave_live || k0 >= w_hi || k0 + BN <= w_lo) return;

        // 32 keys at a time: the score products of the next 32 run on the matrix cores while the vector units form the weights of
        // these. S^T, keys down, queries across: the lane holds its query's keys (i % 4) + 8 (i / 4) + 4 h.
        const auto scores = [&](int kt) {
            f32x16 s{};
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
#pragma unroll
                for (int kj = 0; kj < KT; ++kj) {
                    const vec<E, 8> kf = *reinterpret_cast<const vec<E, 8> *>(
                        &sh.k[kDirect ? buf : kj][32 * kt + col][((2 * i + h) ^ key_swap(col)) * 8]);
#pragma unroll
                    for (int qi = 0; qi < QT; ++qi)
                        if (qi + kj < Tm::kMost) s = mfma32(kf, q[qi][i], s);
                }
            }
            return s;
        };
        f32x16 s = scores(0), ahead{};
#pragma unroll
        for (int kt = 0; kt < NK; ++kt) {
            const int k1 = k0 + 32 * kt;
            const unsigned exists = static_cast<unsigned>(exist >> (32 * kt));
            if (partial) {
                // which of the lane's keys its row may attend to: bit (i % 4) + 8 (i / 4) for register i
                const unsigned may = (exists >> (4 * h)) & below(hi - k1 - 4 * h) & ~below(lo - k1 - 4 * h);
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (!(may & (1u << ((i & 3) + 8 * (i >> 2))))) s[i] = -INFINITY;
            }
            float mx = m;
#pragma unroll
            for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[i]);
            mx = fmaxf(mx, lane_xor<32>(mx, lane));
            if (__ballot((mx - m) * c > kHeadroom<QT>)) {
                const float nb = mx == -INFINITY ? 0.0f : fmaf(-mx, c, kWeightShift<E, QT>);
                const float f = m == -INFINITY ? 0.0f : exp2f(nb - bias);
                m = mx;
                bias = nb;
                l *= f;
#pragma unroll
                for (int i = 0; i < ND; ++i) acc[i] *= f;
            }
            if (kt + 1 < NK) ahead = scores(kt + 1);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], c, bias));
                if (QT > 1) l += s[i];
            }
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                float x[8];
                vec<E, 8> p[QT];
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = s[8 * half + e];
                split<E, QT>(x, p);
                if (QT == 1) l = add_all(p[0], l);  // (what the products sum, so the rounding of the weights cancels in part)
#pragma unroll
                for (int d = 0; d < ND; ++d) {
#pragma unroll
                    for (int kj = 0; kj < KT; ++kj) {
                        const int i = lane & 15, row = 32 * kt + 16 * half + 4 * h + i / 4;
                        const int ch = (4 * d + (lane & 16) / 8 + (i & 3) / 2) ^ value_swap(i / 4);
                        const E *v0 = v_now + kj * BN * D + row * D + ch * 8 + 4 * (i & 1);
                        const vec<E, 4> a0 = lds_columns(v0), a1 = lds_columns(v0 + 8 * D);
                        const vec<E, 8> vf = __builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
                        for (int qi = 0; qi < QT; ++qi)
                            if (qi + kj < Tm::kMost) acc[d] = mfma32(vf, p[qi], acc[d]);
                    }
                }
            }
            s = ahead;
        }
        for (unsigned long long w = partial ? sh.wild[buf] & exist : 0; w; w &= w - 1) {
            const int key = k0 + __builtin_ctzll(w);
            if (key >= lo && key < hi) l = NAN;  // (formula_row takes the row)
        }
    };
    for (int n = 0, k0 = kb; k0 < ke; k0 += BN, ++n) {
        const int buf = n & 1;
        const unsigned long long all = BN == 64 ? ~0ull : 0xffffffffull;
        const unsigned long long exist = scalar(sh.here[n / kTiles & 1][n % kTiles * BN / 64]) >> (BN == 64 ? 0 : n % 2 * 32) & all;
        // An infinite or NaN value would reach rows that mask its key through a product with their weight of zero: where some
        // row of the block masks some key, it goes into the products as zero, and the rows that see its key are done again.
        const bool partial = k0 < full_lo || k0 + BN > full_hi || exist != all;
        if (n % kTiles == kTiles - 1) {
            put_offsets(n / kTiles + 1, next_page);
            next_page = key_page(n / kTiles + 2);
        }
        if constexpr (kDirect) {
            wait_loads();  // the wave's part of this tile
            __syncthreads();
            if (partial) {
#pragma unroll
                for (int i = 0; i < NCH; ++i) {
                    const int ch = tid + 256 * i;
                    vec<C, 8> *p = reinterpret_cast<vec<C, 8> *>(&sh.v[buf][0][0]) + ch;
                    vec<C, 8> x = *p;
                    if (!make_finite<C>(x)) {
                        *p = x;
                        atomicOr(&sh.wild[buf], 1ull << (ch / CH));
                    }
                }
                __syncthreads();
            }
            if (tid == 0) sh.wild[buf ^ 1] = 0;
        } else {
            if (k0 != kb) __syncthreads();  // the last tile has been read
            if (tid == 0) sh.wild[buf ^ 1] = 0;
#pragma unroll
            for (int i = 0; i < NCH; ++i) {
                const int ch = tid + 256 * i, row = ch / CH, at = ch % CH;
                if (partial && !make_finite<C>(vr[i])) atomicOr(&sh.wild[buf], 1ull << row);
                vec<E, 8> terms[KT];
                as_terms<C, E, KT>(kr[i], terms);
#pragma unroll
                for (int n = 0; n < KT; ++n) *reinterpret_cast<vec<E, 8> *>(&sh.k[n][row][(at ^ key_swap(row)) * 8]) = terms[n];
                as_terms<C, E, KT>(vr[i], terms);
#pragma unroll
                for (int n = 0; n < KT; ++n) *reinterpret_cast<vec<E, 8> *>(&sh.v[n][row][(at ^ value_swap(row)) * 8]) = terms[n];
            }
            __syncthreads();
        }
        step(n, k0, partial, exist, &sh.v[kDirect ? buf : 0][0][0], &sh.k[kDirect ? buf ^ 1 : 0][0][0], &sh.v[kDirect ? buf ^ 1 : 0][0][0]);
    }
    l = checked_sum<E>(bias, l + lane_xor<32>(l, lane));
    float z = l * 0.0f;
#pragma unroll
    for (int d = 0; d < ND; ++d) z = not_finite<16>(acc[d], z);
    unsigned long long odd = __ballot(wr0 + col < rows && z != 0.0f);
    odd = (odd | odd >> 32) & 0xffffffffu;  // rows of the wave
    if (wr0 + col < rows && !(odd >> col & 1)) {
        if (a.parts > 1) {
            const int64_t at = (static_cast<int64_t>(token) * a.n_heads + head) * a.parts + blockIdx.y;
            if (h == 0) a.part_ml[at] = make_float2(bias, l);
            float *o = a.part_o + at * D;
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int g = 0; g < 4; ++g)
                    *reinterpret_cast<float4 *>(o + 32 * d + 8 * g + 4 * h) =
                        make_float4(acc[d][4 * g], acc[d][4 * g + 1], acc[d][4 * g + 2], acc[d][4 * g + 3]);
        } else {
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            T *o = static_cast<T *>(a.out) + token * a.out_stride + head * D;
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    float x[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[e] = acc[d][4 * g + e] * inv;
                    store_rounded<T, 4>(o + 32 * d + 8 * g + 4 * h, x);
                }
        }
    }
    if (__builtin_expect(odd == 0, 1)) return;
#pragma unroll 1
    for (; odd; odd &= odd - 1) {
        const int ro = wr0 + __builtin_ctzll(odd), p = t.pos0 + ro / a.group;
        formula_row<T, C, D>(a, t.b, ro, t.first, kvh, max(kb, key_lo(a, p)), min(ke, key_hi(a, p, t.len)));
    }
}

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

int64_t part_row_bytes(const tqhip_kv_cache &c) { return c.head_dim * sizeof(float) + sizeof(float2); }

struct Plan {
    bool few;
    int tiles, parts, span;
};

Plan plan(const tqhip_attn &p, const tqhip_kv_cache &c, const tqhip_seqs &s) {
    const int group = p.n_heads / c.n_kv_heads;
    const int64_t rows = static_cast<int64_t>(s.n_tokens) * group;
    Plan n{};
    // Tiles of 16 rows read the cache once for each; they win up to 32 rows a sequence (64 sequences of up to 4000 keys, 32 heads of
    // 128: 16 rows 140 us, against 182 with tiles of 128; 32 rows 195 and 189; 64 rows 294 and 223), and, whatever the rows, as long
    // as there are few of them in all, because there they come in shorter parts (one sequence of 64 rows on 8 K/V heads 22 us and 32,
    // 128 rows 34 and 34; 448 rows on 2 heads of 64 30 and 41, 1792 rows 79 and 47; 1024 on one of 256 52 and 81).
    n.few = rows <= int64_t{2} * kFewRows * s.n_seqs || (rows + kFewRows - 1) / kFewRows * c.n_kv_heads <= 56;
    n.tiles = static_cast<int>(rows / (n.few ? kFewRows : kTileRows)) + s.n_seqs;
    const int64_t most = static_cast<int64_t>(s.table_stride) * c.page_size;
    const int64_t kv = s.max_kv > 0 ? std::min<int64_t>(s.max_kv, most) : most;
    // keys that one tile reads
    const int64_t seen = p.causal && p.window > 0 ? std::min<int64_t>(kv, int64_t{p.window} + (n.few ? kFewRows : kTileRows)) : kv;
    const int64_t blocks = static_cast<int64_t>(n.tiles) * c.n_kv_heads, cus = device_cu_count();
    const auto up = [](int64_t x, int64_t to) { return (x + to - 1) / to * to; };
    if (n.few) {
        // A workgroup's start and end cost as much as some 500 keys, so parts are as long as two workgroups per CU make them, up to
        // 1024 keys, which evens out ragged lengths. One token of 32 heads over 30000 keys: 35 us in parts of 512, 61 of
        // 128; of 14 heads over 3000: 14 of 128, 31 of 1024; 64 sequences of up to 16000: 423 of 1024, 455 of 512, 428 of 4096.
        const int64_t full = std::max<int64_t>(s.n_seqs, (rows + kFewRows - 1) / kFewRows) * c.n_kv_heads;  // tiles that there are
        n.span = static_cast<int>(std::clamp<int64_t>(up(seen * full / (2 * cus), kFewStep), kFewStep, 1024));
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

size_t plan_bytes(const Plan &n, const tqhip_attn &p, const tqhip_kv_cache &c, const tqhip_seqs &s) {
    if (n.parts == 1) return 0;
    return static_cast<size_t>(s.n_tokens) * p.n_heads * n.parts * part_row_bytes(c);
}

template <typename T, typename C, int D>
void launch_dim(const AttnArgs &a, const Plan &n, hipStream_t s) {
    const int kv_heads = a.n_heads / a.group;
    const dim3 grid(n.tiles * kv_heads, n.parts);
    if (n.few)
        attn_few<T, C, D><<<grid, 256, 0, s>>>(a);
    else
        attn_tiles<T, C, D><<<grid, 256, 0, s>>>(a);
    if (n.parts == 1) return;
    const int rows = a.n_tokens * a.n_heads;
    if (n.parts > 8 && rows <= INT32_MAX / 256)  // (a launch has less than 2^32 threads along x)
        attn_join<T, D, 4><<<rows, 256, 0, s>>>(a);
    else
        attn_join<T, D, 1><<<(rows + 3) / 4, 256, 0, s>>>(a);
}

template <typename T, typename C>
void launch_attn(const AttnArgs &a, const Plan &n, int D, hipStream_t s) {
    if (D == 64)
        launch_dim<T, C, 64>(a, n, s);
    else if (D == 128)
        launch_dim<T, C, 128>(a, n, s);
    else
        launch_dim<T, C, 256>(a, n, s);
}

int check_attn(const tqhip_attn &p, const tqhip_kv_cache &c, const tqhip_seqs &s) {
    const int st = check_cache(c, s);
    if (st != kOk) return st;
    if (!p.q || !p.out || !type_known(p.dtype) || p.n_heads < 1 || p.n_heads % c.n_kv_heads || p.window < 0 ||
        !std::isfinite(p.scale * 1.4426950408889634f) || (p.dtype != TQHIP_F32 && c.dtype != p.dtype))
        return kBadShape;
    if (c.head_dim != 64 && c.head_dim != 128 && c.head_dim != 256) return kBadShape;
    const int qb = type_bytes(p.dtype), cb = type_bytes(c.dtype);
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

int run_attn(const tqhip_attn &p, const tqhip_kv_cache &c, const tqhip_seqs &b, hipStream_t s) {
    int st = check_attn(p, c, b);
    if (st != kOk) return st;
    const Plan n = plan(p, c, b);
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
    if (p.dtype == TQHIP_F16)
        launch_attn<f16, f16>(a, n, c.head_dim, s);
    else if (p.dtype == TQHIP_BF16)
        launch_attn<bf16, bf16>(a, n, c.head_dim, s);
    else if (c.dtype == TQHIP_F32)
        launch_attn<float, float>(a, n, c.head_dim, s);
    else if (c.dtype == TQHIP_F16)
        launch_attn<float, f16>(a, n, c.head_dim, s);
    else
        launch_attn<float, bf16>(a, n, c.head_dim, s);
    return hipGetLastError() == hipSuccess ? kOk : kLaunchFailed;
}

}  // namespace
}  // namespace tqhip

extern "C" {

int tqhip_paged_attention_dev(const tqhip_attn *attn, const tqhip_kv_cache *cache, const tqhip_seqs *seqs,
                              void *stream) {
    if (!attn || !cache || !seqs) return tqhip::kBadShape;
    try {
        return tqhip::run_attn(*attn, *cache, *seqs, static_cast<hipStream_t>(stream));
    } catch (...) {  // (host memory ran out)
        return tqhip::kHipFailed;
    }
}

size_t tqhip_paged_attention_workspace(const tqhip_attn *attn, const tqhip_kv_cache *cache, const tqhip_seqs *seqs) {
    if (!attn || !cache || !seqs || tqhip::check_attn(*attn, *cache, *seqs) != tqhip::kOk) return 0;
    return tqhip::plan_bytes(tqhip::plan(*attn, *cache, *seqs), *attn, *cache, *seqs);
}

int tqhip_paged_attention_plan(const tqhip_attn *attn, const tqhip_kv_cache *cache, const tqhip_seqs *seqs, int *tile_rows,
                               int *parts) {
    if (!attn || !cache || !seqs || !tile_rows || !parts) return tqhip::kBadShape;
    const int st = tqhip::check_attn(*attn, *cache, *seqs);
    if (st != tqhip::kOk) return st;
    const tqhip::Plan n = tqhip::plan(*attn, *cache, *seqs);
    *tile_rows = n.few ? tqhip::kFewRows : tqhip::kTileRows;
    *parts = n.parts;
    return tqhip::kOk;
}

}  // extern "C"
