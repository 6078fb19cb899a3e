// paged_attn8.hip -- attention over a paged cache of 8-bit codes with a scale for each block of tokens and head.
//
// With k_j = a_j x_j and v_j = b_j y_j (x, y codes, a, b the scales of j's block):
//   out = sum_j w_j b_j y_j / sum_j w_j,  w_j = 2^(c a_j q.x_j + bias),  c = scale log2 e.
// A code is an fp16 number without rounding, so q.x_j and the second product run on the matrix cores as over an fp16 cache, and the
// scales meet fp32 numbers: a_j the score, b_j the weight. A weight times its b_j is what has to fit fp16, so the
// running maximum that sets the bias is that of c a_j q.x_j + log2 b_j, and b is taken relative to a power of two near the first
// block's, which the sums get back at the end. Rows that this does not hold (infinities, NaN, scales 2^100 apart) are done by the formula.
//
// Weights times scales are two fp16 terms where the result shows more than one (see Terms).
//
// The cut into tiles of 16, 32 and 128 rows, the parts and their join are those of the other caches (paged_attn.h, paged_attn.hip).
// Few rows are bound by HBM: a key and a value of D bytes and their scales, read once for the rows of a K/V head. Many rows are bound by
// the vector units, which make fp16 of the codes and weights of the scores while the matrix units wait (busy 31 % and 45 % of the time).
//   64 single tokens over up to 16000 i8 keys, 32 heads of 128 over 8 (1.04 GB)     220 us, 4.7 TB/s (f16 keys 390)
//   32 sequences of 5 tokens over up to 9000 e4m3 keys, the same heads (316 MB)       93 us, 3.4 TB/s
//   one token over 3000 keys, 14 heads of 64 over 2                                  13 us, 8 and 3.5 of them kernels
//   752 fp32 tokens over up to 8000 i8 keys, 32 on 8 heads of 128 (72 GFLOP, twice that with two terms)  211 us
//   12577 bf16 tokens of prompts, e4m3, the same heads (707 GFLOP)                  915 us, 773 TFLOP/s
#include "paged_attn.h"

namespace tqhip {
namespace {

// Eight codes as fp16. An i8 becomes the low byte of 1024 + (x + 128), which is subtracted again, two at a time.
template <typename C>
__device__ inline vec<f16, 8> as_halves(unsigned lo, unsigned hi) {
    using h2 = vec<f16, 2>;
    h2 h[4];
    if constexpr (std::is_same_v<C, i8>) {
        const h2 off{static_cast<f16>(1152.0f), static_cast<f16>(1152.0f)};
        lo ^= 0x80808080u;
        hi ^= 0x80808080u;
        h[0] = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, lo, 0x04010400u)) - off;
        h[1] = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, lo, 0x04030402u)) - off;
        h[2] = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, hi, 0x04010400u)) - off;
        h[3] = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, hi, 0x04030402u)) - off;
    } else {
        h[0] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false);
        h[1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true);
        h[2] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false);
        h[3] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true);
    }
    return vec<f16, 8>{h[0][0], h[0][1], h[1][0], h[1][1], h[2][0], h[2][1], h[3][0], h[3][1]};
}

// Eight rows of 16 codes, 8 codes a lane by 16 lanes (two a row), as columns: lane i gets column i's eight.
__device__ inline vec<unsigned, 2> lds_code_columns(const unsigned char *p) {
    using raw = vec<int, 2>;
    return __builtin_bit_cast(vec<unsigned, 2>, __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) raw *)p));
}

// Zeros in the place of e4m3's NaN codes; false if there were any.
__device__ inline bool make_finite_codes(vec<unsigned, 4> &x) {
    bool finite = true;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const unsigned nan = ((x[i] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
        if (nan) {
            finite = false;
            x[i] &= ~((nan >> 7) * 0xffu);
        }
    }
    return finite;
}

// What the values' scales are taken relative to: the power of two of the largest among the wave's lanes that is a number.
__device__ inline float scale_unit(float b) {
    const float top = xor_max_wave(b > 0.0f && b < INFINITY ? b : 0.0f);
    const unsigned e = __float_as_uint(top) & 0x7f800000u;
    return e == 0 ? 1.0f : __uint_as_float(e);
}
// A value's scale relative to the unit, and its log2 for the running maximum. A weight is as much larger than its product with the scale
// as that is small, and has to fit fp32: a scale of 0 is taken as 2^-100 for the maximum (the product is 0 all the same), and one that is further than that from
// the unit makes its rows' sums NaN, so the formula takes them.
__device__ inline float relative_scale(float scale, float per_unit, float &log) {
    const float b = scale * per_unit, x = __builtin_amdgcn_logf(b);
    log = fminf(fmaxf(x, -100.0f), 100.0f);
    return scale == 0.0f || fabsf(x) <= 100.0f ? b : NAN;
}

// A key's scale as the factor of its score. A product of codes times an infinity would be an infinity of its own sign, where elements of either sign
// make no number; and what load_query's least factor and fp32 leave room for are scales of up to 2^60. One past that makes its rows NaN, so the formula takes them.
__device__ inline float key_scale(float scale) { return fabsf(scale) <= 0x1p60f ? scale : NAN; }
// A row of queries so large that its products times its factor pass fp32, or the factor alone, whatever the keys' scales make of them, may have had nothing but minus
// infinities: its sum of 0 says nothing then, and the formula takes it. (Products of queries and codes stay below 2^34, scales below 2^60.)
__device__ inline bool may_overflow(float c) { return c > 0x1p30f; }

// x as it is rounded to fp32, for split: a product whose fp16 form is taken twice, as the first term and to find the rest, must not be rounded
// to fp16 from its exact value once and from its fp32 one the other time (the compiler has an instruction for the former; the terms
// then miss each other by a step of fp16 where the two roundings fall to different sides, one weight in some 10^4).
__device__ inline float as_fp32(float x) {
    asm("" : "+v"(x));
    return x;
}

// A key's scales in LDS: a, log2 b, b.
constexpr int kScaleA = 0, kScaleLog = 1, kScaleB = 2;

// ---- few rows: tiles of 16 rows ------------------------------------------------------------------

// As over the other caches: 32 keys a wave and step, K straight into operand registers (16 codes a lane and load, which are the chunks of
// two products), V into LDS as it is and out of it by transposing reads of bytes.
template <typename T, typename C, int D, int R>
__global__ __launch_bounds__(256, (D == 256 ? 1 : 2)) void attn8_few(AttnArgs a) {
    constexpr int QT = Terms<T, C>::QT, WT = Terms<T, C>::WT;
    constexpr int kRows = R * kFewRows;
    constexpr int ND = D / 16, NS = D / 32, NL = D / 64, CH = D / 16, NV = kFewKeys * CH / 64;
    __shared__ struct {
        union {
            __attribute__((aligned(16))) unsigned char v[4][2][kFewKeys][D];
            float o[4][kRows][D];
        };
        __attribute__((aligned(16))) float by[4][3][kFewKeys];
        float meet[2][4][kRows];
    } sh;

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, col = lane & 15;
    const int kv_heads = a.n_heads / a.group;
    // The heads of a tile follow one another on one XCD, eight tiles at a time on the eight: where a token's heads lie side by side, they
    // read the same pages of memory at about the same time. Which tile goes to which XCD moves on with the eight and with the part, so that neither long
    // sequences nor numbers that name no tile stay with one of them. (64 single tokens and 32 times five of them, the file comment's: 228 and 88 us; each
    // head an XCD of its own 250 and 101; without the moving on 231 and 129.)
    const int tiles = gridDim.x / kv_heads, eights = tiles / 8, x = blockIdx.x, eight = x / (8 * kv_heads), over = x - eights * 8 * kv_heads;
    const int kvh = over < 0 ? x / 8 % kv_heads : over % kv_heads;
    TileRows t;
    if (!find_tile<kRows>(a, over < 0 ? 8 * eight + (x + eight + static_cast<int>(blockIdx.y)) % 8 : 8 * eights + over / kv_heads, t)) return;
    const int rows = t.n * a.group;
    const int last = min(t.r0 + kRows, rows) - 1;
    const int p_first = t.pos0 + t.r0 / a.group, p_last = t.pos0 + last / a.group;
    int ke = key_hi(a, p_last, t.len), kb = max(min(key_lo(a, p_first), ke), 0);  // (a window past the table is empty)
    if (a.parts > 1) {
        kb = max(kb, static_cast<int>(blockIdx.y) * a.span);
        if (static_cast<int>(blockIdx.y) < a.parts - 1) ke = min(ke, (static_cast<int>(blockIdx.y) + 1) * a.span);
        if (kb >= ke) return;
    }
    const int full_lo = key_lo(a, p_last), full_hi = key_hi(a, p_first, t.len);
    // the lane's rows: t.r0 + 16 r + col
    const auto row_of = [&](int r) { return min(t.r0 + kFewRows * r + col, rows - 1); };
    int lo[R], hi[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int pos = t.pos0 + row_of(r) / a.group;
        lo[r] = key_lo(a, pos);
        hi[r] = key_hi(a, pos, t.len);
    }

    const unsigned char *kc = static_cast<const unsigned char *>(a.k) + kvh * a.pages.head_stride + 16 * g;
    const unsigned char *vc = static_cast<const unsigned char *>(a.v) + kvh * a.pages.head_stride;
    // of a value row's chunks of 16 bytes, so that the 32 rows of a transposing read lie in different banks
    const auto swap = [](int row) {
        const int bit1 = row >> 1 & 1, bit2 = row >> 2 & 1, bit4 = row >> 4 & 1;
        return D == 64 ? bit4 | bit2 << 1 : D == 128 ? bit1 | bit4 << 1 | bit2 << 2 : (row & 3) | bit4 << 2 | bit2 << 3;
    };
    vec<unsigned, 4> kr[2][2][NL];
    float2 by[2];
    // The lane's keys of a step are k0 + col and k0 + 16 + col. All loads of the loop are unconditional (a page past the table is its
    // last entry, a row that does not exist is row 0 of page 0): a load under a branch would be waited for with all others.
    const auto pages_of = [&](int k0, int *page) {
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
            const int i = min(a.pages.page_size.quot(k0 + 16 * kt + col), a.pages.table_stride - 1);
            page[kt] = a.pages.table[static_cast<int64_t>(t.b) * a.pages.table_stride + i];
        }
    };
    const auto offsets = [&](int k0, const int *page, int64_t *o, int *scale) {
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
            const int key = k0 + 16 * kt + col;
            o[kt] = key < ke ? row_in_page(a.pages, page[kt], key) : -1;
            const int row = key - a.pages.page_size.quot(key) * static_cast<int>(a.pages.page_size.d);
            scale[kt] = ((o[kt] < 0 ? 0 : page[kt]) * kv_heads + kvh) * a.blocks + a.block.quot(row);
        }
    };
    const auto load_keys = [&](const int64_t *o, vec<unsigned, 4> (*x)[NL]) {
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int j = 0; j < NL; ++j) x[kt][j] = *reinterpret_cast<const vec<unsigned, 4> *>(kc + max(o[kt], int64_t{0}) + 64 * j);
    };
    const auto load_values = [&](const int64_t *o, unsigned char *__restrict__ to) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {  // 64 chunks in order; the row's offset is held by lane `row % 16`
            const int first = 64 * i / CH, row = first + lane / CH;
            const int64_t ro = __shfl(static_cast<long long>(max(o[first / 16], int64_t{0})), row & 15);
            global_to_lds<true>(vc + ro + ((lane % CH) ^ swap(row)) * 16, to + 64 * i * 16);
        }
    };

    int64_t off[2];
    int next[2], at[2];
    float2 by_next[2];
    int k0 = kb + wave * kFewKeys;
    pages_of(k0, next);
    offsets(k0, next, off, at);
    pages_of(k0 + kFewStep, next);
    load_keys(off, kr[0]);
    load_values(off, &sh.v[wave][0][0][0]);
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) by_next[kt] = a.scales[at[kt]];
    vec<f16, 8> q[R][QT][NS];
    float c[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int row = row_of(r), token = t.first + row / a.group, head = kvh * a.group + row % a.group;
        c[r] = load_query<T, f16, QT, NS>(a, static_cast<const T *>(a.q) + token * a.q_stride + head * D + 16 * g, q[r],
                                          [](int i) { return 64 * (i / 2) + 8 * (i % 2); },
                                          [&](float x) {
                                              x = fmaxf(x, lane_xor<16>(x, lane));
                                              return fmaxf(x, lane_xor<32>(x, lane));
                                          });
    }
    const float unit = scale_unit(fmaxf(off[0] >= 0 ? by_next[0].y : 0.0f, off[1] >= 0 ? by_next[1].y : 0.0f)), per_unit = 1.0f / unit;
    f32x4 acc[R][ND];
    float m[R], bias[R], l[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
        for (int i = 0; i < ND; ++i) acc[r][i] = f32x4{};
        m[r] = -INFINITY;
        bias[r] = l[r] = 0.0f;
    }

    // (The restrict pointers tell the compiler that the next step's transfers do not touch the values that are read meanwhile.)
    const auto step = [&](const vec<unsigned, 4> (*k_now)[NL], vec<unsigned, 4> (*k_next)[NL], const unsigned char *__restrict__ v_now,
                          unsigned char *__restrict__ v_next) __attribute__((always_inline)) {
        const unsigned exist = static_cast<unsigned>(__ballot(off[0] >= 0) & 0xffff) |
                               static_cast<unsigned>(__ballot(off[1] >= 0) & 0xffff) << 16;
        const bool partial = k0 < full_lo || k0 + kFewKeys > full_hi || exist != ~0u;
        wait_loads();
        by[0] = by_next[0];
        by[1] = by_next[1];
        offsets(k0 + kFewStep, next, off, at);
        pages_of(k0 + 2 * kFewStep, next);
        load_keys(off, k_next);
        load_values(off, v_next);
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) by_next[kt] = a.scales[at[kt]];
        if (g < 2) {
            const float2 x = g == 0 ? by[0] : by[1];
            float log;
            sh.by[wave][kScaleA][16 * g + col] = key_scale(x.x);
            sh.by[wave][kScaleB][16 * g + col] = relative_scale(x.y, per_unit, log);
            sh.by[wave][kScaleLog][16 * g + col] = log;
        }
        // S^T: the lane holds its rows' scores of keys 16 kt + 4 g + i
        f32x4 s[R][2];
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
            for (int r = 0; r < R; ++r) s[r][kt] = f32x4{};
#pragma unroll
            for (int j = 0; j < NL; ++j)
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const vec<f16, 8> kf = as_halves<C>(k_now[kt][j][2 * half], k_now[kt][j][2 * half + 1]);
#pragma unroll
                    for (int r = 0; r < R; ++r)
#pragma unroll
                        for (int qi = 0; qi < QT; ++qi) s[r][kt] = mfma16(kf, q[r][qi][2 * j + half], s[r][kt]);
                }
        }
        wave_lds_order();
        const auto by_of = [&](int what, int kt) { return *reinterpret_cast<const f32x4 *>(&sh.by[wave][what][16 * kt + 4 * g]); };
        const f32x4 sa[2] = {by_of(kScaleA, 0), by_of(kScaleA, 1)}, lg[2] = {by_of(kScaleLog, 0), by_of(kScaleLog, 1)},
                    b[2] = {by_of(kScaleB, 0), by_of(kScaleB, 1)};
        vec<f16, 8> p[R][WT];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            unsigned may = ~0u;
            if (partial) {
                const int k1 = k0 + 4 * g;
                may = (exist >> (4 * g)) & below(hi[r] - k1) & ~below(lo[r] - k1);
            }
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) s[r][kt] *= sa[kt];
            if (partial) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (!(may & (1u << (16 * (e / 4) + e % 4)))) s[r][e / 4][e % 4] = -INFINITY;
            }
            float mx = m[r];
#pragma unroll
            for (int e = 0; e < 8; ++e) mx = fmaxf(mx, fmaf(s[r][e / 4][e % 4], c[r], lg[e / 4][e % 4]));
            mx = fmaxf(mx, lane_xor<16>(mx, lane));
            mx = fmaxf(mx, lane_xor<32>(mx, lane));
            if (__ballot(mx - m[r] > kHeadroom<WT>)) {
                const float nb = mx == -INFINITY ? 0.0f : kWeightShift<f16, WT> - mx;
                const float f = m[r] == -INFINITY ? 0.0f : exp2f(nb - bias[r]);
                m[r] = mx;
                bias[r] = nb;
                l[r] *= f;
#pragma unroll
                for (int i = 0; i < ND; ++i) acc[r][i] *= f;
            }
            float w[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                w[e] = __builtin_amdgcn_exp2f(fmaf(s[r][e / 4][e % 4], c[r], bias[r]));
                l[r] += w[e];
                w[e] = as_fp32(w[e] * b[e / 4][e % 4]);
            }
            if (partial) {  // (the scale of a masked value may be no number)
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (!(may & (1u << (16 * (e / 4) + e % 4)))) w[e] = 0.0f;
            }
            split<f16, WT>(w, p[r]);
        }
        if constexpr (std::is_same_v<C, e4m3>) {
            if (partial) {  // NaN codes as the infinite and NaN values of attn_tiles
                unsigned wild = 0;
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    vec<unsigned, 4> *chunk = reinterpret_cast<vec<unsigned, 4> *>(const_cast<unsigned char *>(v_now)) + 64 * i + lane;
                    vec<unsigned, 4> x = *chunk;
                    const bool finite = make_finite_codes(x);
                    if (!finite) *chunk = x;
                    unsigned long long bad = __ballot(!finite);  // by chunk: CH of them a row
                    for (int row = 64 * i / CH; bad; ++row, bad >>= CH)
                        if (bad & ((1ull << CH) - 1)) wild |= 1u << row;
                }
                wave_lds_order();
#pragma unroll
                for (int r = 0; r < R; ++r)
                    if (wild & exist & below(hi[r] - k0) & ~below(lo[r] - k0)) l[r] = NAN;  // (formula_row takes the row)
            }
        }
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            const int e = (lane & 15) >> 1, row = 16 * (e >> 2) + 4 * g + (e & 3);
            const vec<unsigned, 2> u = lds_code_columns(v_now + row * D + (d ^ swap(row)) * 16 + 8 * (lane & 1));
            const vec<f16, 8> vf = as_halves<C>(u[0], u[1]);
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int wi = 0; wi < WT; ++wi) acc[r][d] = mfma16(vf, p[r][wi], acc[r][d]);
        }
        k0 += kFewStep;
    };
    unsigned char *v0 = &sh.v[wave][0][0][0], *v1 = &sh.v[wave][1][0][0];
    while (k0 < ke) {
        step(kr[0], kr[1], v0, v1);
        if (k0 >= ke) break;
        step(kr[1], kr[0], v1, v0);
    }
    wait_loads();  // (the loads past the last step: into LDS that is used for other things below)
    // the four waves' sums, brought to the least exponent bias among those that have any
#pragma unroll
    for (int r = 0; r < R; ++r) {
        l[r] += lane_xor<16>(l[r], lane);
        l[r] += lane_xor<32>(l[r], lane);
        l[r] = checked_sum<f16>(bias[r], l[r]);
        if (l[r] == 0.0f && may_overflow(c[r])) l[r] = NAN;
        if (g == 0) {
            sh.meet[0][wave][kFewRows * r + col] = bias[r];
            sh.meet[1][wave][kFewRows * r + col] = l[r];
        }
    }
    __syncthreads();  // (and every wave is done with V)
    float least[R], total[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int row = kFewRows * r + col;
        least[r] = INFINITY, total[r] = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w)
            if (sh.meet[1][w][row] != 0.0f) least[r] = fminf(least[r], sh.meet[0][w][row]);
#pragma unroll
        for (int w = 0; w < 4; ++w)
            if (sh.meet[1][w][row] != 0.0f) total[r] += sh.meet[1][w][row] * exp2f(least[r] - sh.meet[0][w][row]);
        if (l[r] != 0.0f) {
            const float f = exp2f(least[r] - bias[r]) * unit;
#pragma unroll
            for (int d = 0; d < ND; ++d) acc[r][d] *= f;
        }
#pragma unroll
        for (int d = 0; d < ND; ++d) *reinterpret_cast<f32x4 *>(&sh.o[wave][row][16 * d + 4 * g]) = acc[r][d];
    }
    __syncthreads();
    // thread: rows tid / 16 of each 16, every 16th group of four dimensions
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int row = kFewRows * r + (tid >> 4);
        const int r2 = t.r0 + row, token2 = t.first + r2 / a.group, head2 = kvh * a.group + r2 % a.group;
        const float total2 = __shfl(total[r], tid >> 4), least2 = __shfl(least[r], tid >> 4);
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
            const int64_t to = (static_cast<int64_t>(token2) * a.n_heads + head2) * a.parts + blockIdx.y;
            if (a.parts > 1 && (tid & 15) == 0) a.part_ml[to] = make_float2(least2, total2);
            const float inv = total2 == 0.0f ? 0.0f : 1.0f / total2;
#pragma unroll
            for (int i = 0; i < D / 64; ++i) {
                const int d = 4 * (tid & 15) + 64 * i;
                if (a.parts > 1) {
                    *reinterpret_cast<f32x4 *>(a.part_o + to * D + d) = o[i];
                } else {
                    float x[4] = {o[i][0] * inv, o[i][1] * inv, o[i][2] * inv, o[i][3] * inv};
                    store_rounded<T, 4>(static_cast<T *>(a.out) + token2 * a.out_stride + head2 * D + d, x);
                }
            }
        }
        if (__builtin_expect(odd == 0, 1)) continue;
#pragma unroll 1
        for (int i = 0; i < 4; ++i)
            if (odd >> (16 * i) & 0xffff) {
                const int ro = t.r0 + kFewRows * r + 4 * wave + i, p = t.pos0 + ro / a.group;
                formula_row<T, C, D>(a, t.b, ro, t.first, kvh, max(kb, key_lo(a, p)), min(ke, key_hi(a, p, t.len)));
            }
    }
}

// ---- many rows: tiles of 128 rows ---------------------------------------------------------------

// As over the other caches, but a tile's codes pass through registers on their way into LDS, where they are fp16: converted once for the
// four waves. The tile after next is under way while this one is used; the next is converted after it, into the other buffer.
template <typename T, typename C, int D>
struct TileShape8 {
    static constexpr int QT = Terms<T, C>::QT;
    static constexpr int BN = D == 256 && QT > 1 ? 32 : 64;
    static constexpr int kWavesPerSimd = D == 256 ? 1 : 2;
};

template <typename T, typename C, int D>
__global__ __launch_bounds__(256, (TileShape8<T, C, D>::kWavesPerSimd)) void attn8_tiles(AttnArgs a) {
    constexpr int QT = Terms<T, C>::QT, WT = Terms<T, C>::WT, BN = TileShape8<T, C, D>::BN;
    constexpr int CH = D / 16, NCH = BN * CH / 256;  // chunks of 16 codes a row, and a thread
    constexpr int NK = BN / 32, ND = D / 32, kTiles = 256 / BN;
    __shared__ struct {
        __attribute__((aligned(16))) f16 k[2][BN][D];
        __attribute__((aligned(16))) f16 v[2][BN][D];
        __attribute__((aligned(16))) float by[2][3][BN];
        int64_t offs[2][256];           // offsets of the rows of 256 keys, several tiles, and of the next 256
        int scale[2][256];              // places of their scales
        unsigned long long here[2][4];  // which of those keys exist
        unsigned one[2][8];             // groups of 32 of those keys that share their scales: all ones
        unsigned long long wild[3];     // keys of a partly masked tile that have NaN codes
        float unit;
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

    vec<f16, 8> q[QT][D / 16];
    const float c = load_query<T, f16, QT, D / 16>(a, static_cast<const T *>(a.q) + token * a.q_stride + head * D + 8 * h, q,
                                                   [](int i) { return 16 * i; },
                                                   [&](float x) { return fmaxf(x, lane_xor<32>(x, lane)); });
    const unsigned char *kc = static_cast<const unsigned char *>(a.k) + kvh * a.pages.head_stride;
    const unsigned char *vc = static_cast<const unsigned char *>(a.v) + kvh * a.pages.head_stride;
    // Places of a row's chunks of 8 elements (16 bytes), so that the reads below meet every bank once, and the writes, of every other
    // chunk of a row or two by 8 lanes, every second chunk's banks and the ones between (1 % of the time for prompts).
    const auto key_at = [](int row, int ch) { return (D == 64 ? ch ^ (row >> 1 & 7) ^ (row & 1) : ch ^ (ch >> 3 & 1) ^ (row & 15)) * 8; };
    const auto value_at = [](int row, int ch) { return (D == 64 ? ch ^ (row & 3) << 1 ^ (row & 1) : ch ^ (ch >> 3 & 1) ^ (row & 3) << 2) * 8; };
    vec<unsigned, 4> kr[NCH], vr[NCH];
    float2 by;
    // A tile's codes and scales on their way into registers. For a key that does not exist row 0 of page 0 is loaded.
    const auto load_tile = [&](int n) __attribute__((always_inline)) {
        const int slot = n / kTiles & 1, first = n % kTiles * BN;
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            const int ch = tid + 256 * i;
            const int64_t o = sh.offs[slot][first + ch / CH] + ch % CH * 16;
            kr[i] = *reinterpret_cast<const vec<unsigned, 4> *>(kc + o);
            vr[i] = *reinterpret_cast<const vec<unsigned, 4> *>(vc + o);
        }
        by = a.scales[sh.scale[slot][first + tid % BN]];
    };
    const auto exist_of = [&](int n) {
        return scalar(sh.here[n / kTiles & 1][n % kTiles * BN / 64]) >> (BN == 64 ? 0 : n % 2 * 32) & (BN == 64 ? ~0ull : 0xffffffffull);
    };
    const auto partial_at = [&](int k0, unsigned long long exist) {
        return k0 < full_lo || k0 + BN > full_hi || exist != (BN == 64 ? ~0ull : 0xffffffffull);
    };
    // The tile's codes from registers into LDS as fp16, its keys' scales beside them.
    const auto put_tile = [&](int n, float per_unit) __attribute__((always_inline)) {
        const int buf = n & 1;
        if constexpr (std::is_same_v<C, e4m3>) {
            // A NaN value would reach rows that mask its key through a product with their weight of zero: where some row of the
            // block masks some key, it goes into the products as zero, and the rows that see its key are done again.
            if (partial_at(kb + n * BN, exist_of(n))) {
#pragma unroll
                for (int i = 0; i < NCH; ++i)
                    if (!make_finite_codes(vr[i])) atomicOr(&sh.wild[n % 3], 1ull << ((tid + 256 * i) / CH));
            }
        }
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            const int ch = tid + 256 * i, row = ch / CH, at = ch % CH * 2;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                *reinterpret_cast<vec<f16, 8> *>(&sh.k[buf][row][key_at(row, at + e)]) = as_halves<C>(kr[i][2 * e], kr[i][2 * e + 1]);
                *reinterpret_cast<vec<f16, 8> *>(&sh.v[buf][row][value_at(row, at + e)]) = as_halves<C>(vr[i][2 * e], vr[i][2 * e + 1]);
            }
        }
        if (tid < BN) {
            float log;
            sh.by[buf][kScaleA][tid] = key_scale(by.x);
            sh.by[buf][kScaleB][tid] = relative_scale(by.y, per_unit, log);
            sh.by[buf][kScaleLog][tid] = log;
        }
    };
    // 256 keys' pages are looked up while the tiles of the 256 before run, and their offsets put into LDS two tiles before they start.
    const auto key_page = [&](int n) {
        const int key = kb + n * 256 + tid;
        return key < ke ? page_number(a.pages, t.b, key) : -1;
    };
    const auto put_offsets = [&](int n, int page) {
        const int key = kb + n * 256 + tid;
        const int64_t o = row_in_page(a.pages, page, key);
        const unsigned long long m = __ballot(o >= 0);
        const int row = key - a.pages.page_size.quot(key) * static_cast<int>(a.pages.page_size.d);
        sh.offs[n & 1][tid] = max(o, int64_t{0});
        sh.scale[n & 1][tid] = o < 0 ? kvh * a.blocks : (page * kv_heads + kvh) * a.blocks + a.block.quot(row);
        if (lane == 0) sh.here[n & 1][wave] = m;
        const int place = sh.scale[n & 1][tid], first = __shfl(place, lane & 32);
        const unsigned long long same = __ballot(place == first);
        if ((lane & 31) == 0) sh.one[n & 1][tid / 32] = static_cast<unsigned>(same >> (lane & 32));
    };

    f32x16 acc[ND];
#pragma unroll
    for (int i = 0; i < ND; ++i) acc[i] = f32x16{};
    float m = -INFINITY, bias = 0.0f, l = 0.0f;

    put_offsets(0, key_page(0));
    if (tid < 3) sh.wild[tid] = 0;
    __syncthreads();
    int next_page = key_page(1);
    load_tile(0);
    if (wave == 0) {
        const float unit = scale_unit(tid < BN && (exist_of(0) >> tid & 1) ? by.y : 0.0f);
        if (tid == 0) sh.unit = unit;
    }
    __syncthreads();
    const float unit = sh.unit, per_unit = 1.0f / unit;
    put_tile(0, per_unit);
    if (kb + BN < ke) load_tile(1);

    const auto compute = [&](int n, int k0, bool partial, unsigned long long exist) __attribute__((always_inline)) {
        const int buf = n & 1;
        if (!wave_live || k0 >= w_hi || k0 + BN <= w_lo) return;
        // 32 keys at a time: the score products of the next 32 run on the matrix cores while the vector units form the weights of
        // these. S^T, keys down, queries across: the lane holds its query's keys (i % 4) + 8 (i / 4) + 4 h.
        const auto scores = [&](int kt) {
            f32x16 s{};
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
                const vec<f16, 8> kf = *reinterpret_cast<const vec<f16, 8> *>(&sh.k[buf][32 * kt + col][key_at(col, 2 * i + h)]);
#pragma unroll
                for (int qi = 0; qi < QT; ++qi) s = mfma32(kf, q[qi][i], s);
            }
            return s;
        };
        const auto by_of = [&](int what, int kt, int j) { return *reinterpret_cast<const f32x4 *>(&sh.by[buf][what][32 * kt + 8 * j + 4 * h]); };
        f32x16 s = scores(0), ahead{};
#pragma unroll
        for (int kt = 0; kt < NK; ++kt) {
            const int k1 = k0 + 32 * kt;
            // Keys of one scale that all count: their scores' factor is c a, and b goes into the weights' exponent, and out of their sum.
            const float a0 = sh.by[buf][kScaleA][32 * kt], b0 = sh.by[buf][kScaleB][32 * kt], lg0 = sh.by[buf][kScaleLog][32 * kt];
            const bool one = __builtin_amdgcn_readfirstlane(!partial && sh.one[n / kTiles & 1][n % kTiles * NK + kt] == ~0u && a0 >= 0.0f && b0 > 0.0f);
            // else: which of the lane's keys its row may attend to: bit (i % 4) + 8 (i / 4) for register i
            unsigned may = ~0u;
            if (partial) may = (static_cast<unsigned>(exist >> (32 * kt)) >> (4 * h)) & below(hi - k1 - 4 * h) & ~below(lo - k1 - 4 * h);
            float mx;
            if (one) {
                mx = s[0];
#pragma unroll
                for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[i]);
                mx = fmaf(mx, c * a0, lg0);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const f32x4 sa = by_of(kScaleA, kt, j);
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[4 * j + i] *= sa[i];
                }
                if (partial) {
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (!(may & (1u << ((i & 3) + 8 * (i >> 2))))) s[i] = -INFINITY;
                }
                mx = m;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const f32x4 lg = by_of(kScaleLog, kt, j);
#pragma unroll
                    for (int i = 0; i < 4; ++i) mx = fmaxf(mx, fmaf(s[4 * j + i], c, lg[i]));
                }
            }
            mx = fmaxf(m, fmaxf(mx, lane_xor<32>(mx, lane)));
            if (__ballot(mx - m > kHeadroom<WT>)) {
                const float nb = mx == -INFINITY ? 0.0f : kWeightShift<f16, WT> - mx;
                const float f = m == -INFINITY ? 0.0f : exp2f(nb - bias);
                m = mx;
                bias = nb;
                l *= f;
#pragma unroll
                for (int i = 0; i < ND; ++i) acc[i] *= f;
            }
            if (kt + 1 < NK) ahead = scores(kt + 1);
            if (one) {
                const float ca = c * a0, from = bias + lg0;
                float sum = 0.0f;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], ca, from));
                    sum += s[i];
                }
                l = fmaf(sum, __builtin_amdgcn_rcpf(b0), l);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const f32x4 b = by_of(kScaleB, kt, j);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float x = __builtin_amdgcn_exp2f(fmaf(s[4 * j + i], c, bias));
                        l += x;
                        s[4 * j + i] = as_fp32(x * b[i]);
                    }
                }
                if (partial) {  // (the scale of a masked value may be no number)
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (!(may & (1u << ((i & 3) + 8 * (i >> 2))))) s[i] = 0.0f;
                }
            }
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                float x[8];
                vec<f16, 8> p[WT];
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = s[8 * half + e];
                split<f16, WT>(x, p);
#pragma unroll
                for (int d = 0; d < ND; ++d) {
                    const int i = lane & 15, row = 32 * kt + 16 * half + 4 * h + i / 4;
                    const f16 *v0 = &sh.v[buf][row][value_at(i / 4, 4 * d + (lane & 16) / 8 + (i & 3) / 2) + 4 * (i & 1)];
                    const vec<f16, 4> a0 = lds_columns(v0), a1 = lds_columns(v0 + 8 * D);
                    const vec<f16, 8> vf = __builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
                    for (int wi = 0; wi < WT; ++wi) acc[d] = mfma32(vf, p[wi], acc[d]);
                }
            }
            s = ahead;
        }
        if constexpr (std::is_same_v<C, e4m3>)
            for (unsigned long long w = partial ? sh.wild[n % 3] & exist : 0; w; w &= w - 1) {
                const int key = k0 + __builtin_ctzll(w);
                if (key >= lo && key < hi) l = NAN;  // (formula_row takes the row)
            }
    };
    for (int n = 0, k0 = kb; k0 < ke; k0 += BN, ++n) {
        if (n % kTiles == kTiles - 2) {
            put_offsets(n / kTiles + 1, next_page);
            next_page = key_page(n / kTiles + 2);
        }
        __syncthreads();  // this tile is in LDS, and the one before has been read
        if (std::is_same_v<C, e4m3> && tid == 0) sh.wild[(n + 2) % 3] = 0;
        const unsigned long long exist = exist_of(n);
        compute(n, k0, partial_at(k0, exist), exist);
        if (k0 + BN < ke) put_tile(n + 1, per_unit);
        if (k0 + 2 * BN < ke) load_tile(n + 2);
    }
    l = checked_sum<f16>(bias, l + lane_xor<32>(l, lane));
    if (l == 0.0f && may_overflow(c)) l = NAN;
    float z = l * 0.0f;
#pragma unroll
    for (int d = 0; d < ND; ++d) {
        acc[d] *= unit;
        z = not_finite<16>(acc[d], z);
    }
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

// ---- host ----------------------------------------------------------------------------------------

template <typename T, typename C, int D>
void launch_dim(const AttnArgs &a, const Plan &n, hipStream_t s) {
    const dim3 grid(n.tiles * (a.n_heads / a.group), n.parts);
    constexpr int kPair = D == 256 && std::is_same_v<T, float> ? 1 : 2;  // (as plan has it)
    if (n.rows == kFewRows)
        attn8_few<T, C, D, 1><<<grid, 256, 0, s>>>(a);
    else if (n.rows == 2 * kFewRows)
        attn8_few<T, C, D, kPair><<<grid, 256, 0, s>>>(a);
    else
        attn8_tiles<T, C, D><<<grid, 256, 0, s>>>(a);
    launch_join<T, D>(a, n, s);
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
template <typename C>
void launch_attn(int dtype, const AttnArgs &a, const Plan &n, int D, hipStream_t s) {
    if (dtype == TQHIP_F32)
        launch_attn<float, C>(a, n, D, s);
    else if (dtype == TQHIP_F16)
        launch_attn<f16, C>(a, n, D, s);
    else
        launch_attn<bf16, C>(a, n, D, s);
}

int check(const tqhip_attn &p, const tqhip_kv_cache8 &c, const tqhip_seqs &s) {
    const int st = check_cache8(c, s);
    return st == kOk ? check_attn(p, rows_of(c), s, 1) : st;
}

int run(const tqhip_attn &p, const tqhip_kv_cache8 &c, const tqhip_seqs &b, hipStream_t s) {
    const int st = check(p, c, b);
    if (st != kOk) return st;
    const tqhip_kv_cache rows = rows_of(c);
    return run_attn(p, rows, b, plan(p, rows, b, true), s, [&](AttnArgs a, const Plan &n) {
        a.scales = reinterpret_cast<const float2 *>(c.scales);
        a.block = FastDiv(static_cast<uint32_t>(c.block));
        a.blocks = c.page_size / c.block;
        if (c.dtype == TQHIP_I8)
            launch_attn<i8>(p.dtype, a, n, c.head_dim, s);
        else
            launch_attn<e4m3>(p.dtype, a, n, c.head_dim, s);
    });
}

}  // namespace
}  // namespace tqhip

extern "C" {

int tqhip_paged_attention8_dev(const tqhip_attn *attn, const tqhip_kv_cache8 *cache, const tqhip_seqs *seqs, void *stream) {
    if (!attn || !cache || !seqs) return tqhip::kBadShape;
    try {
        return tqhip::run(*attn, *cache, *seqs, static_cast<hipStream_t>(stream));
    } catch (...) {  // (host memory ran out)
        return tqhip::kHipFailed;
    }
}

size_t tqhip_paged_attention8_workspace(const tqhip_attn *attn, const tqhip_kv_cache8 *cache, const tqhip_seqs *seqs) {
    if (!attn || !cache || !seqs || tqhip::check(*attn, *cache, *seqs) != tqhip::kOk) return 0;
    const tqhip_kv_cache rows = tqhip::rows_of(*cache);
    return tqhip::plan_bytes(tqhip::plan(*attn, rows, *seqs, true), *attn, rows, *seqs);
}

int tqhip_paged_attention8_plan(const tqhip_attn *attn, const tqhip_kv_cache8 *cache, const tqhip_seqs *seqs, int *tile_rows, int *parts) {
    if (!attn || !cache || !seqs || !tile_rows || !parts) return tqhip::kBadShape;
    const int st = tqhip::check(*attn, *cache, *seqs);
    if (st != tqhip::kOk) return st;
    const tqhip::Plan n = tqhip::plan(*attn, tqhip::rows_of(*cache), *seqs, true);
    *tile_rows = n.rows;
    *parts = n.parts;
    return tqhip::kOk;
}

}  // extern "C"
