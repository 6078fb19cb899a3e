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
#include "paged_attn.h"

namespace tqhip {
namespace {

// ---- few rows: tiles of 16 rows ------------------------------------------------------------------

// A tile's keys are dealt to the four waves 32 at a time; each wave keeps a softmax of its own, and the four meet at the end, so no
// wave waits for another. K goes from the cache straight into operand registers, V into LDS of the wave's own, whose
// transposing reads turn its rows into columns. Reading the cache is the work (a query row takes 2 to 4 flops a byte), so the loads of
// the next step are issued as soon as this step's have arrived, before anything is computed on them.
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
    const float c = load_query<T, E, QT, NS>(a, static_cast<const T *>(a.q) + token * a.q_stride + head * D + 8 * g, q, [](int i) { return 32 * i; },
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
    const float c = load_query<T, E, QT, D / 16>(a, static_cast<const T *>(a.q) + token * a.q_stride + head * D + 8 * h, q, [](int i) { return 16 * i; },
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

// ---- host ----------------------------------------------------------------------------------------

template <typename T, typename C, int D>
void launch_dim(const AttnArgs &a, const Plan &n, hipStream_t s) {
    const int kv_heads = a.n_heads / a.group;
    const dim3 grid(n.tiles * kv_heads, n.parts);
    if (n.few)
        attn_few<T, C, D><<<grid, 256, 0, s>>>(a);
    else
        attn_tiles<T, C, D><<<grid, 256, 0, s>>>(a);
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

int check(const tqhip_attn &p, const tqhip_kv_cache &c, const tqhip_seqs &s) {
    const int st = check_cache(c, s);
    if (st != kOk) return st;
    if (p.dtype != TQHIP_F32 && c.dtype != p.dtype) return kBadShape;
    return check_attn(p, c, s, type_bytes(c.dtype));
}

int run(const tqhip_attn &p, const tqhip_kv_cache &c, const tqhip_seqs &b, hipStream_t s) {
    const int st = check(p, c, b);
    if (st != kOk) return st;
    return run_attn(p, c, b, plan(p, c, b, false), s, [&](const AttnArgs &a, const Plan &n) {
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
    });
}

}  // namespace
}  // namespace tqhip

extern "C" {

int tqhip_paged_attention_dev(const tqhip_attn *attn, const tqhip_kv_cache *cache, const tqhip_seqs *seqs,
                              void *stream) {
    if (!attn || !cache || !seqs) return tqhip::kBadShape;
    try {
        return tqhip::run(*attn, *cache, *seqs, static_cast<hipStream_t>(stream));
    } catch (...) {  // (host memory ran out)
        return tqhip::kHipFailed;
    }
}

size_t tqhip_paged_attention_workspace(const tqhip_attn *attn, const tqhip_kv_cache *cache, const tqhip_seqs *seqs) {
    if (!attn || !cache || !seqs || tqhip::check(*attn, *cache, *seqs) != tqhip::kOk) return 0;
    return tqhip::plan_bytes(tqhip::plan(*attn, *cache, *seqs, false), *attn, *cache, *seqs);
}

int tqhip_paged_attention_plan(const tqhip_attn *attn, const tqhip_kv_cache *cache, const tqhip_seqs *seqs, int *tile_rows,
                               int *parts) {
    if (!attn || !cache || !seqs || !tile_rows || !parts) return tqhip::kBadShape;
    const int st = tqhip::check(*attn, *cache, *seqs);
    if (st != tqhip::kOk) return st;
    const tqhip::Plan n = tqhip::plan(*attn, *cache, *seqs, false);
    *tile_rows = n.rows;
    *parts = n.parts;
    return tqhip::kOk;
}

}  // extern "C"
