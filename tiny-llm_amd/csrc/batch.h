// batch.h -- what the kernels of a batch of requests share (heads.hip, paged_attn.hip, lora.hip):
// element types, the search of a token's sequence, positions to pages.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <array>
#include <cstdint>
#include <utility>

#include "../../include/tqhip.h"

namespace tqhip {
namespace {

using bf16 = __bf16;
using f16 = _Float16;

template <typename T, int N>
using vec = T __attribute__((ext_vector_type(N)));

inline int type_bytes(int dtype) { return dtype == TQHIP_F32 ? 4 : 2; }
inline bool type_known(int dtype) { return dtype >= TQHIP_F32 && dtype <= TQHIP_BF16; }

// N elements at p (aligned to their size) as floats, and floats rounded to nearest even at p.
template <typename T, int N>
__device__ inline void load_as_float(const T *p, float *out) {
    const vec<T, N> v = *reinterpret_cast<const vec<T, N> *>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = static_cast<float>(v[i]);
}
template <typename T, int N>
__device__ inline void store_rounded(T *p, const float *in) {
    vec<T, N> v;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = static_cast<T>(in[i]);
    *reinterpret_cast<vec<T, N> *>(p) = v;
}

// LDS that only one wave uses: what its lanes wrote is there for all of them (a wave's LDS accesses complete in order; this
// keeps the compiler from reordering them).
__device__ inline void wave_lds_order() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// The sequence b of token t and the token's position in it; false where it is in none. The 64 lanes of a wave search
// together (all call with the same arguments): up to 64 sequences' starts and lengths are one round of loads, and 4096 are
// two and a third, where a bisection waits for 6 and 12 loads one after the other. Whatever the arrays hold, b is in range.
__device__ inline bool find_token(const int *start, const int *len, int n, int t, int &b, int &pos) {
    const int lane = threadIdx.x & 63;
    int lo = 0;
    while (n > 64) {
        const int step = (n + 63) / 64, i = lane * step;
        const int c = __popcll(__ballot(i < n && start[lo + i] <= t));
        if (c == 0) return false;
        lo += (c - 1) * step;
        n = min(step, n - (c - 1) * step);
    }
    const int at = lo + min(lane, n - 1);
    const int first = start[at], end = start[at + 1], kv = len[at];
    const int c = __popcll(__ballot(lane < n && first <= t));
    if (c == 0) return false;
    b = lo + c - 1;
    const int e = __builtin_amdgcn_readlane(end, c - 1);
    pos = max(__builtin_amdgcn_readlane(kv, c - 1), 0) - (e - t);
    return t < e;
}

// The rows of a ragged batch in tiles of BM: a sequence with n tokens has n * per rows (per: rows of a token). Tiles are numbered
// over the batch without a scan of the lengths: sequence b's start at floor(start[b] per / BM) + b, which leaves room for
// ceil(n per / BM) of them, so there are floor(n_tokens per / BM) + n_seqs numbers and some name no tile.
struct Run {
    int b, first, n, r0;  // sequence, its first token, its number of tokens, the tile's first row
};
template <int BM>
__device__ inline bool find_run(const int *q_start, int n_seqs, int n_tokens, int per, int tile, Run &t) {
    const int lane = threadIdx.x & 63;
    int lo = 0, n = n_seqs;
    const auto base = [&](int b) {
        const int64_t s = min(max(q_start[b], 0), n_tokens);
        return static_cast<int>(s * per / BM) + b;
    };
    for (;;) {
        const int step = (n + 63) / 64, i = lane * step;
        const int c = __popcll(__ballot(i < n && base(lo + i) <= tile));
        if (c == 0) return false;
        lo += (c - 1) * step;
        n = min(step, n - (c - 1) * step);
        if (step == 1) break;
    }
    t.b = lo;
    t.first = min(max(q_start[lo], 0), n_tokens);
    t.n = min(max(q_start[lo + 1], 0), n_tokens) - t.first;
    t.r0 = (tile - base(lo)) * BM;
    return t.n > 0 && t.r0 < t.n * per;
}

// Division of 0 <= n < 2^31 by a fixed d >= 1 as a multiplication (Granlund and Montgomery, Division by
// Invariant Integers using Multiplication, 1994): with s = ceil(log2 d) and
// m = floor(2^32 (2^s - d) / d) + 1, n / d = (mulhi(m, n) + n) >> s; the sum stays below 2^32.
struct FastDiv {
    uint32_t m, s, d;
    explicit FastDiv(uint32_t div) : m(0), s(0), d(div) {
        while ((uint64_t{1} << s) < d) ++s;
        m = static_cast<uint32_t>(((uint64_t{1} << 32) * ((uint64_t{1} << s) - d)) / d + 1);
    }
    __device__ inline int quot(int n) const {
        return static_cast<int>((__umulhi(m, static_cast<uint32_t>(n)) + static_cast<uint32_t>(n)) >> s);
    }
};

// A paged cache and a batch's pages as the kernels take them (strides in elements).
struct Pages {
    const int *table;
    int table_stride, n_pages;
    FastDiv page_size;
    int64_t page_stride, token_stride, head_stride;
};

// The page number of position p of sequence b as the table has it (-1 past the table and before position 0), and the element
// offset (head 0) of the position's row, -1 where it does not exist. Two steps, so that a kernel can have the page under way
// while it computes: what is done with a loaded value, even a comparison, waits for it and for every load before it.
__device__ inline int page_number(const Pages &g, int b, int p) {
    const int i = p < 0 ? 0x7fffffff : g.page_size.quot(p);
    return i < g.table_stride ? g.table[static_cast<int64_t>(b) * g.table_stride + i] : -1;
}
__device__ inline int64_t row_in_page(const Pages &g, int page, int p) {
    if (static_cast<unsigned>(page) >= static_cast<unsigned>(g.n_pages)) return -1;
    return page * g.page_stride + (p - g.page_size.quot(p) * static_cast<int>(g.page_size.d)) * g.token_stride;
}
__device__ inline int64_t row_offset(const Pages &g, int b, int p) { return row_in_page(g, page_number(g, b, p), p); }

// The cache's strides with the contiguous layout for zeros; false: less than a head's row apart.
inline bool cache_strides(const tqhip_kv_cache &c, int64_t *page, int64_t *token, int64_t *head) {
    if (c.page_stride == 0 && c.token_stride == 0 && c.head_stride == 0) {
        *head = c.head_dim;
        *token = static_cast<int64_t>(c.n_kv_heads) * c.head_dim;
        *page = *token * c.page_size;
        return true;
    }
    *page = c.page_stride;
    *token = c.token_stride;
    *head = c.head_stride;
    return *page > 0 && *token >= c.head_dim && *head >= c.head_dim;
}

// Whether no two heads' rows share an element, so that writing them is no race: with the axes ordered by stride, a step along one clears
// all that lies along those before it. (Reading rows that share elements is fine.)
inline bool rows_apart(const tqhip_kv_cache &c) {
    std::array<std::pair<int64_t, int>, 3> axis{{{0, c.n_pages}, {0, c.page_size}, {0, c.n_kv_heads}}};
    (void)cache_strides(c, &axis[0].first, &axis[1].first, &axis[2].first);
    std::sort(axis.begin(), axis.end());
    __int128 extent = c.head_dim;
    for (const auto &[stride, n] : axis) {
        if (n == 1) continue;
        if (stride < extent) return false;
        extent += static_cast<__int128>(stride) * (n - 1);
    }
    return true;
}

// Checks of the cache and the batch that kv_append and paged_attention share.
inline int check_cache(const tqhip_kv_cache &c, const tqhip_seqs &s) {
    if (!c.k || !c.v || !type_known(c.dtype) || c.n_pages < 1 || c.page_size < 1 || c.n_kv_heads < 1 || c.head_dim < 1)
        return TQHIP_EBADSHAPE;
    if (s.n_seqs < 1 || s.n_tokens < 1 || !s.q_start || !s.kv_len || !s.block_table || s.table_stride < 1 || s.max_kv < 0)
        return TQHIP_EBADSHAPE;
    int64_t page, token, head;
    if (!cache_strides(c, &page, &token, &head)) return TQHIP_EBADSHAPE;
    // offsets are 64-bit; what has to fit 32 bits, a tile's length to spare, are the positions
    if (static_cast<int64_t>(s.table_stride) * c.page_size > INT32_MAX / 2) return TQHIP_ETOOLARGE;
    return TQHIP_OK;
}

inline Pages make_pages(const tqhip_kv_cache &c, const tqhip_seqs &s) {
    Pages g{s.block_table, s.table_stride, c.n_pages, FastDiv(static_cast<uint32_t>(c.page_size)), 0, 0, 0};
    (void)cache_strides(c, &g.page_stride, &g.token_stride, &g.head_stride);
    return g;
}

}  // namespace
}  // namespace tqhip
