// lora.hip -- the low-rank adapters of many requests beside the projection that they share:
// y_t = base_t + scale[a] * B_a (A_a x_t), a the adapter of t's request.
//
// Two launches. The first forms u = scale A x (few numbers: rank of them per token), the second adds B u to base. A tile
// is a run of tokens of one sequence, so it has one adapter, whatever the order of the adapters over the requests.
// Both are products on the matrix cores in bf16 terms: an fp32 operand (x, u, fp32 weights) is three
// of them (24 bits), an fp16 weight two (all 11 bits, and fp16's range), a bf16 weight one; products below 2^-24 are
// left out. So fp32 results keep fp32's precision at 3 to 6 matrix instructions a product, where the fp32 ones take 16.
#include <algorithm>
#include <type_traits>

#include "batch.h"
#include "tq_common.h"

namespace tqhip {
namespace {

struct LoraArgs {
    const float *x, *base;
    float *y;
    const void *a, *b;
    const float *scale;
    const int *q_start, *adapter;
    float *u;  // [splits][n_tokens][rank]: parts of scale A x, over the parts of K
    int n_tokens, K, M, rank, n_adapters, n_seqs;
    int splits, m_per_block;
};

using f32x4 = vec<float, 4>;
using bf16x8 = vec<bf16, 8>;
__device__ inline f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

constexpr int kUTerms = 3;  // of x and u
template <typename W>
constexpr int kWTerms = std::is_same_v<W, bf16> ? 1 : std::is_same_v<W, f16> ? 2 : 3;

// x as N bf16 terms: all but the last cut off (an infinity is its first term), the last rounded to nearest even.
template <int N>
__device__ inline void bf16_terms(const float *x, bf16x8 *out) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float r = x[i];
#pragma unroll
        for (int n = 0; n < N - 1; ++n) {
            const unsigned u = __float_as_uint(r);
            out[n][i] = __builtin_bit_cast(bf16, static_cast<unsigned short>(u >> 16));
            const float cut = __uint_as_float(u & 0xffff0000u);
            r = r == cut ? 0.0f : r - cut;
        }
        out[N - 1][i] = static_cast<bf16>(r);
    }
}

// Elements at .. at + 7 of a row of n, zeros past its end. WIDE: n is a multiple of 8 and rows are 16-byte aligned.
template <bool WIDE, typename T>
__device__ inline vec<T, 8> load8(const T *row, int at, int n) {
    vec<T, 8> v{};
    if constexpr (WIDE) {
        if (at < n) v = *reinterpret_cast<const vec<T, 8> *>(row + at);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (at + i < n) v[i] = row[at + i];
    }
    return v;
}
template <typename W>
__device__ inline void weight_terms(const vec<W, 8> &w, bf16x8 *out) {
    if constexpr (std::is_same_v<W, bf16>) {
        out[0] = w;
    } else {
        float f[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = static_cast<float>(w[i]);
        bf16_terms<kWTerms<W>>(f, out);
    }
}

__device__ inline int adapter_of(const LoraArgs &p, int b) {
    const int a = p.adapter[b];
    return static_cast<unsigned>(a) < static_cast<unsigned>(p.n_adapters) ? a : -1;
}

// u^T = A x^T for a tile of 16 TT tokens: the lane holds ranks 16 n + 4 g + i of token 16 t + lane % 16. The steps of 32 along K are
// dealt to gridDim.y blocks of four waves; the waves' sums meet in LDS, the blocks' in lora_expand. x is read once.
template <typename W, int NR, int TT, bool WIDE>
__global__ __launch_bounds__(256) void lora_shrink(LoraArgs p) {
    constexpr int BM = 16 * TT;
    __shared__ float sum[4][BM][16 * NR + 4];
    Run t;
    if (!find_run<BM>(p.q_start, p.n_seqs, p.n_tokens, 1, blockIdx.x, t)) return;
    const int ad = adapter_of(p, t.b);
    if (ad < 0) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, col = lane & 15;
    const int steps = (p.K + 31) / 32, workers = 4 * p.splits, worker = blockIdx.y * 4 + wave;
    const int s0 = static_cast<int>(static_cast<int64_t>(steps) * worker / workers);
    const int s1 = static_cast<int>(static_cast<int64_t>(steps) * (worker + 1) / workers);
    const float *x[TT];
#pragma unroll
    for (int j = 0; j < TT; ++j) x[j] = p.x + static_cast<int64_t>(t.first + min(t.r0 + 16 * j + col, t.n - 1)) * p.K;
    const W *a[NR];
#pragma unroll
    for (int n = 0; n < NR; ++n)
        a[n] = static_cast<const W *>(p.a) + (static_cast<int64_t>(ad) * p.rank + min(16 * n + col, p.rank - 1)) * p.K;
    f32x4 acc[NR][TT];
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int j = 0; j < TT; ++j) acc[n][j] = f32x4{};
    for (int s = s0; s < s1; ++s) {
        const int k = 32 * s + 8 * g;
        bf16x8 xt[TT][kUTerms];
#pragma unroll
        for (int j = 0; j < TT; ++j) {
            const vec<float, 8> v = load8<WIDE>(x[j], k, p.K);
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = v[e];
            bf16_terms<kUTerms>(f, xt[j]);
        }
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            bf16x8 wt[kWTerms<W>];
            weight_terms<W>(load8<WIDE>(a[n], k, p.K), wt);
#pragma unroll
            for (int w = 0; w < kWTerms<W>; ++w)
#pragma unroll
                for (int u = 0; u < kUTerms; ++u)
                    if (w + u < 3) {
#pragma unroll
                        for (int j = 0; j < TT; ++j) acc[n][j] = mfma16(wt[w], xt[j][u], acc[n][j]);
                    }
        }
    }
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int j = 0; j < TT; ++j) *reinterpret_cast<f32x4 *>(&sum[wave][16 * j + col][16 * n + 4 * g]) = acc[n][j];
    __syncthreads();
    const float scale = p.scale[ad];
    const int live = min(BM, t.n - t.r0);
    float *u = p.u + (static_cast<int64_t>(blockIdx.y) * p.n_tokens + t.first + t.r0) * p.rank;
    for (int i = threadIdx.x; i < live * p.rank; i += 256) {
        const int row = i / p.rank, c = i - row * p.rank;
        u[i] = scale * ((sum[0][row][c] + sum[1][row][c]) + (sum[2][row][c] + sum[3][row][c]));
    }
}

// y = base + u B^T for a tile of 16 TT tokens and m_per_block outputs, 32 of them per wave and step. Rows of the matrix instruction
// are dealt so that a lane holds outputs 8 g .. 8 g + 7 of the 32 for its token, and four lanes a whole 128-byte line.
template <typename W, int KS, int TT, bool WIDE, bool WIDE_Y>
__global__ __launch_bounds__(256) void lora_expand(LoraArgs p) {
    constexpr int BM = 16 * TT, US = 32 * KS + 8;
    __shared__ __attribute__((aligned(16))) bf16 ut[kUTerms][BM][US];
    Run t;
    if (!find_run<BM>(p.q_start, p.n_seqs, p.n_tokens, 1, blockIdx.x, t)) return;
    const int ad = adapter_of(p, t.b);
    if (ad < 0 && p.base == p.y) return;
    const int live = min(BM, t.n - t.r0);
    const int m_first = blockIdx.y * p.m_per_block, m_end = min(m_first + p.m_per_block, p.M);
    const int64_t token0 = t.first + t.r0;
    if (ad < 0) {
        for (int row = threadIdx.x >> 6; row < live; row += 4)
            for (int m = m_first + (threadIdx.x & 63); m < m_end; m += 64) {
                const int64_t at = (token0 + row) * p.M + m;
                p.y[at] = p.base ? p.base[at] : 0.0f;
            }
        return;
    }
    for (int i = threadIdx.x; i < BM * KS * 4; i += 256) {
        const int row = i / (KS * 4), c = i % (KS * 4) * 8;
        float f[8] = {};
        if (row < live) {
            for (int z = 0; z < p.splits; ++z) {
                const float *u = p.u + (static_cast<int64_t>(z) * p.n_tokens + token0 + row) * p.rank;
                const vec<float, 8> v = load8<WIDE>(u, c, p.rank);
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] += v[e];
            }
        }
        bf16x8 terms[kUTerms];
        bf16_terms<kUTerms>(f, terms);
#pragma unroll
        for (int n = 0; n < kUTerms; ++n) *reinterpret_cast<bf16x8 *>(&ut[n][row][c]) = terms[n];
    }
    __syncthreads();
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, col = lane & 15;
    bf16x8 u[TT][KS][kUTerms];
#pragma unroll
    for (int j = 0; j < TT; ++j)
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int n = 0; n < kUTerms; ++n) u[j][s][n] = *reinterpret_cast<bf16x8 *>(&ut[n][16 * j + col][32 * s + 8 * g]);
    const W *b = static_cast<const W *>(p.b) + static_cast<int64_t>(ad) * p.M * p.rank;
    for (int m0 = m_first + 32 * wave; m0 < m_end; m0 += 128) {
        f32x4 acc[2][TT];
        const int m = m0 + 8 * g;  // the lane's outputs m .. m + 7
#pragma unroll
        for (int j = 0; j < TT; ++j) {
            const float *src = p.base ? p.base + (token0 + min(16 * j + col, live - 1)) * p.M : nullptr;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                acc[h][j] = f32x4{};
                if (!src) continue;
                if (WIDE_Y && m + 4 * h < p.M) acc[h][j] = *reinterpret_cast<const f32x4 *>(src + m + 4 * h);
                if constexpr (!WIDE_Y) {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (m + 4 * h + e < p.M) acc[h][j][e] = src[m + 4 * h + e];
                }
            }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            // row col of the instruction is output 8 (col / 4) + 4 h + col % 4 of the 32
            const int row = m0 + 8 * (col >> 2) + 4 * h + (col & 3);
            const W *br = b + static_cast<int64_t>(min(row, p.M - 1)) * p.rank;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                bf16x8 wt[kWTerms<W>];
                weight_terms<W>(load8<WIDE>(br, 32 * s + 8 * g, p.rank), wt);
#pragma unroll
                for (int w = 0; w < kWTerms<W>; ++w)
#pragma unroll
                    for (int n = 0; n < kUTerms; ++n)
                        if (w + n < 3) {
#pragma unroll
                            for (int j = 0; j < TT; ++j) acc[h][j] = mfma16(wt[w], u[j][s][n], acc[h][j]);
                        }
            }
        }
#pragma unroll
        for (int j = 0; j < TT; ++j) {
            if (16 * j + col >= live) continue;
            float *dst = p.y + (token0 + 16 * j + col) * p.M;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (WIDE_Y && m + 4 * h < p.M) *reinterpret_cast<f32x4 *>(dst + m + 4 * h) = acc[h][j];
                if constexpr (!WIDE_Y) {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (m + 4 * h + e < p.M) dst[m + 4 * h + e] = acc[h][j][e];
                }
            }
        }
    }
}

// ---- host ----------------------------------------------------------------------------------------

struct LoraPlan {
    int few;             // sequences of a token or a few: tiles of 16 tokens
    int shrink_tiles, splits;
    int expand_tiles, m_per_block;
};

int expand_tokens(int rank, bool few) { return few || rank > 128 ? 16 : rank > 64 ? 32 : 64; }

LoraPlan lora_plan(const tqhip_lora &l) {
    LoraPlan n{};
    n.few = l.n_tokens <= 16 * static_cast<int64_t>(l.n_seqs);
    n.shrink_tiles = l.n_tokens / (n.few ? 16 : 32) + l.n_seqs;
    // about two workgroups per CU, of at least two steps of 32 per wave
    const int most = std::max(1, (l.in_dim + 31) / 32 / 8);
    n.splits = std::clamp(2 * device_cu_count() / n.shrink_tiles, 1, most);
    n.expand_tiles = l.n_tokens / expand_tokens(l.rank, n.few) + l.n_seqs;
    const int64_t want = static_cast<int64_t>(l.out_dim) * n.expand_tiles / (4 * device_cu_count());
    n.m_per_block = static_cast<int>(std::clamp<int64_t>((want + 127) / 128 * 128, 128, 2048));
    return n;
}

size_t lora_bytes(const tqhip_lora &l) {
    return static_cast<size_t>(lora_plan(l).splits) * l.n_tokens * l.rank * sizeof(float);
}

int check_lora(const tqhip_lora &l) {
    if (!type_known(l.dtype) || l.n_tokens < 1 || l.in_dim < 1 || l.out_dim < 1 || l.rank < 1 || l.rank > 256 ||
        l.n_adapters < 1 || l.n_seqs < 1 || !l.x || !l.y || !l.a || !l.b || !l.scale || !l.q_start || !l.adapter)
        return kBadShape;
    // tiles in grid.x, blocks of outputs in grid.y; everything else is addressed in 64 bits
    if (static_cast<int64_t>(l.n_tokens) + l.n_seqs > INT32_MAX / 256 || l.out_dim > 65535 * 128 || l.in_dim > INT32_MAX - 64)
        return kTooLarge;
    return kOk;
}

template <typename W, int NR, bool WIDE>
void launch_shrink(const LoraArgs &p, const LoraPlan &n, hipStream_t s) {
    const dim3 grid(n.shrink_tiles, n.splits);
    if (n.few)
        lora_shrink<W, NR, 1, WIDE><<<grid, 256, 0, s>>>(p);
    else
        lora_shrink<W, NR, 2, WIDE><<<grid, 256, 0, s>>>(p);
}

template <typename W, int KS, bool WIDE>
void launch_expand(const LoraArgs &p, const LoraPlan &n, bool wide_y, hipStream_t s) {
    constexpr int TT = KS <= 2 ? 4 : KS == 4 ? 2 : 1;
    const dim3 grid(n.expand_tiles, (p.M + p.m_per_block - 1) / p.m_per_block);
    if (n.few && wide_y)
        lora_expand<W, KS, 1, WIDE, true><<<grid, 256, 0, s>>>(p);
    else if (n.few)
        lora_expand<W, KS, 1, WIDE, false><<<grid, 256, 0, s>>>(p);
    else if (wide_y)
        lora_expand<W, KS, TT, WIDE, true><<<grid, 256, 0, s>>>(p);
    else
        lora_expand<W, KS, TT, WIDE, false><<<grid, 256, 0, s>>>(p);
}

template <typename W>
void launch_lora(const LoraArgs &p, const LoraPlan &n, hipStream_t s) {
    const auto on16 = [](const void *q) { return reinterpret_cast<uintptr_t>(q) % 16 == 0; };
    const bool wide_a = p.K % 8 == 0 && on16(p.x) && on16(p.a), wide_b = p.rank % 8 == 0 && on16(p.b) && on16(p.u);
    const bool wide_y = p.M % 4 == 0 && on16(p.y) && on16(p.base);
    const auto shrink = [&](auto wide) {
        if (p.rank <= 16)
            launch_shrink<W, 1, wide.value>(p, n, s);
        else if (p.rank <= 32)
            launch_shrink<W, 2, wide.value>(p, n, s);
        else if (p.rank <= 64)
            launch_shrink<W, 4, wide.value>(p, n, s);
        else if (p.rank <= 128)
            launch_shrink<W, 8, wide.value>(p, n, s);
        else
            launch_shrink<W, 16, wide.value>(p, n, s);
    };
    const auto expand = [&](auto wide) {
        if (p.rank <= 32)
            launch_expand<W, 1, wide.value>(p, n, wide_y, s);
        else if (p.rank <= 64)
            launch_expand<W, 2, wide.value>(p, n, wide_y, s);
        else if (p.rank <= 128)
            launch_expand<W, 4, wide.value>(p, n, wide_y, s);
        else
            launch_expand<W, 8, wide.value>(p, n, wide_y, s);
    };
    if (wide_a)
        shrink(std::true_type{});
    else
        shrink(std::false_type{});
    if (wide_b)
        expand(std::true_type{});
    else
        expand(std::false_type{});
}

int run_lora(const tqhip_lora &l, hipStream_t s) {
    int st = check_lora(l);
    if (st != kOk) return st;
    const size_t bytes = lora_bytes(l);
    void *ws = l.workspace;
    if (ws && l.workspace_bytes < bytes) return kNoScratch;
    if (!ws && (st = scratch_batch(s, bytes, &ws)) != kOk) return st;
    const LoraPlan n = lora_plan(l);
    const LoraArgs p{l.x, l.base, l.y, l.a, l.b, l.scale, l.q_start, l.adapter, static_cast<float *>(ws), l.n_tokens,
                     l.in_dim, l.out_dim, l.rank, l.n_adapters, l.n_seqs, n.splits, n.m_per_block};
    switch (l.dtype) {
        case TQHIP_F32: launch_lora<float>(p, n, s); break;
        case TQHIP_F16: launch_lora<f16>(p, n, s); break;
        default: launch_lora<bf16>(p, n, s); break;
    }
    return hipGetLastError() == hipSuccess ? kOk : kLaunchFailed;
}

}  // namespace
}  // namespace tqhip

extern "C" {

int tqhip_lora_add_dev(const tqhip_lora *lora, void *stream) {
    if (!lora) return tqhip::kBadShape;
    try {
        return tqhip::run_lora(*lora, static_cast<hipStream_t>(stream));
    } catch (...) {  // (host memory ran out)
        return tqhip::kHipFailed;
    }
}

size_t tqhip_lora_workspace(const tqhip_lora *lora) {
    return lora && tqhip::check_lora(*lora) == tqhip::kOk ? tqhip::lora_bytes(*lora) : 0;
}

}  // extern "C"
