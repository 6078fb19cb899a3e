// lora.hip -- the low-rank adapters of many requests beside the projection that they share:
// y_t = base_t + scale[a] * B_a (A_a x_t), a the adapter of t's request.
//
// Two launches. The first forms u = scale A x (few numbers: rank of them per token), the second adds B u to base. A tile
// is a run of tokens of one sequence, so it has one adapter, whatever the order of the adapters over the requests.
// Both are products on the matrix cores in bf16 terms: an fp32 operand (x, u, fp32 weights) is three
// of them (24 bits), an fp16 weight two (all 11 bits, and fp16's range), a bf16 weight one; products below 2^-24 are
// left out. So fp32 results keep fp32's precision at 3 to 6 matrix instructions a product, where the fp32 ones take 16.
// An infinity is its first term, and no number beside the zero or the other sign of the other operand's next one: results that
// are not finite are formed again by the formula, in 64 bits, by the threads that have them. The loops carry nothing for it.
//
// Both launches are bound by HBM (x once; base and y once) or, with few tokens, by latency. 3555 tokens of 8
// requests, rank 64 in bf16 beside 9728x2560: 26 and 73 us; the second reads base and u, 139 MB, and writes as much, and as its tiles of one
// block of outputs go to all XCDs, each of those reads all of B into its L2, another 60 MB. 64 requests of a token, rank 16 in fp16 beside
// 4096x2560: 5.8 and 7 us. Requests of one token are a tile each, also where they share an adapter: 256 of them, rank 64 beside
// 9728x2560, take 28 and 57 us for one adapter or four.
#include <algorithm>
#include <optional>
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
    int splits;
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

// Elements at .. at + 7 of a row of n, zeros past its end. WIDE: n is a multiple of 8 and rows are 16-byte aligned; the load is
// then unconditional, so that the compiler can count it among those that may stay under way at a wait.
template <bool WIDE, typename T>
__device__ inline vec<T, 8> load8(const T *row, int at, int n) {
    vec<T, 8> v{};
    if constexpr (WIDE) {
        v = *reinterpret_cast<const vec<T, 8> *>(row + min(at, n - 8));
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = at < n ? v[i] : static_cast<T>(0.0f);
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

// u^T = A x^T for a tile of 16 tokens: the lane holds ranks 16 n + 4 g + i of token lane % 16. The steps of 32 along K are dealt to
// the workgroup's waves, whose sums meet in LDS, and to gridDim.y workgroups where there are fewer tiles than CUs, whose sums
// meet in lora_expand. x is read once. The launch lasts as long as one wave's loads one after the other, so the waves are many and
// their steps few: 16 waves of 5 steps at K = 2560. (4 waves, 32 tokens and 4 workgroups a tile took 21 us for 3555 tokens, and
// the four sums of u cost every workgroup of lora_expand as many bytes as its outputs.)
template <int NR>
constexpr int kShrinkWaves = NR <= 4 ? 16 : 8;

template <typename W, int NR, bool WIDE>
__global__ __launch_bounds__(64 * kShrinkWaves<NR>) void lora_shrink(LoraArgs p) {
    constexpr int BM = 16, NW = kShrinkWaves<NR>;
    __shared__ float sum[NW][BM][16 * NR + 4];
    Run t;
    if (!find_run<BM>(p.q_start, p.n_seqs, p.n_tokens, 1, blockIdx.x, t)) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, col = lane & 15;
    const int steps = (p.K + 31) / 32, workers = NW * p.splits, worker = blockIdx.y * NW + wave;
    const int s0 = static_cast<int>(static_cast<int64_t>(steps) * worker / workers);
    const int s1 = static_cast<int>(static_cast<int64_t>(steps) * (worker + 1) / workers);
    const float *x = p.x + static_cast<int64_t>(t.first + min(t.r0 + col, t.n - 1)) * p.K;
    vec<float, 8> xv = load8<WIDE>(x, 32 * s0 + 8 * g, p.K);  // (under way while the adapter is looked up)
    const int ad = adapter_of(p, t.b);
    if (ad < 0) return;
    const W *a = static_cast<const W *>(p.a) + static_cast<int64_t>(ad) * p.rank * p.K;
    vec<W, 8> av[NR];
    const auto load_weights = [&](int s) {
#pragma unroll
        for (int n = 0; n < NR; ++n)
            av[n] = load8<WIDE>(a + static_cast<int64_t>(min(16 * n + col, p.rank - 1)) * p.K, 32 * s + 8 * g, p.K);
    };
    load_weights(s0);
    f32x4 acc[NR];
#pragma unroll
    for (int n = 0; n < NR; ++n) acc[n] = f32x4{};
    for (int s = s0; s < s1; ++s) {
        bf16x8 xt[kUTerms];
        float f[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = xv[e];
        bf16_terms<kUTerms>(f, xt);
        const int ahead = min(s + 1, s1 - 1);  // the next step's operands are under way during this step's products
        xv = load8<WIDE>(x, 32 * ahead + 8 * g, p.K);
        vec<W, 8> now[NR];
#pragma unroll
        for (int n = 0; n < NR; ++n) now[n] = av[n];
        load_weights(ahead);
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            bf16x8 wt[kWTerms<W>];
            weight_terms<W>(now[n], wt);
#pragma unroll
            for (int w = 0; w < kWTerms<W>; ++w)
#pragma unroll
                for (int u = 0; u < kUTerms; ++u)
                    if (w + u < 3) acc[n] = mfma16(wt[w], xt[u], acc[n]);
        }
    }
#pragma unroll
    for (int n = 0; n < NR; ++n) *reinterpret_cast<f32x4 *>(&sum[wave][col][16 * n + 4 * g]) = acc[n];
    __syncthreads();
    const float scale = p.scale[ad];
    const int live = min(BM, t.n - t.r0);
    float *u = p.u + (static_cast<int64_t>(blockIdx.y) * p.n_tokens + t.first + t.r0) * p.rank;
    bool odd = false;
    for (int i = threadIdx.x; i < live * p.rank; i += 64 * NW) {
        const int row = i / p.rank, c = i - row * p.rank;
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; ++w) v += sum[w][row][c];
        odd = odd || v * 0.0f != 0.0f;
        u[i] = scale * v;
    }
    if (!odd) return;
    // the thread's infinite and NaN sums by the formula, over what the workgroup's waves had
    const int64_t k0 = 32 * (static_cast<int64_t>(steps) * blockIdx.y * NW / workers);
    const int64_t k1 = min(32 * (static_cast<int64_t>(steps) * (blockIdx.y + 1) * NW / workers), static_cast<int64_t>(p.K));
#pragma unroll 1
    for (int i = threadIdx.x; i < live * p.rank; i += 64 * NW) {
        const int row = i / p.rank, c = i - row * p.rank;
        if (u[i] * 0.0f == 0.0f) continue;
        const float *xr = p.x + static_cast<int64_t>(t.first + t.r0 + row) * p.K;
        const W *ar = a + static_cast<int64_t>(c) * p.K;
        double v = 0.0;
#pragma unroll 1
        for (int64_t k = k0; k < k1 && v == v; ++k) v += static_cast<double>(xr[k]) * static_cast<float>(ar[k]);
        u[i] = scale * static_cast<float>(v);
    }
}

// One output by the formula.
template <typename W>
__device__ inline float formula_output(const float *base, const float *u, const W *b, int rank, int splits, int64_t split_stride) {
    double v = base ? *base : 0.0f;
#pragma unroll 1
    for (int r = 0; r < rank && v == v; ++r) {
        float u_r = 0.0f;
#pragma unroll 1
        for (int z = 0; z < splits; ++z) u_r += u[z * split_stride + r];
        v += static_cast<double>(u_r) * static_cast<float>(b[r]);
    }
    return static_cast<float>(v);
}

// y = base + u B^T for a tile of 16 TT tokens and 128 S outputs, 32 of them per wave and step: the lane holds outputs
// 4 g + 16 h .. + 3 of a step for token 16 j + lane % 16. All of the wave's base is requested first and under way while u is put
// together, and nothing is stored before it is all there: with the next step's base requested between the stores, in fewer and longer
// workgroups, 8 prompts of up to 600 tokens beside 9728x2560 took 125 us instead of 99 (a load waits for the stores before it,
// and reads and writes take turns at the memory).
template <typename W, int KS, int TT, int S, bool WIDE, bool WIDE_Y>
__global__ __launch_bounds__(256) void lora_expand(LoraArgs p) {
    constexpr int BM = 16 * TT, US = 32 * KS + 8;
    __shared__ __attribute__((aligned(16))) bf16 ut[kUTerms][BM][US];
    Run t;
    if (!find_run<BM>(p.q_start, p.n_seqs, p.n_tokens, 1, blockIdx.x, t)) return;
    const int live = min(BM, t.n - t.r0);
    const int m_first = blockIdx.y * 128 * S, m_end = min(m_first + 128 * S, p.M);
    const int64_t token0 = t.first + t.r0;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, col = lane & 15;
    f32x4 acc[S][2][TT];
#pragma unroll
    for (int j = 0; j < TT; ++j) {
        const float *src = p.base + (token0 + min(16 * j + col, live - 1)) * p.M;
#pragma unroll
        for (int i = 0; i < S; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int m = m_first + 128 * i + 32 * wave + 16 * h + 4 * g;
                acc[i][h][j] = f32x4{};
                if (!p.base) continue;
                if constexpr (WIDE_Y) {
                    acc[i][h][j] = *reinterpret_cast<const f32x4 *>(src + min(m, p.M - 4));
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[i][h][j][e] = src[min(m + e, p.M - 1)];
                }
            }
    }
    const int ad = adapter_of(p, t.b);
    if (ad < 0) {
        if (p.base == p.y) return;
        for (int row = wave; row < live; row += 4)
            for (int m = m_first + lane; m < m_end; m += 64) {
                const int64_t at = (token0 + row) * p.M + m;
                p.y[at] = p.base ? p.base[at] : 0.0f;
            }
        return;
    }
    const W *b = static_cast<const W *>(p.b) + static_cast<int64_t>(ad) * p.M * p.rank;
    vec<W, 8> bv[S][2][KS];
#pragma unroll
    for (int i = 0; i < S; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int s = 0; s < KS; ++s)
                bv[i][h][s] = load8<WIDE>(b + static_cast<int64_t>(min(m_first + 128 * i + 32 * wave + 16 * h + col, p.M - 1)) * p.rank,
                                          32 * s + 8 * g, p.rank);
    for (int i = threadIdx.x; i < BM * KS * 4; i += 256) {
        const int row = i / (KS * 4), c = i % (KS * 4) * 8;
        float f[8] = {};
        if (row < live) {
            for (int z = 0; z < p.splits; z += 4) {  // four parts' loads at a time
                vec<float, 8> v[4];
#pragma unroll
                for (int y = 0; y < 4; ++y)
                    v[y] = load8<WIDE>(p.u + (static_cast<int64_t>(min(z + y, p.splits - 1)) * p.n_tokens + token0 + row) * p.rank, c, p.rank);
#pragma unroll
                for (int y = 0; y < 4; ++y)
#pragma unroll
                    for (int e = 0; e < 8; ++e) f[e] += z + y < p.splits ? v[y][e] : 0.0f;
            }
        }
        bf16x8 terms[kUTerms];
        bf16_terms<kUTerms>(f, terms);
#pragma unroll
        for (int n = 0; n < kUTerms; ++n) *reinterpret_cast<bf16x8 *>(&ut[n][row][c]) = terms[n];
    }
    __syncthreads();
    bf16x8 u[TT][KS][kUTerms];
#pragma unroll
    for (int j = 0; j < TT; ++j)
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int n = 0; n < kUTerms; ++n) u[j][s][n] = *reinterpret_cast<bf16x8 *>(&ut[n][16 * j + col][32 * s + 8 * g]);
#pragma unroll
    for (int i = 0; i < S; ++i) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                bf16x8 wt[kWTerms<W>];
                weight_terms<W>(bv[i][h][s], wt);
#pragma unroll
                for (int w = 0; w < kWTerms<W>; ++w)
#pragma unroll
                    for (int n = 0; n < kUTerms; ++n)
                        if (w + n < 3) {
#pragma unroll
                            for (int j = 0; j < TT; ++j) acc[i][h][j] = mfma16(wt[w], u[j][s][n], acc[i][h][j]);
                        }
            }
        }
    }
    // Which of the lane's groups of 8 outputs are not all finite (or so large that products of pairs are not): they are not stored here,
    // for base may be y.
    unsigned again = 0;
#pragma unroll
    for (int i = 0; i < S; ++i)
#pragma unroll
        for (int j = 0; j < TT; ++j) {
            float z = 0.0f;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int e = 0; e < 4; e += 2) z = fmaf(acc[i][h][j][e], acc[i][h][j][e + 1], z);
            z *= 0.0f;
            again |= static_cast<unsigned>(z != 0.0f) << (i * TT + j);
            if (16 * j + col >= live || z != 0.0f) continue;
            float *dst = p.y + (token0 + 16 * j + col) * p.M;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int m = m_first + 128 * i + 32 * wave + 16 * h + 4 * g;
                if (WIDE_Y && m < p.M) *reinterpret_cast<f32x4 *>(dst + m) = acc[i][h][j];
                if constexpr (!WIDE_Y) {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (m + e < p.M) dst[m + e] = acc[i][h][j][e];
                }
            }
        }
    if (__builtin_expect(again == 0, 1)) return;
#pragma unroll 1
    for (; again; again &= again - 1) {
        const int i = __builtin_ctz(again) / TT, j = __builtin_ctz(again) % TT;
        const int64_t token = token0 + 16 * j + col;
        if (16 * j + col >= live) continue;
#pragma unroll 1
        for (int n = 0; n < 8; ++n) {
            const int m = m_first + 128 * i + 32 * wave + 16 * (n >> 2) + 4 * g + (n & 3);
            if (m >= p.M) continue;
            const int64_t at = token * p.M + m;
            p.y[at] = formula_output(p.base ? p.base + at : nullptr, p.u + token * p.rank, b + static_cast<int64_t>(m) * p.rank, p.rank, p.splits,
                                     static_cast<int64_t>(p.n_tokens) * p.rank);
        }
    }
}

// ---- host ----------------------------------------------------------------------------------------

struct LoraPlan {
    bool few;  // sequences of a token or a few: tiles of 16 tokens
    int shrink_tiles, splits, expand_tiles;
};

constexpr int kLoraSteps = 2;  // of a wave in lora_expand, 1 with few tokens

int expand_tokens(int rank, bool few) { return few || rank > 128 ? 16 : 32; }

LoraPlan lora_plan(const tqhip_lora &l) {
    LoraPlan n{};
    n.few = l.n_tokens <= 16 * static_cast<int64_t>(l.n_seqs);
    n.shrink_tiles = l.n_tokens / 16 + l.n_seqs;
    // fewer tiles than CUs: several workgroups a tile, of at least a step of 32 per wave
    const int most = std::max(1, (l.in_dim + 31) / 32 / (l.rank <= 64 ? kShrinkWaves<4> : kShrinkWaves<8>));
    n.splits = std::clamp(device_cu_count() / n.shrink_tiles, 1, std::min(most, 8));
    n.expand_tiles = l.n_tokens / expand_tokens(l.rank, n.few) + l.n_seqs;
    return n;
}

size_t lora_bytes(const tqhip_lora &l) {
    return static_cast<size_t>(lora_plan(l).splits) * l.n_tokens * l.rank * sizeof(float);
}

int check_lora(const tqhip_lora &l) {
    if (!type_known(l.dtype) || l.n_tokens < 1 || l.in_dim < 1 || l.out_dim < 1 || l.rank < 1 || l.rank > 256 ||
        l.n_adapters < 1 || l.n_seqs < 1 || !l.x || !l.y || !l.a || !l.b || !l.scale || !l.q_start || !l.adapter)
        return kBadShape;
    // tiles of at least 16 tokens in grid.x, of up to 1024 threads, blocks of outputs in grid.y; everything else is addressed in 64 bits
    if (static_cast<int64_t>(l.n_tokens) / 16 + l.n_seqs > INT32_MAX / 1024 || l.n_tokens > INT32_MAX / 16 || l.out_dim > 65535 * 128 ||
        l.in_dim > INT32_MAX - 64)
        return kTooLarge;
    return kOk;
}

template <typename W, int NR, bool WIDE>
void launch_shrink(const LoraArgs &p, const LoraPlan &n, hipStream_t s) {
    lora_shrink<W, NR, WIDE><<<dim3(n.shrink_tiles, n.splits), 64 * kShrinkWaves<NR>, 0, s>>>(p);
}

template <typename W, int KS, bool WIDE>
void launch_expand(const LoraArgs &p, const LoraPlan &n, bool wide_y, hipStream_t s) {
    constexpr int TT = KS <= 4 ? 2 : 1, S = kLoraSteps;
    const int steps = n.few ? 1 : S;
    const dim3 grid(n.expand_tiles, (p.M + 128 * steps - 1) / (128 * steps));
    if (n.few && wide_y)
        lora_expand<W, KS, 1, 1, WIDE, true><<<grid, 256, 0, s>>>(p);
    else if (n.few)
        lora_expand<W, KS, 1, 1, WIDE, false><<<grid, 256, 0, s>>>(p);
    else if (wide_y)
        lora_expand<W, KS, TT, S, WIDE, true><<<grid, 256, 0, s>>>(p);
    else
        lora_expand<W, KS, TT, S, WIDE, false><<<grid, 256, 0, s>>>(p);
}

template <typename W>
void launch_lora(const LoraArgs &p, const LoraPlan &n, hipStream_t s) {
    const auto on16 = [](const void *q) { return reinterpret_cast<uintptr_t>(q) % 16 == 0; };
    const bool wide_a = p.K % 8 == 0 && on16(p.x) && on16(p.a), wide_b = p.rank % 8 == 0 && on16(p.b);
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
    if (reinterpret_cast<uintptr_t>(ws) % 256) return kBadShape;
    if (ws && l.workspace_bytes < bytes) return kNoScratch;
    std::optional<ScratchCall> call;
    if (!ws) {
        call.emplace(s);
        if ((st = call->workspace(bytes, &ws)) != kOk) return st;
    }
    const LoraPlan n = lora_plan(l);
    const LoraArgs p{l.x, l.base, l.y, l.a, l.b, l.scale, l.q_start, l.adapter, static_cast<float *>(ws), l.n_tokens,
                     l.in_dim, l.out_dim, l.rank, l.n_adapters, l.n_seqs, n.splits};
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
