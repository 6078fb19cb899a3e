// append8.hip -- the heads of a batch of tokens finished as in heads.hip, their keys and values going to a paged cache of 8-bit codes with a
// scale for each block of tokens and head.
//
// Of the rows that a call brings to a block: scale = max(largest |x| / top, 2^-60), top 127 or 448, code = x / scale rounded to nearest even. A block that
// has rows already keeps its scale if that is larger; if not, its codes become code * old / new, rounded again. A block that is given an
// infinity or NaN gets a scale of NaN, so all of it is NaN, until it is written anew from its first row.
//
// A wave takes one block's keys, or its values, of one head: that is where the largest is needed, and no other wave touches
// the block's codes or scale. Its rows lie side by side as in heads.hip (a head in D / (2 V) lanes), all of them in registers while they
// fit (32, 16 or 8 fp32 rows of 64, 128 or 256); a larger block is a workgroup's, and one past four times that is read twice. Of blocks of
// few rows it takes several heads side by side.
// Bytes moved are the bound of a long batch, latency (sequence, page, rows, the block's scale) that of a short one. 12520 tokens of 14 + 2 + 2
// heads of 64, 106 MB: 23 to 26 us, 4.1 to 4.6 TB/s, a copy's rate; 61 single tokens: 11 us where two blocks in five get a larger scale, or all of them, and
// the older rows' codes are read and written again; 7 to 8.5 where none does.
// The queries that ride along are the same launch's, finished as heads.h does it (a launch of their own where something is off the vector path).
#include <algorithm>
#include <cmath>

#include "heads.h"

namespace tqhip {
namespace {

constexpr int kAppendThreads = 256;
constexpr float kLeastBlockScale = 0x1p-60f;

struct Append8Args {
    const void *in[2];  // k, v
    int64_t in_stride[2];
    const float *bias[2], *norm;
    unsigned char *cache[2];
    float *scales;
    int n_tokens, heads, rot, dtype, tiles;
    int side;  // heads that a wave takes side by side (a power of two), where KEEP is 1
    float eps;
    double log2_theta;
    const float *inv_freq;
    const int *positions;
    const int *q_start, *kv_len;
    int n_seqs;
    Pages pages;
    FastDiv block;
    int blocks;
};

// The blocks that a batch's new tokens lie in, numbered over the batch without a scan of the lengths: sequence b's start at
// floor(start[b] / block) + 2 b, which leaves room for the floor(n / block) + 2 that n tokens can touch.
struct NewRows {
    int b, token0, pos0, pos1;  // positions [pos0, pos1) of the sequence are new in this block; token0 is pos0's
};
__device__ inline bool find_block(const Append8Args &a, int tile, NewRows &r) {
    const int lane = threadIdx.x & 63;
    int lo = 0, n = a.n_seqs;
    const auto start = [&](int b) { return min(max(a.q_start[b], 0), a.n_tokens); };
    const auto base = [&](int b) { return a.block.quot(start(b)) + 2 * b; };
    for (;;) {
        const int step = (n + 63) / 64, i = lane * step;
        const int c = __popcll(__ballot(i < n && base(lo + i) <= tile));
        if (c == 0) return false;
        lo += (c - 1) * step;
        n = min(step, n - (c - 1) * step);
        if (step == 1) break;
    }
    const int first = start(lo), count = start(lo + 1) - first, kv = max(a.kv_len[lo], 0);
    const int from = max(kv - count, 0), block = static_cast<int>(a.block.d);  // (tokens before position 0 are not written)
    if (count <= 0 || kv == 0) return false;
    const int64_t at = (static_cast<int64_t>(a.block.quot(from)) + tile - base(lo)) * block;
    if (at >= kv) return false;
    r.b = lo;
    r.pos0 = max(static_cast<int>(at), from);
    r.pos1 = static_cast<int>(min(at + block, static_cast<int64_t>(kv)));
    r.token0 = first + r.pos0 - (kv - count);
    return true;
}

// x / scale as the code's bits.
__device__ inline unsigned to_code(float x, int dtype) {
    if (dtype == TQHIP_I8) return static_cast<unsigned>(static_cast<int>(rintf(fminf(fmaxf(x, -127.0f), 127.0f)))) & 0xff;
    const float y = fminf(fmaxf(x, -448.0f), 448.0f);
    return static_cast<unsigned>(__builtin_amdgcn_cvt_pk_fp8_f32(y, y, 0, false)) & 0xff;
}
__device__ inline unsigned four_codes(const float *x, int dtype) {
    return to_code(x[0], dtype) | to_code(x[1], dtype) << 8 | to_code(x[2], dtype) << 16 | to_code(x[3], dtype) << 24;
}
// A word of codes of one scale as those of another.
__device__ inline unsigned recode(unsigned u, float ratio, int dtype) {
    float x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int byte = static_cast<int>(u << (24 - 8 * i)) >> 24;
        x[i] = (dtype == TQHIP_I8 ? static_cast<float>(byte) : __builtin_amdgcn_cvt_f32_fp8(byte, 0)) * ratio;
    }
    return four_codes(x, dtype);
}

// D: head dimension; V: elements per load (1: any rotary dimension and alignment); WAVES: of a block's head; KEEP: rounds of rows held in
// registers, 0: none, they are read and finished twice; 1: the wave's rows are those of `side` heads.
template <typename T, int D, int V, int WAVES, int KEEP>
__device__ inline void append_block(const Append8Args &a) {
    constexpr int LPR = D / (2 * V) < 64 ? D / (2 * V) : 64, NU = D / (2 * V) / LPR, RPW = 64 / LPR;
    const int side = KEEP == 1 ? a.side : 1, per = RPW / side, kRows = per * WAVES;  // rows of a head in the wave, and in a round
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int unit = WAVES == 1 ? blockIdx.x * 4 + wave : blockIdx.x, mine = WAVES == 1 ? 0 : wave;
    const int sub = lane / LPR, row_lane = sub % per;
    const int times = (a.heads + side - 1) / side, tile = unit / (2 * times), kv = unit % (2 * times) / times;
    const int head = unit % times * side + (KEEP == 1 ? sub / per : 0), h = min(head, a.heads - 1);
    NewRows r;
    if (tile >= a.tiles || !find_block(a, tile, r)) return;
    const int page = page_number(a.pages, r.b, r.pos0);
    const int64_t row0 = row_in_page(a.pages, page, r.pos0);
    if (row0 < 0) return;
    const int n = r.pos1 - r.pos0, half = a.rot / 2;

    int at0[NU], at1[NU];
    bool turned[NU];
    double freq[NU][V];
    float bias0[NU][V], bias1[NU][V], norm0[NU][V], norm1[NU][V];
#pragma unroll
    for (int j = 0; j < NU; ++j) {
        const int u = lane % LPR + LPR * j, rot_units = half / V;
        turned[j] = kv == 0 && u < rot_units;
        at0[j] = u < rot_units ? u * V : a.rot + 2 * V * (u - rot_units);
        at1[j] = u < rot_units ? half + u * V : at0[j] + V;
        constexpr double kInvTwoPi = 0.15915494309189535;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const int i = at0[j] + e;
            freq[j][e] = turned[j] ? (a.inv_freq ? static_cast<double>(a.inv_freq[i]) : exp2(-a.log2_theta * i / half)) * kInvTwoPi : 0.0;
            bias0[j][e] = bias1[j][e] = 0.0f;
        }
        if (a.bias[kv]) {
            load_as_float<float, V>(a.bias[kv] + h * D + at0[j], bias0[j]);
            load_as_float<float, V>(a.bias[kv] + h * D + at1[j], bias1[j]);
        }
        if (kv == 0 && a.norm) {
            load_as_float<float, V>(a.norm + at0[j], norm0[j]);
            load_as_float<float, V>(a.norm + at1[j], norm1[j]);
        }
    }
    const T *in = static_cast<const T *>(a.in[kv]) + h * D;
    struct Raw {
        vec<T, V> x0[NU], x1[NU];
    };
    // the row of a round that the lane has part in (past the last: the last again)
    const auto row_of = [&](int round) { return min(round * kRows + mine * per + row_lane, n - 1); };
    const auto load = [&](int round, Raw &x) {
        const T *src = in + static_cast<int64_t>(r.token0 + row_of(round)) * a.in_stride[kv];
#pragma unroll
        for (int j = 0; j < NU; ++j) {
            x.x0[j] = *reinterpret_cast<const vec<T, V> *>(src + at0[j]);
            x.x1[j] = *reinterpret_cast<const vec<T, V> *>(src + at1[j]);
        }
    };
    struct Row {
        float x0[NU][V], x1[NU][V];
    };
    const auto finish = [&](int round, const Raw &raw, Row &x) {
        float sq = 0.0f;
#pragma unroll
        for (int j = 0; j < NU; ++j)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                x.x0[j][e] = static_cast<float>(raw.x0[j][e]) + bias0[j][e];
                x.x1[j][e] = static_cast<float>(raw.x1[j][e]) + bias1[j][e];
                sq += x.x0[j][e] * x.x0[j][e] + x.x1[j][e] * x.x1[j][e];
            }
        if (kv) return;
        if (a.norm) {
#pragma unroll
            for (int d = 1; d < LPR; d *= 2) sq += __shfl_xor(sq, d);
            const float s = 1.0f / sqrtf(sq / D + a.eps);
#pragma unroll
            for (int j = 0; j < NU; ++j)
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    x.x0[j][e] = x.x0[j][e] * s * norm0[j][e];
                    x.x1[j][e] = x.x1[j][e] * s * norm1[j][e];
                }
        }
        const int i = row_of(round), pos = a.positions ? a.positions[r.token0 + i] : r.pos0 + i;
#pragma unroll
        for (int j = 0; j < NU; ++j)
            if (turned[j]) {
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const double w = pos * freq[j][e];
                    float s, c;
                    sincospif(static_cast<float>(2.0 * (w - rint(w))), &s, &c);
                    const float y0 = x.x0[j][e], y1 = x.x1[j][e];
                    x.x0[j][e] = y0 * c - y1 * s;
                    x.x1[j][e] = y1 * c + y0 * s;
                }
            }
    };
    // The largest size as bits, in which infinities and NaN are larger than any number.
    unsigned top = 0;
    const auto take_top = [&](const Row &x) {
#pragma unroll
        for (int j = 0; j < NU; ++j)
#pragma unroll
            for (int e = 0; e < V; ++e)
                top = max(top, max(__float_as_uint(x.x0[j][e]) & 0x7fffffffu, __float_as_uint(x.x1[j][e]) & 0x7fffffffu));
    };
    unsigned char *cache = a.cache[kv] + h * a.pages.head_stride;
    const auto store = [&](int round, const Row &x, float scale, bool bad) {
        const int i = round * kRows + mine * per + row_lane;
        if (i >= n || (KEEP == 1 && head != h)) return;
        unsigned char *dst = cache + row0 + i * a.pages.token_stride;
#pragma unroll
        for (int j = 0; j < NU; ++j) {
            float y0[V], y1[V];
#pragma unroll
            for (int e = 0; e < V; ++e) {
                y0[e] = bad ? 0.0f : x.x0[j][e] / scale;
                y1[e] = bad ? 0.0f : x.x1[j][e] / scale;
            }
            if constexpr (V == 1) {
                dst[at0[j]] = static_cast<unsigned char>(to_code(y0[0], a.dtype));
                dst[at1[j]] = static_cast<unsigned char>(to_code(y1[0], a.dtype));
            } else {
                vec<unsigned, V / 4> u0, u1;
#pragma unroll
                for (int e = 0; e < V; e += 4) {
                    u0[e / 4] = four_codes(y0 + e, a.dtype);
                    u1[e / 4] = four_codes(y1 + e, a.dtype);
                }
                *reinterpret_cast<vec<unsigned, V / 4> *>(dst + at0[j]) = u0;
                *reinterpret_cast<vec<unsigned, V / 4> *>(dst + at1[j]) = u1;
            }
        }
    };

    const int in_page = r.pos0 - a.pages.page_size.quot(r.pos0) * static_cast<int>(a.pages.page_size.d);
    const int blk = a.block.quot(in_page), older = in_page - blk * static_cast<int>(a.block.d);  // rows that the block has already
    float *scale_at = a.scales + 2 * ((static_cast<int64_t>(page) * a.heads + h) * a.blocks + blk) + kv;
    const float old = *scale_at;
    const int rounds = (n + kRows - 1) / kRows;
    Row x[KEEP ? KEEP : 1];
    if constexpr (KEEP > 0) {
        Raw raw[KEEP];
#pragma unroll
        for (int i = 0; i < KEEP; ++i)
            if (i < rounds) load(i, raw[i]);
#pragma unroll
        for (int i = 0; i < KEEP; ++i)
            if (i < rounds) {
                finish(i, raw[i], x[i]);
                take_top(x[i]);
            }
    } else {
        for (int i = 0; i < rounds; ++i) {
            Raw raw;
            load(i, raw);
            finish(i, raw, x[0]);
            take_top(x[0]);
        }
    }
#pragma unroll
    for (int d = 1; d < 64; d *= 2)
        if (KEEP != 1 || d < LPR * per) top = max(top, static_cast<unsigned>(__shfl_xor(static_cast<int>(top), d)));
    if constexpr (WAVES > 1) {
        __shared__ unsigned top_of[WAVES];
        if (lane == 0) top_of[wave] = top;
        __syncthreads();  // (the whole workgroup is here: it has one block and head)
#pragma unroll
        for (int w = 0; w < WAVES; ++w) top = max(top, top_of[w]);
    }
    float scale = fmaxf(__uint_as_float(top) / (a.dtype == TQHIP_I8 ? 127.0f : 448.0f), kLeastBlockScale);
    if (older > 0 && !(old <= scale)) scale = old;  // (larger, or NaN)
    if (top >= 0x7f800000u) scale = NAN;
    const bool bad = !(scale < INFINITY);
    if (older > 0 && scale != old && !bad && (KEEP != 1 || head == h)) {
        // 16 codes a lane
        const float ratio = old / scale;
        constexpr int LANES = D / 16;
        const int lanes = KEEP == 1 ? LPR * per : 64, of = lane % lanes, rows = lanes / LANES;  // (of a head)
        unsigned char *from = cache + row0 - static_cast<int64_t>(older) * a.pages.token_stride;
        for (int i = mine * rows + of / LANES; i < older; i += rows * WAVES) {
            vec<unsigned, 4> *p = reinterpret_cast<vec<unsigned, 4> *>(from + i * a.pages.token_stride + of % LANES * 16);
            vec<unsigned, 4> u = *p;
#pragma unroll
            for (int w = 0; w < 4; ++w) u[w] = recode(u[w], ratio, a.dtype);
            *p = u;
        }
    }
    if constexpr (KEEP > 0) {
#pragma unroll
        for (int i = 0; i < KEEP; ++i)
            if (i < rounds) store(i, x[i], scale, bad);
    } else {
        for (int i = 0; i < rounds; ++i) {
            Raw raw;
            load(i, raw);
            finish(i, raw, x[0]);
            store(i, x[0], scale, bad);
        }
    }
    if (lane % LPR == 0 && row_lane == 0 && mine == 0 && (KEEP != 1 || head == h)) *scale_at = scale;
}

// The first `blocks` workgroups take the keys and values, those after them the queries.
template <typename T, int D, int V, int WAVES, int KEEP>
__global__ __launch_bounds__(kAppendThreads) void append8(Append8Args a, HeadArgs q, int blocks) {
    if (static_cast<int>(blockIdx.x) < blocks)
        append_block<T, D, V, WAVES, KEEP>(a);
    else if constexpr (V > 1)
        finish_heads<T, T, V, D / (2 * V), true>(q, blockIdx.x - blocks);
}

// with_q: the queries are this launch's.
template <typename T, int D, int V, int WAVES, int KEEP>
int launch_append(const Append8Args &a, HeadArgs q, bool with_q, hipStream_t s) {
    const int side = KEEP == 1 ? a.side : 1;
    const int64_t units = static_cast<int64_t>(a.tiles) * 2 * ((a.heads + side - 1) / side), blocks = WAVES == 1 ? (units + 3) / 4 : units;
    const int64_t groups = blocks + (with_q ? plan_heads(q, D / (2 * V)) : 0);
    if (groups > INT32_MAX / kAppendThreads) return kTooLarge;
    append8<T, D, V, WAVES, KEEP><<<static_cast<unsigned>(groups), kAppendThreads, 0, s>>>(a, q, static_cast<int>(blocks));
    return hipGetLastError() == hipSuccess ? kOk : kLaunchFailed;
}

template <typename T, int D>
int launch_append_dim(Append8Args a, const HeadArgs &q, bool with_q, bool wide, hipStream_t s) {
    constexpr int V = 16 / sizeof(T), kRound = 64 / (D / (2 * V));
    if (!wide) return launch_append<T, D, 1, 4, 0>(a, q, false, s);
    const int block = static_cast<int>(a.block.d);
    // Blocks that leave lanes without a row, several heads a wave (7600 tokens of 32 + 8 heads of 128 in blocks of one: bf16 56 us, against 340
    // with a head a wave, fp32 92 and 207; of two 54 and 184, of four 59 and 107).
    while (2 * a.side * block <= kRound && a.side < a.heads) a.side *= 2;
    if (block <= kRound) return launch_append<T, D, V, 1, 1>(a, q, with_q, s);
    // Fewer rounds of 16-bit rows take fewer registers (105 instead of 141; bf16 in blocks of sixteen 52 us and 58). fp32 rows do not.
    if constexpr (sizeof(T) == 2)
        if (block <= 2 * kRound) return launch_append<T, D, V, 1, 2>(a, q, with_q, s);
    if (block <= 4 * kRound) return launch_append<T, D, V, 1, 4>(a, q, with_q, s);
    if (block <= 16 * kRound) return launch_append<T, D, V, 4, 4>(a, q, with_q, s);
    return launch_append<T, D, V, 4, 0>(a, q, with_q, s);
}

template <typename T>
int launch_append_type(const Append8Args &a, const HeadArgs &q, bool with_q, int D, bool wide, hipStream_t s) {
    if (D == 64) return launch_append_dim<T, 64>(a, q, with_q, wide, s);
    if (D == 128) return launch_append_dim<T, 128>(a, q, with_q, wide, s);
    return launch_append_dim<T, 256>(a, q, with_q, wide, s);
}

int run_append8(const tqhip_head_proj &p, const tqhip_kv_cache8 &c, const tqhip_seqs &b, hipStream_t s) {
    int st = check_heads(p);
    if (st != kOk) return st;
    const tqhip_kv_cache rows = rows_of(c);
    if ((st = check_cache8(c, b)) != kOk) return st;
    if ((!p.q) != (!p.q_out) || (p.q && p.n_heads < 1) || !p.k || !p.v || c.n_kv_heads != p.n_kv_heads || c.head_dim != p.head_dim ||
        b.n_tokens != p.n_tokens || !rows_apart(rows))
        return kBadShape;
    if (std::max(p.n_heads, p.n_kv_heads) > kMostHeads) return kTooLarge;
    const int D = c.head_dim;
    if (D != 64 && D != 128 && D != 256) return kBadShape;
    const int64_t row = static_cast<int64_t>(p.n_kv_heads) * D;
    Append8Args a{{p.k, p.v}, {p.k_stride ? p.k_stride : row, p.v_stride ? p.v_stride : row}, {p.k_bias, p.v_bias}, p.k_norm,
                  {static_cast<unsigned char *>(c.k), static_cast<unsigned char *>(c.v)}, c.scales, p.n_tokens, p.n_kv_heads, p.rotary_dim, c.dtype, 0, 1,
                  p.eps, p.rotary_dim && !p.inv_freq ? std::log2(p.theta) : 0.0, p.inv_freq, p.positions, b.q_start, b.kv_len, b.n_seqs,
                  make_pages(rows, b), FastDiv(static_cast<uint32_t>(c.block)), c.page_size / c.block};
    const int64_t tiles = b.n_tokens / c.block + int64_t{2} * b.n_seqs;
    if (2 * tiles * p.n_kv_heads > INT32_MAX / kAppendThreads) return kTooLarge;  // (of any form: nothing is launched before that is known)
    a.tiles = static_cast<int>(tiles);
    if (p.n_tokens > 1 && (a.in_stride[0] < row || a.in_stride[1] < row)) return kBadShape;
    // codes are written, and written again, 16 bytes at a time
    const auto apart = [](const void *q, int64_t stride) { return reinterpret_cast<uintptr_t>(q) % 16 || stride % 16; };
    if (apart(c.k, a.pages.page_stride) || apart(c.v, a.pages.token_stride) || a.pages.head_stride % 16) return kBadShape;
    const int bytes = type_bytes(p.dtype), v = 16 / bytes;
    bool wide = p.rotary_dim % (2 * v) == 0;
    for (int i = 0; i < 2; ++i) wide = wide && !apart(a.in[i], a.in_stride[i] * bytes);
    for (const float *f : {p.k_bias, p.v_bias, p.k_norm}) wide = wide && !apart(f, 0);
    const HeadArgs q = query_args(p, rows, b);
    const int64_t q_row = static_cast<int64_t>(p.n_heads) * D;
    if (p.q && p.n_tokens > 1 && (q.in_stride[0] < q_row || q.out_stride[0] < q_row)) return kBadShape;
    const bool with_q = p.q && wide && wide_queries(p, q);
    if (p.q && !with_q && (st = finish_queries(p, rows, b, s)) != kOk) return st;
    switch (p.dtype) {
        case TQHIP_F32: return launch_append_type<float>(a, q, with_q, D, wide, s);
        case TQHIP_F16: return launch_append_type<f16>(a, q, with_q, D, wide, s);
        default: return launch_append_type<bf16>(a, q, with_q, D, wide, s);
    }
}

}  // namespace
}  // namespace tqhip

extern "C" int tqhip_kv_append8_dev(const tqhip_head_proj *proj, const tqhip_kv_cache8 *cache, const tqhip_seqs *seqs, void *stream) {
    if (!proj || !cache || !seqs) return tqhip::kBadShape;
    return tqhip::run_append8(*proj, *cache, *seqs, static_cast<hipStream_t>(stream));
}
