// verify.hip -- drafted tokens accepted or refused by the target's probabilities, and the token after them drawn, from random
// numbers that the caller gives.
//
// Row t of a sequence has logits l_t and, from a draft model, d_t: p = softmax(l_t / T), q = softmax(d_t / T). The drafted token x = tokens[t + 1]
// is accepted iff u_t q(x) < p(x), which leaves it with probability min(1, p / q). The first row that refuses draws the token in its
// place from r = max(p - q, 0), the row after the last draft from p: so what comes out is distributed as the target alone would have it.
// A draw is the first token whose prefix sum of r exceeds v times r's sum. A T of 0 takes each row's argmax.
//
// Whether a token is drawn or its neighbour turns on prefix sums of some 10^5 terms, so exponentials and sums are in 64 bits: in 32 one draw
// in a hundred would come out differently with the order of the sums.
//
// Reading the rows once and an exponential for each logit are the work. Three launches:
//   row_sums  maximum, sum of exponentials and argmax of every chunk of every row;
//   judge     a sequence's chunks each join the sums of its rows, find the row that ends it, and sum their part of that row's r
//             (the row is read a second time, and comes from behind the L2s again: of many requests more has passed them since than they hold);
//   draw      the chunk and then the token that the draw falls into.
// 64 requests with up to 4 drafts and their model's rows, 151936 fp32 logits (316 MB): 73, 24 and 10 us
// 100 requests with up to 7 drafts of no model, bf16 logits (215 MB, 107 million exponentials): 96, 13 and 9
// one request with 3 drafts: 4.4, 4.0 and 5.8
#include <algorithm>
#include <climits>
#include <optional>

#include "batch.h"
#include "lane_sum.h"
#include "tq_common.h"

namespace tqhip {
namespace {

constexpr int kRowThreads = 256;
constexpr int kDrawThreads = 512;
constexpr int kMaxChunks = 1024;  // (a wave scans a row's)
// Logits of a row that a thread takes, and a workgroup (a chunk).
constexpr int kFewPerThread = 16, kManyPerThread = 32;
template <int PER>
constexpr int kChunk = kRowThreads * PER;

struct Part {
    double sum;  // of exp((l - max) / T); NaN where a logit is NaN or plus infinity
    float max;
    int best;    // its first place; of rows of argmax only
};

// How a sequence's tokens end.
enum Kind : int { kNone = 0, kKnown, kTarget, kRest, kWithout };  // no draw; p; max(p - q, 0); p without x
struct End {
    double max, per_sum, max_q, per_sum_q;  // of the row: p = exp((l - max) / T) per_sum
    int kind, row, x;
};

struct VerifyArgs {
    const void *logits, *draft;
    int64_t stride, draft_stride;
    const int *q_start, *tokens;
    const float *heat, *accept, *pick;
    const int *kv_len, *missing;
    int *past, *out, *n_out;
    float *logprob;
    int n_seqs, n_tokens, vocab, chunks;
    Part *parts;  // [target, draft][n_tokens][chunks]
    double *mass; // [n_seqs][chunks]
    End *ends;    // [n_seqs]
};

// log2 e / T (T = 1 for rows of argmax).
__device__ inline double steepness(const VerifyArgs &a, int b, bool &greedy) {
    const float t = a.heat ? a.heat[b] : 1.0f;
    greedy = !(t > 0.0f);
    return 1.4426950408889634 / (greedy ? 1.0 : static_cast<double>(t));
}

// 2^y for y <= 0, 0 for minus infinity and NaN: (2^f - 1) / f of the fraction f in [-1/2, 1/2] by the polynomial of degree 8 through its values at the
// Chebyshev nodes, so 2^0 is 1, and no other off by more than 3.7e-14 of itself, or by half a step of fp64's subnormals where that is more. The whole part is
// found by an addition that leaves it in the low bits. (18 instructions a logit; with the library's exp, exact to the
// last bit, row_sums takes 119 us for the 64 requests below instead of 72.)
__device__ inline double exp2_below(double y) {
    constexpr double kWhole = 0x1.8p52;
    y = fmax(y, -1100.0);
    const double whole = y + kWhole, f = y - (whole - kWhole);
    double p = 0x1.b638808675ca6p-24;
    p = fma(p, f, 0x1.63d136355f669p-20);
    p = fma(p, f, 0x1.ffcb9515c8f1ap-17);
    p = fma(p, f, 0x1.4308ac85abb17p-13);
    p = fma(p, f, 0x1.5d87fe86fe7ccp-10);
    p = fma(p, f, 0x1.3b2ab7181b74ap-7);
    p = fma(p, f, 0x1.c6b08d7047e52p-5);
    p = fma(p, f, 0x1.ebfbdff823cedp-3);
    p = fma(p, f, 0x1.62e42fefa39efp-1);
    p = fma(p, f, 1.0);
    return __builtin_amdgcn_ldexp(p, __double2loint(whole));
}

// exp((x - max) / T) for x <= max; nothing for minus infinity (and max, where all are).
__device__ inline double weight(double x, double max, double steep) { return exp2_below((x - max) * steep); }

// N elements of a row from i on, minus infinity past its end, which only the row's last chunk has: without a branch for each load, so that none waits
// for another. (Rows start at any element: a vocabulary may be odd.)
template <typename T, int N>
__device__ inline void load_row(const T *row, int i, int n, bool last_chunk, float *x) {
    typedef T any_vec __attribute__((ext_vector_type(N), aligned(sizeof(T))));
    if (!last_chunk) {
        const any_vec v = *reinterpret_cast<const any_vec *>(row + i);
#pragma unroll
        for (int e = 0; e < N; ++e) x[e] = static_cast<float>(v[e]);
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const float y = static_cast<float>(row[min(i + e, n - 1)]);
            x[e] = i + e < n ? y : -INFINITY;
        }
    }
}

// The largest of the wave's 64 values, NaN if one is.
__device__ inline float max_of_wave(float m) {
    const int lane = threadIdx.x & 63;
    m = __builtin_elementwise_maximum(m, lane_xor<32>(m, lane));
    m = __builtin_elementwise_maximum(m, lane_xor<16>(m, lane));
    m = __builtin_elementwise_maximum(m, lane_xor<8>(m, lane));
    m = __builtin_elementwise_maximum(m, lane_xor<4>(m, lane));
    m = __builtin_elementwise_maximum(m, lane_xor<2>(m, lane));
    return __builtin_elementwise_maximum(m, lane_xor<1>(m, lane));
}

// Sum over the workgroup's waves of a value that each wave has summed.
template <int WAVES>
__device__ inline double sum_waves(double s, double *of_wave) {
    if ((threadIdx.x & 63) == 0) of_wave[threadIdx.x >> 6] = s;
    __syncthreads();
    s = of_wave[0];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) s += of_wave[w];
    return s;
}

template <typename T, int PER>
__global__ __launch_bounds__(kRowThreads) void row_sums(VerifyArgs a) {
    constexpr int V = 16 / sizeof(T), WAVES = kRowThreads / 64;
    __shared__ float max_of[WAVES];
    __shared__ double sum_of[WAVES];
    __shared__ int best_of[WAVES];
    const int t = blockIdx.x / a.chunks, chunk = blockIdx.x - t * a.chunks, tid = threadIdx.x;
    int b, end;
    // (a draft model's row is not read where no draft follows; a target's is on its way while its sequence is looked for)
    if (blockIdx.y && (!find_seq(a.q_start, a.n_seqs, t, b, end) || t + 1 == end)) return;
    const T *row = blockIdx.y ? static_cast<const T *>(a.draft) + t * a.draft_stride : static_cast<const T *>(a.logits) + t * a.stride;
    float x[PER];
    const auto load = [&](bool last_chunk) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < PER / V; ++j)
            load_row<T, V>(row, chunk * kChunk<PER> + (j * kRowThreads + tid) * V, a.vocab, last_chunk, x + j * V);
    };
    if (chunk < a.chunks - 1)
        load(false);
    else
        load(true);
    if (!blockIdx.y && !find_seq(a.q_start, a.n_seqs, t, b, end)) return;
    bool greedy;
    const double steep = steepness(a, b, greedy);
    float m = x[0];
#pragma unroll
    for (int i = 1; i < PER; ++i) m = __builtin_elementwise_maximum(m, x[i]);  // (NaN if one is)
    m = max_of_wave(m);
    if ((tid & 63) == 0) max_of[tid >> 6] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; ++w) m = __builtin_elementwise_maximum(m, max_of[w]);
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < PER; ++i) s += weight(x[i], m, steep);
    s = sum_waves<WAVES>(xor_sum_wave(s), sum_of);
    if (!(m < INFINITY)) s = NAN;
    int best = INT_MAX;
    if (greedy && blockIdx.y == 0) {
#pragma unroll
        for (int i = PER - 1; i >= 0; --i)
            if (x[i] == m) best = chunk * kChunk<PER> + (i / V * kRowThreads + tid) * V + i % V;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) best = min(best, __shfl_xor(best, d));
        if ((tid & 63) == 0) best_of[tid >> 6] = best;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < WAVES; ++w) best = min(best, best_of[w]);
    }
    if (tid == 0) a.parts[(static_cast<int64_t>(blockIdx.y) * a.n_tokens + t) * a.chunks + chunk] = Part{s, m, best};
}

// A row's chunks as each lane of a wave has them (one, where there are no more than lanes).
__device__ inline Part load_parts(const VerifyArgs &a, const Part *parts, double steep) {
    const int lane = threadIdx.x & 63;
    Part p = parts[min(lane, a.chunks - 1)];
    if (lane >= a.chunks) p = Part{0.0, -INFINITY, INT_MAX};
    for (int c = lane + 64; c < a.chunks; c += 64) {
        const Part o = parts[c];
        const float m = __builtin_elementwise_maximum(p.max, o.max);
        p.sum = p.sum * weight(p.max, m, steep) + o.sum * weight(o.max, m, steep);
        if (o.max > p.max) p.best = o.best;
        p.max = m;
    }
    return p;
}
// Joined over the wave: maximum, sum (NaN where the row has no probabilities for NaN or plus infinity, 0 for nothing but minus infinity)
// and first place of the maximum.
__device__ inline void join_parts(const Part &p, double steep, double &max, double &sum, int &best) {
    const float m = max_of_wave(p.max);
    sum = xor_sum_wave(p.sum * weight(p.max, m, steep));
    max = m;
    best = p.max == m ? p.best : INT_MAX;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) best = min(best, __shfl_xor(best, d));
}

// What the row that ends a sequence draws from: N logits of each of its rows from element i on, and their weights.
template <typename T, int N>
__device__ inline void load_rows(const VerifyArgs &a, const End &e, int kind, int i, bool last_chunk, float *x, float *y) {
    load_row<T, N>(static_cast<const T *>(a.logits) + e.row * a.stride, i, a.vocab, last_chunk, x);
    if (kind == kRest) load_row<T, N>(static_cast<const T *>(a.draft) + e.row * a.draft_stride, i, a.vocab, last_chunk, y);
}
template <int N>
__device__ inline void weights(const End &e, int kind, double steep, int i, const float *x, const float *y, double *w) {
#pragma unroll
    for (int j = 0; j < N; ++j) w[j] = weight(x[j], e.max, steep) * e.per_sum;
    if (kind == kRest) {
#pragma unroll
        for (int j = 0; j < N; ++j) w[j] = fmax(w[j] - weight(y[j], e.max_q, steep) * e.per_sum_q, 0.0);  // (0 where q is no number)
    } else if (kind == kWithout) {
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (i + j == e.x) w[j] = 0.0;
    }
}

// log p of a token whose logit is l.
__device__ inline float log_chance(double l, const End &e, double steep) {
    return static_cast<float>((l - e.max) * steep * 0.6931471805599453 + log(e.per_sum));
}

// Chunk c's share of the row's p.
__device__ inline double share(const VerifyArgs &a, const End &e, double steep, int c) {
    const Part p = a.parts[static_cast<int64_t>(e.row) * a.chunks + c];
    return p.sum * weight(p.max, e.max, steep) * e.per_sum;
}

template <typename T, int PER>
__global__ __launch_bounds__(kRowThreads) void judge(VerifyArgs a) {
    constexpr int V = 16 / sizeof(T), WAVES = kRowThreads / 64;
    __shared__ End end;
    __shared__ int stop;
    __shared__ double sum_of[WAVES];
    const int b = blockIdx.x / a.chunks, chunk = blockIdx.x - b * a.chunks;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int first = min(max(a.q_start[b], 0), a.n_tokens), n = min(max(a.q_start[b + 1], 0), a.n_tokens) - first;
    // (a sequence without all of its pages has rows over positions that do not exist: it says nothing, and keeps the length it had before the call)
    if (n <= 0 || (a.missing && a.missing[b] > 0)) {
        if (chunk == 0) {
            for (int t = first + tid; t < first + n; t += kRowThreads) {
                a.out[t] = -1;
                if (a.logprob) a.logprob[t] = 0.0f;
            }
            if (tid == 0) {
                a.n_out[b] = 0;
                a.ends[b].kind = kNone;
                if (a.past) a.past[b] = a.kv_len[b] - max(n, 0);
            }
        }
        return;
    }
    bool greedy;
    const double steep = steepness(a, b, greedy);
    if (tid == 0) stop = INT_MAX;
    __syncthreads();
    // four rows at a time, up to the first that ends the sequence: the last one does
    for (int r0 = 0;; r0 += WAVES) {
        const int r = r0 + wave, t = first + r;
        End e{};
        float lp = 0.0f;
        bool ends = false;
        if (r < n) {
            // (all that the row needs is on its way before anything waits)
            const bool more = r + 1 < n;
            const int x = more ? a.tokens[t + 1] : -1;
            const float u = a.accept[t];
            const Part p = load_parts(a, a.parts + static_cast<int64_t>(t) * a.chunks, steep);
            Part d{};
            if (a.draft && more) d = load_parts(a, a.parts + (static_cast<int64_t>(a.n_tokens) + t) * a.chunks, steep);
            const bool drafted = static_cast<unsigned>(x) < static_cast<unsigned>(a.vocab);
            const int safe = drafted ? x : 0;
            const double lx = static_cast<const T *>(a.logits)[t * a.stride + safe];
            const double dx = a.draft && more ? static_cast<double>(static_cast<const T *>(a.draft)[t * a.draft_stride + safe]) : 0.0;
            int best, none;
            double sum, sum_q;
            join_parts(p, steep, e.max, sum, best);
            e.per_sum = 1.0 / sum;
            e.row = t;
            e.x = x;
            ends = true;
            if (!(sum > 0.0)) {
                e.kind = kNone;
                e.x = -1;
            } else if (greedy) {
                e.kind = kKnown;
                ends = x != best;
                e.x = best;
                lp = static_cast<float>(-log(sum));
            } else if (!drafted) {
                e.kind = kTarget;
            } else {
                double q = 1.0;
                e.kind = kWithout;
                if (a.draft) {
                    join_parts(d, steep, e.max_q, sum_q, none);
                    e.per_sum_q = 1.0 / sum_q;
                    q = weight(dx, e.max_q, steep) * e.per_sum_q;
                    e.kind = kRest;
                }
                ends = !(u * q < weight(lx, e.max, steep) * e.per_sum);
                lp = log_chance(lx, e, steep);
            }
        }
        if (ends && lane == 0) atomicMin(&stop, r);
        __syncthreads();
        const int s = stop;
        if (r == s && lane == 0) end = e;
        if (chunk == 0 && lane == 0 && r < n && (r < s || (r == s && e.kind <= kKnown))) {
            a.out[t] = e.x;
            if (a.logprob) a.logprob[t] = lp;
        }
        __syncthreads();
        if (s != INT_MAX) break;
    }
    const End e = end;
    if (chunk == 0) {
        for (int t = e.row + 1 + tid; t < first + n; t += kRowThreads) {
            a.out[t] = -1;
            if (a.logprob) a.logprob[t] = 0.0f;
        }
        if (tid == 0) {
            const int count = e.row - first + 1;
            a.n_out[b] = count;
            if (a.past) a.past[b] = a.kv_len[b] - n + count;
            a.ends[b] = e;
        }
    }
    if (e.kind <= kKnown) return;
    double s = 0.0;
    if (e.kind == kTarget || (e.kind == kWithout && e.x / kChunk<PER> != chunk)) {
        s = share(a, e, steep, chunk);
    } else {
        float x[PER], y[PER];
        double w[PER];
        const auto at = [&](int j) { return chunk * kChunk<PER> + (j * kRowThreads + tid) * V; };
        const auto read = [&](bool last_chunk) __attribute__((always_inline)) {
#pragma unroll
            for (int j = 0; j < PER / V; ++j) load_rows<T, V>(a, e, e.kind, at(j), last_chunk, x + j * V, y + j * V);
        };
        if (chunk < a.chunks - 1)
            read(false);
        else
            read(true);
#pragma unroll
        for (int j = 0; j < PER / V; ++j) weights<V>(e, e.kind, steep, at(j), x + j * V, y + j * V, w + j * V);
#pragma unroll
        for (int i = 0; i < PER; ++i) s += w[i];
        s = sum_waves<WAVES>(xor_sum_wave(s), sum_of);
    }
    if (tid == 0) a.mass[static_cast<int64_t>(b) * a.chunks + chunk] = s;
}

// Inclusive prefix sums over the wave.
__device__ inline double scan_wave(double v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const double y = __shfl_up(v, d);
        if (lane >= d) v += y;
    }
    return v;
}

// A draw among the N weights of each of the wave's lanes, in order: the first weight whose prefix sum (`before` and all those before it counted)
// exceeds the goal, or, where none does because sums were rounded down, the last that is not 0. Its place (lane * N + j) and what is before it.
template <int N>
__device__ inline int pick(const double *w, double goal, double &before) {
    double sum = 0.0;
#pragma unroll
    for (int j = 0; j < N; ++j) sum += w[j];
    double at = before + (scan_wave(sum) - sum), hit_at = 0.0, any_at = 0.0;
    int hit = -1, any = -1;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        if (w[j] > 0.0) {
            if (at + w[j] > goal && hit < 0) hit = j, hit_at = at;
            any = j, any_at = at;
        }
        at += w[j];
    }
    const unsigned long long hits = __ballot(hit >= 0), anys = __ballot(any >= 0);
    if (anys == 0) return 0;
    const int from = hits ? __builtin_ctzll(hits) : 63 - __builtin_clzll(anys);
    before = __shfl(hits ? hit_at : any_at, from);
    return from * N + __shfl(hits ? hit : any, from);
}

template <typename T, int PER>
__global__ __launch_bounds__(kDrawThreads) void draw(VerifyArgs a) {
    constexpr int N = kChunk<PER> / kDrawThreads, WAVES = kDrawThreads / 64, LANE = kMaxChunks / 64;
    __shared__ double sum_of[WAVES], before_of[WAVES];
    __shared__ int place_of[WAVES];
    const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const End e = a.ends[b];
    if (e.kind <= kKnown) return;
    bool greedy;
    const double steep = steepness(a, b, greedy);
    // every wave finds the chunk for itself, a lane `per` chunks in order
    const int per = (a.chunks + 63) / 64;
    int kind = e.kind;
    double mass[LANE], total = 0.0;
    for (int again = 0; again < 2; ++again) {
        double mine = 0.0;
#pragma unroll
        for (int j = 0; j < LANE; ++j) {
            const int c = lane * per + j;
            mass[j] = j >= per || c >= a.chunks ? 0.0 : again ? share(a, e, steep, c) : a.mass[static_cast<int64_t>(b) * a.chunks + c];
            mine += mass[j];
        }
        total = xor_sum_wave(mine);
        if (total > 0.0 || kind == kTarget) break;
        kind = kTarget;  // p and q are the same: p itself
    }
    const double goal = a.pick[b] * total;
    double before = 0.0;
    const int lane_and_chunk = pick<LANE>(mass, goal, before), chunk = lane_and_chunk / LANE * per + lane_and_chunk % LANE;

    const int i0 = chunk * kChunk<PER> + tid * N;
    double w[N], sum = 0.0;
    float x[N], y[N];
    if (chunk < a.chunks - 1)
        load_rows<T, N>(a, e, kind, i0, false, x, y);
    else
        load_rows<T, N>(a, e, kind, i0, true, x, y);
    weights<N>(e, kind, steep, i0, x, y, w);
#pragma unroll
    for (int j = 0; j < N; ++j) sum += w[j];
    sum = xor_sum_wave(sum);
    if (lane == 0) sum_of[wave] = sum;
    __syncthreads();
#pragma unroll
    for (int v = 0; v < WAVES; ++v)
        if (v < wave) before += sum_of[v];
    const double upto = before + sum;
    const int place = pick<N>(w, goal, before);
    if (lane == 0) {
        place_of[wave] = sum > 0.0 ? place : -1;
        before_of[wave] = upto;
    }
    __syncthreads();
    if (tid != 0) return;
    int from = -1;  // the first wave past the goal, or the last that has anything
    for (int v = 0; v < WAVES; ++v)
        if (place_of[v] >= 0) {
            from = v;
            if (before_of[v] > goal) break;
        }
    const int token = chunk * kChunk<PER> + (from < 0 ? 0 : from * 64 * N + place_of[from]);
    a.out[e.row] = token;
    if (a.logprob) a.logprob[e.row] = log_chance(static_cast<const T *>(a.logits)[e.row * a.stride + token], e, steep);
}

// Long chunks spread a workgroup's search, sums and barriers over more logits; short ones spread few rows over more of the
// card. Up to 12 long ones a CU, of 151936 fp32 logits with drafts' rows: one request 17 us short and 20 long, 8 28 and 31, 16 38 and 41, 32 63 and 63, 64 112
// and 105 (64 without drafts 28 and 27).
int64_t rows_of(const tqhip_verify &p) { return static_cast<int64_t>(p.n_tokens) * (p.draft ? 2 : 1); }
int64_t most_few_rows(const tqhip_verify &p) { return int64_t{12} * device_cu_count() * kChunk<kManyPerThread> / p.vocab; }
bool few_rows(const tqhip_verify &p) { return rows_of(p) <= most_few_rows(p); }
int chunks_of(const tqhip_verify &p) {
    const int chunk = few_rows(p) ? kChunk<kFewPerThread> : kChunk<kManyPerThread>;
    return (p.vocab + chunk - 1) / chunk;
}

int check_verify(const tqhip_verify &p) {
    if (!type_known(p.dtype) || p.n_seqs < 1 || p.n_tokens < 1 || p.vocab < 1 || !p.logits || !p.q_start || !p.tokens || !p.accept || !p.pick ||
        !p.out_tokens || !p.n_out || (p.past && !p.kv_len))
        return kBadShape;
    if ((p.logits_stride && p.logits_stride < p.vocab) || (p.draft_stride && p.draft_stride < p.vocab)) return kBadShape;
    const int bytes = type_bytes(p.dtype);
    if ((reinterpret_cast<uintptr_t>(p.logits) | reinterpret_cast<uintptr_t>(p.draft)) % bytes) return kBadShape;
    if (p.vocab > kMaxChunks * kChunk<kFewPerThread>) return kTooLarge;
    const int64_t chunks = chunks_of(p);
    // (a launch has less than 2^32 threads along x)
    if (chunks * std::max(p.n_tokens, p.n_seqs) > INT32_MAX / kRowThreads || p.n_seqs > INT32_MAX / kDrawThreads) return kTooLarge;
    // a sequence's workgroups read its tokens and numbers while the first of them writes
    const auto meet = [](const void *in, int n_in, const void *out, int n_out) {
        const uintptr_t x = reinterpret_cast<uintptr_t>(in), y = reinterpret_cast<uintptr_t>(out);
        return in && out && (x < y ? y - x < 4 * static_cast<uintptr_t>(n_in) : x - y < 4 * static_cast<uintptr_t>(n_out));
    };
    for (const void *in : {static_cast<const void *>(p.tokens), static_cast<const void *>(p.accept)})
        if (meet(in, p.n_tokens, p.out_tokens, p.n_tokens) || meet(in, p.n_tokens, p.logprob, p.n_tokens)) return kBadShape;
    for (const void *out : {static_cast<const void *>(p.out_tokens), static_cast<const void *>(p.logprob)})
        if (meet(p.missing, p.n_seqs, out, p.n_tokens)) return kBadShape;
    if (meet(p.missing, p.n_seqs, p.n_out, p.n_seqs) || meet(p.missing, p.n_seqs, p.past, p.n_seqs)) return kBadShape;
    return kOk;
}

size_t part_bytes(int64_t rows, int n_seqs, size_t chunks) { return chunks * rows * sizeof(Part) + n_seqs * (sizeof(End) + chunks * sizeof(double)); }
size_t verify_bytes(const tqhip_verify &p) { return part_bytes(rows_of(p), p.n_seqs, chunks_of(p)); }
// What this call and every smaller one takes: short chunks are more of them, so the largest call of few rows may take more than one that is larger yet.
size_t verify_room(const tqhip_verify &p) {
    const size_t few_chunks = (p.vocab + kChunk<kFewPerThread> - 1) / kChunk<kFewPerThread>;
    return std::max(verify_bytes(p), part_bytes(std::min(rows_of(p), most_few_rows(p)), p.n_seqs, few_chunks));
}

template <typename T, int PER>
void launch_verify(const VerifyArgs &a, hipStream_t s) {
    row_sums<T, PER><<<dim3(a.chunks * a.n_tokens, a.draft ? 2 : 1), kRowThreads, 0, s>>>(a);
    judge<T, PER><<<a.chunks * a.n_seqs, kRowThreads, 0, s>>>(a);
    draw<T, PER><<<a.n_seqs, kDrawThreads, 0, s>>>(a);
}
template <typename T>
void launch_verify(const VerifyArgs &a, bool few, hipStream_t s) {
    if (few)
        launch_verify<T, kFewPerThread>(a, s);
    else
        launch_verify<T, kManyPerThread>(a, s);
}

int run_verify(const tqhip_verify &p, hipStream_t s) {
    int st = check_verify(p);
    if (st != kOk) return st;
    const size_t bytes = verify_bytes(p);
    void *ws = p.workspace;
    if (reinterpret_cast<uintptr_t>(ws) % 256) return kBadShape;
    if (ws && p.workspace_bytes < bytes) return kNoScratch;
    std::optional<ScratchCall> call;
    if (!ws) {
        call.emplace(s);
        if ((st = call->workspace(bytes, &ws)) != kOk) return st;
    }
    const int chunks = chunks_of(p);
    const bool few = few_rows(p);
    Part *parts = static_cast<Part *>(ws);
    End *ends = reinterpret_cast<End *>(parts + static_cast<size_t>(chunks) * p.n_tokens * (p.draft ? 2 : 1));
    const VerifyArgs a{p.logits, p.draft, p.logits_stride ? p.logits_stride : p.vocab, p.draft_stride ? p.draft_stride : p.vocab, p.q_start, p.tokens,
                       p.temperature, p.accept, p.pick, p.kv_len, p.missing, p.past, p.out_tokens, p.n_out, p.logprob, p.n_seqs, p.n_tokens, p.vocab, chunks,
                       parts, reinterpret_cast<double *>(ends + p.n_seqs), ends};
    if (p.dtype == TQHIP_F32)
        launch_verify<float>(a, few, s);
    else if (p.dtype == TQHIP_F16)
        launch_verify<f16>(a, few, s);
    else
        launch_verify<bf16>(a, few, s);
    return hipGetLastError() == hipSuccess ? kOk : kLaunchFailed;
}

}  // namespace
}  // namespace tqhip

extern "C" {

int tqhip_verify_tokens_dev(const tqhip_verify *verify, void *stream) {
    if (!verify) return tqhip::kBadShape;
    try {
        return tqhip::run_verify(*verify, static_cast<hipStream_t>(stream));
    } catch (...) {  // (host memory ran out)
        return tqhip::kHipFailed;
    }
}

size_t tqhip_verify_tokens_workspace(const tqhip_verify *verify) {
    return verify && tqhip::check_verify(*verify) == tqhip::kOk ? tqhip::verify_room(*verify) : 0;
}

}  // extern "C"
