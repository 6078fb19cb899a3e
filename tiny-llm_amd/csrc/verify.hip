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
// Reading the rows once is the work. Three launches:
//   row_sums  maximum, sum of exponentials and argmax of every chunk of every row;
//   judge     a sequence's chunks each join the sums of its rows, find the row that ends it, and sum their part of that row's r
//             (the row is read a second time, from L2);
//   draw      the chunk and then the token that the draw falls into.
#include <algorithm>
#include <climits>
#include <optional>

#include "batch.h"
#include "lane_sum.h"
#include "tq_common.h"

namespace tqhip {
namespace {

constexpr int kRowThreads = 256;
constexpr int kPerThread = 32;
constexpr int kChunk = kRowThreads * kPerThread;
constexpr int kDrawThreads = 1024;
constexpr int kMaxChunks = 512;  // (one workgroup scans a row's)

struct Part {
    double sum;  // of exp((l - max) / T)
    float max;
    int best;    // its first place; of rows of argmax only
};

// How a sequence's tokens end.
enum Kind : int { kNone = 0, kKnown, kTarget, kRest, kWithout };  // no draw; p; max(p - q, 0); p without x
struct End {
    double max, sum, max_q, sum_q;  // of the row: p = exp((l - max) / T) / sum
    int kind, row, x;
};

struct VerifyArgs {
    const void *logits, *draft;
    int64_t stride, draft_stride;
    const int *q_start, *tokens;
    const float *heat, *accept, *pick;
    const int *kv_len;
    int *past, *out, *n_out;
    float *logprob;
    int n_seqs, n_tokens, vocab, chunks;
    Part *parts;  // [target, draft][n_tokens][chunks]
    double *mass; // [n_seqs][chunks]
    End *ends;    // [n_seqs]
};

__device__ inline double inverse_heat(const VerifyArgs &a, int b, bool &greedy) {
    const float t = a.heat ? a.heat[b] : 1.0f;
    greedy = !(t > 0.0f);
    return greedy ? 1.0 : 1.0 / t;
}

// exp((x - max) / T); nothing for minus infinity, NaN for NaN and plus infinity.
__device__ inline double weight(float x, double max, double inv) { return x == -INFINITY ? 0.0 : exp((x - max) * inv); }

// N elements of a row from i on, minus infinity past its end. (Rows start at any element: a vocabulary may be odd.)
template <typename T, int N>
__device__ inline void load_row(const T *row, int i, int n, float *x) {
    typedef T any_vec __attribute__((ext_vector_type(N), aligned(sizeof(T))));
    if (i + N <= n) {
        const any_vec v = *reinterpret_cast<const any_vec *>(row + i);
#pragma unroll
        for (int e = 0; e < N; ++e) x[e] = static_cast<float>(v[e]);
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) x[e] = i + e < n ? static_cast<float>(row[i + e]) : -INFINITY;
    }
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

template <typename T>
__global__ __launch_bounds__(kRowThreads) void row_sums(VerifyArgs a) {
    constexpr int V = 16 / sizeof(T), WAVES = kRowThreads / 64;
    __shared__ float max_of[WAVES];
    __shared__ double sum_of[WAVES];
    __shared__ int best_of[WAVES];
    const int t = blockIdx.x / a.chunks, chunk = blockIdx.x - t * a.chunks, tid = threadIdx.x;
    if (t < a.q_start[0] || t >= a.q_start[a.n_seqs]) return;
    const int b = last_at_most(a.q_start, a.n_seqs, t);
    if (blockIdx.y && t + 1 == a.q_start[b + 1]) return;  // (no draft after it)
    bool greedy;
    const double inv = inverse_heat(a, b, greedy);
    const T *row = blockIdx.y ? static_cast<const T *>(a.draft) + t * a.draft_stride : static_cast<const T *>(a.logits) + t * a.stride;
    float x[kPerThread];
#pragma unroll
    for (int j = 0; j < kPerThread / V; ++j) load_row<T, V>(row, chunk * kChunk + (j * kRowThreads + tid) * V, a.vocab, x + j * V);
    float m = x[0];
#pragma unroll
    for (int i = 1; i < kPerThread; ++i) m = fmaxf(m, x[i]);
    m = xor_max_wave(m);
    if ((tid & 63) == 0) max_of[tid >> 6] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; ++w) m = fmaxf(m, max_of[w]);
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) s += weight(x[i], m, inv);
    s = sum_waves<WAVES>(xor_sum_wave(s), sum_of);
    int best = INT_MAX;
    if (greedy && blockIdx.y == 0) {
#pragma unroll
        for (int i = kPerThread - 1; i >= 0; --i)
            if (x[i] == m) best = chunk * kChunk + (i / V * kRowThreads + tid) * V + i % V;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) best = min(best, __shfl_xor(best, d));
        if ((tid & 63) == 0) best_of[tid >> 6] = best;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < WAVES; ++w) best = min(best, best_of[w]);
    }
    if (tid == 0) a.parts[(static_cast<int64_t>(blockIdx.y) * a.n_tokens + t) * a.chunks + chunk] = Part{s, m, best};
}

// A row's chunks joined by one wave: maximum, sum and first place of the maximum.
__device__ inline void join_row(const VerifyArgs &a, const Part *parts, double inv, double &max, double &sum, int &best) {
    const int lane = threadIdx.x & 63;
    float m = -INFINITY;
    for (int c = lane; c < a.chunks; c += 64) m = fmaxf(m, parts[c].max);
    m = xor_max_wave(m);
    double s = 0.0;
    best = INT_MAX;
    for (int c = lane; c < a.chunks; c += 64) {
        const Part p = parts[c];
        // a chunk of nothing but minus infinity has a sum of 0, or of NaN where it has one
        s += p.max == -INFINITY ? p.sum : p.sum * exp((static_cast<double>(p.max) - m) * inv);
        if (p.max == m) best = min(best, p.best);
    }
    sum = xor_sum_wave(s);
    max = m;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) best = min(best, __shfl_xor(best, d));
}

// What the row that ends a sequence draws from, at element i.
template <typename T, int N>
__device__ inline void weights(const VerifyArgs &a, const End &e, int kind, double inv, int i, double *w) {
    float x[N];
    load_row<T, N>(static_cast<const T *>(a.logits) + e.row * a.stride, i, a.vocab, x);
#pragma unroll
    for (int j = 0; j < N; ++j) w[j] = weight(x[j], e.max, inv) / e.sum;
    if (kind == kRest) {
        load_row<T, N>(static_cast<const T *>(a.draft) + e.row * a.draft_stride, i, a.vocab, x);
#pragma unroll
        for (int j = 0; j < N; ++j) w[j] = fmax(w[j] - weight(x[j], e.max_q, inv) / e.sum_q, 0.0);  // (0 where q is no number)
    } else if (kind == kWithout) {
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (i + j == e.x) w[j] = 0.0;
    }
}

template <typename T>
__global__ __launch_bounds__(kRowThreads) void judge(VerifyArgs a) {
    constexpr int V = 16 / sizeof(T), WAVES = kRowThreads / 64;
    __shared__ End end;
    __shared__ int stop;
    __shared__ double sum_of[WAVES];
    const int b = blockIdx.x / a.chunks, chunk = blockIdx.x - b * a.chunks;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int first = min(max(a.q_start[b], 0), a.n_tokens), n = min(max(a.q_start[b + 1], 0), a.n_tokens) - first;
    if (n <= 0) {
        if (chunk == 0 && tid == 0) {
            a.n_out[b] = 0;
            a.ends[b].kind = kNone;
            if (a.past) a.past[b] = a.kv_len[b];
        }
        return;
    }
    bool greedy;
    const double inv = inverse_heat(a, b, greedy);
    if (tid == 0) stop = INT_MAX;
    __syncthreads();
    // four rows at a time, up to the first that ends the sequence: the last one does
    for (int r0 = 0;; r0 += WAVES) {
        const int r = r0 + wave, t = first + r;
        End e{};
        float lp = 0.0f;
        bool ends = false;
        if (r < n) {
            int best;
            join_row(a, a.parts + static_cast<int64_t>(t) * a.chunks, inv, e.max, e.sum, best);
            const int x = r + 1 < n ? a.tokens[t + 1] : -1;
            const bool drafted = static_cast<unsigned>(x) < static_cast<unsigned>(a.vocab);
            const double lx = drafted ? static_cast<double>(static_cast<const T *>(a.logits)[t * a.stride + x]) : 0.0;
            e.row = t;
            e.x = x;
            ends = true;
            if (!(e.sum > 0.0)) {
                e.kind = kNone;
                e.x = -1;
            } else if (greedy) {
                e.kind = kKnown;
                ends = x != best;
                e.x = best;
                lp = static_cast<float>(-log(e.sum));
            } else if (!drafted) {
                e.kind = kTarget;
            } else {
                double q = 1.0;
                e.kind = kWithout;
                if (a.draft) {
                    int none;
                    join_row(a, a.parts + (static_cast<int64_t>(a.n_tokens) + t) * a.chunks, inv, e.max_q, e.sum_q, none);
                    q = weight(static_cast<float>(static_cast<const T *>(a.draft)[t * a.draft_stride + x]), e.max_q, inv) / e.sum_q;
                    e.kind = kRest;
                }
                ends = !(a.accept[t] * q < weight(static_cast<float>(lx), e.max, inv) / e.sum);
                lp = static_cast<float>((lx - e.max) * inv - log(e.sum));
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
    if (e.kind == kTarget || (e.kind == kWithout && e.x / kChunk != chunk)) {
        const Part p = a.parts[static_cast<int64_t>(e.row) * a.chunks + chunk];
        s = p.max == -INFINITY ? 0.0 : p.sum * exp((p.max - e.max) * inv) / e.sum;
    } else {
#pragma unroll
        for (int j = 0; j < kPerThread / V; ++j) {
            double w[V];
            weights<T, V>(a, e, e.kind, inv, chunk * kChunk + (j * kRowThreads + tid) * V, w);
#pragma unroll
            for (int i = 0; i < V; ++i) s += w[i];
        }
        s = sum_waves<WAVES>(xor_sum_wave(s), sum_of);
    }
    if (tid == 0) a.mass[static_cast<int64_t>(b) * a.chunks + chunk] = s;
}

// Inclusive prefix sums over the workgroup, and the total.
__device__ inline double scan(double v, double *of_wave, double &total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const double y = __shfl_up(v, d);
        if (lane >= d) v += y;
    }
    if (lane == 63) of_wave[wave] = v;
    __syncthreads();
    double before = 0.0;
    total = 0.0;
#pragma unroll
    for (int w = 0; w < kDrawThreads / 64; ++w) {
        if (w == wave) before = total;
        total += of_wave[w];
    }
    __syncthreads();
    return before + v;
}

template <typename T>
__global__ __launch_bounds__(kDrawThreads) void draw(VerifyArgs a) {
    constexpr int N = kChunk / kDrawThreads;
    __shared__ double of_wave[kDrawThreads / 64], before_chunk;
    __shared__ int found, last;
    const int b = blockIdx.x, tid = threadIdx.x;
    const End e = a.ends[b];
    if (e.kind <= kKnown) return;
    bool greedy;
    const double inv = inverse_heat(a, b, greedy);
    if (tid == 0) found = INT_MAX, last = 0;
    int kind = e.kind;
    double mine = tid < a.chunks ? a.mass[static_cast<int64_t>(b) * a.chunks + tid] : 0.0, total;
    double upto = scan(mine, of_wave, total);
    if (!(total > 0.0) && kind != kTarget) {  // p and q are the same: p itself
        kind = kTarget;
        mine = 0.0;
        if (tid < a.chunks) {
            const Part p = a.parts[static_cast<int64_t>(e.row) * a.chunks + tid];
            if (p.max > -INFINITY) mine = p.sum * exp((p.max - e.max) * inv) / e.sum;
        }
        upto = scan(mine, of_wave, total);
    }
    const double goal = a.pick[b] * total;
    // the first whose prefix exceeds the goal, or (the last sums rounded down) the last that has any weight
    if (mine > 0.0) {
        if (upto > goal) atomicMin(&found, tid);
        atomicMax(&last, tid);
    }
    __syncthreads();
    const int chunk = found == INT_MAX ? last : found;
    if (tid == chunk) before_chunk = upto - mine;
    __syncthreads();
    const double before = before_chunk;
    if (tid == 0) found = INT_MAX, last = chunk * kChunk;
    const int i0 = chunk * kChunk + tid * N;
    double w[N], sum = 0.0;
#pragma unroll
    for (int j = 0; j < N; j += 4) weights<T, 4>(a, e, kind, inv, i0 + j, w + j);
#pragma unroll
    for (int j = 0; j < N; ++j) sum += w[j];
    double at = before + scan(sum, of_wave, total) - sum;
    int hit = INT_MAX, any = -1;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        at += w[j];
        if (w[j] > 0.0) {
            if (at > goal && hit == INT_MAX) hit = i0 + j;
            any = i0 + j;
        }
    }
    if (hit != INT_MAX) atomicMin(&found, hit);
    if (any >= 0) atomicMax(&last, any);
    __syncthreads();
    if (tid == 0) {
        const int x = found == INT_MAX ? last : found;
        a.out[e.row] = x;
        if (a.logprob)
            a.logprob[e.row] = static_cast<float>(
                (static_cast<double>(static_cast<const T *>(a.logits)[e.row * a.stride + x]) - e.max) * inv - log(e.sum));
    }
}

int check_verify(const tqhip_verify &p) {
    if (!type_known(p.dtype) || p.n_seqs < 1 || p.n_tokens < 1 || p.vocab < 1 || !p.logits || !p.q_start || !p.tokens || !p.accept || !p.pick ||
        !p.out_tokens || !p.n_out || (p.past && !p.kv_len))
        return kBadShape;
    if ((p.logits_stride && p.logits_stride < p.vocab) || (p.draft_stride && p.draft_stride < p.vocab)) return kBadShape;
    const int bytes = type_bytes(p.dtype);
    if ((reinterpret_cast<uintptr_t>(p.logits) | reinterpret_cast<uintptr_t>(p.draft)) % bytes) return kBadShape;
    if (p.vocab > kMaxChunks * kChunk) return kTooLarge;
    const int64_t chunks = (p.vocab + kChunk - 1) / kChunk;
    // (a launch has less than 2^32 threads along x)
    if (chunks * std::max(p.n_tokens, p.n_seqs) > INT32_MAX / kRowThreads || p.n_seqs > INT32_MAX / kDrawThreads) return kTooLarge;
    return kOk;
}

size_t verify_bytes(const tqhip_verify &p) {
    const size_t chunks = (p.vocab + kChunk - 1) / kChunk;
    return chunks * p.n_tokens * sizeof(Part) * (p.draft ? 2 : 1) + p.n_seqs * (sizeof(End) + chunks * sizeof(double));
}

template <typename T>
void launch_verify(const VerifyArgs &a, hipStream_t s) {
    row_sums<T><<<dim3(a.chunks * a.n_tokens, a.draft ? 2 : 1), kRowThreads, 0, s>>>(a);
    judge<T><<<a.chunks * a.n_seqs, kRowThreads, 0, s>>>(a);
    draw<T><<<a.n_seqs, kDrawThreads, 0, s>>>(a);
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
    const int chunks = (p.vocab + kChunk - 1) / kChunk;
    Part *parts = static_cast<Part *>(ws);
    End *ends = reinterpret_cast<End *>(parts + static_cast<size_t>(chunks) * p.n_tokens * (p.draft ? 2 : 1));
    const VerifyArgs a{p.logits, p.draft, p.logits_stride ? p.logits_stride : p.vocab, p.draft_stride ? p.draft_stride : p.vocab, p.q_start, p.tokens,
                       p.temperature, p.accept, p.pick, p.kv_len, p.past, p.out_tokens, p.n_out, p.logprob, p.n_seqs, p.n_tokens, p.vocab, chunks,
                       parts, reinterpret_cast<double *>(ends + p.n_seqs), ends};
    if (p.dtype == TQHIP_F32)
        launch_verify<float>(a, s);
    else if (p.dtype == TQHIP_F16)
        launch_verify<f16>(a, s);
    else
        launch_verify<bf16>(a, s);
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
    return verify && tqhip::check_verify(*verify) == tqhip::kOk ? tqhip::verify_bytes(*verify) : 0;
}

}  // extern "C"
