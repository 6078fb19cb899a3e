// page_map.hip -- the pages of a batch of requests from their lengths: block tables and the list of free pages brought to what
// the coming call needs, and the q_start, kv_len, positions and slots that the batch calls and their callers take.
//
// With kv = past + new and need = ceil(kv / page_size), sequence b gives back max(held - need, 0) pages or wants max(need - held, 0).
// Both are prefix sums over the sequences, in their order, so every page's place in the list follows from them:
//   the r-th page given back goes to free_pages[n_free + r], the e-th page taken comes from free_pages[n_free + given - 1 - e].
// Taking may take what has just been given, so the two are phases of one workgroup with a barrier between them.
//
// Nothing here is work: it is latency, a few dependent loads and the scans. 256 requests, a token each: 10 us (as much with a workgroup of 256); 48
// prompts' 830000 tokens and 53000 pages: 16 us, and 6 to 7 for the tokens, which are a launch of their own past 4096.
#include <algorithm>

#include "batch.h"
#include "tq_common.h"

namespace tqhip {
namespace {

constexpr int kMapThreads = 1024;
constexpr int kAtOnce = 16, kLongRun = 16;
constexpr int kMapSeqs = 4096;  // (their prefix sums are in LDS)

struct MapArgs {
    int n_seqs, n_tokens, n_pages, table_stride;
    FastDiv page_size;
    const int *past, *fresh;
    int *table, *held, *free_pages, *n_free;
    int *q_start, *kv_len, *missing, *positions, *slots;
};

// Position and slot of token t of sequence b, whose tokens end before `end`.
__device__ inline void map_token(const MapArgs &a, int t, int b, int end, int kv) {
    const int pos = kv - (end - t);
    int slot = -1;
    if (pos >= 0) {
        const int i = a.page_size.quot(pos);
        const int page = i < a.table_stride ? a.table[static_cast<int64_t>(b) * a.table_stride + i] : -1;
        if (static_cast<unsigned>(page) < static_cast<unsigned>(a.n_pages))
            slot = page * static_cast<int>(a.page_size.d) + pos - i * static_cast<int>(a.page_size.d);
    }
    if (a.positions) a.positions[t] = pos;
    if (a.slots) a.slots[t] = slot;
}
__device__ inline void map_none(const MapArgs &a, int t) {
    if (a.positions) a.positions[t] = -1;
    if (a.slots) a.slots[t] = -1;
}

// Inclusive prefix sums of three numbers over the workgroup, and their totals.
struct Three {
    int64_t x[3];
};
__device__ inline Three scan_three(Three v, Three (*of_wave)[kMapThreads / 64], Three &total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d *= 2)
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            const int64_t y = __shfl_up(static_cast<long long>(v.x[i]), d);
            if (lane >= d) v.x[i] += y;
        }
    if (lane == 63) (*of_wave)[wave] = v;
    __syncthreads();
    total = Three{};
    Three before{};
#pragma unroll 2
    for (int w = 0; w < kMapThreads / 64; ++w)
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            if (w < wave) before.x[i] += (*of_wave)[w].x[i];
            total.x[i] += (*of_wave)[w].x[i];
        }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 3; ++i) v.x[i] += before.x[i];
    return v;
}

__global__ __launch_bounds__(kMapThreads) void map_pages(MapArgs a, bool tokens_too) {
    __shared__ int64_t give_at[kMapSeqs], want_at[kMapSeqs];
    __shared__ int start[kMapSeqs], need_of[kMapSeqs], held_of[kMapSeqs];
    __shared__ Three of_wave[kMapThreads / 64];
    __shared__ int taken;
    const int tid = threadIdx.x;
    const int64_t nf = min(max(*a.n_free, 0), a.n_pages);

    if (tid == 0) taken = 0;
    Three sum{};  // of the sequences so far: tokens, pages given back, pages wanted
    for (int b0 = 0; b0 < a.n_seqs; b0 += kMapThreads) {
        const int b = b0 + tid;
        Three v{};
        if (b < a.n_seqs) {
            const int n = max(a.fresh[b], 0);
            const int kv = static_cast<int>(min(static_cast<int64_t>(max(a.past[b], 0)) + n, static_cast<int64_t>(INT32_MAX)));
            const int held = min(max(a.held[b], 0), a.table_stride);
            const int whole = a.page_size.quot(kv), need = whole + (kv > whole * static_cast<int>(a.page_size.d));
            v = Three{{n, max(held - need, 0), need <= a.table_stride ? max(need - held, 0) : 0}};
            a.kv_len[b] = kv;
            need_of[b] = need;
            held_of[b] = held;
        }
        Three total;
        const Three upto = scan_three(v, &of_wave, total);
        if (b < a.n_seqs) {
            start[b] = static_cast<int>(min(sum.x[0] + upto.x[0] - v.x[0], static_cast<int64_t>(a.n_tokens)));
            a.q_start[b] = start[b];
            give_at[b] = sum.x[1] + upto.x[1] - v.x[1];
            want_at[b] = sum.x[2] + upto.x[2] - v.x[2];
        }
#pragma unroll
        for (int i = 0; i < 3; ++i) sum.x[i] += total.x[i];
    }
    const int end = static_cast<int>(min(sum.x[0], static_cast<int64_t>(a.n_tokens)));
    const int64_t given = sum.x[1], there = min(nf + given, static_cast<int64_t>(a.n_pages));
    __syncthreads();

    // f(b, i, n) for page i of the n that sequence b moves, n(b): by the threads, each with a search for its sequence, where sequences move few, by the waves, a
    // sequence at a time and several pages a lane, where they move many. (53000 pages of 48 prompts: 39 us with a search for each, 17 without.)
    const auto each = [&](int64_t total, const int64_t *at, auto count, auto f) {
        if (total <= int64_t{kLongRun} * a.n_seqs) {
            for (int64_t e = tid; e < total; e += kMapThreads) {
                const int b = last_at_most<int64_t>(at, a.n_seqs, e);
                f(b, static_cast<int>(e - at[b]), INT32_MAX);
            }
            return;
        }
        const int lane = tid & 63;
        for (int b = __builtin_amdgcn_readfirstlane(tid >> 6); b < a.n_seqs; b += kMapThreads / 64)
            for (int i = lane, n = count(b); i < n; i += kAtOnce * 64) f(b, i, n);
    };
    each(given, give_at, [&](int b) { return max(held_of[b] - need_of[b], 0); },
         [&](int b, int i0, int n) {
             int *entry = a.table + static_cast<int64_t>(b) * a.table_stride + need_of[b];
             const int64_t to = nf + give_at[b];
             const auto move = [&](int i, int page) {
                 if (to + i < a.n_pages) a.free_pages[to + i] = page;
                 entry[i] = -1;
             };
             if (n == INT32_MAX) return move(i0, entry[i0]);
             int page[kAtOnce];
#pragma unroll
             for (int k = 0; k < kAtOnce; ++k) page[k] = entry[min(i0 + 64 * k, n - 1)];
#pragma unroll
             for (int k = 0; k < kAtOnce; ++k)
                 if (i0 + 64 * k < n) move(i0 + 64 * k, page[k]);
         });
    __syncthreads();
    // The pages that are there go to the sequences in order, up to the first that they do not suffice for.
    const auto fits = [&](int b) { return want_at[b] + need_of[b] - held_of[b] <= there; };
    each(min(sum.x[2], there), want_at, [&](int b) { return need_of[b] <= a.table_stride && fits(b) ? need_of[b] - held_of[b] : 0; },
         [&](int b, int i0, int n) {
             if (!fits(b)) return;
             int *entry = a.table + static_cast<int64_t>(b) * a.table_stride + held_of[b];
             const int *page = a.free_pages + (there - 1 - want_at[b]);
             if (n == INT32_MAX) {
                 entry[i0] = page[-i0];
                 return;
             }
             int x[kAtOnce];
#pragma unroll
             for (int k = 0; k < kAtOnce; ++k) x[k] = page[-min(i0 + 64 * k, n - 1)];
#pragma unroll
             for (int k = 0; k < kAtOnce; ++k)
                 if (i0 + 64 * k < n) entry[i0 + 64 * k] = x[k];
         });
    for (int b = tid; b < a.n_seqs; b += kMapThreads) {
        const int need = need_of[b], held = held_of[b];
        const bool fits = need <= held || (need <= a.table_stride && want_at[b] + need - held <= there);
        a.held[b] = fits ? need : held;
        a.missing[b] = fits ? 0 : need - held;
        const int64_t upto = b + 1 < a.n_seqs ? want_at[b + 1] : sum.x[2];
        if (upto <= there) atomicMax(&taken, static_cast<int>(upto));
    }
    __syncthreads();
    if (tid == 0) *a.n_free = static_cast<int>(there - taken);
    if (tid == 0) a.q_start[a.n_seqs] = end;
    if (!tokens_too) return;
    for (int t = tid; t < a.n_tokens; t += kMapThreads) {
        if (t >= end) {
            map_none(a, t);
            continue;
        }
        const int b = last_at_most(start, a.n_seqs, t);
        map_token(a, t, b, b + 1 < a.n_seqs ? start[b + 1] : end, a.kv_len[b]);
    }
}

// Four tokens a thread, 256 apart, rarely of two sequences.
__global__ __launch_bounds__(256) void map_tokens(MapArgs a) {
    const int t0 = blockIdx.x * 1024 + threadIdx.x, end = a.q_start[a.n_seqs];
    int b = 0, to = -1, kv = 0;
    for (int t = t0; t < min(t0 + 1024, a.n_tokens); t += 256) {
        if (t >= end) {
            map_none(a, t);
            continue;
        }
        if (t >= to) {
            b = last_at_most<int>(a.q_start, a.n_seqs, t);
            to = a.q_start[b + 1];
            kv = a.kv_len[b];
        }
        map_token(a, t, b, to, kv);
    }
}

int run_map(const tqhip_page_map &p, hipStream_t s) {
    if (p.n_seqs < 1 || p.n_tokens < 0 || p.n_pages < 1 || p.page_size < 1 || p.table_stride < 1 || !p.past || !p.n_new || !p.block_table ||
        !p.n_held || !p.free_pages || !p.n_free || !p.q_start || !p.kv_len || !p.missing)
        return kBadShape;
    if (p.n_seqs > kMapSeqs || static_cast<int64_t>(p.table_stride) * p.page_size > INT32_MAX / 2 ||
        static_cast<int64_t>(p.n_pages) * p.page_size > INT32_MAX || p.n_tokens > INT32_MAX / 2)
        return kTooLarge;
    const MapArgs a{p.n_seqs, p.n_tokens, p.n_pages, p.table_stride, FastDiv(static_cast<uint32_t>(p.page_size)), p.past, p.n_new, p.block_table,
                    p.n_held, p.free_pages, p.n_free, p.q_start, p.kv_len, p.missing, p.positions, p.slots};
    const bool tokens = p.n_tokens > 0 && (p.positions || p.slots), few = p.n_tokens <= 4 * kMapThreads;
    map_pages<<<1, kMapThreads, 0, s>>>(a, tokens && few);
    if (tokens && !few) map_tokens<<<(p.n_tokens + 1023) / 1024, 256, 0, s>>>(a);
    return hipGetLastError() == hipSuccess ? kOk : kLaunchFailed;
}

}  // namespace
}  // namespace tqhip

extern "C" int tqhip_page_map_dev(const tqhip_page_map *map, void *stream) {
    if (!map) return tqhip::kBadShape;
    return tqhip::run_map(*map, static_cast<hipStream_t>(stream));
}
