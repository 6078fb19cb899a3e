// lora.hip -- the low-rank adapters of many requests beside the projection that they share:
// y_t = base_t + scale[a] * B_a (A_a x_t), a the adapter of t's request.
#include <algorithm>

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
    float *u;  // [n_tokens][rank]
    int n_tokens, K, M, rank, n_adapters, n_seqs;
};

__device__ inline int token_adapter(const LoraArgs &p, int t) {
    const int b = last_start_at_or_before(p.q_start, p.n_seqs, t);
    if (b < 0 || t >= p.q_start[b + 1]) return -1;
    const int a = p.adapter[b];
    return static_cast<unsigned>(a) < static_cast<unsigned>(p.n_adapters) ? a : -1;
}

template <typename W>
__global__ __launch_bounds__(256) void lora_shrink(LoraArgs p) {
    const int t = blockIdx.x, lane = threadIdx.x & 63;
    const int a = token_adapter(p, t);
    if (a < 0) return;
    const float *x = p.x + static_cast<int64_t>(t) * p.K;
    for (int r = threadIdx.x >> 6; r < p.rank; r += 4) {
        const W *w = static_cast<const W *>(p.a) + (static_cast<int64_t>(a) * p.rank + r) * p.K;
        float acc = 0.0f;
        for (int k = lane; k < p.K; k += 64) acc += static_cast<float>(w[k]) * x[k];
#pragma unroll
        for (int d = 1; d < 64; d *= 2) acc += __shfl_xor(acc, d);
        if (lane == 0) p.u[static_cast<int64_t>(t) * p.rank + r] = acc * p.scale[a];
    }
}

template <typename W>
__global__ __launch_bounds__(256) void lora_expand(LoraArgs p) {
    const int t = blockIdx.y, m = blockIdx.x * 256 + threadIdx.x;
    const int a = token_adapter(p, t);
    if (m >= p.M) return;
    const int64_t at = static_cast<int64_t>(t) * p.M + m;
    float acc = p.base ? p.base[at] : 0.0f;
    if (a >= 0) {
        const W *w = static_cast<const W *>(p.b) + (static_cast<int64_t>(a) * p.M + m) * p.rank;
        const float *u = p.u + static_cast<int64_t>(t) * p.rank;
        float d = 0.0f;
        for (int r = 0; r < p.rank; ++r) d += static_cast<float>(w[r]) * u[r];
        acc += d;
    }
    p.y[at] = acc;
}

size_t lora_workspace(const tqhip_lora &l) { return static_cast<size_t>(l.n_tokens) * l.rank * sizeof(float); }

int check_lora(const tqhip_lora &l) {
    if (!type_known(l.dtype) || l.n_tokens < 1 || l.in_dim < 1 || l.out_dim < 1 || l.rank < 1 || l.rank > 256 ||
        l.n_adapters < 1 || l.n_seqs < 1 || !l.x || !l.y || !l.a || !l.b || !l.scale || !l.q_start || !l.adapter)
        return kBadShape;
    if (l.n_tokens > 65535) return kTooLarge;
    return kOk;
}

template <typename W>
void launch_lora(const LoraArgs &p, hipStream_t s) {
    lora_shrink<W><<<p.n_tokens, 256, 0, s>>>(p);
    lora_expand<W><<<dim3((p.M + 255) / 256, p.n_tokens), 256, 0, s>>>(p);
}

int run_lora(const tqhip_lora &l, hipStream_t s) {
    int st = check_lora(l);
    if (st != kOk) return st;
    void *ws = l.workspace;
    if (ws && l.workspace_bytes < lora_workspace(l)) return kNoScratch;
    if (!ws && (st = scratch_batch(s, lora_workspace(l), &ws)) != kOk) return st;
    const LoraArgs p{l.x, l.base, l.y, l.a, l.b, l.scale, l.q_start, l.adapter, static_cast<float *>(ws), l.n_tokens,
                     l.in_dim, l.out_dim, l.rank, l.n_adapters, l.n_seqs};
    switch (l.dtype) {
        case TQHIP_F32: launch_lora<float>(p, s); break;
        case TQHIP_F16: launch_lora<f16>(p, s); break;
        default: launch_lora<bf16>(p, s); break;
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
    return lora && tqhip::check_lora(*lora) == tqhip::kOk ? tqhip::lora_workspace(*lora) : 0;
}

}  // extern "C"
