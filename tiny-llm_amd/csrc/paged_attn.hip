// paged_attn.hip -- attention of the new tokens of a batch of sequences over their paged cache.
#include <algorithm>
#include <cmath>

#include "batch.h"
#include "tq_common.h"

namespace tqhip {
namespace {

struct AttnArgs {
    const void *q, *k, *v;
    void *out;
    int64_t q_stride, out_stride;
    const int *q_start, *kv_len;
    int n_seqs, n_tokens, n_heads, group;  // group: query heads per key/value head
    float scale;
    int causal, window;
    Pages pages;
};

// One wave per token and query head, 64 keys at a time.
template <typename T, typename C, int D>
__global__ __launch_bounds__(64) void attn_simple(AttnArgs a) {
    __shared__ float qs[D];
    const int t = blockIdx.x, h = blockIdx.y, lane = threadIdx.x;
    const int b = last_start_at_or_before(a.q_start, a.n_seqs, t);
    if (b < 0) return;
    const int end = a.q_start[b + 1];
    if (t >= end) return;
    const int pos = a.kv_len[b] - (end - t), len = min(a.kv_len[b], a.pages.table_stride * static_cast<int>(a.pages.page_size.d));
    for (int d = lane; d < D; d += 64)
        qs[d] = static_cast<float>((static_cast<const T *>(a.q) + t * a.q_stride + h * D)[d]) * a.scale;
    __syncthreads();
    const int hi = a.causal ? min(pos + 1, len) : len;
    const int lo = a.causal && a.window > 0 ? max(0, pos + 1 - a.window) : 0;
    const C *kc = static_cast<const C *>(a.k) + h / a.group * a.pages.head_stride;
    const C *vc = static_cast<const C *>(a.v) + h / a.group * a.pages.head_stride;
    float m = -INFINITY, l = 0.0f, acc[D / 64] = {};
    for (int j0 = lo; j0 < hi; j0 += 64) {
        const int64_t row = j0 + lane < hi ? row_offset(a.pages, b, j0 + lane) : -1;
        float s = -INFINITY;
        if (row >= 0) {
            s = 0.0f;
            for (int d = 0; d < D; ++d) s += qs[d] * static_cast<float>(kc[row + d]);
        }
        float mx = s;
        for (int d = 1; d < 64; d *= 2) mx = fmaxf(mx, __shfl_xor(mx, d));
        const float mn = fmaxf(m, mx);
        if (mn == -INFINITY) continue;
        const float p = row >= 0 ? expf(s - mn) : 0.0f, f = expf(m - mn);
        m = mn;
        float sum = p;
        for (int d = 1; d < 64; d *= 2) sum += __shfl_xor(sum, d);
        l = l * f + sum;
        for (int i = 0; i < D / 64; ++i) acc[i] *= f;
        for (int j = 0; j < min(64, hi - j0); ++j) {
            const int64_t r = __shfl(row, j);
            const float pj = __shfl(p, j);
            if (r < 0) continue;
            for (int i = 0; i < D / 64; ++i) acc[i] += pj * static_cast<float>(vc[r + lane + 64 * i]);
        }
    }
    T *o = static_cast<T *>(a.out) + t * a.out_stride + h * D;
    for (int i = 0; i < D / 64; ++i) o[lane + 64 * i] = static_cast<T>(l > 0.0f ? acc[i] / l : 0.0f);
}

template <typename T, typename C>
void launch_attn(const AttnArgs &a, int D, hipStream_t s) {
    const dim3 grid(a.n_tokens, a.n_heads);
    if (D == 64)
        attn_simple<T, C, 64><<<grid, 64, 0, s>>>(a);
    else if (D == 128)
        attn_simple<T, C, 128><<<grid, 64, 0, s>>>(a);
    else
        attn_simple<T, C, 256><<<grid, 64, 0, s>>>(a);
}

int check_attn(const tqhip_attn &p, const tqhip_kv_cache &c, const tqhip_seqs &s) {
    const int st = check_cache(c, s);
    if (st != kOk) return st;
    if (!p.q || !p.out || !type_known(p.dtype) || p.n_heads < 1 || p.n_heads % c.n_kv_heads || p.window < 0 ||
        !std::isfinite(p.scale) || (p.dtype != TQHIP_F32 && c.dtype != p.dtype))
        return kBadShape;
    if (c.head_dim != 64 && c.head_dim != 128 && c.head_dim != 256) return kBadShape;
    const int qb = type_bytes(p.dtype), cb = type_bytes(c.dtype);
    int64_t page, token, head;
    (void)cache_strides(c, &page, &token, &head);
    const uintptr_t bases = reinterpret_cast<uintptr_t>(p.q) | reinterpret_cast<uintptr_t>(p.out) |
                            reinterpret_cast<uintptr_t>(c.k) | reinterpret_cast<uintptr_t>(c.v);
    if (bases % 16 || p.q_stride * qb % 16 || p.out_stride * qb % 16 || page * cb % 16 || token * cb % 16 || head * cb % 16)
        return kBadShape;
    const int64_t row = static_cast<int64_t>(p.n_heads) * c.head_dim;
    if (s.n_tokens > 1 && ((p.q_stride && p.q_stride < row) || (p.out_stride && p.out_stride < row))) return kBadShape;
    if (p.n_heads > 65535 || static_cast<int64_t>(s.n_tokens) * p.n_heads > INT32_MAX) return kTooLarge;
    return kOk;
}

int run_attn(const tqhip_attn &p, const tqhip_kv_cache &c, const tqhip_seqs &b, hipStream_t s) {
    const int st = check_attn(p, c, b);
    if (st != kOk) return st;
    const int64_t row = static_cast<int64_t>(p.n_heads) * c.head_dim;
    const AttnArgs a{p.q, c.k, c.v, p.out, p.q_stride ? p.q_stride : row, p.out_stride ? p.out_stride : row, b.q_start,
                     b.kv_len, b.n_seqs, b.n_tokens, p.n_heads, p.n_heads / c.n_kv_heads, p.scale, p.causal,
                     p.window, make_pages(c, b)};
    if (p.dtype == TQHIP_F16)
        launch_attn<f16, f16>(a, c.head_dim, s);
    else if (p.dtype == TQHIP_BF16)
        launch_attn<bf16, bf16>(a, c.head_dim, s);
    else if (c.dtype == TQHIP_F32)
        launch_attn<float, float>(a, c.head_dim, s);
    else if (c.dtype == TQHIP_F16)
        launch_attn<float, f16>(a, c.head_dim, s);
    else
        launch_attn<float, bf16>(a, c.head_dim, s);
    return hipGetLastError() == hipSuccess ? kOk : kLaunchFailed;
}

}  // namespace
}  // namespace tqhip

extern "C" {

int tqhip_paged_attention_dev(const tqhip_attn *attn, const tqhip_kv_cache *cache, const tqhip_seqs *seqs,
                              void *stream) {
    if (!attn || !cache || !seqs) return tqhip::kBadShape;
    return tqhip::run_attn(*attn, *cache, *seqs, static_cast<hipStream_t>(stream));
}

size_t tqhip_paged_attention_workspace(const tqhip_attn *attn, const tqhip_kv_cache *cache, const tqhip_seqs *seqs) {
    (void)attn, (void)cache, (void)seqs;
    return 0;
}

}  // extern "C"
