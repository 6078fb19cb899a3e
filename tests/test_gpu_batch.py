"""The batch calls on the GPU against plain 64-bit forms (batch_ref.py): heads normed and rotated, appended to a paged
cache, attended to, and low-rank adapters, at the sizes, masks and layouts where each can go wrong.

Tolerances. One rounding to a type is off by at most half a step (HALF). In fp32 u = 2^-24:
heads: a result is made of two normed values, each a sum (1 u), a root of a mean of up to 512 squares summed in a tree of
depth <= 14 (at most 8 u after the root), two products (2 u), times a sine or cosine (within 4 u of its argument's: a rounded
half-turn, pi u, and the function's own step), and added (2 u): 20 u of the size of its terms.
attention: a score is D products and sums, at most (D + 4) u of the sum of their sizes, S; e^x multiplies its error, and the
weights enter numerator and denominator: 2 (D + 4) u S; N weights and products summed: at most (N + 16) u each. So within
(2 (D + 4) S + 2 N + 32) u of sum p |v|. f16 / bf16 activations: one rounding of the weights (a bf16 or f16 half step of
sum p |v|) and one of the result. That bound is loose for fp32, where errors are random, so those results are held to a
relative L2 distance of 2^-17 too: a lost 16-bit term of a score or weight is 2^-8 or 2^-11 of it.
lora: K products and sums, then r, of the size of the terms: (K + r + 8) u at most, and 2^-18 of them in L2.
"""
import numpy as np
import pytest

import batch_ref as ref
from batch_ref import HALF, TINY, Batch, Dev, ints

pytestmark = pytest.mark.gpu

F32, F16, BF16 = 0, 1, 2
U = 2.0 ** -24


def f32_buffer(gpu, x):
    return None if x is None else gpu.DeviceBuffer.from_array(np.asarray(x, np.float32))


def ptr(b):
    return None if b is None else b.ptr


def head_inputs(gpu, rng, T, Hq, Hk, D, act, bias, norm, packed=False):
    """q, k, v as the projections leave them (one matrix when packed), and their biases and norms."""
    s = {}
    if packed:
        x = Dev(gpu, rng.standard_normal((T, (Hq + 2 * Hk) * D)), act)
        w = {0: 4, 1: 2, 2: 2}[act]
        cut = {"q": (0, Hq), "k": (Hq, Hk), "v": (Hq + Hk, Hk)}
        s["keep"] = x
        for n, (at, h) in cut.items():
            s[n] = (x.ptr + at * D * w, (Hq + 2 * Hk) * D, x.values[:, at * D:(at + h) * D].reshape(T, h, D))
    else:
        for n, h in (("q", Hq), ("k", Hk), ("v", Hk)):
            x = Dev(gpu, rng.standard_normal((T, h, D)), act)
            s["keep_" + n] = x
            s[n] = (x.ptr, 0, x.values)
    for n, h in (("q", Hq), ("k", Hk), ("v", Hk)):
        b = rng.standard_normal(h * D).astype(np.float32) if bias else None
        s[n + "_bias"] = (b, f32_buffer(gpu, b))
        w = (1 + 0.2 * rng.standard_normal(D)).astype(np.float32) if norm and n != "v" else None
        s[n + "_norm"] = (w, f32_buffer(gpu, w))
    return s


def proj_of(gpu, s, T, Hq, Hk, D, act, rotary, q_out, k_out=None, positions=None, eps=1e-6, theta=1e6, inv_freq=None):
    return gpu.HeadProj(dtype=act, n_tokens=T, n_heads=Hq, n_kv_heads=Hk, head_dim=D, rotary_dim=rotary, q=s["q"][0], k=s["k"][0], v=s["v"][0],
                        q_out=ptr(q_out), k_out=ptr(k_out), q_stride=s["q"][1], k_stride=s["k"][1], v_stride=s["v"][1],
                        q_bias=ptr(s["q_bias"][1]), k_bias=ptr(s["k_bias"][1]), v_bias=ptr(s["v_bias"][1]), q_norm=ptr(s["q_norm"][1]),
                        k_norm=ptr(s["k_norm"][1]), eps=eps, theta=theta, positions=ptr(positions), inv_freq=ptr(inv_freq))


def check_heads(got, want, size, dtype, what):
    bound = 20 * U * size + HALF[dtype] * np.abs(want) * (dtype != F32) + TINY[dtype]
    bad = ~(np.abs(got - want) <= bound)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} off, worst {np.nanmax(np.abs(got - want) / np.maximum(bound, 1e-300)):.2f} bounds"


# Head widths on the vector path (4 to 32 lanes a head) and off it (odd pairs, 24, 80, 512), partial rotation, no rotation;
# one token and more tokens than waves; one matrix of q, k and v; positions far out.
HEADS = [
    (1, 32, 8, 128, F32, False, True, 128, False), (3, 14, 2, 64, F32, True, False, 64, True), (5, 2, 1, 256, F32, False, True, 256, False),
    (77, 4, 4, 32, F32, True, True, 16, False), (9, 3, 1, 24, F32, False, True, 24, False), (6, 2, 2, 80, F32, True, True, 80, False),
    (2, 1, 1, 512, F32, False, True, 512, False), (4, 5, 1, 6, F32, True, True, 2, False), (31, 14, 2, 64, F16, False, True, 64, True),
    (13, 32, 8, 128, BF16, True, True, 32, False), (2500, 7, 1, 128, F32, False, True, 128, True), (9, 2, 1, 256, BF16, False, False, 0, False),
    (4, 3, 1, 2, F16, True, True, 2, False),
]


@pytest.mark.parametrize("T,Hq,Hk,D,act,bias,norm,rotary,packed", HEADS)
def test_qk_norm_rope(gpu, T, Hq, Hk, D, act, bias, norm, rotary, packed):
    rng = np.random.default_rng(T * 7 + D)
    s = head_inputs(gpu, rng, T, Hq, Hk, D, act, bias, norm, packed)
    pos = rng.integers(0, 150000, T)
    pos[0] = 0
    q_out, k_out = Dev(gpu, np.full((T, Hq, D), 7.0), act), Dev(gpu, np.full((T, Hk, D), 7.0), act)
    d_pos = ints(gpu, pos)
    gpu.qk_norm_rope_dev(proj_of(gpu, s, T, Hq, Hk, D, act, rotary, q_out, k_out, d_pos))
    gpu.synchronize()
    for n, out in (("q", q_out), ("k", k_out)):
        want, size = ref.finish_heads(s[n][2], s[n + "_bias"][0], s[n + "_norm"][0], pos, rotary, 1e-6, 1e6)
        check_heads(out.read(), want, size, act, n)


def test_qk_norm_rope_in_place_one_side_and_strided_outputs(gpu):
    T, Hq, Hk, D = 10, 6, 2, 64
    rng = np.random.default_rng(5)
    s = head_inputs(gpu, rng, T, Hq, Hk, D, F32, False, True)
    pos = np.arange(T) * 1000
    d_pos = ints(gpu, pos)
    want_q, size_q = ref.finish_heads(s["q"][2], None, s["q_norm"][0], pos, D, 1e-6, 1e6)
    want_k, size_k = ref.finish_heads(s["k"][2], None, s["k_norm"][0], pos, D, 1e-6, 1e6)
    # q alone, into rows twice as far apart (the gap untouched)
    wide = Dev(gpu, np.full((T, 2 * Hq, D), 3.0), F32)
    p = proj_of(gpu, s, T, Hq, Hk, D, F32, D, wide, None, d_pos)
    p.k, p.q_out_stride = None, 2 * Hq * D
    gpu.qk_norm_rope_dev(p)
    # k alone, in place
    p = proj_of(gpu, s, T, Hq, Hk, D, F32, D, None, None, d_pos)
    p.q, p.k_out = None, p.k
    gpu.qk_norm_rope_dev(p)
    gpu.synchronize()
    got = wide.read()
    check_heads(got[:, :Hq], want_q, size_q, F32, "strided q")
    assert np.all(got[:, Hq:] == 3.0)
    check_heads(s["keep_k"].read(), want_k, size_k, F32, "in-place k")


def test_qk_norm_rope_frequencies_and_unaligned_rows(gpu):
    T, Hq, Hk, D = 7, 2, 1, 64
    rng = np.random.default_rng(6)
    inv = (1e4 ** (-np.arange(D // 2) / (D // 2)) / 8).astype(np.float32)
    pos = rng.integers(0, 1000000, T)
    d_pos, d_inv = ints(gpu, pos), f32_buffer(gpu, inv)
    x = Dev(gpu, rng.standard_normal((T, Hq * D + 1)), F32)  # rows of an odd number of elements, from the second one on
    out = Dev(gpu, np.full((T, Hq, D), 7.0), F32)
    gpu.qk_norm_rope_dev(gpu.HeadProj(dtype=F32, n_tokens=T, n_heads=Hq, n_kv_heads=Hk, head_dim=D, rotary_dim=D, q=x.ptr + 4, q_out=out.ptr,
                                      q_stride=Hq * D + 1, inv_freq=d_inv.ptr, positions=d_pos.ptr))
    gpu.synchronize()
    flat = np.concatenate([x.values.reshape(-1)[1:], [0.0]])
    q = np.stack([flat[t * (Hq * D + 1):t * (Hq * D + 1) + Hq * D] for t in range(T - 1)] + [flat[(T - 1) * (Hq * D + 1):][:Hq * D]]).reshape(T, Hq, D)
    want, size = ref.finish_heads(q, None, None, pos, D, 0, 0, inv)
    check_heads(out.read()[:T - 1], want[:T - 1], size[:T - 1], F32, "inv_freq")


@pytest.mark.parametrize("act,cache", [(F32, F32), (F32, F16), (F32, BF16), (F16, F16), (BF16, BF16)])
@pytest.mark.parametrize("Hq,Hk,D,page,layout", [(14, 2, 64, 48, "token"), (8, 2, 128, 16, "head"), (3, 1, 24, 7, "token")])
def test_kv_append(gpu, act, cache, Hq, Hk, D, page, layout):
    """Sequences with many, one and no new tokens, one with more tokens than positions, missing pages, tokens outside."""
    new, kv = [5, 1, 0, 40, 3, 1], [5, 100, 33, 90, 2, 2 * page + 1]
    b = Batch(gpu, new, kv, page, Hk, D, cache, seed=3, tail=2, lead=1, bad=[(3, 80 // page)], layout=layout)
    T = b.tokens
    s = head_inputs(gpu, b.rng, T, Hq, Hk, D, act, True, True)
    before = b.k.read_bits(), b.v.read_bits()
    q_out = Dev(gpu, np.full((T, Hq, D), 7.0), act)
    gpu.kv_append_dev(proj_of(gpu, s, T, Hq, Hk, D, act, D, q_out), b.c, b.s)
    gpu.synchronize()
    at = b.token_positions()
    pos = np.array([at.get(t, (0, 0))[1] for t in range(T)])
    want_q, size_q = ref.finish_heads(s["q"][2], s["q_bias"][0], s["q_norm"][0], pos, D, 1e-6, 1e6)
    want_k, size_k = ref.finish_heads(s["k"][2], s["k_bias"][0], s["k_norm"][0], pos, D, 1e-6, 1e6)
    want_v, size_v = ref.finish_heads(s["v"][2], s["v_bias"][0], None, pos, 0, 0, 1)
    got_q = q_out.read()
    live = [t for t in at if at[t][1] >= 0]
    dead = [t for t in range(T) if t not in live]
    check_heads(got_q[live], want_q[live], size_q[live], act, "q")
    assert dead and np.all(got_q[dead] == 7.0)
    for dev, old, want, size, what in ((b.k, before[0], want_k, size_k, "k"), (b.v, before[1], want_v, size_v, "v")):
        got, bits = b.rows(dev.read()), b.rows(dev.read_bits())
        old = b.rows(old).copy()
        written = 0
        for t in live:
            pl = b.place(*at[t])
            if pl:
                check_heads(got[pl], want[t], size[t], cache, f"{what} row {at[t]}")
                old[pl] = bits[pl]
                written += 1
        assert 0 < written < len(live)  # (one page is missing)
        assert np.array_equal(old, bits), f"{what}: rows outside the call's positions changed"


def check_attention(gpu, b, act, Hq, causal, window, scale=None, q_std=1.5, stream=None, q_pad=0):
    T, D = b.tokens, b.D
    scale = D ** -0.5 if scale is None else scale
    q = Dev(gpu, q_std * b.rng.standard_normal((T, Hq + q_pad, D)), act)
    out = Dev(gpu, np.full((T, Hq + q_pad, D), 7.0), act)
    gpu.paged_attention_dev(gpu.Attn(dtype=act, n_heads=Hq, q=q.ptr, out=out.ptr, scale=scale, causal=causal, window=window,
                                     q_stride=(Hq + q_pad) * D, out_stride=(Hq + q_pad) * D), b.c, b.s, stream)
    gpu.synchronize()
    want, spread, score, live = ref.attention(b, q.values[:, :Hq], float(np.float32(scale)), causal, window)
    got = out.read()
    dead = np.setdiff1d(np.arange(T), live)
    assert np.all(got[dead] == 7.0) and np.all(got[:, Hq:] == 7.0), "rows outside the call changed"
    got = got[:, :Hq]
    N = max(b.kv)
    bound = (2 * (D + 4) * score + 2 * N + 32) * U * spread
    if act != F32:
        bound = bound + HALF[act] * (spread + np.abs(want)) + TINY[act]
    bad = ~(np.abs(got - want) <= bound)[live]
    assert not bad.any(), f"{bad.sum()} of {bad.size} off, worst {np.nanmax((np.abs(got - want) / np.maximum(bound, 1e-300))[live]):.2f} bounds"
    if act == F32:
        den = np.linalg.norm(want[live])
        assert np.linalg.norm((got - want)[live]) <= 2.0 ** -17 * den


TYPES = [(F32, F32), (F32, F16), (F32, BF16), (F16, F16), (BF16, BF16)]
SHAPES = [(14, 2, 64), (8, 2, 128), (2, 1, 256)]


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("Hq,Hk,D", SHAPES)
def test_attention_single_tokens(gpu, act, cache, Hq, Hk, D):
    """Lengths of zero (more tokens than positions), one, about a tile, and long ones; tokens outside every sequence."""
    kv = [1, 0, 2, 31, 32, 33, 63, 64, 65, 700, 129, 1500]
    b = Batch(gpu, [1] * len(kv), kv, 16, Hk, D, cache, seed=D, tail=2, lead=1)
    check_attention(gpu, b, act, Hq, 1, 0)


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("Hq,Hk,D", SHAPES)
def test_attention_chunks(gpu, act, cache, Hq, Hk, D):
    """Chunks of 0, 1, a few and many tokens over caches that end inside a page, positions before the cache's first."""
    b = Batch(gpu, [70, 1, 0, 5, 129, 4], [70, 90, 12, 300, 400, 2], 48, Hk, D, cache, seed=D + 1, tail=3, layout="head")
    check_attention(gpu, b, act, Hq, 1, 0)


@pytest.mark.parametrize("new", [[1, 1], [40, 3]])
@pytest.mark.parametrize("scale", [0.0, -0.2])
def test_attention_scale_of_zero_and_below(gpu, new, scale):
    b = Batch(gpu, new, [150, 60], 16, 1, 64, F16, seed=20)
    check_attention(gpu, b, F32, 3, 1, 0, scale=scale)


@pytest.mark.parametrize("page", [1, 7, 40, 64, 1000])
def test_attention_page_sizes(gpu, page):
    b = Batch(gpu, [33, 1, 3], [200, 333, 70], page, 2, 64, F16, seed=page)
    check_attention(gpu, b, F32, 6, 1, 0)


@pytest.mark.parametrize("new", [[1, 1, 1, 1], [90, 3, 1, 64]])
@pytest.mark.parametrize("causal,window", [(0, 0), (1, 1), (1, 37), (1, 5000)])
def test_attention_masks(gpu, new, causal, window):
    b = Batch(gpu, new, [600, 77, 1, 64], 16, 1, 128, BF16, seed=window)
    check_attention(gpu, b, F32, 4, causal, window)


@pytest.mark.parametrize("new", [[1, 1, 1], [50, 64, 3]])
def test_attention_missing_pages(gpu, new):
    """Pages outside the cache hold no positions; a sequence of them alone gives zeros."""
    b = Batch(gpu, new, [200, 64, 500], 32, 2, 64, F16, seed=4, bad=[(0, 0), (0, 3), (1, 0), (1, 1), (2, 5), (2, 15)])
    check_attention(gpu, b, F32, 4, 1, 0)


@pytest.mark.parametrize("Hq,Hk", [(1, 1), (5, 5), (20, 1), (33, 1), (64, 8)])
def test_attention_head_groups(gpu, Hq, Hk):
    b = Batch(gpu, [1, 9, 40], [130, 70, 41], 16, Hk, 64, F16, seed=Hq)
    check_attention(gpu, b, F32, Hq, 1, 0)


@pytest.mark.parametrize("new", [[1] * 3, [200] * 2])
@pytest.mark.parametrize("cache", [F16, BF16, F32])
def test_attention_large_scores(gpu, new, cache):
    """Scores of hundreds, of either sign: one weight is near 1, the rest are tiny, and maxima move late."""
    b = Batch(gpu, new, [400 + 17 * i for i in range(len(new))], 16, 1, 64, cache, seed=9)
    check_attention(gpu, b, F32, 4, 1, 0, scale=1.0, q_std=12.0)


@pytest.mark.parametrize("q_std", [1e-20, 1e5, 1e20])
def test_attention_wide_range_queries(gpu, q_std):
    """fp32 queries beyond fp16's range, brought back by the scale."""
    b = Batch(gpu, [1, 70], [100, 200], 16, 2, 64, F16, seed=10)
    check_attention(gpu, b, F32, 4, 1, 0, scale=float(np.float32(0.2 / q_std)), q_std=q_std)


def test_attention_strided_queries_and_a_stream(gpu):
    b = Batch(gpu, [1, 30, 1], [50, 60, 900], 16, 2, 128, BF16, seed=11)
    check_attention(gpu, b, F32, 6, 1, 0, q_pad=3, stream=gpu.Stream())


def test_attention_long_sequence_without_a_length_hint(gpu):
    b = Batch(gpu, [1, 1, 20], [9000, 40, 3000], 16, 1, 64, F16, seed=12)
    b.s.max_kv = 0
    check_attention(gpu, b, F32, 7, 1, 0)


LORA = [  # tokens of each request, adapters of each, K, M, rank
    ([1], [0], 64, 5, 1), ([1] * 9, [0, 3, -1, 2, 2, 7, 1, 0, 3], 896, 130, 16), ([5, 0, 17, 40, 1, 3], [1, 0, 3, -1, 2, 1], 260, 33, 8),
    ([70, 130], [2, 0], 516, 900, 64), ([33], [1], 100, 64, 3), ([3, 200], [0, 1], 1001, 257, 100), ([2, 2], [3, 1], 40, 30, 256),
]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("new,adapter,K,M,r", LORA)
def test_lora_add(gpu, dtype, new, adapter, K, M, r):
    """Adapter 7 is outside the four: as none. Tokens before the first and after the last request keep their y."""
    rng = np.random.default_rng(K + M + r)
    n, starts = 4, 1 + np.concatenate(([0], np.cumsum(new)))
    T = int(starts[-1]) + 2
    x, base = rng.standard_normal((T, K)).astype(np.float32), rng.standard_normal((T, M)).astype(np.float32)
    a, b = Dev(gpu, rng.standard_normal((n, r, K)) / np.sqrt(K), dtype), Dev(gpu, 0.3 * rng.standard_normal((n, M, r)), dtype)
    scale = rng.uniform(0.5, 2, n).astype(np.float32)
    dx, db, ds, dst, dad = f32_buffer(gpu, x), f32_buffer(gpu, base), f32_buffer(gpu, scale), ints(gpu, starts), ints(gpu, adapter)
    want, size = ref.lora(x.astype(np.float64), base.astype(np.float64), a.values, b.values, scale.astype(np.float64), starts, adapter, T)
    inside = slice(1, int(starts[-1]))

    def call(dbase, dy):
        gpu.lora_add_dev(gpu.Lora(dtype=dtype, n_tokens=T, in_dim=K, out_dim=M, rank=r, n_adapters=n, n_seqs=len(new), x=dx.ptr, base=dbase, y=dy,
                                  a=a.ptr, b=b.ptr, scale=ds.ptr, q_start=dst.ptr, adapter=dad.ptr))
        gpu.synchronize()

    def check(got, want, outside, what):
        got = got.reshape(T, M)
        assert np.array_equal(got[0], outside[0]) and np.array_equal(got[-2:], outside[-2:]), f"{what}: rows outside the call changed"
        off = np.abs(got.astype(np.float64) - want)[inside]
        assert np.all(off <= (K + r + 8) * U * size[inside]), what
        assert np.linalg.norm(off) <= 2.0 ** -18 * np.linalg.norm(size[inside]), what

    seven = np.full((T, M), 7.0, np.float32)
    dy = f32_buffer(gpu, seven)
    call(db.ptr, dy.ptr)
    check(dy.download(np.float32, T * M), want, seven, "y = base + delta")
    call(None, dy.ptr)
    check(dy.download(np.float32, T * M), want - base, seven, "y = delta")
    call(db.ptr, db.ptr)
    check(db.download(np.float32, T * M), want, base, "in place")


@pytest.mark.parametrize("cache", [F16, BF16, F32])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_attention_masked_infinities_and_nan(gpu, cache, D):
    """Rows of a chunk's later tokens hold infinities and NaN: the tokens before them must not notice, the ones that see
    them must not be finite in the value's dimension."""
    n, kv = 40, 150
    b = Batch(gpu, [n, 1], [kv, 90], 16, 1, D, cache, seed=13)
    rows = {}
    for p, (where, x) in {120: ("v", np.inf), 133: ("k", np.nan), 140: ("v", np.nan), 149: ("v", -np.inf)}.items():
        pg, r = b.place(0, p)
        dev = b.v if where == "v" else b.k
        full = dev.values
        full[pg, r, 0, 5] = x
        dev.buf.upload(ref.raw(full, cache)[0])
        rows[p] = (where, x)
    q = Dev(gpu, 1.5 * b.rng.standard_normal((b.tokens, 4, D)), F32)
    out = Dev(gpu, np.full((b.tokens, 4, D), 7.0), F32)
    gpu.paged_attention_dev(gpu.Attn(dtype=F32, n_heads=4, q=q.ptr, out=out.ptr, scale=D ** -0.5, causal=1), b.c, b.s)
    gpu.synchronize()
    got = out.read()
    with np.errstate(invalid="ignore"):
        want = ref.attention(b, q.values, float(np.float32(D ** -0.5)), 1, 0)[0]
    first = kv - n  # position of token 0
    clean = [t for t in range(n + 1) if t == n or first + t < 120]
    assert np.linalg.norm(got[clean] - want[clean]) <= 2.0 ** -17 * np.linalg.norm(want[clean])
    one = [t for t in range(n) if 120 <= first + t < 133]  # see the infinity in dimension 5 alone
    keep = np.arange(D) != 5
    assert np.linalg.norm((got - want)[one][..., keep]) <= 2.0 ** -17 * np.linalg.norm(want[one][..., keep])
    assert not np.isfinite(got[one][..., 5]).any()
    assert np.isnan(got[[t for t in range(n) if first + t >= 133]]).all()


def test_kv_append_keys_alone_at_given_positions(gpu):
    """No queries, angles of the caller's positions, no rotation of the rest of the head."""
    b = Batch(gpu, [2, 1, 4], [9, 30, 4], 8, 2, 64, F32, seed=30)
    T = b.tokens
    s = head_inputs(gpu, b.rng, T, 4, 2, 64, F32, False, True)
    pos = np.array([1000, 3, 70000, 0, 5, 6, 9])
    d_pos = ints(gpu, pos)
    p = proj_of(gpu, s, T, 4, 2, 64, F32, 32, None, None, d_pos)
    p.q = None
    gpu.kv_append_dev(p, b.c, b.s)
    gpu.synchronize()
    want, size = ref.finish_heads(s["k"][2], None, s["k_norm"][0], pos, 32, 1e-6, 1e6)
    got_k, got_v = b.k.read(), b.v.read()
    for t, at in b.token_positions().items():
        check_heads(got_k[b.place(*at)], want[t], size[t], F32, f"k of token {t}")
        assert np.array_equal(got_v[b.place(*at)], s["v"][2][t])


def test_positions_past_the_table_do_not_exist(gpu):
    """A cached length beyond the table's pages: the rows past them are neither written nor attended to."""
    b = Batch(gpu, [3, 1], [32, 20], 16, 1, 64, F16, seed=31)  # (the table has three entries a sequence)
    b.kv = [50, 20]
    b.d_kv = ints(gpu, b.kv)
    b.s.kv_len, b.s.max_kv = b.d_kv.ptr, 50
    before = b.k.read_bits()
    s = head_inputs(gpu, b.rng, b.tokens, 2, 1, 64, F32, False, False)
    q_out = Dev(gpu, np.full((b.tokens, 2, 64), 7.0), F32)
    gpu.kv_append_dev(proj_of(gpu, s, b.tokens, 2, 1, 64, F32, 64, q_out), b.c, b.s)
    gpu.synchronize()
    after = b.k.read_bits()
    changed = np.argwhere((before != after).any((2, 3)))
    assert [tuple(c) for c in changed] == [b.place(1, 19)]  # positions 47..49 of sequence 0 are past its pages
    b.k.values, b.v.values = b.k.read(), b.v.read()
    check_attention(gpu, b, F32, 2, 1, 0)


@pytest.mark.parametrize("new,kv", [([1, 1], [700, 2600]), ([300, 64], [900, 2600])])
@pytest.mark.parametrize("window", [0, 50, 2 ** 31 - 1])
@pytest.mark.parametrize("max_kv", [1, 300, 2 ** 31 - 1])
def test_attention_split_by_a_wrong_length(gpu, new, kv, window, max_kv):
    """max_kv decides how the work is split and nothing else, too small and too large ones too."""
    b = Batch(gpu, new, kv, 16, 1, 64, F16, seed=35)
    b.s.max_kv = max_kv
    check_attention(gpu, b, F32, 2, 1, window)


@pytest.mark.parametrize("length", [2 ** 31 - 1, 2 ** 30, -2 ** 31, -1, 0])
@pytest.mark.parametrize("new", [[1, 1], [120, 30]])
@pytest.mark.parametrize("page", [1, 16])
def test_lengths_that_no_table_holds(gpu, length, new, page):
    """A sequence whose window lies past its table, or whose length is no length, gets zeros; the other one is as ever."""
    b = Batch(gpu, new, [150, 140], page, 1, 64, F16, seed=36)
    q, out = Dev(gpu, b.rng.standard_normal((b.tokens, 2, 64)), F32), Dev(gpu, np.full((b.tokens, 2, 64), 7.0), F32)
    attn = gpu.Attn(dtype=F32, n_heads=2, q=q.ptr, out=out.ptr, scale=0.125, causal=1, window=20)
    gpu.paged_attention_dev(attn, b.c, b.s)
    gpu.synchronize()
    want = out.read()
    want[: new[0]] = 0
    b.d_kv.upload(np.int32([length, 140]))
    gpu.paged_attention_dev(attn, b.c, b.s)
    gpu.synchronize()
    assert np.array_equal(out.read(), want)


def test_many_sequences(gpu):
    """More sequences than two rounds of the search cover, most without tokens, and their tokens found by all the calls."""
    rng = np.random.default_rng(32)
    B, D = 5000, 64
    new = (rng.random(B) < 0.03).astype(int)
    new[[0, 63, 64, 4095, 4096, 4999]] = [2, 1, 3, 1, 17, 1]
    kv = np.where(new > 0, rng.integers(0, 12, B) + new, 0)
    b = Batch(gpu, new, kv, 4, 1, D, F32, seed=33, tail=1)
    s = head_inputs(gpu, b.rng, b.tokens, 2, 1, D, F32, False, True)
    q_out = Dev(gpu, np.full((b.tokens, 2, D), 7.0), F32)
    gpu.kv_append_dev(proj_of(gpu, s, b.tokens, 2, 1, D, F32, D, q_out), b.c, b.s)
    gpu.synchronize()
    at = b.token_positions()
    assert len(at) == b.tokens - 1
    pos = np.array([at.get(t, (0, 0))[1] for t in range(b.tokens)])
    want, size = ref.finish_heads(s["k"][2], None, s["k_norm"][0], pos, D, 1e-6, 1e6)
    got = b.k.read()
    for t, a in at.items():
        check_heads(got[b.place(*a)], want[t], size[t], F32, f"token {t}")
    b.k.values, b.v.values = b.k.read(), b.v.read()
    check_attention(gpu, b, F32, 2, 1, 0)
    K, M, r, n = 32, 20, 4, 3
    x, base = rng.standard_normal((b.tokens, K)).astype(np.float32), rng.standard_normal((b.tokens, M)).astype(np.float32)
    a_, b_ = Dev(gpu, rng.standard_normal((n, r, K)), F16), Dev(gpu, rng.standard_normal((n, M, r)), F16)
    scale, of = np.float32([1, 2, 0.5]), rng.integers(-1, n, B)
    dx, db, ds, dof, dy = f32_buffer(gpu, x), f32_buffer(gpu, base), f32_buffer(gpu, scale), ints(gpu, of), f32_buffer(gpu, base)
    gpu.lora_add_dev(gpu.Lora(dtype=F16, n_tokens=b.tokens, in_dim=K, out_dim=M, rank=r, n_adapters=n, n_seqs=B, x=dx.ptr, base=db.ptr, y=dy.ptr,
                              a=a_.ptr, b=b_.ptr, scale=ds.ptr, q_start=b.d_start.ptr, adapter=dof.ptr))
    gpu.synchronize()
    want, size = ref.lora(x.astype(np.float64), base.astype(np.float64), a_.values, b_.values, scale, b.starts, of, b.tokens)
    assert np.all(np.abs(dy.download(np.float32, base.size).reshape(base.shape) - want) <= (K + r + 8) * U * size)


def test_rows_past_4_gib(gpu):
    """Pages more than 2^31 elements apart in one allocation: appended to and attended to."""
    D, page, far = 64, 16, (1 << 31) + 4096
    room = gpu.DeviceBuffer(2 * (far + 2 * page * D))
    start, kv, table = ints(gpu, [0, 20]), ints(gpu, [20]), ints(gpu, [[1, 0]])
    cache = gpu.KvCache(k=room.ptr, v=room.ptr + 2 * page * D, dtype=F16, n_pages=2, page_size=page, n_kv_heads=1, head_dim=D, page_stride=far,
                        token_stride=D, head_stride=D)
    seqs = gpu.Seqs(n_seqs=1, n_tokens=20, q_start=start.ptr, kv_len=kv.ptr, block_table=table.ptr, table_stride=2, max_kv=20)
    rng = np.random.default_rng(34)
    s = head_inputs(gpu, rng, 20, 2, 1, D, F32, False, False)
    q_out, out = Dev(gpu, np.zeros((20, 2, D)), F32), Dev(gpu, np.zeros((20, 2, D)), F32)
    gpu.kv_append_dev(proj_of(gpu, s, 20, 2, 1, D, F32, 0, q_out), cache, seqs)
    gpu.paged_attention_dev(gpu.Attn(dtype=F32, n_heads=2, q=q_out.ptr, out=out.ptr, scale=0.125, causal=1), cache, seqs)
    gpu.synchronize()
    k, v = (s[n][2][:, 0].astype(np.float16).astype(np.float64) for n in ("k", "v"))
    for h in range(2):
        w = np.where(np.tri(20) > 0, s["q"][2][:, h] @ k.T / 8, -np.inf)
        w = np.exp(w - w.max(-1, keepdims=True))
        want = w / w.sum(-1, keepdims=True) @ v
        assert np.linalg.norm(out.read()[:, h] - want) <= 2.0 ** -17 * np.linalg.norm(want)


def test_same_bits_again_and_on_two_streams(gpu):
    """Calls that overlap on two streams, each with scratch of its own, give what each gives alone, again and again."""
    cases = []
    for seed, new, kv in ((40, [1] * 6, [3000, 10, 700, 1, 64, 2100]), (41, [150, 20], [2500, 900])):
        b = Batch(gpu, new, kv, 16, 2, 128, F16, seed=seed)
        q = Dev(gpu, b.rng.standard_normal((b.tokens, 8, 128)), F32)
        out = Dev(gpu, np.zeros((b.tokens, 8, 128)), F32)
        x, y = f32_buffer(gpu, b.rng.standard_normal((b.tokens, 512))), f32_buffer(gpu, np.zeros((b.tokens, 260)))
        a_, b_ = Dev(gpu, b.rng.standard_normal((2, 24, 512)), BF16), Dev(gpu, b.rng.standard_normal((2, 260, 24)), BF16)
        sc, of = f32_buffer(gpu, [1.0, 2.0]), ints(gpu, [i % 2 for i in range(len(new))])
        lo = gpu.Lora(dtype=BF16, n_tokens=b.tokens, in_dim=512, out_dim=260, rank=24, n_adapters=2, n_seqs=len(new), x=x.ptr, y=y.ptr, a=a_.ptr,
                      b=b_.ptr, scale=sc.ptr, q_start=b.d_start.ptr, adapter=of.ptr)
        at = gpu.Attn(dtype=F32, n_heads=8, q=q.ptr, out=out.ptr, scale=0.1, causal=1)
        cases.append((b, at, lo, out, y, gpu.Stream(), (q, x, a_, b_, sc, of)))
    first = []
    for b, at, lo, out, y, stream, _ in cases:
        gpu.paged_attention_dev(at, b.c, b.s, stream)
        gpu.lora_add_dev(lo, stream)
        stream.synchronize()
        first.append((out.read_bits(), y.download(np.int32, b.tokens * 260)))
    for _ in range(4):
        for b, at, lo, out, y, stream, _ in cases * 3:
            gpu.paged_attention_dev(at, b.c, b.s, stream)
            gpu.lora_add_dev(lo, stream)
        for (b, at, lo, out, y, stream, _), (o1, y1) in zip(cases, first):
            stream.synchronize()
            assert np.array_equal(out.read_bits(), o1) and np.array_equal(y.download(np.int32, b.tokens * 260), y1)


def layer_ops(gpu, b, w, bufs, T, Hq, Hk, D, H, act_stride=None):
    """One attention block of a layer for the T tokens of the batch as an op list: q, k, v projections with an adapter beside q, k and v
    appended, attention, o projection. Returns the ops and the structs that they name."""
    proj = gpu.HeadProj(dtype=F32, n_tokens=T, n_heads=Hq, n_kv_heads=Hk, head_dim=D, rotary_dim=D, q=bufs["q"].ptr, k=bufs["k"].ptr, v=bufs["v"].ptr,
                        q_out=bufs["q"].ptr, q_norm=w["qn"].ptr, k_norm=w["kn"].ptr, eps=1e-6, theta=1e6)
    attn = gpu.Attn(dtype=F32, n_heads=Hq, q=bufs["q"].ptr, out=bufs["attn"].ptr, scale=D ** -0.5, causal=1)
    lora = gpu.Lora(dtype=F16, n_tokens=T, in_dim=H, out_dim=Hq * D, rank=8, n_adapters=2, n_seqs=len(b.new), x=bufs["x"].ptr, base=bufs["q"].ptr,
                    y=bufs["q"].ptr, a=w["a"].ptr, b=w["b"].ptr, scale=w["s"].ptr, q_start=b.d_start.ptr, adapter=w["of"].ptr)
    mm = lambda name, x, y, m, k: gpu.Op(gpu.OP_I4_MATMUL, w[name].ptr, bufs[x].ptr, bufs[y].ptr, m, k, T, 64, None, None, None, None, 0)  # noqa: E731
    ops = [mm("wq", "x", "q", Hq * D, H), mm("wk", "x", "k", Hk * D, H), mm("wv", "x", "v", Hk * D, H), gpu.batch_op(gpu.OP_LORA_ADD, lora),
           gpu.batch_op(gpu.OP_KV_APPEND, proj, b.c, b.s), gpu.batch_op(gpu.OP_PAGED_ATTENTION, attn, b.c, b.s), mm("wo", "attn", "y", H, Hq * D)]
    return ops, (proj, attn, lora)


def test_attention_block_of_prompts_and_decode_steps(gpu, orc):
    """The calls together, as a runtime makes them: prompts in one batch, then decode steps replayed from a captured op list whose
    device arrays (lengths, activations) change between replays. Each replay equals the eager list bit for bit, and each stage
    what the stage's plain form gives on the stage's own inputs."""
    Hq, Hk, D, H, steps = 4, 2, 64, 256, 3
    lens = [5, 33, 1]
    rng = np.random.default_rng(50)
    w = {n: gpu.synth_i4(m, k, 64, seed=60 + i) for i, (n, m, k) in enumerate((("wq", Hq * D, H), ("wk", Hk * D, H), ("wv", Hk * D, H), ("wo", H, Hq * D)))}
    host = dict(w)
    w = {n: gpu.DeviceBuffer.from_array(x) for n, x in w.items()}
    a_, b_ = Dev(gpu, rng.standard_normal((2, 8, H)) / 16, F16), Dev(gpu, 0.3 * rng.standard_normal((2, Hq * D, 8)), F16)
    qn, kn = (1 + 0.1 * rng.standard_normal((2, D))).astype(np.float32)
    sc, of = np.float32([1.5, 0.5]), [1, -1, 0]
    w.update(a=a_, b=b_, qn=f32_buffer(gpu, qn), kn=f32_buffer(gpu, kn), s=f32_buffer(gpu, sc), of=ints(gpu, of))

    def plain(b, bufs, x, T):
        """q, k, v after the projections and the adapter, then everything after them, from the i4 oracle and the plain forms."""
        m = lambda n, v, rows, cols: orc.matmul_i4(host[n], np.ascontiguousarray(v, np.float32).ravel(), rows, cols, T, 64).reshape(T, rows)  # noqa: E731
        q = ref.lora(x.astype(np.float64), m("wq", x, Hq * D, H).astype(np.float64), a_.values, b_.values, sc, b.starts, of, T)[0]
        k, v = m("wk", x, Hk * D, H), m("wv", x, Hk * D, H)
        at = b.token_positions()
        pos = np.array([at[t][1] for t in range(T)])
        q = ref.finish_heads(q.reshape(T, Hq, D), None, qn, pos, D, 1e-6, 1e6)[0]
        k = ref.finish_heads(k.astype(np.float64).reshape(T, Hk, D), None, kn, pos, D, 1e-6, 1e6)[0]
        for t in range(T):
            pl = b.place(*at[t])
            b.k.values[pl], b.v.values[pl] = k[t], v[t].reshape(Hk, D)
        o = ref.attention(b, q, D ** -0.5, 1, 0)[0]
        return m("wo", o.reshape(T, Hq * D), H, Hq * D)

    def buffers(T):
        return {n: gpu.DeviceBuffer(4 * T * m) for n, m in (("x", H), ("q", Hq * D), ("k", Hk * D), ("v", Hk * D), ("attn", Hq * D), ("y", H))}

    # prompts: the pages have room for the steps after them
    b = Batch(gpu, lens, [n + steps for n in lens], 16, Hk, D, F16, seed=51, fill=0.0)
    b.kv = list(lens)
    b.d_kv.upload(np.int32(b.kv))
    T = b.tokens
    bufs = buffers(T)
    x = rng.standard_normal((T, H)).astype(np.float32)
    bufs["x"].upload(x)
    stream = gpu.Stream()
    ops, keep = layer_ops(gpu, b, w, bufs, T, Hq, Hk, D, H)
    gpu.run_ops(ops, 1, stream)
    stream.synchronize()
    want = plain(b, bufs, x, T)
    got = bufs["y"].download(np.float32, T * H).reshape(T, H)
    # fp16 operands in the projections: 4e-4 of them in L2 (1e-3 at most), through two of them, and fp16 rows in the cache
    assert np.linalg.norm(got - want) <= 4e-3 * np.linalg.norm(want)

    # decode steps
    b.new, b.starts, b.tokens = [1, 1, 1], np.arange(4), 3
    b.d_start = ints(gpu, b.starts)
    b.s = gpu.Seqs(n_seqs=3, n_tokens=3, q_start=b.d_start.ptr, kv_len=b.d_kv.ptr, block_table=b.d_table.ptr, table_stride=b.stride, max_kv=0)
    bufs = buffers(3)
    ops, keep = layer_ops(gpu, b, w, bufs, 3, Hq, Hk, D, H)
    b.kv = [n + 1 for n in lens]
    b.d_kv.upload(np.int32(b.kv))
    bufs["x"].upload(np.zeros((3, H), np.float32))
    graph = gpu.OpsGraph(ops, stream)
    for step in range(steps):
        b.kv = [n + 1 + step for n in lens]
        b.d_kv.upload(np.int32(b.kv))
        x = rng.standard_normal((3, H)).astype(np.float32)
        bufs["x"].upload(x)
        gpu.run_ops(ops, 1, stream)
        stream.synchronize()
        eager = [bufs["y"].download(np.int32, 3 * H), b.k.read_bits(), b.v.read_bits()]
        for _ in range(2):
            bufs["x"].upload(x)
            graph.launch()
            stream.synchronize()
            again = [bufs["y"].download(np.int32, 3 * H), b.k.read_bits(), b.v.read_bits()]
            assert all(np.array_equal(p, q) for p, q in zip(eager, again)), f"step {step}"
        want = plain(b, bufs, x, 3)
        got = bufs["y"].download(np.float32, 3 * H).reshape(3, H)
        assert np.linalg.norm(got - want) <= 4e-3 * np.linalg.norm(want), f"step {step}"
    graph.close()


class Hip:
    """The runtime's capture calls, which the library does not wrap (a caller that captures for itself has them)."""

    def __init__(self):
        import ctypes
        self.c = ctypes
        self.lib = ctypes.CDLL("libamdhip64.so")

    def begin(self, stream):
        assert self.lib.hipStreamBeginCapture(self.c.c_void_p(stream.ptr), 2) == 0  # relaxed

    def end(self, stream):
        g = self.c.c_void_p()
        assert self.lib.hipStreamEndCapture(self.c.c_void_p(stream.ptr), self.c.byref(g)) == 0
        return g

    def replay(self, g, stream, times):
        e = self.c.c_void_p()
        assert self.lib.hipGraphInstantiate(self.c.byref(e), g, None, None, self.c.c_size_t(0)) == 0
        for _ in range(times):
            assert self.lib.hipGraphLaunch(e, self.c.c_void_p(stream.ptr)) == 0
            stream.synchronize()
        assert self.lib.hipGraphExecDestroy(e) == 0 and self.lib.hipGraphDestroy(g) == 0


def test_own_capture_needs_a_workspace(gpu):
    """Under the caller's own capture the calls that need scratch are refused without a workspace, and run with one."""
    hip, stream = Hip(), gpu.Stream()
    b = Batch(gpu, [1, 1], [3000, 1200], 16, 1, 64, F16, seed=70)
    q, out = Dev(gpu, b.rng.standard_normal((2, 4, 64)), F32), Dev(gpu, np.zeros((2, 4, 64)), F32)
    attn = gpu.Attn(dtype=F32, n_heads=4, q=q.ptr, out=out.ptr, scale=0.125, causal=1)
    x, y = f32_buffer(gpu, b.rng.standard_normal((2, 64))), f32_buffer(gpu, np.zeros((2, 32)))
    a_, b_ = Dev(gpu, b.rng.standard_normal((1, 4, 64)), F16), Dev(gpu, b.rng.standard_normal((1, 32, 4)), F16)
    sc, of = f32_buffer(gpu, [1.0]), ints(gpu, [0, 0])
    lora = gpu.Lora(dtype=F16, n_tokens=2, in_dim=64, out_dim=32, rank=4, n_adapters=1, n_seqs=2, x=x.ptr, y=y.ptr, a=a_.ptr, b=b_.ptr,
                    scale=sc.ptr, q_start=b.d_start.ptr, adapter=of.ptr)
    gpu.paged_attention_dev(attn, b.c, b.s, stream)
    gpu.lora_add_dev(lora, stream)
    stream.synchronize()
    want = out.read_bits(), y.download(np.int32, 64)
    out.buf.upload(np.zeros((2, 4, 64), np.float32))
    y.upload(np.zeros(64, np.float32))
    need = gpu.paged_attention_workspace(attn, b.c, b.s), gpu.lora_workspace(lora)
    assert need[0] > 0 and need[1] > 0
    spaces = [gpu.DeviceBuffer(n) for n in need]
    lib = gpu.lib()
    hip.begin(stream)
    refused = lib.tqhip_paged_attention_dev(attn, b.c, b.s, stream.ptr), lib.tqhip_lora_add_dev(lora, stream.ptr)
    for struct, space, n in ((attn, spaces[0], need[0]), (lora, spaces[1], need[1])):
        struct.workspace, struct.workspace_bytes = space.ptr, n
    ran = lib.tqhip_paged_attention_dev(attn, b.c, b.s, stream.ptr), lib.tqhip_lora_add_dev(lora, stream.ptr)
    g = hip.end(stream)
    assert refused == (gpu.ENOSCRATCH, gpu.ENOSCRATCH) and ran == (0, 0)
    hip.replay(g, stream, 3)
    assert np.array_equal(out.read_bits(), want[0]) and np.array_equal(y.download(np.int32, 64), want[1])
    attn.workspace_bytes -= 1
    lora.workspace_bytes -= 1
    assert lib.tqhip_paged_attention_dev(attn, b.c, b.s, stream.ptr) == gpu.ENOSCRATCH
    assert lib.tqhip_lora_add_dev(lora, stream.ptr) == gpu.ENOSCRATCH


@pytest.mark.parametrize("T", [1, 37])
def test_qk_norm_rope_in_an_op_list(gpu, T):
    """Finishing heads out of place as an op, eager and replayed from a graph with other positions: the direct call's bits."""
    rng = np.random.default_rng(80 + T)
    Hq, Hk, D = 5, 2, 64
    s = head_inputs(gpu, rng, T, Hq, Hk, D, F32, True, True)
    pos = ints(gpu, np.arange(T) + 11)
    outs = [[Dev(gpu, np.zeros((T, h, D)), F32) for h in (Hq, Hk)] for _ in range(2)]
    projs = [proj_of(gpu, s, T, Hq, Hk, D, F32, D, q, k, pos) for q, k in outs]
    stream = gpu.Stream()
    graph = gpu.OpsGraph([gpu.batch_op(gpu.OP_QK_NORM_ROPE, projs[1])], stream)
    for first in (11, 40000, 0):
        pos.upload(np.int32(np.arange(T) + first))
        gpu.qk_norm_rope_dev(projs[0], stream)
        graph.launch()
        stream.synchronize()
        for a, b in zip(*outs):
            assert np.array_equal(a.read_bits(), b.read_bits()), first
        want, size = ref.finish_heads(s["q"][2], s["q_bias"][0], s["q_norm"][0], np.arange(T) + first, D, 1e-6, 1e6)
        check_heads(outs[1][0].read(), want, size, F32, f"q from position {first}")
    graph.close()
