"""Attention over a paged cache of 8-bit codes (tqhip_paged_attention8_dev) against the formula in 64 bits.

Tolerances, with u = 2^-24, as in test_gpu_batch.py: a score is D products and sums and the product with its key's scale, (D + 5) u of its terms'
sizes, S, at most, and e^x doubles that; N weights and products summed, and the product of a weight with its value's scale: 2 N + 40 u. So
within (2 (D + 5) S + 2 N + 40) u of sum p |v|. fp32 activations are two fp16 terms, 2^-22 of an element, which that covers, or 2^-39 of the row's
largest. For weights that is: the largest of a row, times its value's scale, stands at 2^14 at least, and below 2^-14 a second term is off by 2^-25; so each
of N weights by 2^-39 of that largest product, which is at most the largest scale, and the result by as much of the largest code times it (that counts
where the values of the large weights are 0, as codes often are). Beside that fp32 results are held to a relative L2 distance of 2^-17.
f16 / bf16 activations: a weight is rounded to fp16 (2^-11 of sum p |v|), or off by 2^-25 where the largest stands at 2^8: 2^-33 in the place of
2^-39; and the result is rounded to its type."""
import numpy as np
import pytest

import batch_ref as ref
from batch8_ref import E4M3, I8, TOP, Batch8
from batch_ref import HALF, TINY, Dev, ints

pytestmark = pytest.mark.gpu

F32, F16, BF16 = 0, 1, 2
U = 2.0 ** -24


def attend(gpu, b, q, act, Hq, scale, causal=1, window=0, stream=None, pad=0, **kw):
    out = Dev(gpu, np.full(q.shape, 7.0), act)
    gpu.paged_attention8_dev(gpu.Attn(dtype=act, n_heads=Hq, q=q.ptr, out=out.ptr, scale=scale, causal=causal, window=window,
                                      q_stride=(Hq + pad) * b.D, out_stride=(Hq + pad) * b.D, **kw), b.c, b.s, stream)
    gpu.synchronize()
    return out.read()


def bound_of(b, act, want, spread, score):
    N = max(max(b.kv), 1)
    scales = b.scales[..., 1]
    top = TOP[b.dtype] * np.abs(scales[np.isfinite(scales)]).max()
    bound = (2 * (b.D + 5) * score + 2 * N + 40) * U * spread + N * (2.0 ** -39 if act == F32 else 2.0 ** -33) * top
    if act != F32:
        bound = bound + 2.0 ** -11 * spread + HALF[act] * np.abs(want) + TINY[act]
    return bound


def check(gpu, b, act, Hq, causal=1, window=0, scale=None, q_std=1.5, stream=None, pad=0, q=None):
    scale = b.D ** -0.5 if scale is None else scale
    q = Dev(gpu, q_std * b.rng.standard_normal((b.tokens, Hq + pad, b.D)) if q is None else q, act)
    got = attend(gpu, b, q, act, Hq, scale, causal, window, stream, pad)
    want, spread, score, live = ref.attention(b, q.values[:, :Hq], float(np.float32(scale)), causal, window)
    dead = np.setdiff1d(np.arange(b.tokens), live)
    assert np.all(got[dead] == 7.0) and np.all(got[:, Hq:] == 7.0), "rows outside the call changed"
    got = got[:, :Hq]
    bound = bound_of(b, act, want, spread, score)
    bad = ~(np.abs(got - want) <= bound)[live]
    assert not bad.any(), f"{bad.sum()} of {bad.size} off, worst {np.nanmax((np.abs(got - want) / np.maximum(bound, 1e-300))[live]):.2f} bounds"
    if act == F32:
        assert np.linalg.norm((got - want)[live]) <= 2.0 ** -17 * np.linalg.norm(want[live])
    return got


TYPES = [(a, c) for c in (I8, E4M3) for a in (F32, F16, BF16)]
SHAPES = [(14, 2, 64), (8, 2, 128), (2, 1, 256)]
# new tokens, cached positions, query heads, key/value heads: tiles of 16, 32 and (twice) 128 rows, in one part and in several
FORMS = [([3, 9], [9, 100], 2, 1), ([40, 1], [1400, 2100], 4, 2), ([90, 170], [90, 200], 8, 8), ([150, 130], [1700, 900], 8, 8)]


@pytest.mark.parametrize("act,dtype", TYPES)
@pytest.mark.parametrize("Hq,Hk,D", SHAPES)
def test_single_tokens(gpu, act, dtype, Hq, Hk, D):
    """Lengths of zero (more tokens than positions), one, about a tile, and long ones; tokens outside every sequence."""
    kv = [1, 0, 2, 31, 32, 33, 63, 64, 65, 700, 129, 1500]
    check(gpu, Batch8(gpu, [1] * len(kv), kv, 16, Hk, D, dtype, seed=D, tail=2, lead=1), act, Hq)


@pytest.mark.parametrize("act,dtype", TYPES)
@pytest.mark.parametrize("Hq,Hk,D", SHAPES)
def test_chunks(gpu, act, dtype, Hq, Hk, D):
    """Chunks of 0, 1, a few and many tokens over caches that end inside a page, positions before the cache's first."""
    check(gpu, Batch8(gpu, [70, 1, 0, 5, 129, 4], [70, 90, 12, 300, 400, 2], 48, Hk, D, dtype, 24, seed=D + 1, tail=3, layout="head"), act, Hq)


@pytest.mark.parametrize("act,dtype", TYPES)
@pytest.mark.parametrize("new,kv,Hq,Hk", FORMS)
def test_forms(gpu, act, dtype, new, kv, Hq, Hk):
    b = Batch8(gpu, new, kv, 32, Hk, 128, dtype, 8, seed=2, spread=3)
    rows, parts = gpu.paged_attention8_plan(gpu.Attn(dtype=act, n_heads=Hq, q=256, out=256, scale=1.0, causal=1), b.c, b.s)
    i = FORMS.index((new, kv, Hq, Hk))
    assert (rows, parts > 1) == ((16, 32, 128, 128)[i], bool(i % 2))
    check(gpu, b, act, Hq)


@pytest.mark.parametrize("act,dtype", TYPES)
@pytest.mark.parametrize("new,kv,Hq,Hk,D", [([9, 20], [100, 1500], 4, 2, 256), ([300, 170], [700, 200], 4, 2, 256), ([200, 230], [3000, 300], 4, 2, 256), ([300, 170], [700, 200], 6, 2, 64)])
def test_chunks_of_wide_and_narrow_heads(gpu, act, dtype, new, kv, Hq, Hk, D):
    check(gpu, Batch8(gpu, new, kv, 64, Hk, D, dtype, 32, seed=3, spread=2), act, Hq)


@pytest.mark.parametrize("new", [[1, 1, 1], [33, 1, 3], [150, 200, 90]])
@pytest.mark.parametrize("page,block", [(1, 1), (7, 7), (40, 5), (64, 1), (1000, 125), (96, 3)])
def test_page_and_block_sizes(gpu, page, block, new):
    kv = [max(n, m) for n, m in zip(new, [200, 333, 70])]
    check(gpu, Batch8(gpu, new, kv, page, 2, 64, I8, block, seed=page), F32, 6)


@pytest.mark.parametrize("new", [[1, 1, 1, 1], [90, 3, 1, 64], [300, 70, 1, 64]])
@pytest.mark.parametrize("causal,window", [(0, 0), (1, 1), (1, 37), (1, 5000), (1, 2 ** 31 - 1)])
@pytest.mark.parametrize("dtype", [I8, E4M3])
def test_masks(gpu, new, causal, window, dtype):
    check(gpu, Batch8(gpu, new, [600, 77, 1, 64], 16, 4, 128, dtype, seed=window % 100), F32, 16, causal, window)


@pytest.mark.parametrize("new", [[1, 1, 1], [50, 64, 3], [200, 64, 500]])
@pytest.mark.parametrize("dtype", [I8, E4M3])
def test_missing_pages(gpu, new, dtype):
    """Pages outside the cache hold no positions; a sequence of them alone gives zeros."""
    check(gpu, Batch8(gpu, new, [200, 64, 500], 32, 2, 64, dtype, 16, seed=4, bad=[(0, 0), (0, 3), (1, 0), (1, 1), (2, 5), (2, 15)]), F32, 4)


@pytest.mark.parametrize("Hq,Hk", [(1, 1), (5, 5), (20, 1), (33, 1), (64, 8)])
def test_head_groups(gpu, Hq, Hk):
    check(gpu, Batch8(gpu, [1, 9, 40], [130, 70, 41], 16, Hk, 64, E4M3, seed=Hq), BF16, Hq)


@pytest.mark.parametrize("new,kv,Hq,Hk", FORMS)
@pytest.mark.parametrize("dtype", [I8, E4M3])
def test_large_scores(gpu, new, kv, Hq, Hk, dtype):
    """Scores of hundreds, of either sign: one weight is near 1, the rest are tiny, and maxima move late."""
    check(gpu, Batch8(gpu, new, kv, 16, Hk, 64, dtype, seed=9), F32, Hq, scale=1.0, q_std=12.0)


@pytest.mark.parametrize("act,q_std", [(F32, 1e-20), (F32, 1e5), (F32, 1e20), (BF16, 1e-20), (BF16, 1e5), (BF16, 1e30), (F16, 1e4)])
@pytest.mark.parametrize("new", [[1, 70], [200, 300]])
def test_wide_range_queries(gpu, act, q_std, new):
    """Queries beyond fp16's range, brought back by the scale."""
    kv = [max(n, m) for n, m in zip(new, [100, 200])]
    check(gpu, Batch8(gpu, new, kv, 16, 2, 64, I8, seed=10), act, 4, scale=float(np.float32(0.2 / q_std)), q_std=q_std)


@pytest.mark.parametrize("new", [[1, 1], [40, 3], [300, 200]])
@pytest.mark.parametrize("scale", [0.0, -0.2, 1e-30])
@pytest.mark.parametrize("act", [F32, BF16])
def test_scale_of_zero_and_below(gpu, new, scale, act):
    check(gpu, Batch8(gpu, new, [max(150, new[0]), max(60, new[1])], 16, 2, 64, I8, seed=20), act, 4, scale=scale)


def test_strided_queries_and_a_stream(gpu):
    check(gpu, Batch8(gpu, [1, 30, 1], [50, 60, 900], 16, 2, 128, I8, seed=11), F32, 6, pad=3, stream=gpu.Stream())


@pytest.mark.parametrize("new,kv,Hq,Hk", FORMS)
@pytest.mark.parametrize("max_kv", [0, 1, 300, 2 ** 31 - 1])
def test_split_by_a_wrong_length(gpu, new, kv, Hq, Hk, max_kv):
    """max_kv decides how the work is split and nothing else, too small and too large ones too."""
    b = Batch8(gpu, new, kv, 16, Hk, 64, E4M3, seed=35)
    b.s.max_kv = max_kv
    check(gpu, b, F32, Hq, window=50)


@pytest.mark.parametrize("length", [2 ** 31 - 1, 2 ** 30, -2 ** 31, -1, 0])
@pytest.mark.parametrize("new", [[1, 1], [120, 30], [300, 120]])
@pytest.mark.parametrize("page", [1, 16])
def test_lengths_that_no_table_holds(gpu, length, new, page):
    """A sequence whose window lies past its table, or whose length is no length, gets zeros; the other one is as ever."""
    b = Batch8(gpu, new, [300, 140], page, 4, 64, I8, seed=36)
    q = Dev(gpu, b.rng.standard_normal((b.tokens, 4, 64)), F32)
    want = attend(gpu, b, q, F32, 4, 0.125, 1, 20)
    want[: new[0]] = 0
    b.d_kv.upload(np.int32([length, 140]))
    assert np.array_equal(attend(gpu, b, q, F32, 4, 0.125, 1, 20), want)


def wide_scales(b, powers, what):
    """Keys' (0) or values' (1) scales times powers of two, block by block at random."""
    f = 2.0 ** b.rng.choice(powers, b.scales.shape[:3])
    b.scales[..., what] = (b.scales[..., what] * f).astype(np.float32)
    b.put()


@pytest.mark.parametrize("new,kv,Hq,Hk", FORMS)
@pytest.mark.parametrize("act,dtype", TYPES)
@pytest.mark.parametrize("powers", [(0, -6), (0, -30), (-50, 0, 50), (-100, -40, 60)])
def test_values_of_very_different_blocks(gpu, new, kv, Hq, Hk, act, dtype, powers):
    """Values whose scales are powers apart: a weight is held as precisely as its product with its value's scale is large. A weight times scale that
    is 2^-39 of the row's largest (fp32; 2^-33 with 16 bits) is lost beside it: N of them."""
    b = Batch8(gpu, new, kv, 16, Hk, 64, dtype, 4, seed=41)
    wide_scales(b, powers, 1)
    q = Dev(gpu, 1.5 * b.rng.standard_normal((b.tokens, Hq, 64)), act)
    if act == F16 and max(powers) > 15:
        pytest.skip("results past fp16's range")
    got = attend(gpu, b, q, act, Hq, 0.125)
    want, spread, score, live = ref.attention(b, q.values, 0.125, 1, 0)
    top = np.abs(spread).max(-1, keepdims=True)  # (a row's largest product is in its spread)
    bound = (2 * 69 * score + 2 * max(kv) + 40) * U * spread + max(kv) * (2.0 ** -39 if act == F32 else 2.0 ** -33) * 448 * top
    if act != F32:
        bound = bound + 2.0 ** -11 * spread + HALF[act] * np.abs(want) + TINY[act]
    bad = ~(np.abs(got - want) <= bound)[live]
    assert not bad.any(), f"{bad.sum()} of {bad.size} off, worst {np.nanmax((np.abs(got - want) / np.maximum(bound, 1e-300))[live]):.2f} bounds"


@pytest.mark.parametrize("new,kv,Hq,Hk", FORMS)
@pytest.mark.parametrize("dtype", [I8, E4M3])
def test_small_weights_of_large_values(gpu, new, kv, Hq, Hk, dtype):
    """The first block outweighs the others by e^14 or so and its values' scale is 2^-20 of theirs: what it and they add is alike, and both count to
    the last bits."""
    b = Batch8(gpu, new, kv, 16, Hk, 64, dtype, 16, seed=43)
    for s in range(len(kv)):
        page = b.place(s, 0)[0]
        b.codes[0, page, :, :, 0] = 127 if dtype == I8 else 0x7e
        b.scales[page, :, 0, 1] *= 2.0 ** -20
    others = np.ones(b.n_pages, bool)
    others[[b.place(s, 0)[0] for s in range(len(kv))]] = False
    b.codes[0, others, :, :, 0] = 0
    b.put()
    q = 0.5 * b.rng.standard_normal((b.tokens, Hq, 64))
    q[..., 0] = 40.0
    check(gpu, b, F32, Hq, q=q)


@pytest.mark.parametrize("new,kv,Hq,Hk", FORMS)
@pytest.mark.parametrize("dtype", [I8, E4M3])
def test_keys_of_very_different_blocks(gpu, new, kv, Hq, Hk, dtype):
    b = Batch8(gpu, new, kv, 16, Hk, 64, dtype, 4, seed=42)
    wide_scales(b, (0, -20, 3), 0)
    check(gpu, b, F32, Hq)


@pytest.mark.parametrize("new,kv,Hq,Hk", FORMS)
@pytest.mark.parametrize("act,dtype", TYPES)
def test_scales_of_zero(gpu, new, kv, Hq, Hk, act, dtype):
    """Blocks that stand for zeros whatever their codes, of keys and of values: their weights count."""
    b = Batch8(gpu, new, kv, 16, Hk, 64, dtype, 8, seed=44)
    b.scales[b.rng.random(b.scales.shape) < 0.3] = 0.0
    for s in range(len(kv)):
        b.scales[b.place(s, 0)[0]] = 0.0
    b.put()
    check(gpu, b, act, Hq)


@pytest.mark.parametrize("new,kv,Hq,Hk", FORMS)
@pytest.mark.parametrize("what", ["scale of keys", "scale of values", "infinite scale of values", "code"])
@pytest.mark.parametrize("D", [64, 128])
def test_nan_and_infinity(gpu, new, kv, Hq, Hk, what, D):
    """In the block of the last-but-40th position on of each sequence: tokens before it must not notice; a NaN value makes its dimension NaN, a
    NaN key the row. An infinite scale makes its codes infinities of their sign (NaN where they are zero)."""
    b = Batch8(gpu, new, kv, 16, Hk, D, E4M3, 16, seed=45)
    at = [max(0, n - 20) for n in kv]
    for s, p in enumerate(at):
        page, row = b.place(s, p)
        if what == "scale of keys":
            b.scales[page, :, 0, 0] = np.nan
        elif what == "scale of values":
            b.scales[page, :, 0, 1] = np.nan
        elif what == "code":
            b.codes[1, page, row, :, 5] = 0x7f
        else:
            b.scales[page, :, 0, 1] = np.inf
            b.codes[1, page, :, :, 7] = 0x30
            b.codes[1, page, :, :, 8] = 0xb0
    b.put()
    q = Dev(gpu, 1.5 * b.rng.standard_normal((b.tokens, Hq, D)), F32)
    got = attend(gpu, b, q, F32, Hq, D ** -0.5)
    with np.errstate(invalid="ignore"):
        want, spread, score, _ = ref.attention(b, q.values, float(np.float32(D ** -0.5)), 1, 0)
    clean, hit = [], []
    for t, (s, pos) in b.token_positions().items():
        start = at[s] if what == "code" else at[s] // 16 * 16
        (clean if pos < start else hit).append(t)
    assert hit and (clean or min(new) < 40)
    bound = (2 * (D + 5) * score + 2 * max(kv) + 40) * U * spread
    assert np.all(np.abs(got - want)[clean] <= bound[clean])
    g = got[hit]
    if what in ("scale of keys", "scale of values"):
        assert np.isnan(g).all()
    elif what == "code":
        other = np.arange(D) != 5
        assert np.isnan(g[..., 5]).all()
        assert np.all(np.abs(g - want[hit])[..., other] <= bound[hit][..., other])
    else:
        assert np.all(g[..., 7] == np.inf) and np.all(g[..., 8] == -np.inf) and not np.isfinite(g).any()


@pytest.mark.parametrize("new,kv,Hq,Hk", FORMS)
@pytest.mark.parametrize("act,dtype", TYPES)
def test_queries_that_are_not_finite(gpu, new, kv, Hq, Hk, act, dtype):
    """A NaN or infinite query makes its own rows NaN where keys of either sign are seen, and no others."""
    b = Batch8(gpu, new, kv, 16, Hk, 64, dtype, seed=6)
    x = Dev(gpu, 1.5 * b.rng.standard_normal((b.tokens, Hq, 64)), act).values
    want, spread, score, _ = ref.attention(b, x, 0.125, 1, 0)
    last = b.tokens - 1
    odd = (last, 0), (last - 1, 1), (last - 2, 0)
    for (t, h), d, y in zip(odd, (7, 0, 63), (np.nan, np.inf, -np.inf)):
        x[t, h, d] = y
    got = attend(gpu, b, Dev(gpu, x, act), act, Hq, 0.125)
    for t, h in odd:
        assert np.isnan(got[t, h]).all(), (t, h)
        got[t, h] = want[t, h]
    assert np.all(np.abs(got - want) <= bound_of(b, act, want, spread, score))


@pytest.mark.parametrize("new,kv,Hq,Hk", FORMS)
@pytest.mark.parametrize("act,q_std,scale", [(F32, 1e6, 1.0), (F32, 1e9, 1.0), (F32, 3.0, 1e13), (F16, 1e4, 1e4), (BF16, 1e6, 1e4)])
def test_scores_of_millions_and_beyond(gpu, new, kv, Hq, Hk, act, q_std, scale):
    """Keys repeat every 32 positions with one scale, so a row is the mean of the values at its best key's repetitions, which lie in every tile and
    part, unless rounding can decide between the two best keys (scores are off by at most 2 (D + 5) u of their terms' sizes)."""
    D = 64
    b = Batch8(gpu, new, kv, 16, Hk, D, I8, seed=50)
    keys = b.rng.integers(-127, 128, (32, Hk, D)).astype(np.int8).view(np.uint8)
    for s, n in enumerate(kv):
        for p in range(n):
            b.codes[(0, *b.place(s, p))] = keys[p % 32]
    b.scales[..., 0] = 2.0 ** -6
    b.put()
    q = Dev(gpu, q_std * b.rng.standard_normal((b.tokens, Hq, D)), act)
    got = attend(gpu, b, q, act, Hq, scale)
    G, decided = Hq // Hk, 0
    scale = float(np.float32(scale))
    kv_of, vv_of = b.rows(b.k.values), b.rows(b.v.values)
    for t, (s, pos) in b.token_positions().items():
        if pos < 0:
            continue
        pg, r = np.array([b.place(s, p) for p in range(min(kv[s], pos + 1))]).T
        for h in range(Hq):
            kk, vv = kv_of[pg, r, h // G], vv_of[pg, r, h // G]
            z = kk @ q.values[t, h] * scale
            best = z >= z.max() - 1e-9 * abs(z.max())
            off = 2 * (D + 5) * U * (np.abs(kk) @ np.abs(q.values[t, h])).max() * abs(scale)
            if best.all() or z.max() - z[~best].max() > 2 * off + 100:
                decided += 1
                want, spread = vv[best].mean(0), np.abs(vv[best]).mean(0)
                bound = (2 * len(vv) + 40) * U * spread
                if act != F32:
                    bound = bound + 2.0 ** -11 * spread + HALF[act] * np.abs(want) + 2.0 ** -25
                assert np.all(np.abs(got[t, h] - want) <= bound), (t, h)
    assert decided > 0.5 * b.tokens * Hq


def test_a_captured_call_with_its_own_workspace(gpu):
    """Replays attend to the lengths, codes and scales that are there when they run, and nothing past the workspace is written."""
    b = Batch8(gpu, [1, 1], [2100, 1400], 16, 2, 64, I8, seed=60)
    q, out = Dev(gpu, b.rng.standard_normal((2, 4, 64)), F32), Dev(gpu, np.zeros((2, 4, 64)), F32)
    a = gpu.Attn(dtype=F32, n_heads=4, q=q.ptr, out=out.ptr, scale=0.125, causal=1)
    need = gpu.paged_attention8_workspace(a, b.c, b.s)
    assert need > 0
    space = gpu.DeviceBuffer.from_array(np.full(need + 256, 0xA5, np.uint8))
    a.workspace, a.workspace_bytes = space.ptr, need
    stream = gpu.Stream()
    graph = gpu.OpsGraph([gpu.batch_op(gpu.OP_PAGED_ATTENTION8, a, b.c, b.s)], stream)
    for kv, factor in (([2100, 1400], 1.0), ([5, 1399], 2.0), ([0, 700], 0.5), ([2100, 1], 1.0)):
        b.kv = kv
        b.d_kv.upload(np.int32(kv))
        b.scales *= np.float32(factor)
        b.d_scales.upload(b.scales)
        b.stand_for()
        graph.launch()
        stream.synchronize()
        want, spread, score, _ = ref.attention(b, q.values, 0.125, 1, 0)
        assert np.all(np.abs(out.read() - want) <= bound_of(b, F32, want, spread, score)), kv
    graph.close()
    assert np.all(space.download(np.uint8, need + 256)[need:] == 0xA5)
