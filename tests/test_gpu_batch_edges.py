"""The batch calls on the GPU at the ends of their ranges. Tolerances as in test_gpu_batch.py."""
import numpy as np
import pytest

import batch_ref as ref
import test_gpu_batch as base
from batch_ref import HALF, Batch, Dev, ints

pytestmark = pytest.mark.gpu

F32, F16, BF16 = 0, 1, 2
U = 2.0 ** -24

# Sequences (new tokens, cached positions), query heads, key/value heads: 16 rows a tile and 128, in one part and in several.
FEW_ONE = ([3, 9], [9, 100], 2, 1)
FEW_PARTS = ([40, 1], [1400, 2100], 4, 2)
TILES_ONE = ([90, 170], [90, 200], 8, 8)
TILES_PARTS = ([150, 130], [1700, 900], 8, 8)
FORMS = [FEW_ONE, FEW_PARTS, TILES_ONE, TILES_PARTS]


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 30, 5])
@pytest.mark.parametrize("new,kv,Hq,Hk", [([40], [4], 2, 1), ([40, 1], [4, 3000], 2, 1), ([200], [8], 8, 8), ([200, 1], [8, 3000], 8, 8)])
def test_wide_windows_and_positions_before_the_first(gpu, new, kv, Hq, Hk, window):
    """More new tokens than positions: the first ones are before position 0 and get zeros, the rest see what is there."""
    b = Batch(gpu, new, kv, 16, Hk, 64, F16, seed=window % 7)
    base.check_attention(gpu, b, F32, Hq, 1, window)


@pytest.mark.parametrize("new,kv,Hq,Hk", FORMS)
@pytest.mark.parametrize("scale,q_std", [(0.0, 1e-20), (1e-30, 1e-15), (0.0, 1e20)])
def test_scale_of_zero_and_tiny_queries(gpu, new, kv, Hq, Hk, scale, q_std):
    """Every weight is the same, whatever the size of the queries: rows are the mean of the values that they see."""
    b = Batch(gpu, new, kv, 16, Hk, 64, F16, seed=3)
    base.check_attention(gpu, b, F32, Hq, 1, 0, scale=scale, q_std=q_std)


def seen(b, t_pos, g):
    """Keys and values of head g at the positions that a causal row at position t_pos of sequence b sees."""
    batch, seq, pos = b, *t_pos
    places = [batch.place(seq, p) for p in range(0, min(batch.kv[seq], pos + 1))]
    pg, r = np.array([p for p in places if p]).T
    return batch.rows(batch.k.values)[pg, r, g], batch.rows(batch.v.values)[pg, r, g]


def attend(gpu, b, act, Hq, scale, q):
    out = Dev(gpu, np.full(q.shape, 7.0), act)
    gpu.paged_attention_dev(gpu.Attn(dtype=act, n_heads=Hq, q=q.ptr, out=out.ptr, scale=scale, causal=1), b.c, b.s)
    gpu.synchronize()
    return out.read()


@pytest.mark.parametrize("new,kv,Hq,Hk", FORMS)
@pytest.mark.parametrize("act,cache", base.TYPES)
@pytest.mark.parametrize("D", [64, 128])
def test_infinities_that_are_attended_to(gpu, new, kv, Hq, Hk, act, cache, D):
    """As the formula has it, wherever tiles and parts end. A key of minus infinity in a dimension: weight 0 where the query is
    positive there (the value does not count, infinite or not), no number where it is negative. An infinite value: an
    infinity of its sign in its dimension, no number beside one of the other sign, and the other dimensions as ever."""
    b = Batch(gpu, new, kv, 16, Hk, D, cache, seed=5)
    k, v = b.k.values, b.v.values
    for s, n in enumerate(b.kv):
        for p, key, values in ((0, True, {1: np.inf}), (n // 2, False, {2: np.inf, 3: -np.inf}), (n // 3, False, {3: np.inf}), (n - 3, True, {}), (n - 2, False, {4: -np.inf})):
            pg, r = b.place(s, p)
            if key:
                k[pg, r, :, 0] = -np.inf
            for d, x in values.items():
                v[pg, r, :, d] = x
    b.k.buf.upload(ref.raw(k, cache)[0])
    b.v.buf.upload(ref.raw(v, cache)[0])
    q = Dev(gpu, 1.5 * b.rng.standard_normal((b.tokens, Hq, D)), act)
    got = attend(gpu, b, act, Hq, D ** -0.5, q)
    G, kinds = Hq // Hk, set()
    err = size = 0.0
    for t, at in b.token_positions().items():
        for h in range(Hq):
            kk, vv = seen(b, at, h // G)
            with np.errstate(invalid="ignore"):
                s = kk @ q.values[t, h] * float(np.float32(D ** -0.5))
            if not np.all(s < np.inf):
                assert np.isnan(got[t, h]).all(), (t, h, at)
                kinds.add("nan")
                continue
            live = s > -np.inf
            if not live.any():
                assert np.all(got[t, h] == 0), (t, h, at)
                continue
            s, vv = s[live], vv[live]
            p = np.exp(s - s.max())
            p /= p.sum()
            with np.errstate(invalid="ignore"):
                want = p @ vv
            finite = np.isfinite(want)
            assert np.array_equal(np.isnan(got[t, h]), np.isnan(want)) and np.array_equal(got[t, h][np.isinf(want)], want[np.isinf(want)]), (t, h, at, got[t, h, :6], want[:6])
            kinds.update("+" if x > 0 else "-" for x in want[np.isinf(want)])
            spread = p @ np.abs(np.where(np.isfinite(vv), vv, 0))
            fin = np.where(np.isfinite(kk[live]), kk[live], 0)
            score = (np.abs(fin) @ np.abs(q.values[t, h])).max() * D ** -0.5
            bound = (2 * (D + 4) * score + 2 * len(s) + 32) * U * spread
            if act != F32:
                bound = bound + HALF[act] * (spread + np.abs(np.where(finite, want, 0))) + 2.0 ** -25
            assert np.all(np.abs(got[t, h] - want)[finite] <= bound[finite]), (t, h, at)
            err, size = err + np.sum((got[t, h] - want)[finite] ** 2), size + np.sum(want[finite] ** 2)
    assert kinds == {"nan", "+", "-"}
    if act == F32:
        assert np.sqrt(err) <= 2.0 ** -17 * np.sqrt(size)


@pytest.mark.parametrize("new,kv,Hq,Hk", FORMS)
@pytest.mark.parametrize("act,cache", base.TYPES)
def test_queries_that_are_not_finite(gpu, new, kv, Hq, Hk, act, cache):
    """A NaN or infinite query makes its own rows NaN where keys of either sign are seen, and no others: those stay within the bound that
    every row has. (Not the same bits: rows of one wave bring their sums down to a new maximum together, so when one does,
    all have another rounding of a factor and its products, which the N + 16 u of the sums count.)"""
    D = 64
    b = Batch(gpu, new, kv, 16, Hk, D, cache, seed=6)
    x = Dev(gpu, 1.5 * b.rng.standard_normal((b.tokens, Hq, D)), act).values
    want, spread, score, _ = ref.attention(b, x, 0.125, 1, 0)
    bound = (2 * (D + 4) * score + 2 * max(kv) + 32) * U * spread
    if act != F32:
        bound = bound + HALF[act] * (spread + np.abs(want)) + 2.0 ** -25
    last = b.tokens - 1
    odd = (last, 0), (last - 1, 1), (last - 2, 0)
    for (t, h), d, y in zip(odd, (7, 0, 63), (np.nan, np.inf, -np.inf)):
        x[t, h, d] = y
    got = attend(gpu, b, act, Hq, 0.125, Dev(gpu, x, act))
    for t, h in odd:
        assert np.isnan(got[t, h]).all(), (t, h)
        got[t, h] = want[t, h]
    assert np.all(np.abs(got - want) <= bound)


@pytest.mark.parametrize("new,kv,Hq,Hk", FORMS)
@pytest.mark.parametrize("act,cache,q_std,scale", [(F32, F16, 1e6, 1.0), (F32, F16, 1e9, 1.0), (F32, F16, 3.0, 1e13), (F32, BF16, 1e9, -1.0), (F32, F32, 1e15, 1.0),
                                                   (F16, F16, 1e4, 1e2), (F16, F16, 1e4, 1e4), (BF16, BF16, 1e6, 1e4)])
def test_scores_of_millions_and_beyond(gpu, new, kv, Hq, Hk, act, cache, q_std, scale):
    """Scores whose exponents do not fit between two neighbouring fp32 numbers of their size. Keys repeat every 32 positions, so a row
    is the mean of the values at its best key's repetitions, which lie in every tile and part, unless rounding can
    decide between the two best keys (a row's scores are off by at most 2 (D + 4) u of their terms' sizes); such a row lies within its values."""
    D = 64
    b = Batch(gpu, new, kv, 16, Hk, D, cache, seed=int(q_std) % 97)
    keys = ref.raw(b.rng.standard_normal((32, Hk, D)), cache)[1]
    full = b.k.values
    for s, n in enumerate(b.kv):
        for p in range(n):
            pg, r = b.place(s, p)
            full[pg, r] = keys[p % 32]
    b.k.buf.upload(ref.raw(full, cache)[0])
    q = Dev(gpu, q_std * b.rng.standard_normal((b.tokens, Hq, D)), act)
    got = attend(gpu, b, act, Hq, scale, q)
    G, decided = Hq // Hk, 0
    scale = float(np.float32(scale))
    for t, at in b.token_positions().items():
        for h in range(Hq):
            kk, vv = seen(b, at, h // G)
            s = kk @ q.values[t, h] * scale
            top = s.max()
            best = s >= top - 1e-9 * abs(top)
            off = 2 * (D + 4) * U * (np.abs(kk) @ np.abs(q.values[t, h])).max() * abs(scale)
            if best.all() or top - s[~best].max() > 2 * off + 100:
                decided += 1
                want, spread = vv[best].mean(0), np.abs(vv[best]).mean(0)
                bound = (2 * len(vv) + 32) * U * spread
                if act != F32:
                    bound = bound + HALF[act] * (spread + np.abs(want)) + 2.0 ** -25
                assert np.all(np.abs(got[t, h] - want) <= bound), (t, h, at)
            else:
                slack = 1e-5 + (0 if act == F32 else 4 * HALF[act]) * np.abs(vv).max()
                assert np.all((got[t, h] >= vv.min(0) - slack) & (got[t, h] <= vv.max(0) + slack)), (t, h, at)
    assert decided > 0.5 * b.tokens * Hq


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("new,K,M,r", [([1] * 5, 96, 70, 1), ([1] * 5, 100, 33, 8), ([40, 30], 256, 300, 16), ([40, 30], 67, 35, 5), ([40], 2000, 130, 200)])
def test_lora_of_infinities(gpu, dtype, new, K, M, r):
    """Infinite activations and adapter weights go through as the formula has them: infinities of the sum's sign, no number where both
    signs meet; every other token and output is as ever."""
    rng = np.random.default_rng(K + r)
    starts = np.concatenate(([0], np.cumsum(new)))
    T = int(starts[-1])
    x, y0 = rng.standard_normal((T, K)).astype(np.float32), rng.standard_normal((T, M)).astype(np.float32)
    a, b = rng.standard_normal((2, r, K)) / np.sqrt(K), 0.3 * rng.standard_normal((2, M, r))
    b[:, : M // 2] = np.abs(b[:, : M // 2]) * np.sign(a[:, None, :, K - 1])  # (half of the outputs: terms of one sign)
    a, b = Dev(gpu, a, dtype), Dev(gpu, b, dtype)
    x[1, K - 1], x[3, K - 1] = np.inf, -np.inf
    y0[2, 3] = np.inf
    b.values[1, M - 1, 0] = -np.inf
    b.buf.upload(ref.raw(b.values, dtype)[0])
    of = [i % 2 for i in range(len(new))]
    scale = np.float32([1.5, 0.5])
    dx, dy0, ds, dst, dad = base.f32_buffer(gpu, x), base.f32_buffer(gpu, y0), base.f32_buffer(gpu, scale), ints(gpu, starts), ints(gpu, of)
    dy = base.f32_buffer(gpu, np.full((T, M), 7.0))
    gpu.lora_add_dev(gpu.Lora(dtype=dtype, n_tokens=T, in_dim=K, out_dim=M, rank=r, n_adapters=2, n_seqs=len(new), x=dx.ptr, base=dy0.ptr, y=dy.ptr,
                              a=a.ptr, b=b.ptr, scale=ds.ptr, q_start=dst.ptr, adapter=dad.ptr))
    gpu.synchronize()
    got = dy.download(np.float32, T * M).reshape(T, M).astype(np.float64)
    with np.errstate(invalid="ignore"):
        want, size = ref.lora(x.astype(np.float64), y0.astype(np.float64), a.values, b.values, scale.astype(np.float64), starts, of, T)
    finite = np.isfinite(want)
    assert np.isinf(want[1, : M // 2]).all() and (r == 1 or np.isnan(want).any()) and np.isinf(want[2, 3])
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(got[np.isinf(want)], want[np.isinf(want)])
    assert np.all(np.abs(got - want)[finite] <= (K + r + 8) * U * size[finite])
    # in place: the same bits
    bits = dy.download(np.int32, T * M)
    gpu.lora_add_dev(gpu.Lora(dtype=dtype, n_tokens=T, in_dim=K, out_dim=M, rank=r, n_adapters=2, n_seqs=len(new), x=dx.ptr, base=dy0.ptr, y=dy0.ptr,
                              a=a.ptr, b=b.ptr, scale=ds.ptr, q_start=dst.ptr, adapter=dad.ptr))
    gpu.synchronize()
    same = (dy0.download(np.int32, T * M) == bits) | np.isnan(got.ravel())
    assert same.all()


@pytest.mark.parametrize("new,kv,Hq,Hk", FORMS)
@pytest.mark.parametrize("cache", [F16, BF16, F32])
@pytest.mark.parametrize("large", [1e3, 1e5, 1e7])
def test_queries_with_one_large_dimension(gpu, new, kv, Hq, Hk, cache, large):
    """A dimension in which queries are large and keys small: its terms are no larger than the others', so the others' bits count. The
    bound is that of every row, (2 (D + 4) S + 2 N + 32) u of sum p |v|, S the size of the scores' terms. Over an fp16 cache a query element
    is two fp16 terms of a row scaled to below 2^15: the second one is off by 2^-25 at most where it is subnormal, 2^-39 of the row's
    largest element (which is 2^14 at least), so a score by 2^-39 max|q| sum |k| scale more, e, and a result by 2 e of sum p |v|."""
    D = 64
    b = Batch(gpu, new, kv, 16, Hk, D, cache, seed=8)
    k = b.k.values
    k[..., 5] /= large
    bits, b.k.values = ref.raw(k, cache)
    b.k.buf.upload(bits)
    x = 1.5 * b.rng.standard_normal((b.tokens, Hq, D))
    x[..., 5] *= large
    q = Dev(gpu, x, F32)
    got = attend(gpu, b, F32, Hq, 0.125, q)
    want, spread, score, _ = ref.attention(b, q.values, 0.125, 1, 0)
    e = 2.0 ** -39 * np.abs(q.values).max(-1, keepdims=True) * np.nansum(np.abs(b.k.values), -1).max() * 0.125 * (cache == F16)
    assert np.all(np.abs(got - want) <= (2 * (D + 4) * score + 2 * max(kv) + 32) * U * spread + 2 * e * spread)
    assert np.linalg.norm(got - want) <= 2.0 ** -17 * np.linalg.norm(want) + np.linalg.norm(2 * e * spread)


@pytest.mark.parametrize("new,kv,Hq,Hk", FORMS)
@pytest.mark.parametrize("cache", [F16, BF16, F32])
@pytest.mark.parametrize("gap", [12.0, 14.0, 20.0])
def test_a_first_key_with_nearly_all_the_weight(gpu, new, kv, Hq, Hk, cache, gap):
    """The first key outweighs each of the others by e^12 to e^20 or so and its value is zero: the result is made of the small weights.
    Beside the bound of every row: over an fp16 cache a weight is two fp16 terms, the largest weight at 2^14 or above, so a small one is off by 2^-25,
    2^-39 of the largest, and a result by e = 2^-39 sum |v|."""
    D = 64
    b = Batch(gpu, new, kv, 16, Hk, D, cache, seed=9)
    k, v = b.k.values, b.v.values
    k[..., 0] = np.where(np.isnan(k[..., 0]), np.nan, 0.0)
    for s in range(len(kv)):
        place = b.place(s, 0)
        k[place] = 0.0
        k[place][:, 0], v[place] = 1.0, 0.0
    for dev, x in ((b.k, k), (b.v, v)):
        bits, dev.values = ref.raw(x, cache)
        dev.buf.upload(bits)
    x = 0.5 * b.rng.standard_normal((b.tokens, Hq, D))
    x[..., 0] = 8 * gap
    q = Dev(gpu, x, F32)
    got = attend(gpu, b, F32, Hq, 0.125, q)
    want, spread, score, _ = ref.attention(b, q.values, 0.125, 1, 0)
    assert 0 < np.linalg.norm(spread[-1]) < 1e-3 * max(kv)
    e = 2.0 ** -39 * np.nansum(np.abs(v)) * (cache == F16)
    assert np.all(np.abs(got - want) <= (2 * (D + 4) * score + 2 * max(kv) + 32) * U * spread + e)
    # errors of the weights are random, so their sum is that of their squares: sqrt(N) of a half step at most, in each dimension
    typical = 2.0 ** -39 * np.sqrt(max(kv)) * 2 * np.sqrt(want.size) * (cache == F16)
    assert np.linalg.norm(got - want) <= 2.0 ** -17 * np.linalg.norm(want) + typical
