"""Attention over 8-bit codes where keys' scales or scores leave the range of the tiles' numbers, against the formula in 64 bits. Tolerances as in
test_gpu_attention8.py."""
import numpy as np
import pytest

import batch_ref as ref
import test_gpu_attention8 as attention
from batch8_ref import E4M3, I8, Batch8
from batch_ref import HALF, TINY, Dev
from test_gpu_attention8 import BF16, F16, F32, FORMS, TYPES, U, attend, bound_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("new,kv,Hq,Hk", FORMS)
@pytest.mark.parametrize("act,dtype", TYPES)
@pytest.mark.parametrize("what", ["either sign", "either sign, less above", "below", "above", "zero"])
def test_an_infinite_scale_of_keys(gpu, new, kv, Hq, Hk, act, dtype, what):
    """Its codes are infinities of their sign (no number where they are 0): a product with a query of one sign is an infinity (below: a weight of 0,
    above: a row of NaN), with either sign it is no number, whatever the sign of the codes' own product. In the block of the last-but-40th position on."""
    b = Batch8(gpu, new, kv, 16, Hk, 64, dtype, 16, seed=71)
    at = [max(0, n - 20) // 16 * 16 for n in kv]
    plus, minus = (0x05, 0xfb) if dtype == I8 else (0x30, 0xb0)
    for s, p in enumerate(at):
        page = b.place(s, p)[0]
        b.scales[page, :, 0, 0] = np.inf
        b.codes[0, page] = plus if what in ("above", "either sign") else minus
        if what.startswith("either sign"):
            b.codes[0, page, :, :, 1::4] = minus if what == "either sign" else plus
        if what == "zero":
            b.codes[0, page, :, :, 9] = 0
    b.put()
    q = Dev(gpu, np.abs(1.5 * b.rng.standard_normal((b.tokens, Hq, 64))) + 0.1, act)
    got = attend(gpu, b, q, act, Hq, 0.125)
    with np.errstate(invalid="ignore"):
        want = ref.attention(b, q.values, 0.125, 1, 0)[0]
    finite = b.k.values
    finite[~np.isfinite(finite)] = 0.0  # (for the sizes of the other keys' products)
    _, spread, score, _ = ref.attention(b, q.values, 0.125, 1, 0)
    hit = [t for t, (s, pos) in b.token_positions().items() if pos >= at[s]]
    clean = np.setdiff1d(np.arange(b.tokens), hit)
    if what != "below":
        assert np.isnan(want[hit]).all() and np.isnan(got[hit]).all()
    else:
        # (a sequence that begins with the block has nothing else, and its rows are zeros)
        only = [t for t in hit if at[b.token_positions()[t][0]] == 0]
        want[only] = 0.0
        clean = np.arange(b.tokens)
        spread = np.maximum(spread, np.abs(want))
    v = np.nanmax(np.abs(b.v.values))  # (rows that no position uses may be no numbers)
    bound = bound_of(b, act, want, np.maximum(spread, v), score)  # (the reference's spread counts the block's values where the formula has none of them)
    assert not np.isnan(want[clean]).any() and np.all(np.abs(got - want)[clean] <= bound[clean])


@pytest.mark.parametrize("new,kv,Hq,Hk", FORMS)
@pytest.mark.parametrize("dtype", [I8, E4M3])
@pytest.mark.parametrize("act", [F32, BF16])
@pytest.mark.parametrize("power", [50, 70, 110])
def test_large_scales_of_keys_with_small_queries(gpu, new, kv, Hq, Hk, dtype, act, power):
    """Ordinary scores of queries and keys 2^100 from 1, either way."""
    b = Batch8(gpu, new, kv, 16, Hk, 64, dtype, 8, seed=72)
    b.scales[..., 0] *= np.float32(2.0 ** power)
    b.put()
    attention.check(gpu, b, act, Hq, scale=0.125, q_std=1.5 * 2.0 ** -power)


@pytest.mark.parametrize("new,kv,Hq,Hk", FORMS)
@pytest.mark.parametrize("act", [F32, BF16])
def test_scores_below_zero_of_large_queries(gpu, new, kv, Hq, Hk, act):
    """Queries times the scale pass fp32, and keys bring the scores back to some -10^28, all of them below zero: the largest takes it all (unless fp32, in which
    the parts of a row compare theirs, may not tell it from the next)."""
    b = Batch8(gpu, new, kv, 16, Hk, 64, I8, 16, seed=73)
    b.codes[0] = np.maximum(b.codes[0] & 0x7f, 0x10)  # positive, of 16 at least
    b.scales[..., 0] = 2.0 ** -60
    b.put()
    q = Dev(gpu, -1e36 * (0.5 + np.abs(b.rng.standard_normal((b.tokens, Hq, 64)))), act)
    scale = float(np.float32(1e7))
    got = attend(gpu, b, q, act, Hq, scale)
    want, spread, _, _ = ref.attention(b, q.values, scale, 1, 0)
    bound = 2 * U * spread + HALF[act] * np.abs(want) + TINY[act]  # (one value, times its scale, rounded)
    keys, decided = b.k.values, 0
    for t, (s, pos) in b.token_positions().items():
        if pos < 0:
            continue
        pg, r = np.array([b.place(s, p) for p in range(pos + 1)]).T
        for h in range(Hq):
            z = np.sort(keys[pg, r, h // (Hq // Hk)] @ q.values[t, h])
            if pos == 0 or z[-1] - z[-2] > 2.0 ** -22 * abs(z[-1]):
                decided += 1
                assert np.all(np.abs(got[t, h] - want[t, h]) <= bound[t, h]), (t, h)
    assert decided > 0.9 * b.tokens * Hq


@pytest.mark.parametrize("new,kv,Hq,Hk", FORMS)
@pytest.mark.parametrize("dtype", [I8, E4M3])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_f16_rows_are_off_by_their_results_rounding(gpu, new, kv, Hq, Hk, dtype, D):
    """Within fp32's tolerance of the formula before the result is rounded to f16, half a step: no rounding of the weights shows."""
    b = Batch8(gpu, new, kv, 16, Hk, D, dtype, 8, seed=74)
    q = Dev(gpu, 1.5 * b.rng.standard_normal((b.tokens, Hq, D)), F16)
    got = attend(gpu, b, q, F16, Hq, D ** -0.5)
    want, spread, score, _ = ref.attention(b, q.values, float(np.float32(D ** -0.5)), 1, 0)
    before = bound_of(b, F32, want, spread, score)
    assert np.all(np.abs(got - want) <= before + HALF[F16] * (np.abs(want) + before) + TINY[F16])
    rounded = want.astype(np.float16).astype(np.float64)
    assert np.linalg.norm(got - want) <= np.linalg.norm(rounded - want) + 2.0 ** -17 * np.linalg.norm(want)
