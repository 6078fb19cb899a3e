"""The attention kernel of 128-row tiles against the plain 64-bit form, with its keys in one part and in several: head sizes, types, masks,
pages that are missing, lengths past the table, groups of heads. Every test states which kernel it reaches and in how
many parts (tqhip_paged_attention_plan), so that a change of the rule between the kernels cannot move it to the other one
unseen. Tolerances as in test_gpu_batch.py."""
import numpy as np
import pytest

import test_gpu_batch as base
import test_gpu_batch_edges as edges
from batch_ref import Batch, Dev

pytestmark = pytest.mark.gpu

F32, F16, BF16 = 0, 1, 2
AT = 1 << 20  # (the plan reads no pointer)
TILE = 128


def plan(gpu, b, act, Hq, causal=1, window=0):
    return gpu.paged_attention_plan(gpu.Attn(dtype=act, n_heads=Hq, q=AT, out=AT, scale=0.1, causal=causal, window=window), b.c, b.s)


def check(gpu, b, act, Hq, several, causal=1, window=0, **kw):
    rows, parts = plan(gpu, b, act, Hq, causal, window)
    assert rows == TILE and (parts > 1) == several, (rows, parts)
    base.check_attention(gpu, b, act, Hq, causal, window, **kw)


def test_the_forms_of_the_edge_tests(gpu):
    for (new, kv, Hq, Hk), rows, several in zip(edges.FORMS, (16, 16, TILE, TILE), (False, True, False, True)):
        for D in (64, 128, 256):
            got = plan(gpu, Batch(gpu, new, kv, 16, Hk, D, F16), F32, Hq)
            assert got[0] == rows and (got[1] > 1) == several, (new, kv, D, got)


@pytest.mark.parametrize("several", [False, True])
@pytest.mark.parametrize("act,cache", base.TYPES)
@pytest.mark.parametrize("D", [64, 128, 256])
def test_chunks(gpu, act, cache, D, several):
    """Chunks of 0, 1, a few and many tokens over caches that end inside a page, positions before the cache's first, tokens outside."""
    kv = [1500, 90, 12, 300, 700, 2] if several else [130, 90, 12, 300, 400, 2]
    b = Batch(gpu, [130, 1, 0, 5, 129, 4], kv, 48, 8, D, cache, seed=D + 1, tail=3, lead=2, layout="head")
    check(gpu, b, act, 8, several)


@pytest.mark.parametrize("several", [False, True])
@pytest.mark.parametrize("cache,D", [(F16, 64), (BF16, 128), (F32, 64), (F16, 256)])
@pytest.mark.parametrize("causal,window", [(0, 0), (1, 1), (1, 37), (1, 200), (1, 5000)])
def test_masks(gpu, causal, window, cache, D, several):
    b = Batch(gpu, [90, 3, 1, 164], [1300, 77, 1, 640] if several else [400, 77, 1, 164], 16, 8, D, cache, seed=window)
    check(gpu, b, F32, 8, several, causal, window)


@pytest.mark.parametrize("several", [False, True])
@pytest.mark.parametrize("cache,D", [(F16, 64), (BF16, 128), (F32, 128), (BF16, 256)])
@pytest.mark.parametrize("causal", [0, 1])
def test_missing_pages(gpu, cache, D, causal, several):
    """Pages outside the cache hold no positions; a sequence of them alone gives zeros."""
    b = Batch(gpu, [150, 64, 33], [1200 if several else 200, 64, 500], 32, 8, D, cache, seed=4,
              bad=[(0, 0), (0, 3), (0, 5), (1, 0), (1, 1), (2, 5), (2, 15)] + ([(0, i) for i in range(16, 33)] if several else []))
    check(gpu, b, F32, 8, several, causal)


@pytest.mark.parametrize("several", [False, True])
@pytest.mark.parametrize("act,cache", [(F32, F16), (F32, F32), (BF16, BF16)])
def test_infinities_at_heads_of_256(gpu, act, cache, several):
    new, kv, Hq, Hk = edges.TILES_PARTS if several else edges.TILES_ONE
    edges.test_infinities_that_are_attended_to(gpu, new, kv, Hq, Hk, act, cache, 256)


@pytest.mark.parametrize("window", [0, 50, 2 ** 31 - 1])
@pytest.mark.parametrize("max_kv,several", [(1, False), (600, True), (2 ** 31 - 1, True)])
def test_split_by_a_wrong_length(gpu, window, max_kv, several):
    """max_kv decides how the work is split and nothing else, too small and too large ones too."""
    b = Batch(gpu, [300, 64], [900, 2600], 16, 8, 64, F16, seed=35)
    b.s.max_kv = max_kv
    check(gpu, b, F32, 8, several, 1, window)


@pytest.mark.parametrize("length", [2 ** 31 - 1, 2 ** 30, -2 ** 31, -1, 0])
@pytest.mark.parametrize("several", [False, True])
@pytest.mark.parametrize("window", [20, 2 ** 31 - 1])
def test_lengths_that_no_table_holds(gpu, length, several, window):
    """A sequence whose window lies past its table, or whose length is no length, gets zeros (with a window of everything, the table's
    rows where its length is past them); the other one is as ever."""
    b = Batch(gpu, [120, 130], [1504 if several else 160, 140], 16, 8, 64, F16, seed=36)  # (whole pages)
    assert plan(gpu, b, F32, 8, 1, window) == (TILE, 3 if several else 1)
    q, out = Dev(gpu, b.rng.standard_normal((b.tokens, 8, 64)), F32), Dev(gpu, np.full((b.tokens, 8, 64), 7.0), F32)
    attn = gpu.Attn(dtype=F32, n_heads=8, q=q.ptr, out=out.ptr, scale=0.125, causal=1, window=window)
    gpu.paged_attention_dev(attn, b.c, b.s)
    gpu.synchronize()
    want = out.read()
    b.d_kv.upload(np.int32([length, 140]))
    gpu.paged_attention_dev(attn, b.c, b.s)
    gpu.synchronize()
    got = out.read()
    if window == 20 or length <= 0:
        want[:120] = 0
        assert np.array_equal(got, want)
    else:  # (every token of the first sequence sees all pages of its row of the table)
        assert np.array_equal(got[120:], want[120:])
        b.kv = [length, 140]
        for t in (0, 119):
            kk, vv = seen_of_table(b, 0)
            for h in range(8):
                s = kk[:, h] @ q.values[t, h] * 0.125
                p = np.exp(s - s.max())
                assert np.linalg.norm(got[t, h] - p @ vv[:, h] / p.sum()) <= 2.0 ** -17 * np.linalg.norm(p @ vv[:, h] / p.sum())


def seen_of_table(b, s):
    """Keys and values at all rows of a sequence's pages that were filled."""
    rows = [(pg, r) for i, pg in enumerate(b.table[s]) if 0 <= pg < b.n_pages for r in range(b.page)]
    k, v = b.k.values, b.v.values
    pg, r = np.array(rows).T
    return k[pg, r], v[pg, r]


@pytest.mark.parametrize("Hq,Hk,new", [(14, 2, [100, 30]), (5, 5, [200]), (20, 1, [40, 33]), (33, 1, [41]), (64, 8, [30, 9]), (3, 1, [340])])
@pytest.mark.parametrize("several", [False, True])
def test_head_groups(gpu, Hq, Hk, new, several):
    b = Batch(gpu, new, [(1100 if several else 150) + n for n in new], 16, Hk, 64, F16, seed=Hq)
    check(gpu, b, F32, Hq, several)


@pytest.mark.parametrize("page", [1, 7, 40, 64, 1000])
def test_page_sizes(gpu, page):
    b = Batch(gpu, [133, 1, 30], [700, 333, 70], page, 8, 64, F16, seed=page)
    check(gpu, b, F32, 8, True)
