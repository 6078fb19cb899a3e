"""Strides of a paged cache that kv_append takes and refuses, without a GPU: a refusal is TQHIP_EBADSHAPE, and a call that passes the
checks is made to end at a later one (more new tokens' heads than a launch holds, TQHIP_ETOOLARGE), so that nothing is launched."""
import itertools

import pytest

AT = 1 << 20  # a 16-byte aligned address that nothing reads
TOKENS = 2 ** 31 - 1


def append(tqa, n_pages, page_size, n_kv_heads, head_dim, page, token, head):
    proj = tqa.HeadProj(dtype=0, n_tokens=TOKENS, n_heads=8192, n_kv_heads=n_kv_heads, head_dim=head_dim, q=AT, k=AT, v=AT, q_out=AT, eps=1e-6)
    cache = tqa.KvCache(k=AT, v=AT, dtype=1, n_pages=n_pages, page_size=page_size, n_kv_heads=n_kv_heads, head_dim=head_dim, page_stride=page,
                        token_stride=token, head_stride=head)
    seqs = tqa.Seqs(n_seqs=1, n_tokens=TOKENS, q_start=AT, kv_len=AT, block_table=AT, table_stride=1)
    return tqa.lib().tqhip_kv_append_dev(proj, cache, seqs, None)


# pages, rows a page, heads, head size, strides of page, row and head
APART = [
    (4, 16, 2, 64, 0, 0, 0), (4, 16, 2, 64, 2048, 128, 64), (4, 16, 2, 64, 2048, 64, 1024), (4, 16, 2, 64, 128, 512, 64), (4, 16, 2, 64, 4096, 256, 128),
    (4, 16, 2, 64, 1024, 64, 4096), (1, 16, 2, 64, 1, 128, 64), (4, 1, 2, 64, 128, 64, 64), (4, 16, 1, 64, 1024, 64, 64), (4, 3, 2, 64, 400, 130, 64),
    (1 << 20, 1 << 10, 8, 512, 1 << 40, 1 << 20, 512),
]
SHARED = [
    (4, 16, 2, 64, 2048, 64, 64), (4, 16, 2, 64, 8, 128, 64), (4, 16, 2, 64, 2047, 128, 64), (4, 16, 2, 64, 2048, 127, 64), (4, 16, 2, 64, 2048, 64, 1023),
    (4, 16, 2, 64, 127, 512, 64), (2, 2, 2, 64, 64, 64, 64), (2, 1, 1, 64, 63, 64, 64), (2 ** 31 - 1, 2, 1, 64, 2 ** 62, 2 ** 62, 64),
]


@pytest.mark.parametrize("layout", APART)
def test_rows_that_are_apart_are_taken(tqa, layout):
    assert append(tqa, *layout) == tqa.ETOOLARGE


@pytest.mark.parametrize("layout", SHARED)
def test_rows_that_share_elements_are_refused(tqa, layout):
    assert append(tqa, *layout) == tqa.EBADSHAPE


def test_small_layouts_against_their_elements(tqa):
    """No layout of a small family that is taken shares an element between two rows."""
    taken = 0
    for page, token, head in itertools.product(range(2, 14), repeat=3):
        rows = sorted(p * page + t * token + h * head for p in range(2) for t in range(2) for h in range(2))
        apart = all(b - a >= 2 for a, b in zip(rows, rows[1:]))
        status = append(tqa, 2, 2, 2, 2, page, token, head)
        assert status in (tqa.ETOOLARGE, tqa.EBADSHAPE)
        if status == tqa.ETOOLARGE:
            taken += 1
            assert apart, (page, token, head)
    assert taken > 100
