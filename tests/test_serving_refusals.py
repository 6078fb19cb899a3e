"""What the calls of a server's step refuse, before anything is launched: no GPU is needed (and none of these calls gets that far)."""
import pytest

F32, F16, BF16, I8, E4M3 = 0, 1, 2, 3, 4
AT = 1 << 20  # an aligned address that nothing reads
INT_MAX = 2 ** 31 - 1


def page_map(tqa, **kw):
    d = dict(n_seqs=2, n_tokens=3, n_pages=8, page_size=16, table_stride=4, past=AT, n_new=AT, block_table=AT, n_held=AT, free_pages=AT, n_free=AT,
             q_start=AT, kv_len=AT, missing=AT, positions=AT, slots=AT)
    return tqa.lib().tqhip_page_map_dev(tqa.PageMap(**{**d, **kw}), None)


@pytest.mark.parametrize("kw", [dict(n_seqs=0), dict(n_seqs=-1), dict(n_tokens=-1), dict(n_pages=0), dict(page_size=0), dict(table_stride=0)] +
                         [{n: None} for n in ("past", "n_new", "block_table", "n_held", "free_pages", "n_free", "q_start", "kv_len", "missing")])
def test_page_map_refuses(tqa, kw):
    assert page_map(tqa, **kw) == -1


@pytest.mark.parametrize("kw", [dict(n_seqs=4097), dict(table_stride=INT_MAX), dict(n_pages=INT_MAX), dict(page_size=1 << 30), dict(n_tokens=INT_MAX)])
def test_page_map_too_large(tqa, kw):
    assert page_map(tqa, **kw) == -3


def test_null_structs(tqa):
    assert tqa.lib().tqhip_page_map_dev(None, None) == -1


def verify(tqa, **kw):
    d = dict(dtype=F32, n_seqs=2, n_tokens=3, vocab=100, logits=AT, draft=AT, q_start=AT, tokens=AT, temperature=AT, accept=AT, pick=AT, kv_len=AT,
             past=AT, out_tokens=2 * AT, n_out=AT, logprob=2 * AT)
    return tqa.lib().tqhip_verify_tokens_dev(tqa.Verify(**{**d, **kw}), None)


@pytest.mark.parametrize("kw", [dict(dtype=3), dict(dtype=-1), dict(n_seqs=0), dict(n_tokens=0), dict(vocab=0), dict(logits_stride=99), dict(draft_stride=-100),
                                dict(kv_len=None), dict(logits=AT + 2), dict(dtype=F16, draft=AT + 1), dict(workspace=AT + 16, workspace_bytes=1 << 30)] +
                         [{n: None} for n in ("logits", "q_start", "tokens", "accept", "pick", "out_tokens", "n_out")] +
                         [dict(out_tokens=AT), dict(out_tokens=AT + 8), dict(logprob=AT - 8), dict(tokens=2 * AT), dict(accept=2 * AT, logprob=None)])
def test_verify_refuses(tqa, kw):
    assert verify(tqa, **kw) == -1


@pytest.mark.parametrize("kw", [dict(vocab=(1 << 22) + 1), dict(n_tokens=INT_MAX), dict(n_seqs=INT_MAX), dict(vocab=1 << 22, n_tokens=1 << 15)])
def test_verify_too_large(tqa, kw):
    assert verify(tqa, **kw) == -3


def test_verify_workspace(tqa):
    assert verify(tqa, workspace=AT, workspace_bytes=64) == -7
    assert tqa.lib().tqhip_verify_tokens_dev(None, None) == -1 and tqa.lib().tqhip_verify_tokens_workspace(None) == 0
    assert tqa.verify_tokens_workspace(tqa.Verify(dtype=9)) == 0


PROJ = dict(dtype=F32, n_tokens=3, n_heads=4, n_kv_heads=2, head_dim=64, rotary_dim=64, q=AT, k=AT, v=AT, q_out=AT, eps=1e-6, theta=1e6)
CACHE = dict(k=AT, v=AT, scales=AT, dtype=I8, n_pages=4, page_size=16, block=8, n_kv_heads=2, head_dim=64)
SEQS = dict(n_seqs=2, n_tokens=3, q_start=AT, kv_len=AT, block_table=AT, table_stride=4)
ATTN = dict(dtype=F32, n_heads=4, q=AT, out=AT, scale=0.125, causal=1)


def append8(tqa, p={}, c={}, s={}):
    return tqa.lib().tqhip_kv_append8_dev(tqa.HeadProj(**{**PROJ, **p}), tqa.KvCache8(**{**CACHE, **c}), tqa.Seqs(**{**SEQS, **s}), None)


def attention8(tqa, a={}, c={}, s={}):
    return tqa.lib().tqhip_paged_attention8_dev(tqa.Attn(**{**ATTN, **a}), tqa.KvCache8(**{**CACHE, **c}), tqa.Seqs(**{**SEQS, **s}), None)


SHARED8 = [dict(c=dict(dtype=d)) for d in (0, 1, 2, 5, -1)] + [dict(c={n: None}) for n in ("k", "v", "scales")] + \
          [dict(c=dict(n_pages=0)), dict(c=dict(page_size=0)), dict(c=dict(block=0)), dict(c=dict(block=-8)), dict(c=dict(block=5)), dict(c=dict(block=32)),
           dict(c=dict(scales=AT + 4)), dict(c=dict(head_dim=96)), dict(c=dict(page_stride=-1)), dict(c=dict(token_stride=64)), dict(c=dict(k=AT + 8)),
           dict(c=dict(v=AT + 1)), dict(c=dict(page_stride=4096, token_stride=136, head_stride=64)), dict(s=dict(n_seqs=0)), dict(s=dict(q_start=None)),
           dict(s=dict(kv_len=None)), dict(s=dict(block_table=None)), dict(s=dict(table_stride=0)), dict(s=dict(max_kv=-1))]


@pytest.mark.parametrize("kw", SHARED8 + [dict(p=dict(k=None)), dict(p=dict(v=None)), dict(p=dict(n_kv_heads=4)), dict(p=dict(head_dim=128)), dict(p=dict(dtype=3)),
                                          dict(s=dict(n_tokens=4)), dict(p=dict(q_out=None)), dict(p=dict(v_stride=8)), dict(p=dict(q_stride=8)),
                                          dict(p=dict(rotary_dim=66)), dict(p=dict(theta=0.0)), dict(p=dict(eps=-1.0)), dict(p=dict(n_heads=0)),
                                          dict(c=dict(page_stride=1024, token_stride=128, head_stride=64))])
def test_kv_append8_refuses(tqa, kw):
    assert append8(tqa, **kw) == -1


@pytest.mark.parametrize("kw", SHARED8 + [dict(a=dict(q=None)), dict(a=dict(out=None)), dict(a=dict(dtype=3)), dict(a=dict(n_heads=3)), dict(a=dict(n_heads=0)),
                                          dict(a=dict(window=-1)), dict(a=dict(scale=float("nan"))), dict(a=dict(q=AT + 4)), dict(a=dict(out_stride=128)),
                                          dict(a=dict(q_stride=258)), dict(a=dict(workspace=AT + 16, workspace_bytes=1 << 40)), dict(s=dict(n_tokens=0))])
def test_paged_attention8_refuses(tqa, kw):
    assert attention8(tqa, **kw) == -1


def test_8_bits_too_large(tqa):
    for call in (append8, attention8):
        assert call(tqa, s=dict(table_stride=INT_MAX)) == -3
        assert call(tqa, c=dict(n_pages=INT_MAX)) == -3
    assert append8(tqa, p=dict(n_tokens=INT_MAX), s=dict(n_tokens=INT_MAX)) == -3
    assert append8(tqa, p=dict(n_heads=8193)) == -3
    assert append8(tqa, s=dict(n_seqs=INT_MAX)) == -3
    assert attention8(tqa, s=dict(n_tokens=INT_MAX)) == -3
    assert attention8(tqa, s=dict(n_seqs=INT_MAX)) == -3


def test_8_bits_nulls_and_workspace(tqa):
    lib = tqa.lib()
    assert lib.tqhip_kv_append8_dev(None, None, None, None) == -1 and lib.tqhip_paged_attention8_dev(None, None, None, None) == -1
    assert lib.tqhip_paged_attention8_workspace(None, None, None) == 0 and lib.tqhip_paged_attention8_plan(None, None, None, None, None) == -1
    a, c = tqa.Attn(**ATTN), tqa.KvCache8(**CACHE)
    s = tqa.Seqs(**{**SEQS, "table_stride": 2000, "n_tokens": 1})
    need = tqa.paged_attention8_workspace(a, c, s)
    assert need > 0
    a.workspace, a.workspace_bytes = AT, need - 1
    assert lib.tqhip_paged_attention8_dev(a, c, s, None) == -7
    c.block = 7
    assert tqa.paged_attention8_workspace(a, c, s) == 0
