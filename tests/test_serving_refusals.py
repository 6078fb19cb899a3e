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
             past=AT, out_tokens=AT, n_out=AT, logprob=AT)
    return tqa.lib().tqhip_verify_tokens_dev(tqa.Verify(**{**d, **kw}), None)


@pytest.mark.parametrize("kw", [dict(dtype=3), dict(dtype=-1), dict(n_seqs=0), dict(n_tokens=0), dict(vocab=0), dict(logits_stride=99), dict(draft_stride=-100),
                                dict(kv_len=None), dict(logits=AT + 2), dict(dtype=F16, draft=AT + 1), dict(workspace=AT + 16, workspace_bytes=1 << 30)] +
                         [{n: None} for n in ("logits", "q_start", "tokens", "accept", "pick", "out_tokens", "n_out")])
def test_verify_refuses(tqa, kw):
    assert verify(tqa, **kw) == -1


@pytest.mark.parametrize("kw", [dict(vocab=(1 << 22) + 1), dict(n_tokens=INT_MAX), dict(n_seqs=INT_MAX), dict(vocab=1 << 22, n_tokens=1 << 15)])
def test_verify_too_large(tqa, kw):
    assert verify(tqa, **kw) == -3


def test_verify_workspace(tqa):
    assert verify(tqa, workspace=AT, workspace_bytes=64) == -7
    assert tqa.lib().tqhip_verify_tokens_dev(None, None) == -1 and tqa.lib().tqhip_verify_tokens_workspace(None) == 0
    assert tqa.verify_tokens_workspace(tqa.Verify(dtype=9)) == 0
