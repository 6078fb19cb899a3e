"""Which attention kernel a call takes, from the host's numbers alone (no GPU is needed): 16-row tiles up to 32 rows a sequence or
56 tiles in all, 128-row tiles beyond."""
import pytest

AT = 1 << 20


def plan(tqa, n_tokens, n_seqs, Hq, Hk, D=64, **kw):
    attn = tqa.Attn(dtype=0, n_heads=Hq, q=AT, out=AT, scale=0.1, causal=1, **kw)
    cache = tqa.KvCache(k=AT, v=AT, dtype=1, n_pages=4, page_size=16, n_kv_heads=Hk, head_dim=D)
    seqs = tqa.Seqs(n_seqs=n_seqs, n_tokens=n_tokens, q_start=AT, kv_len=AT, block_table=AT, table_stride=64, max_kv=500)
    return tqa.paged_attention_plan(attn, cache, seqs)


@pytest.mark.parametrize("tokens,seqs,Hq,Hk,rows", [
    (1, 1, 14, 2, 16), (64, 64, 32, 8, 16), (64, 64, 64, 2, 16), (512, 64, 32, 8, 16), (513, 64, 32, 8, 128), (112, 1, 8, 8, 16), (113, 1, 8, 8, 128),
    (896, 1, 1, 1, 16), (897, 1, 1, 1, 128), (8192, 2, 32, 8, 128), (129, 1, 14, 2, 128),
])
def test_the_rule_between_the_kernels(tqa, tokens, seqs, Hq, Hk, rows):
    got = plan(tqa, tokens, seqs, Hq, Hk)
    assert got[0] == rows and 1 <= got[1] <= 512


def test_refusals(tqa):
    lib = tqa.lib()
    assert lib.tqhip_paged_attention_plan(None, None, None, None, None) == tqa.EBADSHAPE
    with pytest.raises(RuntimeError):
        plan(tqa, 1, 1, 3, 2)
    with pytest.raises(RuntimeError):
        plan(tqa, 1, 1, 4, 2, D=96)
    with pytest.raises(RuntimeError):
        plan(tqa, 1, 1, 4, 2, window=-1)


@pytest.mark.parametrize("tokens,seqs", [(1, 1), (256, 256), (2048, 256), (4096, 4096)])
def test_workspace_of_many_rows_beside_a_long_sequence(tqa, tokens, seqs):
    """Parts get longer where rows are many: a workspace of some 128 MB, not one of gigabytes."""
    attn = tqa.Attn(dtype=0, n_heads=32, q=AT, out=AT, scale=0.1, causal=1)
    cache = tqa.KvCache(k=AT, v=AT, dtype=1, n_pages=4, page_size=16, n_kv_heads=8, head_dim=128)
    batch = tqa.Seqs(n_seqs=seqs, n_tokens=tokens, q_start=AT, kv_len=AT, block_table=AT, table_stride=8192, max_kv=131072)
    rows, parts = tqa.paged_attention_plan(attn, cache, batch)
    need = tqa.paged_attention_workspace(attn, cache, batch)
    assert rows == 16 and need <= 128 << 20
    assert need == (0 if parts == 1 else parts * tokens * 32 * (4 * 128 + 8))
