"""What the batch calls refuse, before anything is launched: no GPU is needed (and none of these calls gets that far)."""
import pytest

F32, F16, BF16 = 0, 1, 2
AT = 1 << 20  # a 16-byte aligned address that nothing reads
INT_MAX = 2 ** 31 - 1


@pytest.fixture
def calls(tqa):
    lib = tqa.lib()
    proj = dict(dtype=F32, n_tokens=3, n_heads=4, n_kv_heads=2, head_dim=64, rotary_dim=64, q=AT, k=AT, v=AT, q_out=AT, k_out=AT, eps=1e-6,
                theta=1e6, positions=AT)
    cache = dict(k=AT, v=AT, dtype=F16, n_pages=4, page_size=16, n_kv_heads=2, head_dim=64)
    seqs = dict(n_seqs=2, n_tokens=3, q_start=AT, kv_len=AT, block_table=AT, table_stride=4)
    attn = dict(dtype=F32, n_heads=4, q=AT, out=AT, scale=0.125, causal=1)
    lora = dict(dtype=F16, n_tokens=3, in_dim=64, out_dim=8, rank=4, n_adapters=2, n_seqs=2, x=AT, base=AT, y=AT, a=AT, b=AT, scale=AT,
                q_start=AT, adapter=AT)

    def rope(**kw):
        return lib.tqhip_qk_norm_rope_dev(tqa.HeadProj(**{**proj, **kw}), None)

    def append(p={}, c={}, s={}):
        return lib.tqhip_kv_append_dev(tqa.HeadProj(**{**proj, **p}), tqa.KvCache(**{**cache, **c}), tqa.Seqs(**{**seqs, **s}), None)

    def attention(a={}, c={}, s={}):
        return lib.tqhip_paged_attention_dev(tqa.Attn(**{**attn, **a}), tqa.KvCache(**{**cache, **c}), tqa.Seqs(**{**seqs, **s}), None)

    def add(**kw):
        return lib.tqhip_lora_add_dev(tqa.Lora(**{**lora, **kw}), None)

    return dict(rope=rope, append=append, attention=attention, lora=add, lib=lib)


def test_null_structs(calls):
    lib = calls["lib"]
    assert lib.tqhip_qk_norm_rope_dev(None, None) == -1
    assert lib.tqhip_kv_append_dev(None, None, None, None) == -1
    assert lib.tqhip_paged_attention_dev(None, None, None, None) == -1
    assert lib.tqhip_lora_add_dev(None, None) == -1
    assert lib.tqhip_paged_attention_workspace(None, None, None) == 0 and lib.tqhip_lora_workspace(None) == 0


@pytest.mark.parametrize("kw", [dict(dtype=3), dict(dtype=-1), dict(n_tokens=0), dict(n_heads=0), dict(n_kv_heads=-1), dict(head_dim=63), dict(head_dim=0),
                                dict(head_dim=514), dict(rotary_dim=66), dict(rotary_dim=3), dict(rotary_dim=-2), dict(q=None), dict(q_out=None),
                                dict(q=None, q_out=None, k=None, k_out=None), dict(k_out=None), dict(positions=None), dict(theta=0.0),
                                dict(theta=float("nan")), dict(eps=-1.0), dict(eps=float("nan")), dict(q_stride=100), dict(k_out_stride=64), dict(q_stride=-256)])
def test_qk_norm_rope_refuses(calls, kw):
    assert calls["rope"](**kw) == -1


SHARED = [dict(c=dict(dtype=5)), dict(c=dict(k=None)), dict(c=dict(v=None)), dict(c=dict(n_pages=0)), dict(c=dict(page_size=0)),
          dict(c=dict(page_stride=-1)), dict(c=dict(token_stride=64)), dict(c=dict(page_stride=2048, token_stride=32, head_stride=64)),
          dict(s=dict(n_seqs=0)), dict(s=dict(q_start=None)), dict(s=dict(kv_len=None)), dict(s=dict(block_table=None)), dict(s=dict(table_stride=0)),
          dict(s=dict(max_kv=-1))]


@pytest.mark.parametrize("kw", SHARED + [dict(p=dict(k=None)), dict(p=dict(v=None)), dict(p=dict(n_kv_heads=4)), dict(p=dict(head_dim=128)),
                                         dict(p=dict(dtype=BF16)), dict(s=dict(n_tokens=4)), dict(p=dict(q_out=None)), dict(p=dict(v_stride=8))])
def test_kv_append_refuses(calls, kw):
    assert calls["append"](**kw) == -1


@pytest.mark.parametrize("kw", SHARED + [dict(a=dict(q=None)), dict(a=dict(out=None)), dict(a=dict(dtype=7)), dict(a=dict(dtype=BF16)), dict(a=dict(n_heads=3)),
                                         dict(a=dict(n_heads=0)), dict(a=dict(window=-1)), dict(a=dict(scale=float("inf"))), dict(c=dict(head_dim=96)),
                                         dict(a=dict(q=AT + 4)), dict(a=dict(out=AT + 8)), dict(c=dict(k=AT + 2)), dict(a=dict(q_stride=258)),
                                         dict(a=dict(out_stride=128)), dict(c=dict(page_stride=4096, token_stride=129, head_stride=64)),
                                         dict(s=dict(n_tokens=0))])
def test_paged_attention_refuses(calls, kw):
    assert calls["attention"](**kw) == -1


@pytest.mark.parametrize("kw", [dict(dtype=4), dict(n_tokens=0), dict(in_dim=0), dict(out_dim=0), dict(rank=0), dict(rank=257), dict(n_adapters=0), dict(n_seqs=0),
                                dict(x=None), dict(y=None), dict(a=None), dict(b=None), dict(scale=None), dict(q_start=None), dict(adapter=None)])
def test_lora_refuses(calls, kw):
    assert calls["lora"](**kw) == -1


def test_too_large(calls):
    assert calls["attention"](s=dict(table_stride=INT_MAX)) == -3
    assert calls["append"](s=dict(table_stride=INT_MAX)) == -3
    assert calls["rope"](n_tokens=INT_MAX, n_heads=2) == -3
    assert calls["rope"](n_heads=INT_MAX // 64) == -3
    assert calls["rope"](n_heads=8193, head_dim=2, rotary_dim=2) == -3
    assert calls["append"](p=dict(n_tokens=INT_MAX), s=dict(n_tokens=INT_MAX)) == -3
    assert calls["attention"](s=dict(n_tokens=INT_MAX)) == -3
    assert calls["attention"](s=dict(n_seqs=INT_MAX)) == -3
    assert calls["lora"](n_tokens=INT_MAX) == -3
    assert calls["lora"](n_seqs=INT_MAX) == -3


def test_misaligned_workspace(calls):
    assert calls["attention"](a=dict(workspace=AT + 16, workspace_bytes=1 << 40)) == -1
    assert calls["lora"](workspace=AT + 16, workspace_bytes=1 << 40) == -1


def test_workspace_of_a_short_window_in_a_long_cache(calls):
    """The split of the keys is bounded: a table of 2^30 positions and one token ask for some hundred parts, not for millions."""
    import tiny_llm_amd as tqa
    a = tqa.Attn(dtype=F32, n_heads=4, q=AT, out=AT, scale=0.125, causal=1, window=16)
    c = tqa.KvCache(k=AT, v=AT, dtype=F16, n_pages=1, page_size=1 << 20, n_kv_heads=2, head_dim=64)
    s = tqa.Seqs(n_seqs=1, n_tokens=1, q_start=AT, kv_len=AT, block_table=AT, table_stride=1023)
    assert 0 < tqa.paged_attention_workspace(a, c, s) <= 1 << 20
    a.window = INT_MAX
    assert 0 < tqa.paged_attention_workspace(a, c, s) <= 1 << 20


def test_too_small_a_workspace(calls):
    assert calls["lora"](workspace=AT, workspace_bytes=4) == -7
