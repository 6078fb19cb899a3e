"""How attention over codes of 8 bits is cut, from the host's numbers alone (no GPU is needed): tiles of few rows up to 64 rows a sequence or 112
tiles of 16 in all, of 32 rows where sequences have more than 16 (16 on heads of 256 with fp32 activations), 128-row tiles beyond."""
import pytest

AT = 1 << 20
F32, F16, BF16, I8, E4M3 = 0, 1, 2, 3, 4


@pytest.mark.parametrize("cache", [I8, E4M3])
@pytest.mark.parametrize("tokens,seqs,Hq,Hk,D,rows,wide", [
    (1, 1, 14, 2, 64, 16, 16), (64, 64, 32, 8, 128, 16, 16), (128, 32, 32, 8, 128, 16, 16), (160, 32, 32, 8, 128, 32, 32), (512, 32, 32, 8, 128, 32, 32),
    (513, 32, 32, 8, 128, 128, 128), (56, 1, 32, 8, 128, 32, 32), (57, 1, 32, 8, 128, 128, 128), (128, 1, 14, 2, 64, 32, 32), (129, 1, 14, 2, 64, 128, 128),
    (512, 1, 32, 8, 128, 128, 128), (896, 1, 2, 1, 256, 32, 16), (897, 1, 2, 1, 256, 128, 128), (2400, 1, 1, 1, 256, 128, 128), (20, 1, 2, 1, 256, 32, 16),
])
def test_the_rule_between_the_kernels(tqa, tokens, seqs, Hq, Hk, D, rows, wide, cache):
    for act, want in ((BF16, rows), (F16, rows), (F32, wide)):
        attn = tqa.Attn(dtype=act, n_heads=Hq, q=AT, out=AT, scale=0.1, causal=1)
        codes = tqa.KvCache8(k=AT, v=AT, scales=AT, dtype=cache, n_pages=4, page_size=16, block=16, n_kv_heads=Hk, head_dim=D)
        batch = tqa.Seqs(n_seqs=seqs, n_tokens=tokens, q_start=AT, kv_len=AT, block_table=AT, table_stride=64, max_kv=500)
        got = tqa.paged_attention8_plan(attn, codes, batch)
        assert got[0] == want and 1 <= got[1] <= 512
