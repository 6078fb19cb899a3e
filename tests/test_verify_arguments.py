"""What the verification of drafts refuses of its `missing` argument, before anything is launched, and the workspace that it asks for: no GPU is needed (and
no call gets that far)."""
import pytest

F32 = 0
AT = 1 << 20  # an aligned address that nothing reads


def verify(tqa, **kw):
    d = dict(dtype=F32, n_seqs=2, n_tokens=30, vocab=100, logits=AT, draft=AT, q_start=AT, tokens=AT, temperature=AT, accept=AT, pick=AT, kv_len=AT,
             past=AT, out_tokens=2 * AT, n_out=3 * AT, logprob=4 * AT, missing=5 * AT, workspace=AT, workspace_bytes=64)
    return tqa.lib().tqhip_verify_tokens_dev(tqa.Verify(**{**d, **kw}), None)


@pytest.mark.parametrize("at", [2 * AT, 2 * AT + 29 * 4, 2 * AT - 4, 3 * AT, 3 * AT + 4, 4 * AT + 116, AT, AT - 4])
def test_missing_over_an_output_is_refused(tqa, at):
    assert verify(tqa, missing=at) == -1


@pytest.mark.parametrize("at", [None, 5 * AT, 2 * AT - 8, 2 * AT + 30 * 4, 3 * AT + 8, 4 * AT - 8, AT + 8])
def test_missing_beside_the_outputs_is_not(tqa, at):
    assert verify(tqa, missing=at) == -7  # (the workspace is too small, which is looked at last)


@pytest.mark.parametrize("vocab", [1, 999, 4096, 4097, 9001, 24576, 24577, 98304, 100001, 151936])
@pytest.mark.parametrize("draft", [AT, None])
def test_one_workspace_for_smaller_calls(tqa, vocab, draft):
    """Short chunks give way to long ones as rows grow (from 98304 logits a CU on): a workspace for some tokens and sequences does for fewer, and
    for those without a draft."""
    def need(tokens, seqs, draft=draft):
        return tqa.verify_tokens_workspace(tqa.Verify(dtype=F32, n_seqs=seqs, n_tokens=tokens, vocab=vocab, logits=AT, draft=draft, q_start=AT, tokens=AT,
                                                      accept=AT, pick=AT, out_tokens=2 * AT, n_out=3 * AT))

    tokens = sorted({1, 2, 3, 5, 11, 12, 13, 23, 24, 25, 26, 97, 98, 99, 196, 197, 198, 500, 4000})
    for seqs in (1, 7, 600):
        rooms = [need(n, seqs) for n in tokens]
        assert rooms == sorted(rooms) and rooms[0] > 0
        assert all(need(n, max(1, seqs // 2)) <= r and need(n, seqs, None) <= r for n, r in zip(tokens, rooms))
