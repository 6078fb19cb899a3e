"""What the verification of drafts refuses of its `missing` argument, before anything is launched: no GPU is needed (and no call gets that far)."""
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
