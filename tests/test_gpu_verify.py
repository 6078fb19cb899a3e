"""Drafted tokens accepted, refused and replaced (tqhip_verify_tokens_dev), against the rules written out row by row in 64 bits.

Tokens and counts are equal. That asks for random numbers that do not fall on a border: both sides sum up to 2^18 terms of at most 1 in 64
bits, in different orders, so their prefix sums differ by at most 2^18 2^-53 = 2^-35 of the sum, and single probabilities by that of themselves; the
forms below assert that no number is nearer to a border than 2^-30 of the sum, or of the two sides of a comparison (inputs are seeded, and such a case would be drawn with probability 2^-12 each).
Log probabilities are rounded to fp32 once, 2^-24 of themselves; in 64 bits they are exact to 2^-40 beside it.
"""
import numpy as np
import pytest

from batch_ref import Dev, ints

pytestmark = pytest.mark.gpu

F32, F16, BF16 = 0, 1, 2
NEAR = 2.0 ** -30
INF = np.inf


def softmax(row, T):
    """(probabilities, their logarithms), or None where the row has none."""
    top = row.max()
    if not np.isfinite(top):
        return None
    with np.errstate(invalid="ignore"):  # (minus infinity over an infinite T)
        z = np.where(row == -INF, -INF, (row - top) / T)
    total = np.exp(z).sum()
    return np.exp(z) / total, z - np.log(total)


def expect(starts, logits, draft, tokens, heat, accept, pick, vocab):
    """-> (out_tokens, logprob, n_out) over the tokens of the sequences; -2 where a token is in none."""
    n_tokens = len(tokens)
    out, lps, count = np.full(n_tokens, -2, np.int64), np.full(n_tokens, np.nan), np.zeros(len(starts) - 1, np.int64)
    for b in range(len(starts) - 1):
        T, first, end = float(heat[b]), int(starts[b]), int(starts[b + 1])
        out[first:end], lps[first:end] = -1, 0.0
        greedy = not T > 0
        for t in range(first, end):
            count[b] += 1
            sm = softmax(logits[t], 1.0 if greedy else T)
            if sm is None:
                break
            p, lp = sm
            x = int(tokens[t + 1]) if t + 1 < end else -1
            drafted = 0 <= x < vocab
            if greedy:
                out[t] = int(np.argmax(logits[t]))
                lps[t] = lp[out[t]]
                if x == out[t]:
                    continue
                break
            q = None
            if drafted:
                q = np.zeros(vocab)
                q[x] = 1.0
                if draft is not None:
                    sq = softmax(draft[t], T)
                    q = None if sq is None else sq[0]
                u = float(np.float32(accept[t]))
                if q is not None:
                    assert u == 0 or abs(u * q[x] - p[x]) > NEAR * max(u * q[x], p[x])
                    if u * q[x] < p[x]:
                        out[t], lps[t] = x, lp[x]
                        continue
            w = p if q is None else np.maximum(p - q, 0.0)
            if w.sum() <= 0:
                w = p
            upto = np.cumsum(w)
            goal = float(np.float32(pick[b])) * upto[-1]
            live = upto[np.diff(upto, prepend=0) > 0]
            assert len(live) == 1 or np.abs(live[:-1] - goal).min() > NEAR * upto[-1]
            out[t] = min(int(np.searchsorted(upto, goal, side="right")), int(np.flatnonzero(w > 0)[-1]))
            lps[t] = lp[out[t]]
            break
    return out, lps, count


class Case:
    """Rows, drafts drawn from the draft model's rows, random numbers; `lead` and `tail` tokens of no sequence around them."""

    def __init__(self, gpu, counts, vocab, dtype=F32, dense=True, heat=None, seed=0, lead=0, tail=0, pad=0, std=2.0, near=0.5):
        self.gpu, self.vocab, self.dtype, self.pad = gpu, vocab, dtype, pad
        rng = self.rng = np.random.default_rng(seed)
        self.starts = lead + np.concatenate(([0], np.cumsum(counts))).astype(np.int64)
        n = self.n = int(self.starts[-1]) + tail
        self.logits = rng.standard_normal((n, vocab + pad)) * std
        self.draft = self.logits + near * rng.standard_normal((n, vocab + pad)) if dense else None
        self.heat = np.ones(len(counts), np.float32) if heat is None else np.asarray(heat, np.float32)
        self.accept, self.pick = rng.random(n).astype(np.float32), rng.random(len(counts)).astype(np.float32)
        self.tokens = rng.integers(0, vocab, n)
        for t in range(n - 1):
            row = (self.draft if dense else self.logits)[t, :vocab]
            self.tokens[t + 1] = np.argmax(row + rng.gumbel(size=vocab))

    def put(self):
        """To the device (rows are rounded to their type here)."""
        gpu = self.gpu
        self.d_logits = Dev(gpu, self.logits, self.dtype)
        self.d_draft = None if self.draft is None else Dev(gpu, self.draft, self.dtype)
        self.bufs = dict(q_start=ints(gpu, self.starts), tokens=ints(gpu, self.tokens), out_tokens=ints(gpu, np.full(self.n, -2)),
                         n_out=ints(gpu, np.full(len(self.heat), -2)), kv_len=ints(gpu, 1000 + np.arange(len(self.heat))), past=ints(gpu, np.full(len(self.heat), -2)))
        self.bufs |= {n: gpu.DeviceBuffer.from_array(x.astype(np.float32)) for n, x in
                      (("temperature", self.heat), ("accept", self.accept), ("pick", self.pick), ("logprob", np.full(self.n, np.nan)))}
        stride = self.vocab + self.pad if self.pad else 0
        self.v = gpu.Verify(dtype=self.dtype, n_seqs=len(self.heat), n_tokens=self.n, vocab=self.vocab, logits=self.d_logits.ptr,
                            draft=None if self.draft is None else self.d_draft.ptr, logits_stride=stride, draft_stride=stride,
                            **{n: b.ptr for n, b in self.bufs.items()})
        return self

    def read(self):
        b = self.bufs
        return (b["out_tokens"].download(np.int32, self.n), b["logprob"].download(np.float32, self.n), b["n_out"].download(np.int32, len(self.heat)),
                b["past"].download(np.int32, len(self.heat)))

    def want(self):
        V = self.vocab
        return expect(self.starts, self.d_logits.values[:, :V], None if self.draft is None else self.d_draft.values[:, :V], self.tokens, self.heat,
                      self.accept, self.pick, V)

    def check(self):
        out, lp, count, past = self.read()
        want, want_lp, want_count = self.want()
        assert np.array_equal(count, want_count), (count, want_count)
        assert np.array_equal(out, want)
        assert np.array_equal(np.isnan(lp), np.isnan(want_lp))
        fine = ~np.isnan(want_lp)
        assert np.all(np.abs(lp[fine] - want_lp[fine]) <= (2.0 ** -24 + 2.0 ** -40) * np.abs(want_lp[fine]) + 2.0 ** -40)
        assert np.array_equal(past, 1000 + np.arange(len(count)) - np.diff(self.starts) + want_count)
        return out, count

    def run(self):
        self.put()
        self.gpu.verify_tokens_dev(self.v)
        self.gpu.lib().tqhip_synchronize()
        return self.check()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("dense", [True, False])
@pytest.mark.parametrize("vocab", [1, 2, 63, 1000, 8191, 8192, 8193, 20011])
def test_rows_against_the_formula(gpu, vocab, dense, dtype):
    counts = [5, 1, 0, 3, 9, 2, 0, 6]
    heat = [1.0, 0.7, 1.0, 1.5, 0.9, 0.0, 1.0, 0.2]
    Case(gpu, counts, vocab, dtype, dense, heat, seed=vocab + dtype, lead=2, tail=3).run()


@pytest.mark.parametrize("dense", [True, False])
def test_the_benchmark_s_vocabulary(gpu, dense):
    _, count = Case(gpu, [5, 5, 4, 1], 151936, F32, dense, [1.0, 0.8, 0.0, 0.6], seed=3, std=3.0).run()
    assert count[0] >= 1


@pytest.mark.parametrize("pad", [1, 8, 77])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strides_and_odd_rows(gpu, pad, dtype):
    c = Case(gpu, [3, 4, 2], 1001, dtype, True, seed=pad, pad=pad)
    c.logits[:, 1001:], c.draft[:, 1001:] = np.nan, INF  # (what lies between the rows is not theirs)
    c.run()


def test_no_drafts_is_a_plain_draw(gpu):
    Case(gpu, [1] * 70, 5000, F32, False, np.linspace(0, 2, 70), seed=5).run()


def test_many_drafts_of_one_request(gpu):
    c = Case(gpu, [300], 50, F32, True, seed=7, near=0.01)
    c.accept[:200] = 0.0
    _, count = c.run()
    assert count[0] > 200


def test_all_accepted_and_none(gpu):
    c = Case(gpu, [6, 6], 3000, F32, True, seed=9)
    c.accept[:6] = 0.0
    c.accept[6:] = 1.0 - 2.0 ** -24
    c.tokens[7] = np.argmax(c.draft[6, :3000] - c.logits[6, :3000])
    _, count = c.run()
    assert count.tolist() == [6, 1]


def test_drafts_of_other_lengths(gpu):
    """A token outside the vocabulary ends the drafts: the draw before it is from p."""
    for bad in (-1, 400, 2 ** 31 - 1, -2 ** 31):
        c = Case(gpu, [5, 5, 5], 400, F32, True, [1.0, 0.5, 0.0], seed=11)
        c.accept[:] = 0.0
        for b in range(3):
            c.tokens[5 * b + 3] = bad
        c.tokens[11] = np.argmax(c.logits[10])
        c.tokens[12] = np.argmax(c.logits[11])
        _, count = c.run()
        assert count.tolist() == [3, 3, 3]


def test_the_same_rows_accept_everything(gpu):
    """p = q: u p < p whenever p > 0."""
    c = Case(gpu, [8, 8], 700, F32, True, seed=13, near=0.0)
    c.accept[:] = 0.5
    _, count = c.run()
    assert count.tolist() == [8, 8]


def test_nothing_left_draws_from_p(gpu):
    """One token has all of p and of q, and is refused only by a number of 1: max(p - q, 0) is nothing."""
    c = Case(gpu, [2], 40, F32, True, seed=15)
    c.logits[:], c.draft[:] = -INF, -INF
    c.logits[:, 17], c.draft[:, 17] = 3.0, 1.0
    c.tokens[:] = 17
    c.accept[:] = 1.0
    c.put()
    gpu.verify_tokens_dev(c.v)
    gpu.lib().tqhip_synchronize()
    out, lp, count, _ = c.read()
    assert out.tolist() == [17, -1] and count[0] == 1 and lp[0] == 0.0


def test_masked_logits(gpu):
    """Tokens of minus infinity are never drawn, also where whole chunks of the row are."""
    c = Case(gpu, [4, 4, 4, 1], 30000, F32, True, [1.0, 0.0, 2.0, 1.0], seed=17)
    c.logits[:, :9000] = -INF
    c.logits[:, 16000:29000] = -INF
    c.draft[:, 16384:24576] = -INF
    for t in range(1, 13):
        c.tokens[t] = np.argmax(c.draft[t - 1])
    out, _ = c.run()
    got = out[out >= 0]
    assert np.all((got >= 9000) & ((got < 16000) | (got >= 29000)))


@pytest.mark.parametrize("what", [np.nan, INF])
def test_rows_without_probabilities(gpu, what):
    """As a target such a row ends its sequence with -1, as a draft it refuses and the draw is from p; others do not notice."""
    c = Case(gpu, [4, 4, 4, 4, 4], 9000, F32, True, [1.0, 1.0, 0.0, 1.0, 1.0], seed=19)
    c.accept[:] = 0.0
    c.logits[1, 8500] = what
    c.draft[5, 3] = what
    c.tokens[9], c.tokens[10] = np.argmax(c.logits[8]), np.argmax(c.logits[9])
    c.logits[10, 0] = what
    c.logits[12] = -INF
    c.draft[17] = -INF
    out, count = c.run()
    assert count.tolist() == [2, 2, 3, 1, 2]
    assert out[1] == -1 and out[10] == -1 and out[12] == -1 and out[5] >= 0 and out[17] >= 0


def test_greedy_takes_the_first_of_equals(gpu):
    c = Case(gpu, [4, 1, 1], 20000, BF16, False, [0.0, -1.0, np.nan], seed=21)
    c.logits = np.round(c.logits)
    c.logits[0, [30, 8000, 8300, 19999]] = 40.0
    c.logits[1, [8192, 8193]] = 41.0
    c.logits[4, [19998, 19999]] = 42.0
    c.tokens[1:4] = [30, 8193, 5]
    out, count = c.run()
    assert out[:2].tolist() == [30, 8192] and count.tolist() == [2, 1, 1] and out[4] == 19998


@pytest.mark.parametrize("heat", [1e-30, 1e-4, 1e30, INF])
def test_far_temperatures(gpu, heat):
    c = Case(gpu, [3, 1], 500, F32, False, [heat, heat], seed=23)
    c.tokens[1] = np.argmax(c.logits[0])
    c.logits[:, 7] = -INF if heat == INF else c.logits[:, 7]
    c.run()


def test_what_comes_out_is_distributed_as_the_target(gpu):
    """20000 requests with one draft each, drawn from q: the first token out is distributed as p. A count of n p has a standard
    deviation of sqrt(n p (1 - p)); five of them are passed once in 10^6."""
    n, p, q = 20000, np.array([0.5, 0.2, 0.05, 0.25]), np.array([0.1, 0.3, 0.4, 0.2])
    c = Case(gpu, [2] * n, 4, F32, True, seed=25)
    c.logits[:], c.draft[:] = np.log(p), np.log(q)
    c.tokens[1::2] = c.rng.choice(4, n, p=q)
    c.put()
    gpu.verify_tokens_dev(c.v)
    gpu.lib().tqhip_synchronize()
    out, _, count, _ = c.read()
    share = np.bincount(out[::2], minlength=4) / n
    assert np.all(np.abs(share - p) < 5 * np.sqrt(p * (1 - p) / n)), share
    kept = np.minimum(p, q).sum()
    assert abs((count == 2).mean() - kept) < 5 * np.sqrt(kept * (1 - kept) / n)


def test_optional_outputs_and_defaults(gpu):
    c = Case(gpu, [3, 2], 300, F32, True, seed=27).put()
    c.v.temperature = c.v.logprob = c.v.past = c.v.kv_len = None
    gpu.verify_tokens_dev(c.v)
    gpu.lib().tqhip_synchronize()
    out, lp, count, past = c.read()
    want, _, want_count = c.want()
    assert np.array_equal(out, want) and np.array_equal(count, want_count) and np.all(np.isnan(lp)) and np.all(past == -2)


def test_a_captured_call_with_its_own_workspace(gpu):
    """Replays read the rows and numbers that are there when they run; past may be kv_len itself; nothing past the workspace is written."""
    a, b = (Case(gpu, [4, 2, 5], 9001, F32, True, [1.0, 0.0, 0.8], seed=s).put() for s in (29, 31))
    need = gpu.verify_tokens_workspace(a.v)
    assert 0 < need < 1 << 20
    space = gpu.DeviceBuffer.from_array(np.full(need + 256, 0xA5, np.uint8))
    assert space.ptr % 256 == 0
    a.v.workspace, a.v.workspace_bytes, a.v.past = space.ptr, need, a.v.kv_len
    stream = gpu.Stream()
    graph = gpu.OpsGraph([gpu.batch_op(gpu.OP_VERIFY_TOKENS, a.v)], stream)
    for c in (a, b, a):
        a.d_logits.buf.upload(c.d_logits.values.astype(np.float32))
        a.d_draft.buf.upload(c.d_draft.values.astype(np.float32))
        for n, x in (("tokens", c.tokens.astype(np.int32)), ("accept", c.accept), ("pick", c.pick), ("temperature", c.heat)):
            a.bufs[n].upload(x)
        a.bufs["kv_len"].upload(np.full(3, 50, np.int32))
        graph.launch()
        stream.synchronize()
        want, _, count = c.want()
        out, _, got, _ = a.read()
        assert np.array_equal(out, want) and np.array_equal(got, count)
        assert np.array_equal(a.bufs["kv_len"].download(np.int32, 3), 50 - np.array([4, 2, 5]) + count)
    graph.close()
    assert np.all(space.download(np.uint8, need + 256)[need:] == 0xA5)
