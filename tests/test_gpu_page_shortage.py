"""A server's steps whose pages run out: the lengths stay on the device, where the verification of one step leaves them and the page map of the next
reads them, and no sequence ever attends to positions that were not written for it. Tolerances as in the calls' own tests."""
import numpy as np
import pytest

import batch_ref as ref
import test_gpu_append8 as append
import test_gpu_attention8 as attention
import test_gpu_page_map as pages
import test_gpu_verify as verify
from batch8_ref import E4M3, I8
from batch_ref import ints
from test_gpu_server_step import F32, Cache

pytestmark = pytest.mark.gpu


def held_back(want, starts, missing):
    """verify.expect's answer where the sequences that lack pages say nothing."""
    toks, lps, counts = (x.copy() for x in want)
    for b in np.flatnonzero(missing > 0):
        toks[starts[b]:starts[b + 1]], lps[starts[b]:starts[b + 1]], counts[b] = -1, 0.0, 0
    return toks, lps, counts


@pytest.mark.parametrize("counts,vocab,dense", [([5, 1, 0, 3, 9, 2], 1000, True), ([5, 1, 0, 3, 9, 2], 9001, False), ([1] * 70, 300, False), ([300, 2, 300], 50, True)])
def test_sequences_that_lack_pages_say_nothing(gpu, counts, vocab, dense):
    """Every second one (and its neighbours are as ever): no tokens, and the length of before the call."""
    c = verify.Case(gpu, counts, vocab, F32, dense, np.linspace(0, 1.5, len(counts)), seed=vocab, lead=2, tail=3).put()
    missing = np.where(np.arange(len(counts)) % 2 == 0, 3, 0)
    missing[-1] = -5  # (no number of pages)
    d_missing = ints(gpu, missing)
    c.v.missing = d_missing.ptr
    want, lps, count = held_back(c.want(), c.starts, missing)
    for past in ("past", "kv_len"):
        c.v.past = c.bufs[past].ptr  # (past may be kv_len)
        gpu.verify_tokens_dev(c.v)
        gpu.synchronize()
        out, lp, n_out, _ = c.read()
        assert np.array_equal(out, want) and np.array_equal(n_out, count)
        fine = ~np.isnan(lps)
        assert np.array_equal(np.isnan(lp), ~fine) and np.all(np.abs(lp - lps)[fine] <= (2.0 ** -24 + 2.0 ** -40) * np.abs(lps[fine]) + 2.0 ** -40)
        assert np.array_equal(c.bufs[past].download(np.int32, len(counts)), 1000 + np.arange(len(counts)) - np.diff(c.starts) + count)
    c.v.missing = None
    c.bufs["kv_len"].upload((1000 + np.arange(len(counts))).astype(np.int32))
    c.v.past = c.bufs["past"].ptr
    gpu.verify_tokens_dev(c.v)
    gpu.synchronize()
    c.check()


@pytest.mark.parametrize("own_past", [True, False])
@pytest.mark.parametrize("dtype", [I8, E4M3])
def test_steps_while_pages_run_out(gpu, dtype, own_past):
    """Twelve pages for five requests of up to 70 positions. Only the numbers of new tokens (and the end of a request) come from the host; own_past: kv_len
    is an array of its own, else it is past. A request that found no pages is given its tokens again."""
    n, page, block, Hq, Hk, D, V, T, stride, n_pages = 5, 8, 4, 4, 2, 64, 300, 40, 12, 12
    rng = np.random.default_rng(dtype)
    host = pages.Server(n, stride, n_pages, page, 1)
    dev = pages.Device(gpu, host, n_pages, T)
    if not own_past:
        dev.map.kv_len = dev.map.past
    c = Cache(gpu, n, n_pages, page, block, Hk, D, dtype, stride)
    c.s = gpu.Seqs(n_seqs=n, n_tokens=T, q_start=dev.map.q_start, kv_len=dev.map.kv_len, block_table=dev.map.block_table, table_stride=stride)
    zeros = lambda *shape: gpu.DeviceBuffer.from_array(np.zeros(shape, np.float32))  # noqa: E731
    x = {"q": zeros(T, Hq, D), "k": zeros(T, Hk, D), "v": zeros(T, Hk, D), "out": zeros(T, Hq, D), "logits": zeros(T, V), "draft": zeros(T, V),
         "accept": zeros(T), "pick": zeros(n), "heat": zeros(n), "logprob": zeros(T)}
    d_tokens, d_out, d_count = (ints(gpu, np.zeros(m)) for m in (T, T, n))
    proj = gpu.HeadProj(dtype=F32, n_tokens=T, n_heads=Hq, n_kv_heads=Hk, head_dim=D, q=x["q"].ptr, k=x["k"].ptr, v=x["v"].ptr, q_out=x["q"].ptr)
    attn = gpu.Attn(dtype=F32, n_heads=Hq, q=x["q"].ptr, out=x["out"].ptr, scale=D ** -0.5, causal=1)
    judge = gpu.Verify(dtype=F32, n_seqs=n, n_tokens=T, vocab=V, logits=x["logits"].ptr, draft=x["draft"].ptr, q_start=dev.map.q_start, tokens=d_tokens.ptr,
                       temperature=x["heat"].ptr, accept=x["accept"].ptr, pick=x["pick"].ptr, kv_len=dev.map.kv_len, past=dev.map.past,
                       out_tokens=d_out.ptr, n_out=d_count.ptr, logprob=x["logprob"].ptr, missing=dev.map.missing)
    stream = gpu.Stream()
    graph = gpu.OpsGraph([gpu.batch_op(gpu.OP_PAGE_MAP, dev.map), gpu.batch_op(gpu.OP_KV_APPEND8, proj, c.c, c.s),
                          gpu.batch_op(gpu.OP_PAGED_ATTENTION8, attn, c.c, c.s), gpu.batch_op(gpu.OP_VERIFY_TOKENS, judge)], stream)
    written = {}  # (page, row) -> the request and position that its row was last written for
    request = list(range(n))
    again = np.zeros(n, bool)
    new, short, partly, served = np.zeros(n, np.int64), 0, 0, 0
    for step in range(40):
        past = dev.read("past").astype(np.int64)
        fresh = rng.integers(0, 8, n) if step == 0 else rng.integers(0, 5, n)
        ends = np.flatnonzero((past > 60) | ((rng.random(n) < 0.08) & (past > 0)))
        if len(ends):  # requests that ended: others take their places
            past[ends], again[ends] = 0, False
            dev.bufs["past"].upload(np.concatenate((past, np.full(4, 77))).astype(np.int32))
            for b in ends:
                request[b] = 100 * step + int(b)
        new = np.where(again, new, fresh)
        dev.bufs["n_new"].upload(np.concatenate((new, np.full(4, 77))).astype(np.int32))
        data = {m: rng.standard_normal((T, h, D)).astype(np.float32) for m, h in (("q", Hq), ("k", Hk), ("v", Hk))}
        logits = (3 * rng.standard_normal((T, V))).astype(np.float32)
        draft = (logits + 0.3 * rng.standard_normal((T, V))).astype(np.float32)
        tokens = np.concatenate(([0], np.argmax(draft[:-1] + rng.gumbel(size=(T - 1, V)), -1)))
        heat = np.where(np.arange(n) == 2, 0.0, 1.0).astype(np.float32)
        accept, pick = rng.random(T).astype(np.float32), rng.random(n).astype(np.float32)
        for m, y in {**data, "logits": logits, "draft": draft, "accept": accept, "pick": pick, "heat": heat}.items():
            x[m].upload(y)
        d_tokens.upload(tokens.astype(np.int32))
        before = c.read().codes.copy(), c.scales.copy()
        graph.launch()
        stream.synchronize()
        want = host.step(past, new, T)
        count, after = d_count.download(np.int32, n), dev.read("past").copy()
        dev.check(host, {k: y for k, y in want.items() if own_past or k != "kv_len"})
        ready = want["missing"] == 0
        # what the sequences that are ready attend to was written for them, in this step or one before
        for t, slot in enumerate(want["slots"]):
            b = int(np.searchsorted(want["q_start"], t, side="right")) - 1
            if slot >= 0:
                written[divmod(int(slot), page)] = (request[b], int(want["positions"][t]))
        for b in np.flatnonzero(ready):
            for p in range(int(want["kv_len"][b])):
                assert written.get((int(host.table[b, p // page]), p % page)) == (request[b], p), (step, b, p)
        c.new, c.kv, c.starts, c.tokens, c.table = list(new), list(want["kv_len"]), want["q_start"], T, host.table
        c.codes, c.scales = before
        append.plain_append(c, data["k"], data["v"])
        codes, scales = c.codes, c.scales
        c.read()
        assert append.same(c.scales, scales) and append.same_codes(c, codes), step
        got = x["out"].download(np.float32, T * Hq * D).reshape(T, Hq, D).astype(np.float64)
        out, spread, score, live = ref.attention(c, data["q"].astype(np.float64), float(np.float32(D ** -0.5)), 1, 0)
        bound = (2 * (D + 5) * score + 2 * max(max(c.kv), 1) + 40) * attention.U * spread + max(c.kv) * 2.0 ** -39 * 448 * np.nanmax(c.scales)
        assert np.all(np.abs(got - out)[live] <= bound[live]), step
        toks, lps, counts = held_back(verify.expect(want["q_start"], logits.astype(np.float64), draft.astype(np.float64), tokens, heat, accept, pick, V),
                                      want["q_start"], want["missing"])
        end = int(want["q_start"][-1])
        assert np.array_equal(d_out.download(np.int32, T)[:end], toks[:end]) and np.array_equal(count, counts)
        assert np.array_equal(after, np.where(ready, past + counts, past)), step
        short += int((~ready).sum())
        partly += int((~ready & (past % page > 0)).sum())
        served += int((again & ready).sum())
        again = ~ready
    assert short > 5 and partly > 3 and served > 3  # (it did run short, also inside a page, and requests were served later)
    graph.close()
