"""A server's step of page map, append, attention and verification, captured once and replayed without the host knowing a length, against their forms;
and two threads that call on one stream. Tolerances as in the calls' own tests."""
import threading

import numpy as np
import pytest

import batch_ref as ref
import test_gpu_append8 as append
import test_gpu_attention8 as attention
import test_gpu_page_map as pages
import test_gpu_verify as verify
from batch8_ref import E4M3, I8, Batch8
from batch_ref import Dev, ints

pytestmark = pytest.mark.gpu

F32 = 0


class Cache(Batch8):
    """Batch8's forms over arrays that a page map fills."""

    def __init__(self, tq, n_seqs, n_pages, page, block, Hk, D, dtype, stride):
        self.tq, self.page, self.Hk, self.D, self.dtype, self.block, self.layout = tq, page, Hk, D, dtype, block, "token"
        self.n_blocks, self.n_pages, self.stride, self.rng = page // block, n_pages, stride, np.random.default_rng(0)
        self.codes = np.full((2, n_pages, page, Hk, D), 0x7f, np.uint8)
        self.scales = np.full((n_pages, Hk, self.n_blocks, 2), np.nan, np.float32)
        self.put()


@pytest.mark.parametrize("dtype", [I8, E4M3])
def test_captured_steps_of_a_server(gpu, dtype):
    n, page, block, Hq, Hk, D, V, T, stride, n_pages = 5, 8, 4, 4, 2, 64, 300, 40, 12, 33
    rng = np.random.default_rng(dtype)
    host = pages.Server(n, stride, n_pages, page, 1)
    dev = pages.Device(gpu, host, n_pages, T)
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
                       out_tokens=d_out.ptr, n_out=d_count.ptr, logprob=x["logprob"].ptr)
    stream = gpu.Stream()
    graph = gpu.OpsGraph([gpu.batch_op(gpu.OP_PAGE_MAP, dev.map), gpu.batch_op(gpu.OP_KV_APPEND8, proj, c.c, c.s),
                          gpu.batch_op(gpu.OP_PAGED_ATTENTION8, attn, c.c, c.s), gpu.batch_op(gpu.OP_VERIFY_TOKENS, judge)], stream)
    past, accepted = np.zeros(n, np.int64), 0
    for step in range(14):
        new = rng.integers(0, 8, n) if step == 0 else rng.integers(0, 5, n)
        if step % 5 == 4:
            past[step % n] = 0  # a request ended, another takes its place
        dev.lengths(past, new)
        data = {m: rng.standard_normal((T, h, D)).astype(np.float32) for m, h in (("q", Hq), ("k", Hk), ("v", Hk))}
        logits = (3 * rng.standard_normal((T, V))).astype(np.float32)
        draft = (logits + 0.3 * rng.standard_normal((T, V))).astype(np.float32)
        tokens = np.concatenate(([0], np.argmax(draft[:-1] + rng.gumbel(size=(T - 1, V)), -1)))
        heat = np.where(np.arange(n) == 2, 0.0, 1.0).astype(np.float32)
        accept, pick = rng.random(T).astype(np.float32), rng.random(n).astype(np.float32)
        for m, y in {**data, "logits": logits, "draft": draft, "accept": accept, "pick": pick, "heat": heat}.items():
            x[m].upload(y)
        d_tokens.upload(tokens.astype(np.int32))
        x["out"].upload(np.full((T, Hq, D), 7.0, np.float32))
        before = c.read().codes.copy(), c.scales.copy()
        graph.launch()
        stream.synchronize()
        # the page map
        want = host.step(past, new, T)
        count = d_count.download(np.int32, n)
        after = dev.read("past").copy()
        dev.check(host, want)
        # the append, from the state before
        c.new, c.kv, c.starts, c.tokens, c.table = list(new), list(want["kv_len"]), want["q_start"], T, host.table
        c.codes, c.scales = before
        append.plain_append(c, data["k"], data["v"])
        codes, scales = c.codes, c.scales
        c.read()
        assert append.same(c.scales, scales) and append.same_codes(c, codes), step
        # attention over what is there
        got = x["out"].download(np.float32, T * Hq * D).reshape(T, Hq, D).astype(np.float64)
        out, spread, score, live = ref.attention(c, data["q"].astype(np.float64), float(np.float32(D ** -0.5)), 1, 0)
        bound = (2 * (D + 5) * score + 2 * max(max(c.kv), 1) + 40) * attention.U * spread + max(c.kv) * 2.0 ** -39 * 448 * np.nanmax(c.scales)
        assert np.all(np.abs(got - out)[live] <= bound[live]), step
        assert np.all(got[np.setdiff1d(np.arange(T), live)] == 7.0)
        # and the verdict, which shortens the sequences
        toks, lps, counts = verify.expect(want["q_start"], logits.astype(np.float64), draft.astype(np.float64), tokens, heat, accept, pick, V)
        end = int(want["q_start"][-1])
        assert np.array_equal(d_out.download(np.int32, T)[:end], toks[:end]) and np.array_equal(count, counts)
        past = want["kv_len"] - new + counts
        assert np.array_equal(after, past)
        accepted += int(np.maximum(counts - 1, 0).sum())
        past = np.where(want["missing"] > 0, np.minimum(past, host.held * page), past)
    assert accepted > 5
    graph.close()


def test_threads_that_share_a_stream(gpu):
    """Attention in parts and verification take the stream's scratch in turn."""
    stream = gpu.Stream()
    a = Batch8(gpu, [1, 1], [2100, 900], 16, 2, 64, I8, seed=1)
    q = Dev(gpu, a.rng.standard_normal((2, 4, 64)), F32)
    b = verify.Case(gpu, [4, 2, 5], 9001, F32, True, [1.0, 0.0, 0.8], seed=2).put()
    want, spread, score, _ = ref.attention(a, q.values, 0.125, 1, 0)
    outs = [Dev(gpu, np.zeros((2, 4, 64)), F32) for _ in range(40)]
    errors = []

    def attend():
        try:
            for o in outs:
                gpu.paged_attention8_dev(gpu.Attn(dtype=F32, n_heads=4, q=q.ptr, out=o.ptr, scale=0.125, causal=1), a.c, a.s, stream)
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    def judge():
        try:
            for _ in range(40):
                gpu.verify_tokens_dev(b.v, stream)
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=f) for f in (attend, judge, judge)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    stream.synchronize()
    assert not errors
    bound = attention.bound_of(a, F32, want, spread, score)
    assert all(np.all(np.abs(o.read() - want) <= bound) for o in outs)
    b.check()


def test_a_call_under_a_capture_of_the_caller_s_needs_a_workspace(gpu):
    """Scratch of the stream may not be recorded into a graph that the library does not own."""
    torch = pytest.importorskip("torch")
    b = verify.Case(gpu, [3], 500, F32, True, seed=3).put()
    space = torch.empty(gpu.verify_tokens_workspace(b.v) + 256, dtype=torch.uint8, device="cuda")
    graph, codes = torch.cuda.CUDAGraph(), []
    with torch.cuda.graph(graph):
        s = torch.cuda.current_stream().cuda_stream
        codes.append(gpu.lib().tqhip_verify_tokens_dev(b.v, s))
        b.v.workspace, b.v.workspace_bytes = space.data_ptr(), space.numel()
        codes.append(gpu.lib().tqhip_verify_tokens_dev(b.v, s))
    assert codes == [-7, 0]
    for _ in range(3):
        b.bufs["out_tokens"].upload(np.full(b.n, -2, np.int32))
        b.bufs["kv_len"].upload(np.int32([1000]))
        graph.replay()
        torch.cuda.synchronize()
        b.check()
