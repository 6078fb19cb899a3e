"""Block tables, free pages, positions and slots from the lengths of requests (tqhip_page_map_dev), against the rules written out one
page at a time. Everything is whole numbers, so everything is equal."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


class Server:
    """Pages of some sequences, kept by hand."""

    def __init__(self, n_seqs, stride, n_pages, page, seed=0):
        self.page, self.stride = page, stride
        self.table = np.full((n_seqs, stride), -1, np.int64)
        self.held = np.zeros(n_seqs, np.int64)
        self.free = np.random.default_rng(seed).permutation(n_pages).astype(np.int64)
        self.n_free = n_pages

    def copy(self):
        other = object.__new__(Server)
        other.__dict__ = {k: v.copy() if isinstance(v, np.ndarray) else v for k, v in self.__dict__.items()}
        return other

    def step(self, past, new, n_tokens):
        kv = np.asarray(past, np.int64) + new
        need = -(-kv // self.page)
        for b in range(len(kv)):
            for j in range(need[b], self.held[b]):
                self.free[self.n_free] = self.table[b, j]
                self.n_free += 1
                self.table[b, j] = -1
            self.held[b] = min(self.held[b], need[b])
        missing, dry = np.zeros(len(kv), np.int64), False
        for b in range(len(kv)):
            want = need[b] - self.held[b]
            if need[b] > self.stride:
                missing[b] = want
                continue
            dry = dry or want > self.n_free
            if dry:
                missing[b] = want
                continue
            for j in range(self.held[b], need[b]):
                self.n_free -= 1
                self.table[b, j] = self.free[self.n_free]
            self.held[b] = need[b]
        start = np.concatenate(([0], np.cumsum(new)))
        pos, slot = np.full(n_tokens, -1, np.int64), np.full(n_tokens, -1, np.int64)
        for b in range(len(kv)):
            at = np.arange(start[b], start[b + 1])
            p = kv[b] - (start[b + 1] - at)
            pos[at] = p
            pg = np.where(p // self.page < self.stride, self.table[b, np.minimum(p // self.page, self.stride - 1)], -1)
            slot[at] = np.where(pg >= 0, pg * self.page + p % self.page, -1)
        return dict(q_start=start, kv_len=kv, missing=missing, positions=pos, slots=slot)


class Device:
    """The same state on the GPU, with guard words after every array."""

    def __init__(self, gpu, host, n_pages, n_tokens):
        self.gpu, self.n_pages, self.n_tokens = gpu, n_pages, n_tokens
        n = len(host.held)
        free = np.full(n_pages, -7)
        free[:host.n_free] = host.free[:host.n_free]
        self.bufs = {"block_table": host.table, "n_held": host.held, "free_pages": free, "n_free": [host.n_free], "q_start": np.full(n + 1, -9),
                     "kv_len": np.full(n, -9), "missing": np.full(n, -9), "positions": np.full(n_tokens, -9), "slots": np.full(n_tokens, -9),
                     "past": np.zeros(n), "n_new": np.zeros(n)}
        self.size = {k: np.size(v) for k, v in self.bufs.items()}
        self.bufs = {k: gpu.DeviceBuffer.from_array(np.concatenate((np.asarray(v, np.int32).reshape(-1), np.full(4, 77, np.int32)))) for k, v in self.bufs.items()}
        self.map = gpu.PageMap(n_seqs=n, n_tokens=n_tokens, n_pages=n_pages, page_size=host.page, table_stride=host.stride,
                               **{k: b.ptr for k, b in self.bufs.items()})

    def lengths(self, past, new):
        for name, x in (("past", past), ("n_new", new)):
            self.bufs[name].upload(np.concatenate((np.asarray(x, np.int32), np.full(4, 77, np.int32))))

    def read(self, name):
        x = self.bufs[name].download(np.int32, self.size[name] + 4)
        assert np.all(x[-4:] == 77), name
        return x[:-4]

    def check(self, host, want):
        for name, x in want.items():
            assert np.array_equal(self.read(name), x), name
        assert self.read("n_free")[0] == host.n_free
        assert np.array_equal(self.read("n_held"), host.held)
        assert np.array_equal(self.read("block_table").reshape(host.table.shape), host.table)
        assert np.array_equal(self.read("free_pages")[:host.n_free], host.free[:host.n_free])
        pages = np.concatenate((host.table[host.table >= 0], host.free[:host.n_free]))
        assert len(set(pages.tolist())) == len(pages) == self.n_pages  # none lost, none twice


def steps(gpu, n_seqs, stride, n_pages, page, lengths, n_tokens, seed=0):
    host = Server(n_seqs, stride, n_pages, page, seed)
    dev = Device(gpu, host, n_pages, n_tokens)
    for past, new in lengths:
        dev.lengths(past, new)
        gpu.page_map_dev(dev.map)
        gpu.lib().tqhip_synchronize()
        dev.check(host, host.step(past, new, n_tokens))
    return host, dev


@pytest.mark.parametrize("page", [1, 7, 16, 64])
@pytest.mark.parametrize("n_seqs", [1, 3, 64, 65, 300, 1025, 4096])
def test_a_server_s_life(gpu, n_seqs, page):
    """Prompts, decode steps, refused drafts, ended and new requests; what the pages do not suffice for."""
    rng = np.random.default_rng(n_seqs * 100 + page)
    stride, most = 12, 11 * page
    n_pages = max(4, n_seqs * 5)
    host = Server(n_seqs, stride, n_pages, page)
    n_tokens = n_seqs * (3 * page + 8) + 3
    dev = Device(gpu, host, n_pages, n_tokens)
    past = np.zeros(n_seqs, np.int64)
    for step in range(12):
        kind = rng.integers(0, 6, n_seqs) if step else np.full(n_seqs, 0)
        new = np.select([kind == 0, kind <= 2, kind == 3], [rng.integers(0, 3 * page + 1, n_seqs), 1, 5], 0)
        past = np.where(kind == 5, 0, np.where(kind == 4, np.maximum(past - rng.integers(0, 6, n_seqs), 0), past))
        new = np.minimum(new, np.maximum(most - past, 0))
        dev.lengths(past, new)
        gpu.page_map_dev(dev.map)
        gpu.lib().tqhip_synchronize()
        want = host.step(past, new, n_tokens)
        dev.check(host, want)
        past = np.where(want["missing"] == 0, past + new, np.minimum(past, host.held * page))


@pytest.mark.parametrize("n_tokens", [0, 1, 4095, 4096, 4097, 9000])
def test_tokens_by_one_launch_or_two(gpu, n_tokens):
    new = np.array([0, n_tokens // 2, 0, n_tokens - n_tokens // 2 - min(n_tokens, 1), 0])
    host, dev = steps(gpu, 5, 700, 2000, 16, [(np.array([5, 0, 33, 16, 0]), new)], max(n_tokens, 1))
    if n_tokens > 1:
        assert dev.read("slots")[n_tokens - 1] == -1 and dev.read("slots")[n_tokens - 2] >= 0


@pytest.mark.parametrize("n_seqs", [1, 7, 40])
def test_long_runs_of_pages(gpu, n_seqs):
    """Long prompts come, end, and others come into their pages: hundreds of pages of a sequence, given and taken."""
    rng = np.random.default_rng(n_seqs)
    lengths = rng.integers(1000, 6000, n_seqs)
    some = np.where(np.arange(n_seqs) % 3 == 0, lengths, 0)
    zero = np.zeros(n_seqs, np.int64)
    steps(gpu, n_seqs, 900, 1000 * n_seqs, 7, [(zero, lengths), (some, lengths - some), (zero, zero), (zero, some), (zero, lengths[::-1]), (zero, zero + 6000)], 6000 * n_seqs)


def test_pages_given_back_serve_the_same_call(gpu):
    host, _ = steps(gpu, 3, 8, 8, 4, [([0, 0, 0], [20, 12, 0]), ([0, 12, 0], [0, 0, 20])], 40)
    assert host.n_free == 0 and host.held.tolist() == [0, 3, 5]


def test_in_order_until_one_does_not_fit(gpu):
    """The second lacks a page, so the fourth gets none although its one is there; the third needs none."""
    host, dev = steps(gpu, 4, 8, 6, 4, [([0, 0, 0, 0], [8, 0, 4, 0]), ([8, 0, 2, 0], [4, 12, 1, 3])], 40)
    assert dev.read("missing").tolist() == [0, 3, 0, 1] and host.held.tolist() == [3, 0, 1, 0] and host.n_free == 2
    assert dev.read("slots")[4:16].tolist() == [-1] * 12


def test_longer_than_the_table(gpu):
    """Such a sequence gets nothing and holds nobody up; its positions that do exist have their slots."""
    host, dev = steps(gpu, 3, 4, 20, 4, [([0, 0, 0], [4, 6, 4]), ([4, 6, 4], [4, 30, 4])], 40)
    assert dev.read("missing").tolist() == [0, 7, 0] and host.held.tolist() == [2, 2, 2]
    assert (dev.read("slots")[4:34] >= 0).sum() == 2


def test_without_positions_and_slots(gpu):
    host = Server(2, 4, 8, 4)
    dev = Device(gpu, host, 8, 6)
    dev.map.positions = dev.map.slots = None
    dev.lengths([0, 0], [5, 1])
    gpu.page_map_dev(dev.map)
    gpu.lib().tqhip_synchronize()
    want = host.step([0, 0], [5, 1], 6)
    want["positions"] = want["slots"] = np.full(6, -9)
    dev.check(host, want)


def test_numbers_that_make_no_sense(gpu):
    """Negative lengths are 0, counts outside their arrays the nearest inside; more tokens than n_tokens end there."""
    host = Server(3, 4, 8, 4)
    dev = Device(gpu, host, 8, 6)
    dev.lengths([-5, 3, 2 ** 31 - 1], [5, -1, 2 ** 31 - 1])
    dev.bufs["n_free"].upload(np.array([10 ** 9] + [77] * 4, np.int32))
    gpu.page_map_dev(dev.map)
    gpu.lib().tqhip_synchronize()
    assert dev.read("q_start").tolist() == [0, 5, 5, 6]
    assert dev.read("kv_len").tolist() == [5, 3, 2 ** 31 - 1]
    assert dev.read("n_held").tolist() == [2, 1, 0] and dev.read("n_free")[0] == 5
    assert dev.read("missing")[2] == 2 ** 29
    assert np.all(dev.read("slots")[:5] >= 0) and dev.read("slots")[5] == -1
    dev.bufs["n_held"].upload(np.array([10 ** 9, -3, 0] + [77] * 4, np.int32))
    dev.bufs["n_free"].upload(np.array([-4] + [77] * 4, np.int32))
    dev.lengths([0, 0, 0], [0, 0, 0])
    gpu.page_map_dev(dev.map)
    gpu.lib().tqhip_synchronize()
    assert dev.read("n_held").tolist() == [0, 0, 0] and dev.read("n_free")[0] == 4


def test_a_captured_step_and_the_next(gpu):
    """One captured call walks a server through steps: it reads the lengths that are there when it runs, kv_len is the next step's past."""
    n, page, stride, n_pages, n_tokens = 70, 4, 9, 700, 400
    host = Server(n, stride, n_pages, page)
    dev = Device(gpu, host, n_pages, n_tokens)
    dev.map.kv_len = dev.map.past
    rng = np.random.default_rng(1)
    past, new = np.zeros(n, np.int64), rng.integers(0, 5, n)
    stream = gpu.Stream()
    dev.lengths(past, np.zeros(n))
    graph = gpu.OpsGraph([gpu.batch_op(gpu.OP_PAGE_MAP, dev.map)], stream)
    for _ in range(6):
        new = rng.integers(0, 6, n)
        dev.lengths(past, new)
        graph.launch()
        stream.synchronize()
        want = host.step(past, new, n_tokens)
        assert np.array_equal(dev.read("past"), want.pop("kv_len"))
        dev.check(host, want)
        past = past + new
    graph.close()
