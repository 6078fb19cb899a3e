"""Plain 64-bit forms of the batch calls (tqhip_qk_norm_rope_dev, tqhip_kv_append_dev, tqhip_paged_attention_dev,
tqhip_lora_add_dev) and the device state of a ragged batch, for their tests."""
import numpy as np
import torch

TORCH = {0: torch.float32, 1: torch.float16, 2: torch.bfloat16}
HALF = {0: 2.0 ** -24, 1: 2.0 ** -11, 2: 2.0 ** -8}  # half a step of the type, relative
TINY = {0: 0.0, 1: 2.0 ** -25, 2: 0.0}               # half a step of fp16's subnormals


def raw(x, dtype):
    """A float64 array rounded to the type: its bits as numpy, and its values in float64."""
    t = torch.from_numpy(np.ascontiguousarray(x, np.float64)).to(TORCH[dtype])
    bits = t.numpy() if dtype == 0 else t.view(torch.int16).numpy()
    return bits, t.double().numpy()


def values(bits, dtype):
    if dtype == 0:
        return bits.astype(np.float64)
    return torch.from_numpy(bits.view(np.int16)).view(TORCH[dtype]).double().numpy()


def bits_dtype(dtype):
    return np.float32 if dtype == 0 else np.int16


class Dev:
    """A device array of one of the three types made from float64 values."""

    def __init__(self, tq, x, dtype):
        self.tq, self.dtype, self.shape = tq, dtype, np.shape(x)
        bits, self.values = raw(x, dtype)
        self.buf = tq.DeviceBuffer.from_array(bits)
        self.ptr = self.buf.ptr

    def read(self):
        n = int(np.prod(self.shape))
        return values(self.buf.download(bits_dtype(self.dtype), n), self.dtype).reshape(self.shape)

    def read_bits(self):
        return self.buf.download(np.int32 if self.dtype == 0 else np.int16, int(np.prod(self.shape))).reshape(self.shape)


def ints(tq, x):
    return tq.DeviceBuffer.from_array(np.asarray(x, np.int32))


def finish_heads(x, bias, norm, positions, rotary, eps, theta, inv_freq=None):
    """(tokens, heads, D) float64 -> (result, size): size bounds the terms that each result is made of."""
    T, H, D = x.shape
    size = np.abs(x)
    if bias is not None:
        b = np.asarray(bias, np.float64).reshape(H, D)
        x, size = x + b, size + np.abs(b)
    if norm is not None:
        r = 1.0 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
        x, size = x * r * norm, size * r * np.abs(norm)
    half = rotary // 2
    if half:
        f = theta ** (-2.0 * np.arange(half) / rotary) if inv_freq is None else np.asarray(inv_freq, np.float64)
        ang = np.asarray(positions, np.float64)[:, None, None] * f
        c, s = np.cos(ang), np.sin(ang)
        x0, x1 = x[..., :half].copy(), x[..., half:rotary].copy()
        x = x.copy()
        x[..., :half], x[..., half:rotary] = x0 * c - x1 * s, x1 * c + x0 * s
        t = size[..., :half] + size[..., half:rotary]
        size = size.copy()
        size[..., :half] = size[..., half:rotary] = t
    return x, size


class Batch:
    """A ragged batch over a paged cache: `new` tokens and `kv` positions of each sequence, shuffled pages. `tail` tokens
    follow the last sequence, `lead` come before the first; pages in `bad` (pairs sequence, page index) are missing. Cache rows
    that no position of a sequence uses hold NaN. `layout`: "token" ([page][row][head][dim]) or "head" ([page][head][row][dim])."""

    def __init__(self, tq, new, kv, page, Hk, D, cache, seed=0, tail=0, lead=0, bad=(), layout="token", spare=2, fill=None):
        self.tq, self.new, self.kv, self.page, self.Hk, self.D, self.cache = tq, list(new), list(kv), page, Hk, D, cache
        rng = self.rng = np.random.default_rng(seed)
        self.starts = lead + np.concatenate(([0], np.cumsum(new))).astype(np.int64)
        self.tokens = int(self.starts[-1]) + tail
        per = [-(-n // page) for n in kv]
        self.n_pages = sum(per) + spare
        order = rng.permutation(self.n_pages)
        self.stride = max(1, max(per)) + 1
        self.table = np.full((len(new), self.stride), -1, np.int64)
        at = 0
        for i, n in enumerate(per):
            self.table[i, :n] = order[at:at + n]
            at += n
        for b, i in bad:
            self.table[b, i] = -1 if (b + i) % 2 else self.n_pages + 5
        self.layout = layout
        shape = (self.n_pages, page, Hk, D)
        k, v = np.full(shape, np.nan), np.full(shape, np.nan)
        for b, n in enumerate(kv):
            for p in range(n):
                pg = self.table[b, p // page]
                if 0 <= pg < self.n_pages:
                    k[pg, p % page] = rng.standard_normal((Hk, D)) if fill is None else fill
                    v[pg, p % page] = rng.standard_normal((Hk, D)) if fill is None else fill
        if layout == "head":
            k, v = k.transpose(0, 2, 1, 3), v.transpose(0, 2, 1, 3)
        self.k, self.v = Dev(tq, k, cache), Dev(tq, v, cache)
        self.d_start, self.d_kv, self.d_table = ints(tq, self.starts), ints(tq, self.kv), ints(tq, self.table)
        strides = dict(page_stride=page * Hk * D, token_stride=D, head_stride=page * D) if layout == "head" else {}
        self.c = tq.KvCache(k=self.k.ptr, v=self.v.ptr, dtype=cache, n_pages=self.n_pages, page_size=page, n_kv_heads=Hk, head_dim=D, **strides)
        self.s = tq.Seqs(n_seqs=len(new), n_tokens=self.tokens, q_start=self.d_start.ptr, kv_len=self.d_kv.ptr, block_table=self.d_table.ptr,
                         table_stride=self.stride, max_kv=max(kv))

    def rows(self, x):
        """A cache array as [page][row][head][dim]."""
        return x.transpose(0, 2, 1, 3) if self.layout == "head" else x

    def place(self, b, p):
        pg = self.table[b, p // self.page] if 0 <= p < self.stride * self.page else -1
        return (int(pg), p % self.page) if 0 <= pg < self.n_pages else None

    def token_positions(self):
        """(sequence, position) of every token of a sequence, by token."""
        out = {}
        for b in range(len(self.new)):
            n = self.new[b]
            for i in range(n):
                out[int(self.starts[b]) + i] = (b, self.kv[b] - n + i)
        return out


def attention(batch, q, scale, causal, window):
    """q (tokens, Hq, D) float64. -> (out, spread, score, places): spread = sum p |v|, score = the largest sum |q k| scale of a
    row (bounds of the rounding errors), rows of tokens that are in a sequence."""
    T, Hq, D = q.shape
    G = Hq // batch.Hk
    k, v = batch.rows(batch.k.values), batch.rows(batch.v.values)
    out, spread, score = np.zeros_like(q), np.zeros_like(q), np.zeros((T, Hq, 1))
    at = batch.token_positions()
    for t, (b, pos) in at.items():
        lo, hi = 0, batch.kv[b]
        if causal:
            hi = min(hi, pos + 1)
            lo = max(0, pos + 1 - window) if window else 0
        places = [pl for pl in (batch.place(b, p) for p in range(lo, hi)) if pl]
        if not places:
            continue
        pg, r = np.array(places).T
        for g in range(batch.Hk):
            kk, vv = k[pg, r, g], v[pg, r, g]
            qq = q[t, g * G:(g + 1) * G]
            s = qq @ kk.T * scale
            p = np.exp(s - s.max(-1, keepdims=True))
            p /= p.sum(-1, keepdims=True)
            out[t, g * G:(g + 1) * G] = p @ vv
            spread[t, g * G:(g + 1) * G] = p @ np.abs(vv)
            score[t, g * G:(g + 1) * G, 0] = (np.abs(qq) @ np.abs(kk).T * abs(scale)).max(-1)
    return out, spread, score, np.array(sorted(at), np.int64)


def lora(x, base, a, b, scale, starts, adapter, tokens):
    """-> (y, size): size bounds the terms of each result. Rows of tokens in no sequence are the base's."""
    y = np.zeros((tokens, b.shape[1])) if base is None else base.copy()
    size = np.abs(y)
    for i, ad in enumerate(adapter):
        if 0 <= ad < a.shape[0]:
            at = slice(int(starts[i]), int(starts[i + 1]))
            y[at] += scale[ad] * ((x[at] @ a[ad].T) @ b[ad].T)
            size[at] += abs(scale[ad]) * ((np.abs(x[at]) @ np.abs(a[ad]).T) @ np.abs(b[ad]).T)
    return y, size
