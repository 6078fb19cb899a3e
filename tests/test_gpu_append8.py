"""Heads finished into a paged cache of 8-bit codes (tqhip_kv_append8_dev).

Without norm, bias and rotation every number is exactly that of the rules in fp32: scale = max(largest / top, 2^-60), code = x / scale rounded to
nearest even, code * (old / new) rounded again where a block's scale grows. Those tests ask for the same bits.
With them, a finished element is off by 20 u of the size of its terms (test_gpu_batch.py), so a scale by as much of the largest size in its
block / top, and one rounding; an element then lies within half a step of its code's type, times the scale that was stored: 1/2 (i8), 2^-4 of
itself or 2^-10 (e4m3); the division rounds once more, u of itself."""
import numpy as np
import pytest

import batch_ref as ref
import test_gpu_batch as base
from batch8_ref import E4M3, I8, LEAST, TOP, Batch8, from_codes, to_codes
from batch_ref import Dev, ints

pytestmark = pytest.mark.gpu

F32, F16, BF16 = 0, 1, 2
U = 2.0 ** -24


def plain_append(b, k, v):
    """The rules on b.codes and b.scales (in place), from float32 rows by token."""
    at = b.token_positions()
    by_block = {}
    for t, (s, pos) in at.items():
        pl = b.place(s, pos)
        if pos >= 0 and pl:
            by_block.setdefault((pl[0], pl[1] // b.block), []).append((pl[1], t))
    for (page, blk), rows in by_block.items():
        first = min(r for r, _ in rows)
        for h in range(b.Hk):
            for i, x in enumerate((k, v)):
                new = np.stack([x[t, h] for _, t in rows])
                top = np.float32(np.abs(new).max())
                scale = np.maximum(top / np.float32(TOP[b.dtype]), LEAST)
                old = b.scales[page, h, blk, i]
                if first > blk * b.block and not old <= scale:
                    scale = old
                if not top < np.inf:
                    scale = np.float32(np.nan)
                if first > blk * b.block and scale != old and scale < np.inf:
                    at_rows = b.codes[i, page, blk * b.block:first, h]
                    at_rows[:] = to_codes(from_codes(at_rows, b.dtype).astype(np.float32) * (old / scale), b.dtype)
                for (r, _), y in zip(rows, new):
                    b.codes[i, page, r, h] = to_codes(y / scale, b.dtype) if scale < np.inf else 0
                b.scales[page, h, blk, i] = scale


def call(gpu, b, s, Hq, act, rotary=0, q_out=None, **kw):
    p = base.proj_of(gpu, s, b.tokens, Hq, b.Hk, b.D, act, rotary, q_out, **kw)
    if q_out is None:
        p.q = None
    gpu.kv_append8_dev(p, b.c, b.s)
    gpu.synchronize()


def same(got, want):
    return np.array_equal(np.ascontiguousarray(got).view(np.uint8), np.ascontiguousarray(want).view(np.uint8)) or \
        (got.dtype == np.float32 and np.array_equal(got, want, equal_nan=True))


def same_codes(b, want):
    """The same codes; zeros of either sign are the same number (a bias of 0 makes +0 of -0)."""
    got = b.codes
    zeros = (got & 0x7f == 0) & (want & 0x7f == 0) & (b.dtype == E4M3)
    return bool(np.all((got == want) | zeros))


# Pages and blocks (rows of a block in a wave's registers, in a workgroup's, read twice; odd ones), heads, layouts.
FORMS = [(16, 16, 2, 64, "token"), (48, 24, 2, 64, "head"), (64, 64, 1, 128, "token"), (128, 128, 1, 256, "token"), (200, 200, 1, 64, "head"), (300, 300, 1, 128, "token"),
         (7, 7, 3, 128, "token"), (6, 1, 2, 64, "token"), (30, 10, 8, 128, "head"), (20, 5, 1, 256, "token"),
         (12, 1, 5, 128, "head"), (12, 2, 3, 64, "token"), (9, 3, 9, 64, "head"), (8, 4, 4, 128, "token"), (5, 1, 8, 256, "token")]  # (several heads a wave)


@pytest.mark.parametrize("dtype", [I8, E4M3])
@pytest.mark.parametrize("act", [F32, F16, BF16])
@pytest.mark.parametrize("page,block,Hk,D,layout", FORMS)
def test_codes_and_scales_to_the_bit(gpu, page, block, Hk, D, layout, act, dtype):
    """Sequences with many, one and no new tokens, one with more tokens than positions, missing pages, tokens outside; rows and
    blocks that are not the call's stay as they were, whatever they hold."""
    new, kv = [5, 1, 0, 40, 3, 1, 350], [5, 100, 33, 90, 2, 2 * page + 1, 600]
    b = Batch8(gpu, new, kv, page, Hk, D, dtype, block, seed=page + D, tail=2, lead=1, bad=[(3, 80 // page)], layout=layout)
    s = base.head_inputs(gpu, b.rng, b.tokens, 2, Hk, D, act, False, False)
    k, v = (s[n][2].astype(np.float32) for n in "kv")
    call(gpu, b, s, 2, act)
    want_codes, want_scales = b.codes.copy(), b.scales.copy()
    b.codes, b.scales = want_codes, want_scales
    plain_append(b, k, v)
    want_codes, want_scales = b.codes, b.scales
    b.read()
    assert same(b.scales, want_scales)
    assert same_codes(b, want_codes), np.argwhere(b.codes != want_codes)[:5]


@pytest.mark.parametrize("dtype", [I8, E4M3])
@pytest.mark.parametrize("page,block,D", [(16, 16, 64), (32, 8, 128), (150, 150, 64), (24, 12, 256), (12, 3, 64), (16, 4, 128)])
def test_token_by_token(gpu, page, block, D, dtype):
    """Tokens of growing, shrinking and zero size, one or a few at a time: a block's scale only grows until it is begun anew, after lengths
    have gone back (refused drafts) too."""
    rng = np.random.default_rng(page)
    b = Batch8(gpu, [3, 3], [3 * page, 3 * page], page, 2, D, dtype, block, seed=1)
    b.scales[:] = np.nan
    b.codes[:] = 0x7f
    b.put()
    length = [0, 0]
    sizes = [0.0, 1.0, 1e-30, 3.0, 0.5, 7.0, 1e4, 2.0, 1e-3]
    for step in range(40):
        new = [int(rng.integers(0, 4)), int(rng.integers(1, 4))]
        length = [max(0, n - int(rng.integers(0, 3))) if step % 7 == 6 else n for n in length]
        if step == 30:
            length = [0, page - 1]
        length = [min(n + m, 3 * page) for n, m in zip(length, new)]
        b.new, b.kv = new, length
        b.starts = np.concatenate(([0], np.cumsum(new))).astype(np.int64)
        b.tokens = int(b.starts[-1])
        b.d_start, b.d_kv = ints(gpu, b.starts), ints(gpu, length)
        b.s = gpu.Seqs(n_seqs=2, n_tokens=b.tokens, q_start=b.d_start.ptr, kv_len=b.d_kv.ptr, block_table=b.d_table.ptr, table_stride=b.stride)
        s = {}
        for n, h in (("q", 1), ("k", 2), ("v", 2)):
            x = Dev(gpu, rng.standard_normal((b.tokens, h, D)) * sizes[step % len(sizes)], F32)
            s[n], s["keep_" + n], s[n + "_bias"], s[n + "_norm"] = (x.ptr, 0, x.values), x, (None, None), (None, None)
        call(gpu, b, s, 1, F32)
        plain_append(b, *(s[n][2].astype(np.float32) for n in "kv"))
        codes, scales = b.codes, b.scales
        b.read()
        assert same(b.scales, scales), step
        assert same_codes(b, codes), step


@pytest.mark.parametrize("dtype", [I8, E4M3])
@pytest.mark.parametrize("act", [F32, F16, BF16])
@pytest.mark.parametrize("Hq,Hk,D,page,block,rotary,packed", [(14, 2, 64, 48, 24, 64, True), (8, 2, 128, 16, 16, 128, False), (2, 1, 256, 64, 64, 64, False),
                                                              (3, 1, 64, 40, 40, 6, False), (2, 2, 128, 512, 512, 128, False), (2, 1, 256, 6, 3, 0, True), (6, 3, 64, 8, 2, 64, True),
                                                              (5, 5, 128, 8, 1, 64, False)])
def test_finished_heads(gpu, Hq, Hk, D, page, block, rotary, packed, act, dtype):
    new, kv = [5, 1, 0, 40, 3, 1], [5, 100, 33, 90, 2, 2 * page + 1]
    b = Batch8(gpu, new, kv, page, Hk, D, dtype, block, seed=3, tail=2, lead=1)
    s = base.head_inputs(gpu, b.rng, b.tokens, Hq, Hk, D, act, True, True, packed)
    q_out = Dev(gpu, np.full((b.tokens, Hq, D), 7.0), act)
    call(gpu, b, s, Hq, act, rotary, q_out)
    at = b.token_positions()
    pos = np.array([at.get(t, (0, 0))[1] for t in range(b.tokens)])
    want_q, size_q = ref.finish_heads(s["q"][2], s["q_bias"][0], s["q_norm"][0], pos, rotary, 1e-6, 1e6)
    rows = (ref.finish_heads(s["k"][2], s["k_bias"][0], s["k_norm"][0], pos, rotary, 1e-6, 1e6), ref.finish_heads(s["v"][2], s["v_bias"][0], None, pos, 0, 0, 1))
    got_q = q_out.read()
    live = [t for t in at if at[t][1] >= 0]
    dead = [t for t in range(b.tokens) if t not in live]
    base.check_heads(got_q[live], want_q[live], size_q[live], act, "q")
    assert dead and np.all(got_q[dead] == 7.0)
    old_scales = b.scales.copy()
    b.read()
    blocks = {}
    for t in live:
        page_, row = b.place(*at[t])
        blocks.setdefault((page_, row // block), []).append((row, t))
    for (pg, blk), tokens in blocks.items():
        first = min(r for r, _ in tokens)
        for i, (want, size) in enumerate(rows):
            for h in range(Hk):
                scale = float(b.scales[pg, h, blk, i])
                w, z = np.stack([want[t, h] for _, t in tokens]), np.stack([size[t, h] for _, t in tokens])
                top = np.abs(w).max() / TOP[dtype]
                slack = 20 * U * z.max() / TOP[dtype] + 2 * U * top
                kept = float(old_scales[pg, h, blk, i]) if first > blk * block else 0.0
                assert abs(scale - max(top, kept)) <= slack, (pg, blk, h, i, scale, top, kept)
                got = from_codes(np.stack([b.codes[i, pg, r, h] for r, _ in tokens]), dtype) * scale
                half = 0.5 * scale if dtype == I8 else np.maximum(2.0 ** -4 * np.abs(w), 2.0 ** -10 * scale)
                assert np.all(np.abs(got - w) <= half * (1 + 2.0 ** -10) + 20 * U * z + 2 * U * np.abs(w) + slack * TOP[dtype]), (pg, blk, h, i)


@pytest.mark.parametrize("dtype", [I8, E4M3])
@pytest.mark.parametrize("block", [1, 4, 8, 64])
def test_infinities_and_nan(gpu, block, dtype):
    """Such an element makes its block and head NaN, K or V alone, until the block is begun anew; other blocks and heads do not notice."""
    page = 64
    b = Batch8(gpu, [30, 1], [30, 70], page, 2, 64, dtype, block, seed=7)
    s = base.head_inputs(gpu, b.rng, b.tokens, 1, 2, 64, F32, False, False)
    k, v = s["k"][2], s["v"][2]
    k[3, 1, 5], v[20, 0, 63], v[30, 1, 0] = np.nan, -np.inf, np.inf
    for n, x in (("k", k), ("v", v)):
        s["keep_" + n].buf.upload(x.astype(np.float32))
    call(gpu, b, s, 1, F32)
    plain_append(b, k.astype(np.float32), v.astype(np.float32))
    codes, scales = b.codes, b.scales
    b.read()
    assert same(b.scales, scales) and same_codes(b, codes)
    assert np.isnan(b.scales).sum() == np.isnan(scales).sum() >= 3
    # one more row: still NaN; from the block's first row on: numbers again
    pg, r = b.place(0, 3)
    for kv, nan in (([31, 70], True), ([5, 70], False)):
        n = 1 if nan else 5
        b.new, b.kv = [n, 0], kv
        b.starts = np.array([0, n, n])
        b.tokens = n
        b.d_start, b.d_kv = ints(gpu, b.starts), ints(gpu, kv)
        b.s = gpu.Seqs(n_seqs=2, n_tokens=n, q_start=b.d_start.ptr, kv_len=b.d_kv.ptr, block_table=b.d_table.ptr, table_stride=b.stride)
        t = base.head_inputs(gpu, b.rng, n, 1, 2, 64, F32, False, False)
        call(gpu, b, t, 1, F32)
        b.read()
        if block == 64 or not nan:
            assert np.isnan(b.scales[pg, 1, r // block, 0]) == nan


def test_the_largest_and_smallest_numbers(gpu):
    """Blocks of fp32's largest, smallest and no numbers: the scale's floor, nothing overflows."""
    b = Batch8(gpu, [4], [4], 4, 1, 64, I8, 1, seed=9)
    x = Dev(gpu, np.stack([np.full(64, 3.4e38), np.full(64, 1e-45), np.zeros(64), np.full(64, 2.0 ** -60)])[:, None], F32)
    s = {n: (x.ptr, 0, x.values) for n in "qkv"} | {n + e: (None, None) for n in "qkv" for e in ("_bias", "_norm")}
    call(gpu, b, s, 1, F32)
    plain_append(b, x.values.astype(np.float32), x.values.astype(np.float32))
    codes, scales = b.codes, b.scales
    b.read()
    assert same(b.scales, scales) and same_codes(b, codes)
    assert np.all(b.codes[0, b.place(0, 0)[0]][0] == 127) and np.all(b.scales[b.place(0, 0)[0]][0, 1:3] == LEAST)


def test_unaligned_heads_and_given_positions(gpu):
    """Rows of an odd number of elements, angles of the caller's positions and frequencies, keys without norm."""
    T, D = 9, 128
    b = Batch8(gpu, [T], [T + 3], 4, 1, D, I8, 2, seed=11)
    inv = (1e4 ** (-np.arange(20) / 20)).astype(np.float32)
    d_inv, pos = base.f32_buffer(gpu, inv), np.array([100000, 5, 0, 7, 7, 90, 3, 2, 1])
    d_pos = ints(gpu, pos)
    x = Dev(gpu, b.rng.standard_normal((T, D + 1)), F32)
    flat = np.concatenate([x.values.reshape(-1), [0.0]])
    k = np.stack([flat[1 + t * (D + 1):][:D] for t in range(T)])[:, None]
    room = Dev(gpu, flat, F32)
    gpu.kv_append8_dev(gpu.HeadProj(dtype=F32, n_tokens=T, n_kv_heads=1, head_dim=D, rotary_dim=40, k=room.ptr + 4, v=room.ptr, k_stride=D + 1,
                                    v_stride=D + 1, inv_freq=d_inv.ptr, positions=d_pos.ptr), b.c, b.s)
    gpu.synchronize()
    b.read()
    want, size = ref.finish_heads(k, None, None, pos, 40, 0, 0, inv)
    for t, at in b.token_positions().items():
        pg, r = b.place(*at)
        scale = float(b.scales[pg, 0, r // 2, 0])
        assert np.all(np.abs(b.k.values[pg, r] - want[t]) <= 0.5 * scale * (1 + 2.0 ** -10) + 20 * U * size[t].max() * 2), t
        assert np.all(np.abs(b.v.values[pg, r, 0] - x.values[t, :D]) <= 0.5 * float(b.scales[pg, 0, r // 2, 1]) * (1 + 2.0 ** -10))


def test_many_sequences(gpu):
    """More sequences than two rounds of the search cover, most without tokens."""
    rng = np.random.default_rng(32)
    B = 5000
    new = (rng.random(B) < 0.03).astype(int)
    new[[0, 63, 64, 4095, 4096, 4999]] = [2, 1, 3, 1, 17, 1]
    kv = np.where(new > 0, rng.integers(0, 12, B) + new, 0)
    b = Batch8(gpu, new, kv, 4, 1, 64, I8, 4, seed=33, tail=1)
    s = base.head_inputs(gpu, b.rng, b.tokens, 1, 1, 64, F32, False, False)
    call(gpu, b, s, 1, F32)
    plain_append(b, *(s[n][2].astype(np.float32) for n in "kv"))
    codes, scales = b.codes, b.scales
    b.read()
    assert same(b.scales, scales) and same_codes(b, codes)


def test_rows_past_4_gib(gpu):
    """Pages more than 2^32 bytes apart in one allocation: appended to, attended to."""
    D, page, far = 64, 16, (1 << 32) + 4096
    room = gpu.DeviceBuffer(far + 4 * page * D)
    scales = base.f32_buffer(gpu, np.full(4, np.nan))
    start, kv, table = ints(gpu, [0, 20]), ints(gpu, [20]), ints(gpu, [[1, 0]])
    cache = gpu.KvCache8(k=room.ptr, v=room.ptr + 2 * page * D, scales=scales.ptr, dtype=I8, n_pages=2, page_size=page, block=page, n_kv_heads=1, head_dim=D,
                         page_stride=far, token_stride=D, head_stride=D)
    seqs = gpu.Seqs(n_seqs=1, n_tokens=20, q_start=start.ptr, kv_len=kv.ptr, block_table=table.ptr, table_stride=2, max_kv=20)
    rng = np.random.default_rng(34)
    s = base.head_inputs(gpu, rng, 20, 2, 1, D, F32, False, False)
    q_out, out = Dev(gpu, np.zeros((20, 2, D)), F32), Dev(gpu, np.zeros((20, 2, D)), F32)
    gpu.kv_append8_dev(base.proj_of(gpu, s, 20, 2, 1, D, F32, 0, q_out), cache, seqs)
    gpu.paged_attention8_dev(gpu.Attn(dtype=F32, n_heads=2, q=q_out.ptr, out=out.ptr, scale=0.125, causal=1), cache, seqs)
    gpu.synchronize()
    held = []
    for n in "kv":
        x = s[n][2][:, 0].astype(np.float32)
        by = np.repeat([np.abs(x[:16]).max(), np.abs(x[16:]).max()], [16, 4]).astype(np.float32) / np.float32(127)
        held.append(np.rint(x / by[:, None]).astype(np.float64) * by[:, None].astype(np.float64))
    for h in range(2):
        w = np.where(np.tri(20) > 0, s["q"][2][:, h] @ held[0].T / 8, -np.inf)
        w = np.exp(w - w.max(-1, keepdims=True))
        want = w / w.sum(-1, keepdims=True) @ held[1]
        assert np.linalg.norm(out.read()[:, h] - want) <= 2.0 ** -17 * np.linalg.norm(want)
