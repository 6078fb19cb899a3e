"""The operators of a server's step around an 8-bit paged cache, as cases that can be timed and compared.

A case is one of four kinds:

  pages      block tables, page counts, positions and slots of a batch from the lengths of its requests, with a list of free pages
  append     the query, key and value heads of a batch finished, keys and values into pages of 8 bits with a scale for each block of tokens
             and head
  attention  the new tokens of each sequence (one, a few drafted ones, or a chunk) over such pages
  verify     drafted tokens accepted or refused by the target's probabilities, and the token after them drawn, from given random numbers

Head layouts are those of the model sizes that this repository's benchmark and tests use: 14 query and 2 key/value heads of
64, 32 and 8 of 128, 2 and 1 of 256; the vocabulary is its benchmark's. Lengths follow from the case alone, data from the seed.
"""
import importlib.util
import math
import os
import random
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8, "e4m3": torch.float8_e4m3fn}
CODES = {"f32": 0, "f16": 1, "bf16": 2, "i8": 3, "e4m3": 4}
BYTES = {"f32": 4, "f16": 2, "bf16": 2, "i8": 1, "e4m3": 1}
TOP = {"i8": 127.0, "e4m3": 448.0}
LEAST_SCALE = 2.0 ** -60
SMALL = dict(heads=14, kv_heads=2, dim=64)
LARGE = dict(heads=32, kv_heads=8, dim=128)
WIDE = dict(heads=2, kv_heads=1, dim=256)
VOCAB = 151936
EPS = 1e-6
THETA = 1e6


def _package():
    if "tiny_llm_amd" not in sys.modules:
        spec = importlib.util.spec_from_file_location("tiny_llm_amd", os.path.join(ROOT, "tiny-llm_amd", "__init__.py"))
        mod = importlib.util.module_from_spec(spec)
        sys.modules["tiny_llm_amd"] = mod
        spec.loader.exec_module(mod)
    return sys.modules["tiny_llm_amd"]


def listed():
    return [
        # A decode step of 256 requests: one sequence in sixteen needs a page more, some have ended and give theirs back. Latency bound.
        dict(name="pages_decode", kind="pages", seqs=256, new=1, past=4000, page=16, ended=9),
        # 48 prompts come in at once (some 800000 tokens) while other requests end.
        dict(name="pages_prompts", kind="pages", seqs=61, new=26000, past=900, page=16, ended=13),
        # A decode step of 61 requests into e4m3 pages of 16 positions, a scale for each of them: partly filled blocks.
        dict(name="append8_decode", kind="append", seqs=61, new=1, past=4000, act="f32", cache="e4m3", page=16, block=16, norm=True, bias=False,
             rotary=128, **LARGE),
        # Ragged prompts of the 0.5B-sized model (biases, no norms) into int8 pages of 48 positions, scales for 24.
        dict(name="append8_prompts", kind="append", seqs=5, new=3001, past=700, act="f32", cache="i8", page=48, block=24, norm=False, bias=True,
             rotary=64, **SMALL),
        # One decode token of the 0.5B-sized model over 3000 int8 positions: the smallest attention call.
        dict(name="attn8_one_token", kind="attention", seqs=1, new=1, past=3000, act="f32", cache="i8", page=64, block=32, causal=True, window=0, **SMALL),
        # A decode step of 64 requests of ragged lengths: reading the cache is the work.
        dict(name="attn8_decode", kind="attention", seqs=64, new=1, past=16000, act="f32", cache="i8", page=16, block=16, causal=True, window=0, **LARGE),
        # Four drafted tokens and the one before them of 32 requests in bfloat16, e4m3 pages.
        dict(name="attn8_drafts", kind="attention", seqs=32, new=5, past=9000, act="bf16", cache="e4m3", page=32, block=32, causal=True, window=0, **LARGE),
        # Chunks of four prompts that continue over what is cached.
        dict(name="attn8_chunks", kind="attention", seqs=4, new=257, past=8000, act="f32", cache="i8", page=32, block=32, causal=True, window=0, **LARGE),
        # Two long prompts from empty caches, bfloat16 activations over e4m3 pages: the matrix products are the work.
        dict(name="attn8_prompts", kind="attention", seqs=2, new=8192, past=0, act="bf16", cache="e4m3", page=64, block=64, causal=True, window=0, **LARGE),
        # One request's three drafted tokens.
        dict(name="verify_one", kind="verify", seqs=1, drafts=3, vocab=VOCAB, logits="f32", dense=True),
        # Four drafted tokens of 64 requests (some have fewer) with the draft model's logits; one request in eight is greedy.
        dict(name="verify_batch", kind="verify", seqs=64, drafts=4, vocab=VOCAB, logits="f32", dense=True),
        # Drafts looked up in the prompts (no distribution of theirs) of 100 requests, logits in bfloat16.
        dict(name="verify_lookup", kind="verify", seqs=100, drafts=7, vocab=VOCAB, logits="bf16", dense=False),
    ]


def _spread(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(("pages", "append", "append", "attention", "attention", "attention", "verify", "verify"))
    if kind == "pages":
        seqs = _spread(rng, 1, 1000)
        return dict(kind=kind, seqs=seqs, new=rng.choice((1, _spread(rng, 2, max(3, 800000 // seqs)))), past=_spread(rng, 1, 4000),
                    page=rng.choice((16, 32, 64, _spread(rng, 7, 200))), ended=rng.randint(0, seqs // 4))
    if kind == "verify":
        vocab = rng.choice((VOCAB, _spread(rng, 1000, 150000)))
        seqs, drafts = _spread(rng, 1, 100), rng.randint(0, 5)
        return dict(kind=kind, seqs=seqs, drafts=drafts, vocab=vocab, logits=rng.choice(("f32", "f32", "f16", "bf16")), dense=rng.random() < 0.6)
    heads = rng.choice((SMALL, LARGE, WIDE))
    act, cache = rng.choice(("f32", "f16", "bf16")), rng.choice(("i8", "e4m3"))
    block = rng.choice((8, 16, 32, 64, _spread(rng, 1, 100)))
    page = block * rng.choice((1, 1, 2, 3))
    if kind == "append":
        norm = rng.random() < 0.5
        seqs = _spread(rng, 1, 100)
        return dict(kind=kind, seqs=seqs, new=rng.choice((1, _spread(rng, 1, 8000 // seqs))), past=_spread(rng, 1, 4000), act=act, cache=cache,
                    page=page, block=block, norm=norm, bias=not norm, rotary=rng.choice((heads["dim"], heads["dim"], heads["dim"] // 4)), **heads)
    if rng.random() < 0.5:
        seqs = _spread(rng, 1, 64)
        new, past = rng.choice((1, 1, rng.randint(2, 8))), _spread(rng, 10, 12000)
    else:
        seqs = _spread(rng, 1, 8)
        new, past = _spread(rng, 2, 4000 // seqs), _spread(rng, 1, 3000)
    causal = rng.random() < 0.85
    return dict(kind=kind, seqs=seqs, new=new, past=past, act=act, cache=cache, page=page, block=block, causal=causal,
                window=_spread(rng, 30, 2000) if causal and rng.random() < 0.3 else 0, **heads)


def _lengths(case):
    """(new tokens, cached positions before them) of each sequence: the first has the case's own, the others ragged shares of them."""
    rng = random.Random("%d %d %d" % (case["seqs"], case["new"], case["past"]))
    new, past = [case["new"]], [case["past"]]
    for _ in range(case["seqs"] - 1):
        new.append(case["new"] if case["new"] <= 8 else rng.randint(case["new"] // 3 + 1, case["new"]))
        past.append(rng.randint(case["past"] // 20, case["past"]))
    return new, past


def _ended(case):
    """Lengths of a page-map case: (new, past, pages held before). The last `ended` sequences have ended: nothing stays and nothing comes."""
    new, past = _lengths(case)
    held = [-(-p // case["page"]) for p in past]
    for i in range(case["seqs"] - case["ended"], case["seqs"]):
        new[i] = past[i] = 0
    return new, past, held


def _drafts(case):
    """Tokens of each sequence: the one before the drafts and its drafts, one sequence in four with fewer."""
    rng = random.Random("%d %d" % (case["seqs"], case["drafts"]))
    return [1 + case["drafts"]] + [1 + (rng.randint(0, case["drafts"]) if rng.random() < 0.25 else case["drafts"]) for _ in range(case["seqs"] - 1)]


def work(case):
    if case["kind"] == "pages":
        new, past, held = _ended(case)
        need = [-(-(n + p) // case["page"]) for n, p in zip(new, past)]
        moved = sum(abs(a - b) for a, b in zip(need, held))
        return dict(bytes=4 * (7 * case["seqs"] + 2 * sum(new) + 2 * moved), flops=8 * sum(new))
    if case["kind"] == "verify":
        rows = _drafts(case)
        read = sum(rows) + (sum(rows) - len(rows) if case["dense"] else 0)
        return dict(bytes=read * case["vocab"] * BYTES[case["logits"]] + 24 * sum(rows), flops=4 * read * case["vocab"])
    Hq, Hk, D, act = case["heads"], case["kv_heads"], case["dim"], BYTES[case["act"]]
    new, past = _lengths(case)
    tokens = sum(new)
    if case["kind"] == "append":
        blocks = sum((p + n - 1) // case["block"] - p // case["block"] + 1 for n, p in zip(new, past))
        return dict(bytes=tokens * D * (act * (2 * Hq + 2 * Hk) + 2 * Hk) + 8 * blocks * Hk, flops=(14 if case["norm"] else 9) * tokens * (Hq + Hk) * D)
    pairs = rows = 0
    for n, p in zip(new, past):
        w = case["window"]
        if not case["causal"]:
            pairs, rows = pairs + n * (n + p), rows + n + p
        elif not w:
            pairs, rows = pairs + n * p + n * (n + 1) // 2, rows + n + p
        else:
            pairs += sum(min(w, p + i + 1) for i in range(n))
            rows += n + min(p, w - 1)
    return dict(bytes=2 * tokens * Hq * D * act + 2 * rows * Hk * D + 8 * rows * Hk // case["block"], flops=4 * pairs * Hq * D)


def _starts(new):
    out = [0]
    for n in new:
        out.append(out[-1] + n)
    return out


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 1000003 + 29)

    def normal(*shape, dtype=torch.float32, std=1.0, mean=0.0):
        return (torch.randn(*shape, generator=g, device="cuda") * std + mean).to(dtype)

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    def shuffled(n):
        return torch.randperm(n, generator=g, device="cuda").to(torch.int32)

    s = dict(case=case)
    if case["kind"] == "pages":
        new, past, held = _ended(case)
        need = [-(-(n + p) // case["page"]) for n, p in zip(new, past)]
        more = sum(max(a - b, 0) for a, b in zip(need, held))
        stride = max(max(need), max(held)) + 3
        pages = sum(held) + more + 5
        order = shuffled(pages)
        table = torch.full((case["seqs"], stride), -1, dtype=torch.int32, device="cuda")
        table.masked_scatter_(torch.arange(stride, device="cuda") < ints(held)[:, None], order[:sum(held)])
        free = torch.full((pages,), -1, dtype=torch.int32, device="cuda")
        free[:pages - sum(held)] = order[sum(held):]
        # the state that a server keeps, in one array: tables, pages held, free pages, their number
        s.update(past=ints(past), new=ints(new), stride=stride, pages=pages, tokens=sum(new),
                 kept=torch.cat((table.reshape(-1), ints(held), free, ints([pages - sum(held)]))))
        return s
    if case["kind"] == "verify":
        rows = _drafts(case)
        n, V, dt = sum(rows), case["vocab"], DTYPES[case["logits"]]
        starts = ints(_starts(rows))
        seq = torch.repeat_interleave(torch.arange(case["seqs"], device="cuda"), ints(rows))
        heat = (0.6 + 0.5 * torch.rand(case["seqs"], generator=g, device="cuda")) * (torch.arange(case["seqs"], device="cuda") % 8 != 5)
        logits = normal(n, V, std=3.0)
        draft = 0.9 * logits + normal(n, V, std=0.9)
        warm = torch.where(heat > 0, heat, 1.0)[seq][:, None]
        race = torch.rand(n, V, generator=g, device="cuda").clamp_(1e-20, 1 - 1e-7).log_().neg_().log_().neg_()  # the draft model's own draw
        drawn = (draft.to(dt).float() / warm + race * (heat[seq] > 0)[:, None]).argmax(-1).to(torch.int32)
        tokens = torch.cat((torch.randint(0, V, (1,), generator=g, device="cuda").to(torch.int32), drawn[:-1]))
        s.update(logits=logits.to(dt), draft=draft.to(dt) if case["dense"] else None, starts=starts, tokens=tokens, heat=heat,
                 accept=torch.rand(n, generator=g, device="cuda"), pick=torch.rand(case["seqs"], generator=g, device="cuda"))
        return s
    Hq, Hk, D, act = case["heads"], case["kv_heads"], case["dim"], DTYPES[case["act"]]
    new, past = _lengths(case)
    tokens = sum(new)
    kv = [n + p for n, p in zip(new, past)]
    per = [-(-n // case["page"]) for n in kv]
    pages, blocks = sum(per) + 3, case["page"] // case["block"]
    order = shuffled(pages)
    table = torch.full((case["seqs"], max(per)), -1, dtype=torch.int32, device="cuda")
    table.masked_scatter_(torch.arange(max(per), device="cuda") < ints(per)[:, None], order[:sum(per)])
    s.update(q_start=ints(_starts(new)), kv_len=ints(kv), table=table, max_new=max(new), max_kv=max(kv))
    # keys and values of unit size or so, as codes whose block's largest is near the type's
    top = TOP[case["cache"]]
    codes = normal(2, pages, case["page"], Hk, D, std=top / 3.4).clamp_(-top, top)
    s["codes"] = codes.round_().to(torch.int8) if case["cache"] == "i8" else codes.to(torch.float8_e4m3fn)
    s["scales"] = (torch.rand(pages, Hk, blocks, 2, generator=g, device="cuda") + 0.5) * (3.4 / top)
    if case["kind"] == "attention":
        s["q"] = normal(tokens, Hq, D, dtype=act, std=1.5)
        return s
    s.update(q=normal(tokens, Hq * D, dtype=act), k=normal(tokens, Hk * D, dtype=act), v=normal(tokens, Hk * D, dtype=act))
    for n, h in (("q", Hq), ("k", Hk), ("v", Hk)):
        s[n + "_bias"] = normal(h * D, std=0.5) if case["bias"] else None
    for n in ("q", "k"):
        s[n + "_norm"] = normal(D, std=0.1, mean=1.0) if case["norm"] else None
    return s


def _stand_for(codes, scales):
    """What a cache holds, from [2][page][row][head][dim] codes and [page][head][block][2] scales: e4m3 codes are numbers as they are, next to
    their scales; int8 ones are multiplied out (in fp16)."""
    if codes.dtype != torch.int8:
        return codes, scales
    n, P, page, Hk, D = codes.shape
    by = scales.half().permute(3, 0, 2, 1)
    return codes.view(n, P, by.shape[2], -1, Hk, D) * by[:, :, :, None, :, None], scales


# ---- the plain forms ---------------------------------------------------------------------------

def _finished(x, heads, D, bias, norm, positions, rotary):
    """(tokens, heads * D) projections with bias, norm and rotation, in 32 bits (the angles in 64)."""
    x = x.float()
    if bias is not None:
        x = x + bias
    x = x.reshape(-1, heads, D)
    if norm is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * norm
    half = rotary // 2
    freq = THETA ** (-torch.arange(half, device=x.device, dtype=torch.float64) / half)
    angle = (positions.double()[:, None] * freq)[:, None, :]
    c, s = torch.cos(angle).float(), torch.sin(angle).float()
    x0, x1 = x[..., :half], x[..., half:rotary]
    return torch.cat((x0 * c - x1 * s, x1 * c + x0 * s, x[..., rotary:]), -1)


def _token_places(s, tokens):
    """(sequence, position in the cache) of each token."""
    t = torch.arange(tokens, device="cuda")
    starts = s["q_start"].long()
    seq = torch.searchsorted(starts[1:], t, right=True)
    return seq, s["kv_len"].long()[seq] - starts[seq + 1] + t


def _to_codes(x, kind):
    """x / scale rounded to nearest even."""
    x = x.clamp(-TOP[kind], TOP[kind])
    return x.round().to(torch.int8) if kind == "i8" else x.to(torch.float8_e4m3fn)


def _plain_pages(s):
    case, N, stride, P = s["case"], s["case"]["seqs"], s["stride"], s["pages"]
    table, held, free, n_free = s["kept"].long().split((N * stride, N, P, 1))
    table = table.view(N, stride)
    new, kv = s["new"].long(), s["past"].long() + s["new"].long()
    need = (kv + case["page"] - 1) // case["page"]
    give = (held - need).clamp(min=0)
    want = torch.where(need <= stride, (need - held).clamp(min=0), 0)
    j = torch.arange(stride, device="cuda")
    given = (j >= need[:, None]) & (j < held[:, None])
    place = torch.where(given, n_free + (give.cumsum(0) - give - need)[:, None] + j, P)
    free = torch.cat((free, free[:1])).scatter(0, place.view(-1), table.reshape(-1))[:P]
    there, upto = n_free + give.sum(), want.cumsum(0)
    got = want * (upto <= there)
    taken = (j >= held[:, None]) & (j < (held + got)[:, None])
    source = (there - 1 - (upto - want - held)[:, None] - j).clamp(0, P - 1)
    table = torch.where(taken, free[source], torch.where(given, -1, table))
    starts = torch.cat((torch.zeros(1, dtype=torch.int64, device="cuda"), new.cumsum(0)))
    t = torch.arange(s["tokens"], device="cuda")
    seq = torch.searchsorted(starts[1:], t, right=True)
    pos = kv[seq] - starts[seq + 1] + t
    page = table[seq, pos // case["page"]]
    slot = torch.where(page >= 0, page * case["page"] + pos % case["page"], -1)
    missing = torch.where(need <= stride, want - got, need - held)
    return [x.to(torch.int32) for x in (torch.cat((table.view(-1), torch.minimum(need, held + got), free, there - got.sum())), starts, kv, pos, slot, missing)]


def _plain_verify(s):
    case, V = s["case"], s["case"]["vocab"]
    starts = s["starts"].long()
    n = s["tokens"].shape[0]
    t = torch.arange(n, device="cuda")
    seq = torch.searchsorted(starts[1:], t, right=True)
    greedy, heat = (s["heat"] == 0)[seq], torch.where(s["heat"] > 0, s["heat"], 1.0).double()[seq][:, None]

    def chances(x):
        x = x.double() / heat
        e = torch.exp(x - x.amax(-1, keepdim=True))
        return e / e.sum(-1, keepdim=True)

    p, best = chances(s["logits"]), s["logits"].argmax(-1)
    drafted = t + 1 < starts[seq + 1]
    x = s["tokens"].long()[(t + 1).clamp(max=n - 1)]
    q = chances(s["draft"]) if case["dense"] else (torch.arange(V, device="cuda") == x[:, None]).double()
    px, qx = (y.gather(1, x[:, None])[:, 0] for y in (p, q))
    yes = drafted & torch.where(greedy, x == best, s["accept"].double() * qx < px)
    count = torch.full((case["seqs"],), n, device="cuda").scatter_reduce(0, seq, torch.where(yes, n, t - starts[seq]), "amin")
    last = starts[:-1] + count
    rest = torch.where(drafted[last][:, None], (p[last] - q[last]).clamp(min=0), p[last])
    upto = rest.cumsum(-1)
    drawn = (upto <= s["pick"].double()[:, None] * upto[:, -1:]).sum(-1).clamp(max=V - 1)
    drawn = torch.where(s["heat"] == 0, best[last], drawn)
    i = t - starts[seq]
    out = torch.where(i < count[seq], x, torch.where(i == count[seq], drawn[seq], -1))
    logprob = torch.where(out >= 0, p.gather(1, out.clamp(min=0)[:, None])[:, 0].log(), 0.0)
    return out.to(torch.int32), (count + 1).to(torch.int32), logprob.float()


def _plain_append(s):
    case = s["case"]
    Hq, Hk, D, kind, page, block = case["heads"], case["kv_heads"], case["dim"], case["cache"], case["page"], case["block"]
    tokens = s["q"].shape[0]
    seq, pos = _token_places(s, tokens)
    q, k = (_finished(s[n], h, D, s[n + "_bias"], s[n + "_norm"], pos, case["rotary"]) for n, h in (("q", Hq), ("k", Hk)))
    v = s["v"].float() if s["v_bias"] is None else s["v"].float() + s["v_bias"]
    x = torch.stack((k, v.reshape(-1, Hk, D)))
    codes, scales = s["codes"], s["scales"]
    P, per = codes.shape[1], page // block
    table, starts = s["table"].long(), s["q_start"].long()
    rows = codes.view(2, P * page, Hk, D).view(torch.int8)  # (stored through a view that indexing takes)
    by = scales.permute(3, 0, 2, 1).reshape(2, P * per, Hk)  # a copy: [2][block][head]
    row = table[seq, pos // page] * page + pos % page
    at = row // block
    largest = torch.zeros_like(by).scatter_reduce(1, at[None, :, None].expand(2, tokens, Hk), x.abs().amax(-1), "amax")
    # A block keeps its old scale, where that is larger, if it has older rows: a sequence's first block may. Others forget theirs.
    old = by.clone()
    new = torch.maximum(largest / TOP[kind], torch.tensor(LEAST_SCALE, device="cuda"))
    first = s["kv_len"].long() - (starts[1:] - starts[:-1])
    head = first // block * block
    older = head[:, None] + torch.arange(block, device="cuda") < first[:, None]  # [sequence][row of its first block]
    old_at = (table.gather(1, (head // page)[:, None])[:, 0] * page + head % page) // block
    touched, kept = torch.zeros(P * per, device="cuda").scatter(0, at, 1.0), torch.zeros(P * per, device="cuda").scatter(0, old_at, older[:, 0].float())
    new = torch.where(kept[None, :, None] > 0, torch.maximum(new, old), new)
    now = torch.where(touched[None, :, None] > 0, new, old)
    old_rows = (old_at * block)[:, None] + torch.arange(block, device="cuda")
    held = codes.view(2, P * page, Hk, D).view(torch.int8)[:, old_rows].view(codes.dtype)
    again = _to_codes(held.float() * (old[:, old_at] / now[:, old_at])[:, :, None, :, None], kind)
    rows[:, old_rows] = torch.where(older[None, :, :, None, None], again.view(torch.int8), held.view(torch.int8))
    rows[:, row] = _to_codes(x / now[:, at][..., None], kind).view(torch.int8)
    scales.copy_(now.view(2, P, per, Hk).permute(1, 3, 2, 0))
    return (q.to(DTYPES[case["act"]]), *_stand_for(codes, scales))


def _plain_attention(s):
    # every sequence padded to the longest
    case = s["case"]
    Hq, Hk, D, act = case["heads"], case["kv_heads"], case["dim"], DTYPES[case["act"]]
    tokens = s["q"].shape[0]
    seq, _ = _token_places(s, tokens)
    B, n, L = case["seqs"], s["max_new"], s["max_kv"]
    starts = s["q_start"].long()
    count = starts[1:] - starts[:-1]
    at = torch.arange(n, device="cuda")
    q = s["q"].float()[(starts[:-1, None] + at).clamp(max=tokens - 1)]
    j = torch.arange(L, device="cuda")
    page, row = s["table"].long()[:, j // case["page"]].clamp(min=0), j % case["page"]
    stored = s["codes"].view(torch.int8)

    def rows(i):  # B, Hk, L, D
        by = s["scales"][page, :, row // case["block"], i]
        return (stored[i][page, row].view(s["codes"].dtype).float() * by[..., None]).permute(0, 2, 1, 3)

    G = Hq // Hk
    q = q.reshape(B, n, Hk, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, G * n, D)
    scores = (q @ rows(0).transpose(-1, -2).contiguous()).reshape(B, Hk, G, n, L) * (1 / math.sqrt(D))
    p = (s["kv_len"].long() - count)[:, None] + at
    seen = (j < s["kv_len"][:, None, None]).expand(B, n, L)
    if case["causal"]:
        seen = seen & (j <= p[:, :, None])
        if case["window"]:
            seen = seen & (j > p[:, :, None] - case["window"])
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    scores -= scores.amax(-1, keepdim=True).clamp(min=-1e30)
    scores.exp_()
    total = scores.sum(-1, keepdim=True)
    o = (scores.reshape(B, Hk, G * n, L) @ rows(1).contiguous()).reshape(B, Hk, G, n, D) / total.clamp(min=1e-30)
    return o.permute(0, 3, 1, 2, 4).reshape(B * n, Hq, D)[seq * n + torch.arange(tokens, device="cuda") - starts[seq]].to(act)


PLAIN = {"pages": _plain_pages, "append": _plain_append, "attention": _plain_attention, "verify": _plain_verify}


# ---- the framework's operators ----------------------------------------------------------------

def _at(t):
    return None if t is None else t.data_ptr()


def _own_pages(tq, s, stream):
    N, stride, P, tokens = s["case"]["seqs"], s["stride"], s["pages"], s["tokens"]
    kept = s["kept"].clone()  # (a server goes on from its state; here every pass starts from the same)
    out = torch.empty(3 * N + 1 + 2 * tokens, dtype=torch.int32, device="cuda")
    starts, kv, missing, pos, slot = out.split((N + 1, N, N, tokens, tokens))
    at = kept.data_ptr()
    tq.page_map_dev(tq.PageMap(n_seqs=N, n_tokens=tokens, n_pages=P, page_size=s["case"]["page"], table_stride=stride, past=s["past"].data_ptr(),
                               n_new=s["new"].data_ptr(), block_table=at, n_held=at + 4 * N * stride, free_pages=at + 4 * N * (stride + 1),
                               n_free=at + 4 * (N * (stride + 1) + P), q_start=starts.data_ptr(), kv_len=kv.data_ptr(), missing=missing.data_ptr(),
                               positions=pos.data_ptr(), slots=slot.data_ptr()), stream)
    return [kept, starts, kv, pos, slot, missing]


def _own_verify(tq, s, stream):
    case, n = s["case"], s["tokens"].shape[0]
    out, count = torch.empty(n, dtype=torch.int32, device="cuda"), torch.empty(case["seqs"], dtype=torch.int32, device="cuda")
    logprob = torch.empty(n, dtype=torch.float32, device="cuda")
    tq.verify_tokens_dev(tq.Verify(dtype=CODES[case["logits"]], n_seqs=case["seqs"], n_tokens=n, vocab=case["vocab"], logits=s["logits"].data_ptr(),
                                   draft=_at(s["draft"]), q_start=s["starts"].data_ptr(), tokens=s["tokens"].data_ptr(),
                                   temperature=s["heat"].data_ptr(), accept=s["accept"].data_ptr(), pick=s["pick"].data_ptr(),
                                   out_tokens=out.data_ptr(), n_out=count.data_ptr(), logprob=logprob.data_ptr()), stream)
    return out, count, logprob


def _cache(tq, s):
    case, codes = s["case"], s["codes"]
    cache = tq.KvCache8(k=codes[0].data_ptr(), v=codes[1].data_ptr(), scales=s["scales"].data_ptr(), dtype=CODES[case["cache"]], n_pages=codes.shape[1],
                        page_size=case["page"], block=case["block"], n_kv_heads=case["kv_heads"], head_dim=case["dim"])
    return cache, tq.Seqs(n_seqs=case["seqs"], n_tokens=s["q"].shape[0], q_start=s["q_start"].data_ptr(), kv_len=s["kv_len"].data_ptr(),
                          block_table=s["table"].data_ptr(), table_stride=s["table"].shape[1], max_kv=s["max_kv"])


def _own_append(tq, s, stream):
    case, tokens = s["case"], s["q"].shape[0]
    out = torch.empty((tokens, case["heads"], case["dim"]), dtype=s["q"].dtype, device="cuda")
    proj = tq.HeadProj(dtype=CODES[case["act"]], n_tokens=tokens, n_heads=case["heads"], n_kv_heads=case["kv_heads"], head_dim=case["dim"],
                       rotary_dim=case["rotary"], q=s["q"].data_ptr(), k=s["k"].data_ptr(), v=s["v"].data_ptr(), q_out=out.data_ptr(),
                       q_bias=_at(s["q_bias"]), k_bias=_at(s["k_bias"]), v_bias=_at(s["v_bias"]), q_norm=_at(s["q_norm"]), k_norm=_at(s["k_norm"]),
                       eps=EPS, theta=THETA)
    tq.kv_append8_dev(proj, *_cache(tq, s), stream)
    return (out, *_stand_for(s["codes"], s["scales"]))


def _own_attention(tq, s, stream):
    case = s["case"]
    out = torch.empty_like(s["q"])
    tq.paged_attention8_dev(tq.Attn(dtype=CODES[case["act"]], n_heads=case["heads"], q=s["q"].data_ptr(), out=out.data_ptr(),
                                    scale=1 / math.sqrt(case["dim"]), causal=int(case["causal"]), window=case["window"]), *_cache(tq, s), stream)
    return out


OWN = {"pages": _own_pages, "append": _own_append, "attention": _own_attention, "verify": _own_verify}


def run(state):
    kind = state["case"]["kind"]
    if own:
        return OWN[kind](_package(), state, torch.cuda.current_stream().cuda_stream)
    return PLAIN[kind](state)


# ---- the definitions in 64 bits ------------------------------------------------------------------

def _head64(x, bias, norm, position, rotary):
    """Tokens' heads (tokens, heads, D) in float64."""
    x = x.double() + (0 if bias is None else bias.double().reshape(x.shape[-2:]))
    if norm is not None:
        x = x * norm.double() * (x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS).rsqrt()
    y, half = x.clone(), rotary // 2
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=x.device),
                       position.double()[..., None, None] * torch.exp(-math.log(THETA) * 2 / rotary * torch.arange(half, device=x.device, dtype=torch.float64)))
    z = torch.complex(x[..., :half].contiguous(), x[..., half:rotary].contiguous()) * turn
    y[..., :half], y[..., half:rotary] = z.real, z.imag
    return y


def _exact_verify(s):
    """Log probabilities of the tokens given out: sequence by sequence, token by token."""
    starts, heat, given = s["starts"].tolist(), s["heat"].tolist(), s["tokens"].tolist()
    out = torch.zeros(starts[-1], dtype=torch.float64, device="cuda")
    for b, T in enumerate(heat):
        for t in range(starts[b], starts[b + 1]):
            lp = torch.log_softmax(s["logits"][t].double() / (T or 1.0), -1)
            x = given[t + 1] if t + 1 < starts[b + 1] else None
            lq = None if x is None or s["draft"] is None else torch.log_softmax(s["draft"][t].double() / (T or 1.0), -1)
            if T == 0:
                token = int(s["logits"][t].argmax())
                yes = token == x
            else:
                yes = x is not None and float(s["accept"][t]) * (1.0 if lq is None else math.exp(float(lq[x]))) < math.exp(float(lp[x]))
                token = x
                if not yes:
                    weight = lp.exp()
                    if lq is not None:
                        weight = (weight - lq.exp()).clamp(min=0)
                    elif x is not None:
                        weight[x] = 0
                    upto = weight.cumsum(0)
                    token = int(torch.searchsorted(upto, upto[-1:] * s["pick"][b].double(), right=True).clamp(max=len(upto) - 1))
            out[t] = lp[token]
            if not yes:
                break
    return None, None, out


def _exact_append(s):
    case = s["case"]
    Hq, Hk, D, kind, page, block = case["heads"], case["kv_heads"], case["dim"], case["cache"], case["page"], case["block"]
    starts, lens, table = s["q_start"].tolist(), s["kv_len"].tolist(), s["table"].tolist()
    places = torch.cat([torch.arange(lens[i] - (starts[i + 1] - starts[i]), lens[i], device="cuda") for i in range(case["seqs"])])

    def finished(n, h):
        return torch.cat([_head64(x, s[n + "_bias"], s[n + "_norm"], at, case["rotary"]) for x, at in zip(s[n].reshape(-1, h, D).split(1024), places.split(1024))])

    v = s["v"].double().reshape(-1, Hk, D)
    x = torch.stack((finished("k", Hk), v if s["v_bias"] is None else v + s["v_bias"].double().reshape(Hk, D)))
    codes, scales = s["codes"].double(), s["scales"].double()

    def rounded(y):
        return y.round() if kind == "i8" else y.clamp(-448, 448).float().to(torch.float8_e4m3fn).double()

    for i in range(case["seqs"]):
        p = lens[i] - (starts[i + 1] - starts[i])
        while p < lens[i]:
            end = min(lens[i], p // block * block + block)
            pg, r0 = table[i][p // page], p // block * block % page
            part = x[:, starts[i + 1] - (lens[i] - p):starts[i + 1] - (lens[i] - end)]  # [2][row][head][dim]
            by = part.abs().amax((1, 3)) / TOP[kind]  # [2][head]
            old = scales[pg, :, r0 // block].t().clone()
            r = p % page
            if r > r0:
                by = torch.maximum(by, old)
                codes[:, pg, r0:r] = rounded(codes[:, pg, r0:r] * (old / by)[:, None, :, None])
            scales[pg, :, r0 // block] = by.t()
            codes[:, pg, r:r + end - p] = part / by[:, None, :, None] if kind == "e4m3" else rounded(part / by[:, None, :, None])
            p = end
    if kind == "i8":
        per = page // block
        codes = codes.view(2, -1, per, block, Hk, D) * scales.permute(3, 0, 2, 1)[:, :, :, None, :, None]
    return finished("q", Hq), codes, scales


def exact(case, seed):
    if case["kind"] == "pages":
        return None
    s = prepare(case, seed)
    if case["kind"] == "verify":
        return _exact_verify(s)
    if case["kind"] == "append":
        return _exact_append(s)
    Hq, Hk, D, page, block = case["heads"], case["kv_heads"], case["dim"], case["page"], case["block"]
    starts, lens, table = s["q_start"].tolist(), s["kv_len"].tolist(), s["table"].long()
    flat = s["codes"].view(torch.int8).view(2, -1, Hk, D)
    out = torch.zeros((s["q"].shape[0], Hq, D), dtype=torch.float64, device="cuda")
    for i in range(case["seqs"]):
        n, L = starts[i + 1] - starts[i], lens[i]
        j = torch.arange(L, device="cuda")
        pg = table[i, j // page]
        rows = pg * page + j % page
        ahead = j[None, :] - torch.arange(L - n, L, device="cuda")[:, None]
        hidden = (ahead > 0) | ((ahead <= -case["window"]) if case["window"] else False) if case["causal"] else torch.zeros_like(ahead, dtype=torch.bool)
        for g in range(Hk):
            k, v = (flat[c][rows, g].view(s["codes"].dtype).double() * s["scales"][pg, g, j % page // block, c].double()[:, None] for c in (0, 1))
            for h in range(g * Hq // Hk, (g + 1) * Hq // Hk):
                weight = (s["q"][starts[i]:starts[i + 1], h].double() @ k.T.contiguous() / math.sqrt(D)).masked_fill(hidden, -math.inf)
                out[starts[i]:starts[i + 1], h] = torch.softmax(weight, -1) @ v
    return out
