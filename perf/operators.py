"""The operators of a serving step over a paged key-value cache, as they are measured: rotary positions written with K and V
into the cache, attention over it, eviction by accumulated attention weight, and verification of drafted tokens.

A batch is `nseq` sequences; sequence b has the new rows row_start[b] .. row_start[b + 1] (one for a single token, more with
drafted ones) and lens[b] cache entries, its new rows among them.  The cache is the framework's: pages
[page][2 (k, v)][kv_heads][page_tokens][hd] and one row of page ids per sequence.

`run` is one pass through one operator: with `own` the framework's call, without it the same from elementary torch operations.
"""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # a few chats that each take one token: latency
        dict(name="attend, four short chats", op="attend", nseq=4, heads=32, kv_heads=8, hd=128, length=701, page=64, rows=1, q="bf16", kv="bf16", window=0, collect=False),
        # one user with a long document; few sequences, so the length has to be cut
        dict(name="attend, one long document", op="attend", nseq=1, heads=16, kv_heads=4, hd=128, length=130001, page=64, rows=1, q="bf16", kv="bf16", window=0, collect=False),
        # the framework's dense decoder in a ragged batch: fp32 activations, fp16 cache, a kv head per q head
        dict(name="attend, ragged batch", op="attend", nseq=48, heads=32, kv_heads=32, hd=128, length=3001, page=64, rows=1, q="f32", kv="f16", window=0, collect=False),
        # drafted tokens scored together, eight q heads a kv head: up to 48 rows against each cache entry
        dict(name="attend, drafted tokens", op="attend", nseq=24, heads=16, kv_heads=2, hd=64, length=20011, page=16, rows=6, q="f16", kv="f16", window=0, collect=False),
        # a bounded cache that keeps count of what its entries are worth
        dict(name="attend, weights collected", op="attend", nseq=16, heads=32, kv_heads=8, hd=128, length=8193, page=64, rows=1, q="bf16", kv="bf16", window=0, collect=True),
        # one token of a few chats
        dict(name="append, four tokens", op="append", nseq=4, heads=32, kv_heads=8, hd=128, page=64, rows=1, first=700, q="bf16", kv="bf16", rot=128, layout="half", scaling="none", factor=1.0, book=True),
        # a chunk of several long prompts, positions stretched, a quarter of the head left as it is
        dict(name="append, prompt chunk", op="append", nseq=8, heads=32, kv_heads=16, hd=128, page=64, rows=1023, first=120000, q="f32", kv="f16", rot=96, layout="interleaved", scaling="yarn", factor=32.0, book=False),
        # every step of a full cache: one entry has to go
        dict(name="evict, one of 2049", op="evict", nseq=16, kv_heads=8, hd=128, length=2049, page=64, kv="bf16", keep=2048, sinks=4, recent=256),
        # long prompts brought down to a quarter
        dict(name="evict, long prompts", op="evict", nseq=4, kv_heads=8, hd=128, length=60001, page=64, kv="f16", keep=15000, sinks=4, recent=1000),
        # one chat with four drafted tokens
        dict(name="verify, one chat", op="verify", nseq=1, rows=5, vocab=32000, dtype="f32", temperature=1.0, draft=True),
        # a batch with a draft model
        dict(name="verify, batch", op="verify", nseq=32, rows=8, vocab=128000, dtype="bf16", temperature=0.8, draft=True),
        # drafts looked up in the prompt, greedy; rows of an odd length
        dict(name="verify, greedy", op="verify", nseq=64, rows=4, vocab=50003, dtype="f16", temperature=0.0, draft=False),
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


MOST = {}


def _bounded(op, make):
    """The first of make()'s cases that costs no more than the largest listed one of its operator."""
    if not MOST:
        for c in listed():
            MOST[c["op"]] = max(MOST.get(c["op"], 0), _cost(c))
    while True:
        c = make()
        if _cost(c) <= MOST[op]:
            return c


def _cost(c):
    if c["op"] == "attend":  # entries to read, and scores that the plain form holds
        return _entries(c) * c["kv_heads"] * c["hd"] + 16 * c["nseq"] * c["rows"] * c["heads"] * c["length"]
    return work(c)["bytes"]


def draw(rng):
    op = rng.choice(("attend", "attend", "append", "evict", "verify"))
    kv_heads = rng.choice((1, 2, 4, 8, 16, 32))
    types = rng.choice((("bf16", "bf16"), ("f16", "f16"), ("f32", "f16"), ("f32", "bf16"), ("f32", "f32")))
    if op == "attend":
        def make():
            return dict(op=op, nseq=_log(rng, 1, 64), heads=kv_heads * rng.choice((1, 2, 3, 4, 8, 16)), kv_heads=kv_heads, hd=rng.choice((64, 128)), length=_log(rng, 8, 131072),
                        page=rng.choice((16, 24, 64, 128)), rows=rng.choice((1, 1, 1, 2, 4, 5, 8)), q=types[0], kv=types[1], window=rng.choice((0, 0, 0, 1024)), collect=rng.random() < 0.25)
    elif op == "append":
        def make():
            hd = rng.choice((64, 128))
            scaling = rng.choice(("none", "linear", "ntk", "yarn"))
            return dict(op=op, nseq=_log(rng, 1, 64), heads=kv_heads * rng.choice((1, 2, 3, 4, 8)), kv_heads=kv_heads, hd=hd, page=rng.choice((16, 24, 64, 128)), rows=_log(rng, 1, 2048),
                        first=_log(rng, 1, 1000000), q=types[0], kv=types[1], rot=rng.choice((hd, hd, hd // 2, hd // 4, hd - 16)), layout=rng.choice(("half", "interleaved")),
                        scaling=scaling, factor=1.0 if scaling == "none" else rng.choice((2.0, 8.0, 32.0)), book=rng.random() < 0.5)
    elif op == "evict":
        def make():
            length = _log(rng, 40, 131072)
            keep = rng.choice((length - 1, max(8, length // 2), max(8, length // 8), max(8, int(length * rng.uniform(0.1, 0.95)))))
            return dict(op=op, nseq=_log(rng, 1, 64), kv_heads=kv_heads, hd=rng.choice((64, 128)), length=length, page=rng.choice((16, 24, 64, 128)), kv=types[1], keep=keep,
                        sinks=rng.choice((0, 4)), recent=rng.choice((0, keep // 8, keep // 2 - 4)))
    else:
        def make():
            return dict(op=op, nseq=_log(rng, 1, 64), rows=rng.choice((1, 2, 4, 5, 6, 8)), vocab=_log(rng, 500, 200000), dtype=rng.choice(("f32", "f16", "bf16")),
                        temperature=rng.choice((0.0, 0.6, 1.0, 1.0)), draft=rng.random() < 0.6)
    return _bounded(op, make)


def _lengths(c):
    """Lengths from a third of `length` up to it (one sequence: `length` itself), every sequence's new rows among them."""
    n = c["nseq"]
    if c["op"] == "evict":
        return [c["length"] if n == 1 or b % 4 else max(1, c["length"] * 2 // 3) for b in range(n)]
    return [max(min(c["rows"], c["length"]), c["length"] - c["length"] * 2 * b // (3 * n)) for b in range(n)]


def _rows(c):
    """New rows per sequence: `rows`, or one, two .. `rows` in turn where they are drafts."""
    return [c["rows"] if c["rows"] == 1 or c["nseq"] == 1 or c["op"] == "append" else 1 + (b * 5 + c["rows"] - 1) % c["rows"] for b in range(c["nseq"])]


def _entries(c):
    window = c.get("window", 0)
    return sum(min(n, window + r - 1) if window else n for n, r in zip(_lengths(c), _rows(c)))


def work(case):
    c, size = case, {"f32": 4, "f16": 2, "bf16": 2}
    if c["op"] == "attend":
        rows, pairs = sum(_rows(c)), sum(min(n, c["window"] or n) * r for n, r in zip(_lengths(c), _rows(c)))
        moved = 2 * _entries(c) * c["kv_heads"] * c["hd"] * size[c["kv"]] + rows * c["heads"] * (2 * c["hd"] * size[c["q"]] + 4)
        moved += 8 * _entries(c) * c["kv_heads"] if c["collect"] else 0
        return {"bytes": moved, "flops": 4 * pairs * c["heads"] * c["hd"]}
    if c["op"] == "append":
        rows = sum(_rows(c))
        moved = rows * c["hd"] * ((2 * c["heads"] + 2 * c["kv_heads"]) * size[c["q"]] + 2 * c["kv_heads"] * size[c["kv"]]) + rows * (4 + 8 * c["kv_heads"] * c["book"])
        return {"bytes": moved, "flops": 3 * rows * c["rot"] * (c["heads"] + c["kv_heads"])}
    if c["op"] == "evict":  # the expected number of kept entries that lie behind the first `keep`
        total = sum(_lengths(c))
        kept = sum(min(n, c["keep"]) for n in _lengths(c))
        pushed = sum(c["keep"] * (n - c["keep"]) / n for n in _lengths(c) if n > c["keep"])
        return {"bytes": c["kv_heads"] * (8 * total + 8 * kept + pushed * 4 * c["hd"] * size[c["kv"]]), "flops": 0}
    rows = sum(_rows(c))
    return {"bytes": (rows + (rows - c["nseq"]) * c["draft"] * (c["temperature"] > 0)) * c["vocab"] * size[c["dtype"]] + 16 * rows, "flops": 2 * rows * c["vocab"]}


# ------------------------------------------------------------------------------------------------ their inputs
def _starts(counts):
    at = [0]
    for n in counts:
        at.append(at[-1] + n)
    return torch.tensor(at, dtype=torch.int32, device="cuda")


def _pages(c, lengths, g, values):
    """A pool with the sequences' pages in no order, their table, and unused places in both."""
    need = [-(-n // c["page"]) for n in lengths]
    most, spare = max(need) + 1, 3
    ids = torch.randperm(sum(need) + spare, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(c["nseq"], most, dtype=torch.int32, device="cuda")
    has = torch.arange(most, device="cuda")[None] < torch.tensor(need, device="cuda")[:, None]
    table[has] = ids[: sum(need)]
    shape = (sum(need) + spare, 2, c["kv_heads"], c["page"], c["hd"])
    pool = torch.empty(shape, dtype=DTYPES[c["kv"]], device="cuda")
    if values:
        step = max(1, (1 << 27) // (pool.numel() // shape[0]))
        for at in range(0, shape[0], step):
            pool[at:at + step] = torch.randn(pool[at:at + step].shape, generator=g, device="cuda")
    else:
        pool.zero_()
    return pool, table


def _frequencies(c):
    """Angles per position, in 64 bits: base 10000, and what stretches them for contexts `factor` times as long as 4096."""
    half, base, f = c["rot"] // 2, 10000.0, c["factor"]
    i = torch.arange(half, dtype=torch.float64)
    if c["scaling"] == "ntk":
        base = base * f ** (c["rot"] / (c["rot"] - 2)) if c["rot"] > 2 else base
    freq = base ** (-2.0 * i / c["rot"])
    magnitude = 1.0
    if c["scaling"] == "linear":
        freq = freq / f
    if c["scaling"] == "yarn":  # pairs that turn over 32 times in the original context stay, under once: stretched, between: blended
        def pair(turns):
            return c["rot"] * math.log(4096 / (turns * 2 * math.pi)) / (2 * math.log(base))
        low, high = max(math.floor(pair(32.0)), 0), min(math.ceil(pair(1.0)), c["rot"] - 1)
        ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
        freq = freq / f * ramp + freq * (1 - ramp)
        magnitude = 0.1 * math.log(f) + 1.0
    return freq.cuda(), magnitude


def prepare(case, seed):
    c = case
    g = torch.Generator("cuda").manual_seed(seed)
    order = random.Random(seed)
    normal = lambda *shape: torch.randn(shape, generator=g, device="cuda")  # noqa: E731
    s = dict(case=c)
    if c["op"] == "verify":
        counts = _rows(c)
        order.shuffle(counts)
        rows, vocab = sum(counts), c["vocab"]
        s.update(row_start=_starts(counts), max_rows=c["rows"], rows=rows)
        target = normal(rows, vocab) * 2.5
        seq = torch.repeat_interleave(torch.arange(c["nseq"], device="cuda"), torch.tensor(counts, device="cuda"))
        drafted = torch.ones(rows, dtype=torch.bool, device="cuda")
        drafted[s["row_start"][1:].long() - 1] = False  # the last row of a sequence has no draft behind it
        near = target + normal(rows, vocab) * 0.7
        heat = max(c["temperature"], 0.3) if c["draft"] else 0.4
        noise = -torch.log(-torch.log(torch.rand(near.shape, generator=g, device="cuda").clamp(1e-20, 1 - 1e-7)))
        draft = near.to(DTYPES[c["dtype"]])
        tokens = torch.zeros(rows, dtype=torch.int32, device="cuda")  # the pending token, then the drafted ones
        guess = (draft.float() / heat + noise * (1.0 if c["temperature"] else 0.3)).argmax(1).to(torch.int32)
        tokens[torch.nonzero(drafted)[:, 0] + 1] = guess[drafted]
        s.update(target=target.to(DTYPES[c["dtype"]]), draft=draft if c["draft"] else None, tokens=tokens, seq=seq)
        s.update(uniforms=torch.rand(rows, generator=g, device="cuda"), draws=torch.rand(c["nseq"], generator=g, device="cuda"))
        return s
    if c["op"] == "append":
        lengths, counts = [c["rows"] + min(c["first"], 40) + 7 * (b % 5) for b in range(c["nseq"])], _rows(c)
        order.shuffle(lengths)
        s["row_start"] = _starts(counts)
        rows, heads, kv = sum(counts), c["heads"], c["kv_heads"]
        fused = normal(rows, (heads + 2 * kv) * c["hd"]).to(DTYPES[c["q"]])  # what a fused projection leaves
        s["q"], s["k"], s["v"] = (fused[:, a * c["hd"]:z * c["hd"]].unflatten(1, (-1, c["hd"])) for a, z in ((0, heads), (heads, heads + kv), (heads + kv, heads + 2 * kv)))
        s["positions"] = (torch.arange(rows, device="cuda") % c["rows"] + c["first"] + order.randrange(1000)).to(torch.int32)
    else:
        lengths = _lengths(c)
        order.shuffle(lengths)
    s["pool"], s["table"] = _pages(c, lengths, g, c["op"] != "append")
    s["lens"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    s["longest"] = max(lengths)
    cap = s["table"].shape[1] * c["page"]
    if c["op"] == "append":
        s["freq"], s["magnitude"] = _frequencies(c)
    if c["op"] == "attend":
        counts = _rows(c)
        order.shuffle(counts)
        s["row_start"] = _starts(counts)
        s["q"] = (normal(sum(counts), c["heads"], c["hd"]) * 1.5).to(DTYPES[c["q"]])
    if c["op"] == "evict" or c.get("collect") or c.get("book"):
        s["weight"] = torch.exp(normal(c["nseq"], c["kv_heads"], cap) * 1.5) * 0.01
        s["position"] = (torch.arange(cap, device="cuda", dtype=torch.int32) * 2).expand(c["nseq"], c["kv_heads"], cap).contiguous()
    if own:
        from rustane_b200 import ops
        s["cache"] = ops.PagedCache(s["pool"], s["table"], s["lens"], s.get("weight"), s.get("position"))
        if c["op"] == "append":
            s["rope"] = ops.Rope(c["rot"], base=10000.0, layout=c["layout"], scaling=c["scaling"], factor=c["factor"], original=4096)
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    s, c = state, state["case"]
    if c["op"] == "attend":
        got = _attend_own(s, c) if own else _attend(s, c)
        return (*got, s["weight"]) if c["collect"] else got
    if c["op"] == "append":
        got = _append_own(s, c) if own else _append(s, c)
        return (got, s["pool"], s["weight"], s["position"]) if c["book"] else (got, s["pool"])
    if c["op"] == "evict":
        return (*(_evict_own(s, c) if own else _evict(s, c)), s["pool"])
    return _verify_own(s, c) if own else _verify(s, c)


def _attend_own(s, c):
    from rustane_b200 import ops
    return ops.paged_attention(s["cache"], s["q"], s["row_start"], c["rows"], window=c["window"], collect=c["collect"], lse=True)


def _append_own(s, c):
    from rustane_b200 import ops
    return ops.rope_append(s["cache"], s["rope"], s["q"], s["k"], s["v"], s["positions"], s["row_start"])


def _evict_own(s, c):
    from rustane_b200 import ops
    return ops.cache_evict(s["cache"], c["keep"], sinks=c["sinks"], recent=c["recent"])


def _verify_own(s, c):
    from rustane_b200 import ops
    return ops.verify_drafts(s["target"], s["tokens"], s["row_start"], c["rows"], s["uniforms"], s["draws"], draft=s["draft"], temperature=c["temperature"])


def _places(s, rows):
    """Of every new row its sequence, which of the sequence's rows it is, and its place in the cache."""
    start = s["row_start"].long()
    row = torch.arange(rows, device="cuda")
    seq = torch.searchsorted(start, row, right=True) - 1
    of = row - start[seq]
    return seq, of, s["lens"].long()[seq] - (start[seq + 1] - start[seq]) + of


def _attend(s, c):
    nseq, heads, kv, hd, most = c["nseq"], c["heads"], c["kv_heads"], c["hd"], c["rows"]
    q, longest, page = s["q"], s["longest"], c["page"]
    group, rows = heads // kv, q.shape[0]
    pages = s["pool"][s["table"][:, : -(-longest // page)].long()].movedim(3, 1).flatten(2, 2)  # [nseq, kv, pages, 2, page, hd]
    k = pages[:, :, :, 0].flatten(2, 3)[:, :, :longest].float()
    v = pages[:, :, :, 1].flatten(2, 3)[:, :, :longest].float()
    del pages
    seq, of, _ = _places(s, rows)
    start = s["row_start"].long()
    counts = start[1:] - start[:-1]
    padded = torch.zeros(nseq, most, heads, hd, device="cuda")
    padded[seq, of] = q.float()
    padded = padded.view(nseq, most, kv, group, hd).transpose(1, 2).reshape(nseq, kv, most * group, hd)
    scores = (padded @ k.transpose(2, 3)) * (1.0 / math.sqrt(hd))
    place = (s["lens"].long() - counts)[:, None] + torch.arange(most, device="cuda")  # of the queries
    entry = torch.arange(longest, device="cuda")
    seen = entry <= place[:, :, None]
    if c["window"]:
        seen &= entry > place[:, :, None] - c["window"]
    seen = seen & (torch.arange(most, device="cuda")[None, :, None] < counts[:, None, None])
    seen = seen[:, None, :, None].expand(nseq, 1, most, group, longest).reshape(nseq, 1, most * group, longest)
    scores = torch.where(seen, scores, torch.full((), -math.inf, device="cuda"))
    top = scores.amax(3, keepdim=True)
    top = torch.where(torch.isfinite(top), top, torch.zeros_like(top))
    p = torch.exp(scores - top)
    del scores
    total = p.sum(3, keepdim=True)
    some = total > 0
    p = p / torch.where(some, total, torch.ones_like(total))
    out = (p @ v).view(nseq, kv, most, group, hd).transpose(1, 2).reshape(nseq, most, heads, hd)
    lse = (top + torch.log(total))[..., 0].view(nseq, kv, most, group).transpose(1, 2).reshape(nseq, most, heads)
    if c["collect"]:
        s["weight"][:, :, :longest] += p.sum(2)
    return out[seq, of].to(q.dtype), lse[seq, of]


def _append(s, c):
    rot, magnitude = c["rot"], s["magnitude"]
    rows = s["q"].shape[0]
    angle = s["positions"].double()[:, None] * s["freq"]
    cos, sin = (torch.cos(angle) * magnitude).float()[:, None], (torch.sin(angle) * magnitude).float()[:, None]

    def turned(x):
        x = x.float()
        if c["layout"] == "half":
            a, b = x[..., : rot // 2], x[..., rot // 2: rot]
            return torch.cat([a * cos - b * sin, a * sin + b * cos, x[..., rot:]], -1)
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        return torch.cat([torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2), x[..., rot:]], -1)

    seq, _, place = _places(s, rows)
    page = s["table"][seq, place // c["page"]].long()
    s["pool"][page, 0, :, place % c["page"]] = turned(s["k"]).to(s["pool"].dtype)
    s["pool"][page, 1, :, place % c["page"]] = s["v"].to(s["pool"].dtype)
    if c["book"]:
        s["weight"][seq, :, place] = 0.0
        s["position"][seq, :, place] = s["positions"][:, None].expand(rows, c["kv_heads"])
    return turned(s["q"]).to(s["q"].dtype)


def _evict(s, c):
    """The `keep` entries that are protected or heaviest stay (of equals the first ones); those of them that lie behind the
    first `keep` places fill the holes there, in order.  The bookkeeping comes back new; K and V move in the pool."""
    keep, kv, page = c["keep"], c["kv_heads"], c["page"]
    weight, position = s["weight"], s["position"]
    nseq, cap = weight.shape[0], weight.shape[2]
    entry = torch.arange(cap, device="cuda")
    live = (entry < s["lens"].long()[:, None, None]).expand_as(weight)
    newest = torch.where(live, position, torch.full_like(position, -1)).amax(2, keepdim=True).long()
    protected = (position < c["sinks"]) | (position.long() > newest - c["recent"])
    key = torch.where(protected, torch.full_like(weight, math.inf), weight)
    key = torch.where(live, key, torch.full_like(weight, -math.inf))
    rank = torch.empty(nseq, kv, cap, dtype=torch.long, device="cuda")
    rank.scatter_(2, torch.sort(key, dim=2, descending=True, stable=True).indices, entry.expand(nseq, kv, cap).contiguous())
    kept = live & (rank < keep)
    source, hole = kept & (entry >= keep), ~kept & live & (entry < keep)
    full = (s["lens"].long() > keep)[:, None, None]
    a, b = torch.nonzero(source & full), torch.nonzero(hole & full)  # both in the order of (sequence, head, place)
    pages = s["table"].long()
    at = (pages[a[:, 0], a[:, 2] // page], a[:, 1], a[:, 2] % page)
    to = (pages[b[:, 0], b[:, 2] // page], b[:, 1], b[:, 2] % page)
    s["pool"][to[0], :, to[1], to[2]] = s["pool"][at[0], :, at[1], at[2]]
    new_weight, new_position = weight.clone(), position.clone()
    new_weight[b[:, 0], b[:, 1], b[:, 2]] = weight[a[:, 0], a[:, 1], a[:, 2]]
    new_position[b[:, 0], b[:, 1], b[:, 2]] = position[a[:, 0], a[:, 1], a[:, 2]]
    return torch.clamp(s["lens"], max=keep), new_weight, new_position


def _verify(s, c):
    """Draft j of a sequence stays where u q(x) < p(x); the first that does not is replaced by a draw from max(p - q, 0), and
    where all stay one more token is drawn from the last row.  Temperature 0: p and q are one at their largest logit."""
    rows, vocab, nseq = s["rows"], c["vocab"], c["nseq"]
    start, seq = s["row_start"].long(), s["seq"]
    row = torch.arange(rows, device="cuda")
    last = row == start[seq + 1] - 1
    following = torch.where(last, torch.zeros_like(row), s["tokens"].long()[torch.clamp(row + 1, max=rows - 1)])  # the token drafted behind each row

    def probabilities(x):
        x = x.double() / c["temperature"]
        e = torch.exp(x - x.amax(1, keepdim=True))
        return e / e.sum(1, keepdim=True)

    if c["temperature"] == 0:
        best = s["target"].float().argmax(1)
        good = best == following
    else:
        p = probabilities(s["target"])
        px = p[row, following]
        if s["draft"] is not None:
            q = probabilities(s["draft"])
            qx = q[row, following]
        else:
            qx = torch.ones_like(px)
        good = s["uniforms"].double() * qx < px
    good = good & ~last
    run_ = torch.cumsum((~good).long(), 0)  # a row is reached while no row of its sequence before it failed
    before = run_ - (~good).long()
    reached = before == before[start[seq]]
    accepted = torch.zeros(nseq, dtype=torch.long, device="cuda").index_add_(0, seq, (good & reached).long())
    end = start[:-1] + accepted  # the row that the last token is drawn from
    if c["temperature"] == 0:
        drawn = best[end]
    else:
        pe = p[end]
        if s["draft"] is None:
            left = pe.clone()
            left[torch.arange(nseq, device="cuda"), following[end]] = 0.0
        else:
            left = (pe - q[end]).clamp(min=0.0)
        left = torch.where(last[end][:, None], pe, left)
        sums = torch.cumsum(left, 1)
        drawn = (sums <= s["draws"].double()[:, None] * sums[:, -1:]).sum(1).clamp(max=vocab - 1)
    of = row - start[seq]
    tokens = torch.where(of < accepted[seq], following, torch.where(of == accepted[seq], drawn[seq], torch.full_like(row, -1)))
    return accepted.to(torch.int32), tokens.to(torch.int32)


# ------------------------------------------------------------------------------------------------ the same in 64 bits
def exact(case, seed):
    c = case
    if c["op"] == "attend" and _cost(c) > 4e9:
        return None
    s = prepare(c, seed)
    return {"attend": _exact_attend, "append": _exact_append, "evict": _exact_evict, "verify": _exact_verify}[c["op"]](s, c)


def _exact_attend(s, c):
    group, hd = c["heads"] // c["kv_heads"], c["hd"]
    starts, lens = s["row_start"].tolist(), s["lens"].tolist()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    weight = s["weight"].double() if c["collect"] else None
    for b in range(c["nseq"]):
        n, r0, r1 = lens[b], starts[b], starts[b + 1]
        if n == 0 or r0 == r1:
            continue
        pages = s["pool"][s["table"][b, : -(-n // c["page"])].long()]
        q = s["q"][r0:r1].double()
        where = torch.arange(n - (r1 - r0), n, device="cuda")[:, None]
        slots = torch.arange(n, device="cuda")[None]
        hidden = slots > where
        if c["window"]:
            hidden |= where - slots >= c["window"]
        for h in range(c["kv_heads"]):
            keys = pages[:, 0, h].reshape(-1, hd)[:n].double()
            values = pages[:, 1, h].reshape(-1, hd)[:n].double()
            x = torch.einsum("rgd,td->rgt", q[:, h * group:(h + 1) * group], keys) / hd ** 0.5
            x.masked_fill_(hidden[:, None], -math.inf)
            norm = torch.logsumexp(x, 2)
            w = torch.exp(x - norm[..., None])
            out[r0:r1, h * group:(h + 1) * group] = torch.einsum("rgt,td->rgd", w, values)
            lse[r0:r1, h * group:(h + 1) * group] = norm
            if weight is not None:
                weight[b, h, :n] += w.sum((0, 1))
    return (out, lse, weight) if c["collect"] else (out, lse)


def _exact_append(s, c):
    rot, starts = c["rot"], s["row_start"].tolist()
    pool = s["pool"].double()
    z = torch.polar(torch.full_like(s["freq"], s["magnitude"]).expand(len(s["positions"]), -1), s["positions"].double()[:, None] * s["freq"])

    def spun(x):
        x = x.double()
        head = x[..., :rot]
        pairs = head.unflatten(-1, (2, -1)).transpose(-1, -2) if c["layout"] == "half" else head.unflatten(-1, (-1, 2))
        y = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * z[:, None])
        return torch.cat([(y.transpose(-1, -2) if c["layout"] == "half" else y).flatten(-2), x[..., rot:]], -1)

    k, v = spun(s["k"]), s["v"].double()
    for b, n in enumerate(s["lens"].tolist()):
        r0, r1 = starts[b], starts[b + 1]
        slot = torch.arange(n - (r1 - r0), n, device="cuda")
        page, off = s["table"][b].long()[slot // c["page"]], slot % c["page"]
        for h in range(c["kv_heads"]):
            pool[page, 0, h, off] = k[r0:r1, h]
            pool[page, 1, h, off] = v[r0:r1, h]
            if c["book"]:
                s["weight"][b, h, slot] = 0
                s["position"][b, h, slot] = s["positions"][r0:r1]
    return (spun(s["q"]), pool, s["weight"].double(), s["position"]) if c["book"] else (spun(s["q"]), pool)


def _exact_evict(s, c):
    keep = c["keep"]
    lens, weight, position, pool = s["lens"].tolist(), s["weight"].double().cpu(), s["position"].cpu(), s["pool"]
    new_w, new_p = weight.clone(), position.clone()
    for b, n in enumerate(lens):
        if n <= keep:
            continue
        for h in range(c["kv_heads"]):
            w, p = weight[b, h, :n].clone(), position[b, h, :n].long()
            w[(p < c["sinks"]) | (p > int(p.max()) - c["recent"])] = math.inf
            stay = torch.zeros(n, dtype=torch.bool)
            stay[torch.argsort(-w, stable=True)[:keep]] = True
            come, go = torch.nonzero(stay[keep:])[:, 0] + keep, torch.nonzero(~stay[:keep])[:, 0]
            new_w[b, h, go], new_p[b, h, go] = weight[b, h, come], position[b, h, come]
            table = s["table"][b].long()
            a, z = come.cuda(), go.cuda()
            pool[table[z // c["page"]], :, h, z % c["page"]] = pool[table[a // c["page"]], :, h, a % c["page"]]
    return torch.tensor([min(n, keep) for n in lens], dtype=torch.int32), new_w, new_p, pool


def _exact_verify(s, c):
    starts, heat = s["row_start"].tolist(), c["temperature"]
    tokens, uniforms, draws = s["tokens"].tolist(), s["uniforms"].tolist(), s["draws"].tolist()
    accepted, out = [], []
    for b in range(c["nseq"]):
        r0, n = starts[b], starts[b + 1] - starts[b]
        got, left = [], None
        for j in range(n):
            logits = s["target"][r0 + j].double()
            if heat == 0:
                p = torch.zeros_like(logits)
                p[int(torch.nonzero(logits == logits.max())[0])] = 1.0
            else:
                p = torch.softmax(logits / heat, 0)
            left = p
            if j == n - 1:
                break
            x = tokens[r0 + j + 1]
            if heat == 0:
                q = p * 0
                stays = bool(p[x] > 0)
            else:
                if s["draft"] is None:
                    q = torch.zeros_like(p)
                    q[x] = 1.0
                else:
                    q = torch.softmax(s["draft"][r0 + j].double() / heat, 0)
                stays = bool(uniforms[r0 + j] * q[x] < p[x])
            if not stays:
                left = torch.clamp(p - q, min=0)
                break
            got.append(x)
        sums = torch.cumsum(left, 0)
        accepted.append(len(got))
        extra = int(torch.searchsorted(sums, draws[b] * sums[-1:], right=True)[0])
        got.append(min(extra, c["vocab"] - 1))
        out += got + [-1] * (n - len(got))
    return torch.tensor(accepted, dtype=torch.int32), torch.tensor(out, dtype=torch.int32)
