"""The operators of a serving step over paged caches, driven from the device, as cases to be timed.

Pages of an F16 or BF16 cache are shared by the requests of a server. A step of all of them passes

- map:    request lengths to pages: each request's table of pages grows or shrinks to its length,
          and every new token gets its slot, its position and its place among the step's rows;
- append: the new rows of K and V, rounded into their slots;
- attend: attention over the pages, for one new token of each request, for a few drafted ones and
          for prompts; with a window and some first tokens that stay visible, or over everything;
- verify: drafted tokens against the target's probabilities, from given random numbers, and the
          token that follows them.

`draw` takes more of each: one to 64 requests, other head counts and widths, page sizes, lengths
from one token to 131073, windows and sinks, padded steps, vocabularies.
"""
import math
import random

import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
VOCAB = 151936


def listed():
    return [
        # the next token of 24 conversations: tables of up to 64 k tokens, a page taken now and then
        dict(name="map_step_24", op="map", n=24, page=64, longest=65536, most=1, tokens=24),
        # a server takes up waiting prompts, others end or are taken back: 300 requests
        dict(name="map_prompts_300", op="map", n=300, page=64, longest=16384, most=200, tokens=32768),
        # the new rows of 24 conversations
        dict(name="append_step_24", op="append", rows=24, heads=2, dim=256, page=64, type="bf16"),
        # the rows of a long prompt
        dict(name="append_prompt_8001", op="append", rows=8001, heads=2, dim=256, page=64, type="f16"),
        # one user's next token, early in a chat
        dict(name="attend_token_1k", op="attend", n=1, tokens=1, each=1, longest=1025, heads=16, kv_heads=2, dim=256, page=64, type="f16", window=0, sinks=0, gated=False, pad=0),
        # the next token of 24 conversations of any length
        dict(name="attend_serve_24", op="attend", n=24, tokens=24, each=1, longest=65536, heads=16, kv_heads=2, dim=256, page=64, type="bf16", window=0, sinks=0, gated=False, pad=0),
        # one user's next token behind a very long document
        dict(name="attend_long_131073", op="attend", n=1, tokens=1, each=1, longest=131073, heads=16, kv_heads=2, dim=256, page=256, type="bf16", window=0, sinks=0, gated=False, pad=0),
        # five tokens of 16 endless conversations verified at once: a window and the first tokens
        dict(name="attend_drafts_16_window", op="attend", n=16, tokens=80, each=5, longest=65536, heads=16, kv_heads=2, dim=256, page=64, type="f16", window=4096, sinks=4, gated=True, pad=0),
        # a chunk of a prompt behind what is cached of it
        dict(name="attend_chunk_512", op="attend", n=1, tokens=512, each=512, longest=16896, heads=16, kv_heads=2, dim=256, page=64, type="bf16", window=0, sinks=0, gated=True, pad=0),
        # three prompts of one step, with a window
        dict(name="attend_prompts_8001_window", op="attend", n=3, tokens=8001, each=0, longest=8001, heads=16, kv_heads=2, dim=256, page=64, type="f16", window=1024, sinks=4, gated=True, pad=0),
        # one conversation's five drafted tokens, drafted greedily
        dict(name="verify_1x5_greedy", op="verify", n=1, k=5, vocab=VOCAB, sampled=False, ragged=False),
        # five drafted tokens of 24 conversations
        dict(name="verify_24x5", op="verify", n=24, k=5, vocab=VOCAB, sampled=True, ragged=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = {m: max(work(c)[m] for c in listed()) for m in ("bytes", "flops")}
    while True:  # one that costs no more than the listed ones
        c = _draw(rng)
        if all(work(c)[m] <= x for m, x in most.items()):
            return c


def _draw(rng):
    op = rng.choice(["map", "append", "attend", "attend", "attend", "verify"])
    page = rng.choice([32, 64, 64, 128, 256])
    if op == "map":
        n, most = _log(rng, 1, 1000), rng.choice([1, 1, 5, _log(rng, 2, 400)])
        return dict(op=op, n=n, page=page, longest=_log(rng, 32, min(65536, 10_000_000 // n)), most=most, tokens=n * most + rng.randrange(64))
    heads, kv_heads, dim = rng.choice([(16, 2, 256), (16, 2, 256), (32, 8, 128), (28, 4, 128), (8, 1, 64), (6, 6, 128), (12, 2, 256)])
    kind = rng.choice(["f16", "bf16"])
    if op == "append":
        return dict(op=op, rows=_log(rng, 1, 8001), heads=kv_heads, dim=dim, page=page, type=kind)
    if op == "verify":
        return dict(op=op, n=_log(rng, 1, 24), k=rng.choice([0, 1, 2, 3, 4, 5]), vocab=rng.choice([VOCAB, _log(rng, 1000, VOCAB)]),
                    sampled=rng.random() < 0.6, ragged=rng.random() < 0.4)
    window = rng.choice([0, 0, _log(rng, 1, 8192)])
    sinks = rng.choice([0, 4, _log(rng, 1, 300)]) if window else 0
    c = dict(op=op, heads=heads, kv_heads=kv_heads, dim=dim, page=page, type=kind, window=window, sinks=sinks, gated=rng.random() < 0.5)
    if rng.random() < 0.6:  # tokens of many, one or a few drafted ones each
        n, each = _log(rng, 1, 64), rng.choice([1, 1, 1, 2, 5, 8])
        return dict(c, n=n, each=each, tokens=n * each, longest=_log(rng, each, min(131073, 1_500_000 // n)), pad=rng.choice([0, 0, rng.randrange(1, 9)]))
    n = _log(rng, 1, 8)
    tokens = _log(rng, 2 * n, 8001)
    longest = max(tokens, _log(rng, tokens, min(32768, max(tokens, 60_000_000 // tokens))))
    return dict(c, n=n, each=0, tokens=tokens, longest=longest, pad=rng.choice([0, 0, rng.randrange(1, 100)]))


# ---- inputs

class _Draws:
    """Seeded draws on the GPU."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(seed * 1000003 + 29)

    def normal(self, *shape):
        return torch.randn(shape, generator=self.g, device="cuda")

    def uniform(self, *shape):
        return torch.rand(shape, generator=self.g, device="cuda")

    def below(self, most, *shape):
        return torch.randint(0, most, shape, generator=self.g, device="cuda")

    def order(self, n):
        return torch.randperm(n, generator=self.g, device="cuda")


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _prepare_map(c, seed):
    r, d = random.Random(seed * 7919 + 3), _Draws(seed)
    n, page = c["n"], c["page"]
    width = -(-(c["longest"] + c["most"]) // page)
    lens = [_log(r, 1, c["longest"]) for _ in range(n)]
    held = [-(-x // page) for x in lens]
    steps = []
    for turn in range(2):  # what is asked for now, and in the next step
        room, ask = c["tokens"], []
        for i, x in enumerate(lens):
            at = r.random()
            # most go on by some tokens; one ends; one is taken back to half of it
            kept, new = (0, 0) if at < 0.04 else (x // 2, 0) if at < 0.1 else (x, r.randint(1, c["most"]))
            new = min(new, room)
            room -= new
            ask.append((kept, new))
        steps.append((_int32([a for a, _ in ask]), _int32([b for _, b in ask])))
    total = sum(held)
    pages = n * width + 8
    ids = d.order(pages).to(torch.int32)
    at = torch.arange(width, device="cuda")
    held = _int32(held)
    first = torch.cumsum(held, 0) - held
    tables = torch.where(at < held[:, None], ids[(first[:, None] + at).clamp(max=pages - 1)], -1)
    free = torch.cat([ids[total:], ids.new_full((total,), -1)])
    return dict(c, steps=steps, turn=0, tables=tables, held=held, free=free, count=_int32([pages - total]))


def _split(r, total, n):
    """n positive numbers that add up to `total`."""
    cuts = sorted(r.sample(range(1, total), n - 1))
    return [b - a for a, b in zip([0] + cuts, cuts + [total])]


def _prepare_attend(c, seed):
    r, d = random.Random(seed * 7919 + 5), _Draws(seed)
    n, page, heads, kv, dim = c["n"], c["page"], c["heads"], c["kv_heads"], c["dim"]
    new = [c["each"]] * n if c["each"] else _split(r, c["tokens"], n)
    lens = [c["longest"] if i == 0 else max(q, _log(r, min(q + 64, c["longest"]), c["longest"])) for i, q in enumerate(new)]
    if c["each"] == 0 and c["longest"] == c["tokens"]:  # whole prompts, nothing cached before
        lens = list(new)
    held = [-(-x // page) for x in lens]
    pages = sum(held) + 3
    ids, at = d.order(pages).to(torch.int32), torch.arange(max(held), device="cuda")
    count = _int32(held)
    first = torch.cumsum(count, 0) - count
    tables = torch.where(at < count[:, None], ids[(first[:, None] + at).clamp(max=pages - 1)], -1)
    t = TYPES[c["type"]]
    k, v = (torch.empty(pages, page, kv, dim, dtype=t, device="cuda").normal_(generator=d.g) for _ in range(2))
    rows = c["tokens"] + c["pad"]
    # queries of differing reach: some heads look at few keys, others at all
    q = d.normal(rows, heads, 2 * dim if c["gated"] else dim) * torch.exp(0.5 * d.normal(1, heads, 1))
    starts = [0]
    for x in new:
        starts.append(starts[-1] + x)
    return dict(c, q=q[..., :dim], k=k, v=v, tables=tables, lens=_int32(lens), starts=_int32(starts), new=new, keys=lens,
                scale=dim ** -0.5, out=torch.zeros(rows, heads, dim, device="cuda"))


def prepare(case, seed):
    c, d = case, _Draws(seed)
    if c["op"] == "map":
        return _prepare_map(c, seed)
    if c["op"] == "attend":
        return _prepare_attend(c, seed)
    if c["op"] == "append":
        rows, heads, dim, page, t = c["rows"], c["heads"], c["dim"], c["page"], TYPES[c["type"]]
        pages = -(-rows // page) + max(4, rows // page // 8)
        slots = d.order(pages * page)[:rows] if rows < 256 else (d.order(pages)[:, None] * page + torch.arange(page, device="cuda")).reshape(-1)[:rows]
        # the projection's output: q, k and v of a token beside each other
        x = d.normal(rows, 4 * heads, dim)
        k, v = (torch.zeros(pages, page, heads, dim, dtype=t, device="cuda") for _ in range(2))
        return dict(c, new_k=x[:, 2 * heads:3 * heads], new_v=x[:, 3 * heads:], slots=slots.clone(), k=k, v=v)
    n, k, vocab = c["n"], c["k"], c["vocab"]
    # a temperature of one, and what is hardly likely cut off
    logits = 3 * d.normal(n, k + 1, vocab)
    p = torch.softmax(logits, -1)
    p = torch.where(p < 1e-6, 0.0, p)
    p = p / p.sum(-1, keepdim=True)
    guess = torch.softmax(logits[:, :k] + 0.5 * d.normal(n, k, vocab), -1)
    if c["sampled"]:
        drafts = (torch.log(guess) - torch.log(-torch.log(d.uniform(n, k, vocab).clamp_(1e-9, 1 - 1e-7)))).argmax(-1) if k else d.below(1, n, k)
    else:
        drafts = guess.argmax(-1) if k else d.below(1, n, k)
    return dict(c, target=p, guess=guess if c["sampled"] else None, drafts=drafts.to(torch.int32), u=d.uniform(n, k + 1),
                counts=d.below(k + 1, n).to(torch.int32) if c["ragged"] else None)


# ---- the framework's calls

def _run_own(s):
    import paramecia_amd as pk
    if s["op"] == "map":
        lens, add = s["steps"][s["turn"] % 2]
        s["turn"] += 1
        m = pk.map_pages(lens, add, s["tables"], s["held"], s["free"], s["count"], s["page"], s["tokens"])
        return dict(slots=m.slots, positions=m.positions, starts=m.starts, totals=m.totals, status=m.status, **_map_state(s))
    if s["op"] == "append":
        pk.append_pages(s["new_k"], s["new_v"], s["slots"], s["k"], s["v"])
        return s["k"], s["v"]
    if s["op"] == "attend":
        return pk.attend_pages(s["q"], s["k"], s["v"], s["tables"], s["lens"], s["scale"], starts=None if s["each"] == 1 and s["pad"] == 0 else s["starts"],
                               window=s["window"], sinks=s["sinks"], out=s["out"])
    return pk.verify_drafts(s["target"], s["drafts"], s["u"], draft_probs=s["guess"], n_drafts=s["counts"])


def _map_state(s):
    return dict(tables=s["tables"], held=s["held"], free=s["free"], count=s["count"])


# ---- the plain forms

def _map_plain(s):
    lens, add = s["steps"][s["turn"] % 2]
    s["turn"] += 1
    tables, held, free, page, most = s["tables"], s["held"], s["free"], s["page"], s["tokens"]
    total = lens + add
    need = (total + page - 1) // page
    give, take = (held - need).clamp(min=0), (need - held).clamp(min=0)
    at = torch.arange(tables.shape[1], device="cuda")
    given = (at >= need[:, None]) & (at < held[:, None])
    taken = (at >= held[:, None]) & (at < need[:, None])
    starts = torch.cat([add.new_zeros(1), torch.cumsum(add, 0)])
    stack = s["count"] + give.sum()  # the stack's height with the pages that come back on it
    ok = (need.max() <= tables.shape[1]) & (take.sum() <= stack) & (starts[-1] <= most) & (stack <= free.shape[0]) & (lens.min() >= 0) & (add.min() >= 0)
    order = torch.cumsum(given.reshape(-1), 0) - 1 + s["count"]
    back = torch.where(given.reshape(-1) & ok, order, free.shape[0])
    free = torch.cat([free, free[:1]]).scatter_(0, back, tables.reshape(-1))[:-1]
    order = stack - torch.cumsum(taken.reshape(-1), 0)
    mine = torch.where(taken.reshape(-1) & ok, free[order.clamp(0, free.shape[0] - 1)], tables.reshape(-1)).view_as(tables)
    s["free"].copy_(free)
    s["tables"].copy_(mine)
    s["held"].copy_(torch.where(ok, need, held))
    s["count"].copy_(torch.where(ok, stack - take.sum(), s["count"]))
    starts = torch.where(ok, starts, 0).to(torch.int32)
    t = torch.arange(most, dtype=torch.int32, device="cuda")
    b = (torch.searchsorted(starts, t, right=True) - 1).clamp(max=lens.shape[0] - 1)
    live = t < starts[-1]
    position = torch.where(live, lens[b] + t - starts[b], 0)
    slots = torch.where(live, mine[b, (position // page).clamp(max=mine.shape[1] - 1)].long() * page + position % page, -1)
    return dict(slots=slots, positions=position.to(torch.int32), starts=starts, totals=torch.where(ok, total, lens), status=(1 - ok.int()).view(1), **_map_state(s))


def _append_plain(s):
    t = TYPES[s["type"]]
    s["k"].view(-1, s["heads"], s["dim"])[s["slots"]] = s["new_k"].to(t)
    s["v"].view(-1, s["heads"], s["dim"])[s["slots"]] = s["new_v"].to(t)
    return s["k"], s["v"]


def _softmax_plain(score, seen):
    score = torch.where(seen, score.clamp(-100, 100), -math.inf)
    top = score.amax(-1, keepdim=True)
    w = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    return w / w.sum(-1, keepdim=True).clamp(min=1e-30)


def _tokens_plain(s):
    """A few queries of each request, all requests at once: the keys that they see are gathered first."""
    n, each, kv, dim, window, sinks = s["n"], s["each"], s["kv_heads"], s["dim"], s["window"], s["sinks"]
    group = s["heads"] // kv
    if window and max(s["keys"]) > window + each + sinks:
        near = s["lens"][:, None] - (window + each - 1) + torch.arange(window + each - 1, device="cuda")
        at = torch.cat([torch.arange(sinks, device="cuda").expand(n, sinks), torch.where(near >= sinks, near, -1)], 1)
    else:
        at = torch.arange(max(s["keys"]), device="cuda").expand(n, -1)
    live = (at >= 0) & (at < s["lens"][:, None])
    at = torch.where(live, at, 0)
    rows = torch.gather(s["tables"], 1, at // s["page"]).long() * s["page"] + at % s["page"]
    k, v = (x.view(-1, kv, dim)[rows].transpose(1, 2).float() for x in (s["k"], s["v"]))  # [n, kv, keys, dim]
    q = s["q"][:n * each].reshape(n, each, kv, group, dim).permute(0, 2, 1, 3, 4).reshape(n, kv, each * group, dim)
    position = s["lens"][:, None] - each + torch.arange(each, device="cuda")
    seen = live[:, None] & (at[:, None] <= position[..., None])
    if window:
        seen &= (at[:, None] > position[..., None] - window) | (at[:, None] < sinks)
    seen = seen[:, None, :, None].expand(n, 1, each, group, -1).reshape(n, 1, each * group, -1)
    w = _softmax_plain((q @ k.transpose(2, 3).contiguous()) * s["scale"], seen)
    out = (w @ v).view(n, kv, each, group, dim).permute(0, 2, 1, 3, 4)
    s["out"][:n * each] = out.reshape(n * each, s["heads"], dim)
    return s["out"]


def _prompts_plain(s):
    kv, dim, page, first = s["kv_heads"], s["dim"], s["page"], 0
    for i, (new, keys) in enumerate(zip(s["new"], s["keys"])):
        at = torch.arange(keys, device="cuda")
        rows = s["tables"][i, at // page].long() * page + at % page
        k, v = (x.view(-1, kv, dim)[rows].transpose(0, 1).float() for x in (s["k"], s["v"]))  # [kv, keys, dim]
        q = s["q"][first:first + new].reshape(new, kv, -1, dim).transpose(0, 1).reshape(kv, -1, dim)
        position = keys - new + torch.arange(new, device="cuda")[:, None]
        seen = at <= position
        if s["window"]:
            seen &= (at > position - s["window"]) | (at < s["sinks"])
        seen = seen.repeat_interleave(s["heads"] // kv, 0)
        w = _softmax_plain((q @ k.transpose(1, 2).contiguous()) * s["scale"], seen)
        s["out"][first:first + new] = (w @ v).view(kv, new, -1, dim).transpose(0, 1).reshape(new, s["heads"], dim)
        first += new
    return s["out"]


def _verify_plain(s):
    p, q, k = s["target"], s["guess"], s["k"]
    b = torch.arange(s["n"], device="cuda")
    i = torch.arange(k, device="cuda")
    counts = torch.full_like(b, k) if s["counts"] is None else s["counts"].long()
    x = s["drafts"].long()
    mine = torch.gather(p[:, :k], 2, x[..., None])[..., 0].double()
    theirs = torch.ones_like(mine) if q is None else torch.gather(q, 2, x[..., None])[..., 0].double()
    ok = (s["u"][:, :k].double() * theirs < mine) & (i < counts[:, None])
    accepted = torch.cumprod(ok.long(), 1).sum(1)
    row = p[b, accepted].double()  # in 64 bits: a sum's border decides on a token
    if k:
        stopped, last = accepted < counts, accepted.clamp(max=k - 1)
        away = torch.nn.functional.one_hot(x[b, last], s["vocab"]).double() if q is None else q[b, last].double()
        rest = torch.where(stopped[:, None], (row - away).clamp(min=0), row)
        row = torch.where((rest > 0).any(1, keepdim=True), rest, row)
    run = torch.cumsum(row, 1)
    token = (run > s["u"][:, k:].double() * run[:, -1:]).long().argmax(1)
    j = torch.arange(k + 1, device="cuda")
    drafted = torch.cat([x, x.new_zeros(s["n"], 1)], 1)
    tokens = torch.where(j < accepted[:, None], drafted, torch.where(j == accepted[:, None], token[:, None], -1))
    return tokens.to(torch.int32), accepted.to(torch.int32)


def run(state):
    if own:
        return _run_own(state)
    if state["op"] == "attend":
        return (_tokens_plain if state["each"] and state["each"] <= 16 else _prompts_plain)(state)
    return {"map": _map_plain, "append": _append_plain, "verify": _verify_plain}[state["op"]](state)


def _seen(position, window, sinks):
    """How many keys a query at `position` sees."""
    if not window or position + 1 <= window:
        return position + 1
    return window + min(sinks, position + 1 - window)


def work(case):
    c = case
    if c["op"] == "map":
        return {"bytes": 4 * 7 * c["n"] + 12 * c["tokens"] + 8 * c["n"] * c["most"] // c["page"], "flops": 10 * (c["n"] + c["tokens"])}
    if c["op"] == "append":
        m = 2 * c["rows"] * c["heads"] * c["dim"]
        return {"bytes": 6 * m + 8 * c["rows"], "flops": m}
    if c["op"] == "verify":
        rows = c["n"] * (1.0 + c["sampled"])
        return {"bytes": 4 * rows * c["vocab"] + 16 * c["n"] * (c["k"] + 1), "flops": 4 * c["n"] * c["vocab"]}
    # the first request has the longest length, the others' are drawn over their logarithm; the keys that a request's queries see are read once
    n, w, s, each = c["n"], c["window"], c["sinks"], c["each"] or c["tokens"] / c["n"]
    cap = w + s + each - 1 if w else math.inf  # keys that a request's queries see at most
    low, high = (each, each) if not c["each"] and c["longest"] == c["tokens"] else (min(each + 64, c["longest"]), c["longest"])
    spread = math.log(high / low)
    mean = min(low, cap) if spread < 1e-6 else low if cap <= low else (min(cap, high) - low + (cap * math.log(high / cap) if cap < high else 0)) / spread
    keys = min(high, cap) + (n - 1) * mean
    pairs = keys * each if each <= 16 else n * each * (_seen(high - 1, w, s) + _seen(max(0, high - each), w, s)) / 2
    return {"bytes": 4 * keys * c["kv_heads"] * c["dim"] + 8 * c["tokens"] * c["heads"] * c["dim"], "flops": 4 * pairs * c["heads"] * c["dim"]}


# ---- the definitions in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return {"map": _map_exact, "append": _append_exact, "attend": _attend_exact, "verify": _verify_exact}[case["op"]](s)


def _map_exact(s):
    """Request by request, with the free pages as a list."""
    lens, add = (x.tolist() for x in s["steps"][0])
    tables, held, free = s["tables"].tolist(), s["held"].tolist(), s["free"].tolist()
    stack, page = free[:s["count"].item()], s["page"]
    for b, (x, y) in enumerate(zip(lens, add)):
        stack += tables[b][-(-(x + y) // page):held[b]]
    free[:len(stack)] = stack
    slots, positions, starts = [], [], [0]
    for b, (x, y) in enumerate(zip(lens, add)):
        need = -(-(x + y) // page)
        for j in range(held[b], need):
            tables[b][j] = stack.pop()
        held[b] = need
        positions += range(x, x + y)
        slots += [tables[b][p // page] * page + p % page for p in range(x, x + y)]
        starts.append(starts[-1] + y)
    behind = s["tokens"] - len(slots)
    t = lambda v, dtype=torch.int32: torch.tensor(v, dtype=dtype, device="cuda")  # noqa: E731
    return dict(slots=t(slots + [-1] * behind, torch.int64), positions=t(positions + [0] * behind), starts=t(starts), totals=t([x + y for x, y in zip(lens, add)]),
                status=t([0]), tables=t(tables), held=t(held), free=t(free), count=t([len(stack)]))


def _append_exact(s):
    got = []
    for plane, new in ((s["k"], s["new_k"]), (s["v"], s["new_v"])):
        x = plane.double().flatten(0, 1)
        x.index_copy_(0, s["slots"], new.double().contiguous())
        got.append(x.view(plane.shape))
    return tuple(got)


def _attend_exact(s):
    out, group, starts = s["out"].double(), s["heads"] // s["kv_heads"], s["starts"].tolist()
    for i, (first, end) in enumerate(zip(starts, starts[1:])):
        length = s["keys"][i]
        pages = s["tables"][i, :-(-length // s["page"])].long()
        j = torch.arange(length, device="cuda")
        for h in range(s["kv_heads"]):
            k, v = (x[pages, :, h].double().flatten(0, 1)[:length] for x in (s["k"], s["v"]))
            for a in range(first, end, 1024):  # some queries at a time
                z = min(end, a + 1024)
                position = torch.arange(length - (end - a), length - (end - z), device="cuda")[:, None]
                hidden = j > position
                if s["window"]:
                    hidden = hidden | ((j <= position - s["window"]) & (j >= s["sinks"]))
                for g in range(h * group, (h + 1) * group):
                    score = torch.clamp(s["scale"] * (s["q"][a:z, g].double() @ k.T), -100, 100).masked_fill(hidden, -math.inf)
                    out[a:z, g] = torch.softmax(score, -1) @ v
    return out


def _verify_exact(s):
    tokens, accepted = [], []
    for b in range(s["n"]):
        count = s["k"] if s["counts"] is None else int(s["counts"][b])
        drafts, u = s["drafts"][b].tolist(), s["u"][b].tolist()
        taken = 0
        while taken < count and u[taken] * (1.0 if s["guess"] is None else s["guess"][b, taken, drafts[taken]].item()) < s["target"][b, taken, drafts[taken]].item():
            taken += 1
        row = s["target"][b, taken].double().cpu()
        if taken < count:
            rest = row.clone()
            if s["guess"] is None:
                rest[drafts[taken]] = max(0.0, row[drafts[taken]].item() - 1)
            else:
                rest = torch.maximum(row - s["guess"][b, taken].double().cpu(), torch.zeros(()).double())
            row = rest if rest.sum() > 0 else row
        total = torch.cumsum(row, 0)
        token = int(torch.searchsorted(total, u[s["k"]] * total[-1].item(), right=True))
        tokens.append(drafts[:taken] + [token] + [-1] * (s["k"] - taken))
        accepted.append(taken)
    t = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    return t(tokens), t(accepted)
