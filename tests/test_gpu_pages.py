"""The operators over pages that tables on the device name, against plain forms in 64 bits
(pages_checks.py): request lengths to pages and slots, new rows into their slots, attention
over block tables with windows and sinks, drafted tokens; and a serving step of all of them.
The reference has these steps for one sequence (paramecia-model/src/qwen3_next.rs:431-509,
2492-2605, 2755-2762)."""
import math
import random
import sys

import pytest

torch = pytest.importorskip("torch")

from pages_checks import attend64, map_pages64, verify64  # noqa: E402

pytestmark = pytest.mark.gpu

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def say(*a):
    print(*a, flush=True)
    sys.stdout.flush()


@pytest.fixture(scope="module")
def pk():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import paramecia_amd
    paramecia_amd.lib()
    return paramecia_amd


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------ pages from lengths
class Tables:
    """Requests that hold some pages, on the device and as lists."""

    def __init__(self, r, n, width, page, spare, lens):
        self.page, self.lens = page, lens
        self.held = [-(-x // page) for x in lens]
        ids = list(range(sum(self.held) + spare))
        r.shuffle(ids)
        self.rows = []
        for h in self.held:
            self.rows.append([ids.pop() for _ in range(h)] + [-7] * (width - h))
        self.stack = ids
        self.capacity = sum(self.held) + spare
        self.t, self.h = i32(self.rows), i32(self.held)
        self.free = i32(self.stack + [-9] * (self.capacity - len(self.stack)))
        self.count = i32([len(self.stack)])

    def step(self, pk, lens, add, max_tokens, capacity=None, out=None):
        got = pk.map_pages(i32(lens), i32(add), self.t, self.h, self.free, self.count, self.page, max_tokens, out=out)
        want = map_pages64(lens, add, self.rows, self.held, self.stack, self.page, self.capacity, max_tokens)
        status, self.rows, self.held, self.stack, slots, positions, starts, totals = want
        assert got.status.tolist() == [status]
        assert self.count.tolist() == [len(self.stack)] and self.h.tolist() == self.held
        assert self.free.tolist()[:len(self.stack)] == self.stack
        for mine, theirs, h in zip(self.t.tolist(), self.rows, self.held):
            assert mine[:h] == theirs[:h]
        assert got.starts.tolist() == starts and got.totals.tolist() == totals
        assert got.slots.dtype is torch.int64 and got.slots.tolist() == slots and got.positions.tolist() == positions
        return got


@pytest.mark.parametrize("n,longest,page,most,max_tokens", [
    (1, 1, 32, 1, 1),
    (24, 5000, 64, 1, 24),
    (64, 700, 32, 40, 64 * 40 + 5),      # rows behind the last request
    (300, 900, 64, 100, 20000),          # slots by a launch of their own
    (1024, 300, 32, 3, 4096),
    (1025, 300, 32, 3, 4097),            # more requests than threads
    (4500, 100, 64, 5, 4500 * 5),        # starts that do not fit LDS
    (3, 70000, 1024, 9000, 30000),       # one request takes many pages
    (256, 2000, 64, 4, 1024),            # a thread a request, slots in the same launch
    (257, 2000, 32, 4, 1024),
    (256, 2000, 32, 5, 1025),            # and in one of their own
    (1025, 100, 32, 1, 1000),
    (4097, 70, 32, 1, 700),              # starts that do not fit LDS, few rows
    (5000, 70, 32, 0, 0),
])
def test_map_over_steps(pk, n, longest, page, most, max_tokens):
    say("map", n, longest, page, most)
    r = random.Random(n)
    lens = [r.randint(0, longest) for _ in range(n)]
    width = -(-(longest + 4 * most) // page) + 1
    t = Tables(r, n, width, page, spare=2 * n + 4 * n * most // page + 8, lens=lens)
    out = None
    for _ in range(4):
        keep = [x if r.random() < 0.8 else r.randint(0, x) for x in lens]  # rewinds, and ends
        add, room = [], max_tokens
        for _ in keep:
            a = min(room, r.choice([0, 1, most, r.randint(0, most)]))
            room -= a
            add.append(a)
        out = t.step(pk, keep, add, max_tokens, out=out)
        lens = [a + b for a, b in zip(keep, add)]


def test_map_refuses_as_a_whole(pk):
    r = random.Random(3)
    t = Tables(r, 4, 4, 32, spare=2, lens=[40, 0, 96, 5])
    ok = [40, 0, 96, 5]
    t.step(pk, ok, [0, 65, 0, 0], 100)                       # three pages of two
    t.step(pk, ok, [33, 32, 0, 28], 200)                     # one page too many, by all of them
    t.step(pk, ok, [0, 0, 33, 0], 100)                       # five pages of a table of four
    t.step(pk, ok, [1, 1, 1, 1], 3)                          # more rows than the step has
    t.step(pk, [-1, 0, 96, 5], [0, 0, 0, 0], 100)
    t.step(pk, ok, [0, -1, 0, 0], 100)
    t.step(pk, [2 ** 31 - 1, 0, 96, 5], [1, 0, 0, 0], 100)   # a sum past 32 bits
    assert t.held == [2, 0, 3, 1] and len(t.stack) == 2
    t.step(pk, ok, [24, 64, 0, 0], 100)                      # and what fits still goes
    t.step(pk, [0, 0, 0, 0], [0, 0, 0, 0], 0)                # all end; a step without rows
    assert len(t.stack) == t.capacity
    t.count += 1                                             # a stack higher than its memory
    got = pk.map_pages(i32(ok), i32([0] * 4), t.t, t.h, t.free, t.count, 32, 8)
    assert got.status.tolist() == [3] and t.h.tolist() == [0] * 4


# ------------------------------------------------------------------ rows into slots
@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("n,heads,dim,strided", [(1, 2, 256, False), (24, 2, 256, True), (1001, 8, 128, True),
                                                 (33, 1, 64, False), (7, 3, 20, True), (5, 1, 7, False)])
def test_append(pk, kind, n, heads, dim, strided):
    say("append", kind, n, heads, dim)
    g, t = gen(n), TYPES[kind]
    pages, page = -(-n // 32) + 3, 32
    x = torch.randn(n, 3 * heads, dim, device="cuda", generator=g) * torch.exp(3 * torch.randn(n, 1, 1, device="cuda", generator=g))
    x[0, 0, :4] = torch.tensor([math.inf, -math.inf, 1e30, 65519.996])
    k, v = x[:, :heads], x[:, heads:2 * heads]
    if not strided:
        k, v = k.contiguous(), v.contiguous()
    kp, vp = (torch.randn(pages, page, heads, dim, device="cuda", generator=g).to(t) for _ in range(2))
    slots = torch.randperm(pages * page, device="cuda", generator=g)[:n].clone()
    if n > 4:
        slots[2] = -1
        slots[3] = -5
    want = [p.clone().view(-1, heads, dim) for p in (kp, vp)]
    live = slots >= 0
    for p, new in zip(want, (k, v)):
        p[slots[live]] = new[live].to(t)
    pk.append_pages(k, v, slots, kp, vp)
    for p, w in zip((kp, vp), want):
        assert torch.equal(p.view(-1, heads, dim).view(torch.int16), w.view(torch.int16))
    assert pk.lib().pkv_device_status() == 0


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_append_rounds_as_the_cache(pk, kind):
    g = gen(5)
    q = pk.KvCacheQuantization.F16 if kind == "f16" else pk.KvCacheQuantization.BF16
    cache = pk.PreallocatedQuantizedKvCache(1, 2, 64, 64, q)
    bits = torch.randint(-2 ** 31, 2 ** 31 - 1, (1, 2, 64, 64), device="cuda", generator=g).to(torch.int32)
    x = bits.view(torch.float32)  # any value: subnormal, infinite, far past the type
    x = torch.where(torch.isnan(x), 1.0, x)
    cache.append_quantized(x, -x)
    want = [b.view(TYPES[kind]).view(64, 2, 64) for b in cache.raw_bytes()]
    kp, vp = (torch.zeros(2, 32, 2, 64, dtype=TYPES[kind], device="cuda") for _ in range(2))
    rows = x[0].transpose(0, 1)
    pk.append_pages(rows, -rows, torch.arange(64, device="cuda"), kp, vp)
    for p, w in zip((kp, vp), want):
        assert torch.equal(p.view(64, 2, 64).view(torch.int16), w.view(torch.int16))


def test_append_past_the_pages_is_reported(pk):
    kp, vp = (torch.ones(1, 32, 1, 64, dtype=torch.float16, device="cuda") for _ in range(2))
    k = torch.zeros(3, 1, 64, device="cuda")
    pk.append_pages(k, k, torch.tensor([32, 1 << 40, 5], device="cuda"), kp, vp)
    assert pk.lib().pkv_device_status() != 0 and b"slot" in pk.lib().pkv_last_error()
    assert pk.lib().pkv_device_status() == 0
    assert int((kp == 0).sum()) == 64 and int((kp[0, 5] == 0).sum()) == 64


# ------------------------------------------------------------------ attention
class Case:
    """Requests over pages in any order: lens and new rows as lists."""

    def __init__(self, seed, lens, new, heads, kv, dim, kind, page=32, pad=0, spread=1.0, gated=False, spare=2):
        g = gen(seed)
        self.lens, self.new, self.heads = lens, new, heads
        held = [-(-x // page) for x in lens]
        n_pages = sum(held) + spare
        order = torch.randperm(n_pages, generator=g, device="cuda").tolist()
        width = max(max(held), 1) + 1
        self.tables = i32([[order.pop() for _ in range(h)] + [-1] * (width - h) for h in held])
        self.k, self.v = (torch.randn(n_pages, page, kv, dim, device="cuda", generator=g).to(TYPES[kind]) for _ in range(2))
        rows = sum(new) + pad
        q = torch.randn(rows, heads, 2 * dim if gated else dim, device="cuda", generator=g) * spread
        self.q = q[..., :dim]
        self.starts = i32([sum(new[:i]) for i in range(len(new) + 1)])
        self.out = torch.randn(rows, heads, dim, device="cuda", generator=g)
        self.scale = dim ** -0.5
        self.page = page

    def run(self, pk, window=0, sinks=0, starts=True, out=None):
        return pk.attend_pages(self.q, self.k, self.v, self.tables, i32(self.lens), self.scale, starts=self.starts if starts else None,
                               window=window, sinks=sinks, out=self.out.clone() if out is None else out)

    def check(self, pk, window=0, sinks=0, starts=True):
        want, bound = attend64(self.q, self.k, self.v, self.tables, self.lens, self.scale, self.starts, window, sinks, self.out)
        got = self.run(pk, window, sinks, starts)
        assert torch.isfinite(got).all()
        off = (got.double() - want).abs()
        behind = int(self.starts[-1])
        assert torch.equal(got[behind:], self.out[behind:])
        worst = float((off / bound.clamp(min=1e-30))[:behind].max()) if behind else 0.0
        say("   worst share of the bound", round(worst, 4))
        assert worst <= 1.0
        return got


SHAPES = [(16, 2, 256), (8, 1, 64), (32, 8, 128), (28, 4, 128), (6, 6, 128), (12, 2, 256), (2, 2, 64)]


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv,dim", SHAPES)
def test_tokens(pk, kind, heads, kv, dim):
    """One token each: no key, one, blocks that end anywhere, more than a workgroup's share."""
    say("tokens", kind, heads, kv, dim)
    Case(1, [1, 0, 31, 32, 33, 64, 65, 100, 1000, 2, 4097], [1] * 11, heads, kv, dim, kind).check(pk, starts=False)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 4), (31, 0), (32, 1), (33, 33), (64, 100), (300, 4), (5000, 4), (96, 2000)])
def test_windows(pk, kind, window, sinks):
    say("windows", kind, window, sinks)
    for heads, kv, dim in ((16, 2, 256), (8, 1, 64)):
        Case(2, [1, 0, 31, 33, 300, 1000, 2049], [1] * 7, heads, kv, dim, kind, page=64).check(pk, window, sinks)
    Case(3, [40, 700, 9, 300], [40, 13, 9, 1], 28, 4, 128, kind, page=64, pad=3).check(pk, window, sinks)
    Case(4, [600, 200], [500, 200], 16, 2, 256, kind).check(pk, window, sinks)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv,dim", SHAPES)
@pytest.mark.parametrize("lens,new", [
    ([5, 100, 33, 2000], [5, 5, 5, 5]),           # drafted tokens
    ([1, 0, 77, 640], [1, 0, 8, 3]),              # and requests without any
    ([130, 17, 1000], [130, 17, 150]),            # prompts
    ([3, 2, 0, 50], [5, 2, 4, 7]),                # more rows than keys: the first see nothing
])
def test_rows(pk, kind, heads, kv, dim, lens, new):
    say("rows", kind, heads, kv, dim, lens, new)
    Case(5, lens, new, heads, kv, dim, kind, pad=2, gated=True).check(pk)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv,dim", [(64, 1, 64), (20, 1, 128), (96, 2, 256), (33, 11, 64)])
def test_heads_of_a_kv_head(pk, kind, heads, kv, dim):
    """More query heads than a row tile holds, and numbers that no tile divides by."""
    say("heads", kind, heads, kv, dim)
    Case(19, [70, 1, 0, 333], [1, 1, 1, 1], heads, kv, dim, kind).check(pk, 40, 2)
    Case(20, [70, 500], [3, 41], heads, kv, dim, kind).check(pk)


def test_largest_window_and_sinks(pk):
    """A window and sinks as large as they can be see everything."""
    c = Case(21, [300, 5, 0, 90], [20, 5, 3, 90], 16, 2, 256, "f16")
    want = c.run(pk)
    for window, sinks in ((2 ** 31 - 1, 0), (2 ** 31 - 1, 2 ** 31 - 1), (1, 2 ** 31 - 1), (7, 300)):
        assert torch.equal(c.run(pk, window, sinks), want)
    c = Case(22, [300, 5, 0, 90], [1] * 4, 16, 2, 256, "bf16")
    want = c.run(pk)
    for window, sinks in ((2 ** 31 - 1, 0), (2 ** 31 - 1, 2 ** 31 - 1), (1, 2 ** 31 - 1)):
        assert torch.equal(c.run(pk, window, sinks), want)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("new", [1, 25])
def test_queries_that_are_no_numbers(pk, kind, new):
    """NaN makes its own row NaN, an infinite one scores that are clamped or NaN; zeros weigh all
    keys alike. Other rows keep their bits where no piece is made again, their values where one is."""
    c = Case(23, [200, 150], [new, new], 16, 2, 256, kind)
    c.q = c.q.clone()
    clean = c.run(pk)
    c.q[0, 3, 7] = math.nan
    c.q[new, 11] = 0
    got = c.run(pk)
    assert torch.isnan(got[0, 3]).all()
    keep = torch.ones_like(got, dtype=torch.bool)
    keep[0, 3], keep[new, 11] = False, False
    assert torch.isfinite(got[keep]).all() and ((got - clean)[keep].abs() <= 1e-5).all()
    p = 150 - new
    rows = [int(c.tables[1, j // c.page]) * c.page + j % c.page for j in range(p + 1)]
    mean = c.v.view(-1, 2, 256)[rows, 1].double().mean(0)
    assert ((got[new, 11].double() - mean).abs() <= 1e-5).all()


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("spread", [0.01, 4.0, 40.0])
def test_scores_small_and_clamped(pk, kind, spread):
    """Scores near nothing, dominant keys, and many past the clamp at 100."""
    say("spread", kind, spread)
    c = Case(6, [700, 90, 2100], [1, 1, 1], 16, 2, 256, kind, spread=spread)
    c.check(pk, starts=False)
    Case(7, [300, 90], [200, 30], 16, 2, 256, kind, spread=spread).check(pk)


def parts(x, n, kind):
    """x as the sum of n roundings to kind, in 64 bits."""
    total = torch.zeros_like(x)
    for _ in range(n):
        total += (x - total).to(TYPES[kind]).double()
    return total


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("new", [1, 3, 5, 60])
@pytest.mark.parametrize("top", [0.5, 16.0])
def test_precision_of_queries_and_weights(pk, kind, dim, new, top):
    """Keys and values that are unit vectors: a score is one query element, an output one weight, so
    that what is off is the roundings alone and a part of a query or a weight less would show.

    In half steps of f32 (E), scores of at most `top` in log2 units: a query's element is off by 2
    (its factor and the product) and 4 (its parts, F16's 22 bits), a score by 3 more (a part's product at a time) and
    the exponent's difference by 2 more: 11 top E, times ln 2 below 8 top E of a weight, 2 of exp2, 4 of the
    weight's parts, 3 of its sum over parts. The sum below it: 8 top + 2 each, a lane adds 8 weights a
    block of 32 keys and four lanes meet: keys / 4 + 2. A larger maximum and a join: 4 a block and 8; the
    quotient 4. F16's weights, of 2048 and more for the largest, end at 2^-25: 2^-36 of the sum."""
    say("precision", kind, dim, new, top)
    lens = [64, 60, 64]
    c = Case(25, lens, [new] * 3, 8, 1, dim, kind)
    c.k.zero_()
    for b, length in enumerate(lens):
        for j in range(length):
            c.k[int(c.tables[b, j // 32]), j % 32, 0, j] = 1
    c.v = c.k.clone()
    unit = c.scale * math.log2(math.e)
    c.q = (torch.rand(c.q.shape, device="cuda", generator=gen(3)) * 2 - 1).mul(top / unit)
    want, _ = attend64(c.q, c.k, c.v, c.tables, lens, c.scale, c.starts, 0, 0, c.out)
    bound = (16 * top + 45 + 64 / 4 + 4 * 3) * 2.0 ** -24 * want + 2.0 ** -36
    got = c.run(pk)
    off = (got.double() - want).abs()
    say("   worst share of the bound", round(float((off / bound).max()), 3))
    assert (off <= bound).all()
    # the bound would see a part less of the weights (of few bits for small scores), or of the queries
    few = 1 if kind == "f16" else 2
    if top < 1:
        total = parts(want / want.amax(-1, keepdim=True), few, kind) * want.amax(-1, keepdim=True)
        assert ((total - want).abs() > bound).any()
    else:
        c.q = parts(c.q.double() * unit, few, kind) / unit
        less, _ = attend64(c.q, c.k, c.v, c.tables, lens, c.scale, c.starts, 0, 0, c.out)
        assert ((less - want).abs() > bound).any()


def mix(seed):
    """Requests, heads, pages and masks drawn together."""
    r = random.Random(seed)
    kv, group = r.choice([1, 1, 2, 2, 3, 8]), r.choice([1, 2, 3, 4, 7, 8, 8, 16, 20])
    dim, kind, page = r.choice([64, 128, 256]), r.choice(["f16", "bf16"]), r.choice([32, 64, 128, 512])
    most = r.choice([1, 6, 30, 300])
    n = r.choice([1, 2, 3, 7, 24, 64, 65, 90]) if most < 10 else r.choice([1, 2, 5, 9])
    longest = r.choice([3, 70, 700, 3000])
    new = [1 if most == 1 else r.randrange(0, most + 1) for _ in range(n)]
    lens = [(m if r.random() < 0.85 else 0) + r.randrange(0, longest) for m in new]
    window = r.choice([0, 0, 1, 5, 31, 32, 33, 200, 1000])
    return lens, new, group * kv, kv, dim, kind, page, window, r.choice([0, 1, 4, 40, 300])


@pytest.mark.parametrize("seed", range(40))
def test_mixes(pk, seed):
    lens, new, heads, kv, dim, kind, page, window, sinks = mix(seed)
    say("mix", seed, len(lens), sum(lens), sum(new), heads, kv, dim, kind, page, window, sinks)
    c = Case(seed, lens, new, heads, kv, dim, kind, page=page, pad=seed % 3 + 1, spread=[0.2, 1, 6][seed % 3], gated=seed % 2 == 0)
    got = c.check(pk, window, sinks)
    assert torch.equal(c.run(pk, window, sinks), got)


@pytest.mark.parametrize("kind,mag", [("f16", 6e4), ("f16", 1e-6), ("bf16", 1e30), ("bf16", 1e-30)])
def test_values_near_the_ends_of_their_type(pk, kind, mag):
    c = Case(8, [500, 40], [1, 1], 16, 2, 256, kind)
    c.v = (torch.rand(c.v.shape, device="cuda", generator=gen(1)) * 2 - 1).mul(mag).to(TYPES[kind])
    c.check(pk, starts=False)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf, 65504.0])
@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("dim,new", [(256, 1), (64, 1), (128, 9), (256, 40)])
def test_what_is_not_seen_may_be_anything(pk, kind, bad, dim, new):
    """Rows behind a request's end, keys between the sinks and the window (in blocks that are
    read and in pages that are gone), and tokens that later queries see."""
    say("unseen", kind, bad, dim, new)
    c = Case(9, [500, 70, 33], [new, new, min(new, 33)], 4, 2, dim, kind)
    window, sinks = 50, 3
    k, v = c.k.clone(), c.v.clone()
    for b, (length, rows) in enumerate(zip(c.lens, c.new)):
        seen = torch.zeros(c.tables.shape[1] * c.page, dtype=torch.bool)
        for p in range(length - rows, length):
            seen[max(0, p - window + 1):p + 1] = True
            seen[:min(sinks, p + 1)] = True
        for j in range(c.tables.shape[1] * c.page):
            page = int(c.tables[b, j // c.page])
            if page >= 0 and not seen[j]:
                k[page, j % c.page] = bad
                v[page, j % c.page] = bad
    clean = c.check(pk, window, sinks)
    c.k, c.v = k, v
    got = c.run(pk, window, sinks)
    # (the pieces that meet a NaN are made again in plain products: equal up to both bounds)
    _, bound = attend64(c.q, c.k.nan_to_num(0, 0, 0), c.v.nan_to_num(0, 0, 0), c.tables, c.lens, c.scale, c.starts, window, sinks, c.out)
    assert torch.isfinite(got).all()
    assert ((got.double() - clean.double()).abs() <= 2 * bound + 1e-30).all()
    # pages that no query sees are not even looked up
    gone = c.tables.clone()
    for b, (length, rows) in enumerate(zip(c.lens, c.new)):
        first = max(0, length - rows - window + 1) // c.page
        gone[b, -(-sinks // c.page):max(first, 1)] = 1 << 30
    c.tables = gone
    again = c.run(pk, window, sinks)
    assert torch.equal(again, got) and pk.lib().pkv_device_status() == 0


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("new", [1, 20])
def test_infinities_and_nan_that_are_seen(pk, kind, new):
    """What the formula gives in f32: a NaN score or value makes its rows NaN, an infinite
    value infinite ones, an infinite score is clamped; other rows and requests stay."""
    c = Case(10, [300, 300, 300, 300], [new] * 4, 16, 2, 256, kind)
    at = lambda b, j: (int(c.tables[b, j // c.page]), j % c.page)  # noqa: E731
    clean = c.run(pk)
    c.k[at(0, 7)][0, 5] = math.nan
    c.v[at(1, 290)][1, 9] = math.inf
    c.k[at(2, 3)][0] = 0
    c.k[at(2, 3)][0, 0] = math.inf
    got = c.run(pk).view(4, new, 16, 256)
    clean = clean.view(4, new, 16, 256)
    assert torch.isnan(got[0, :, :8]).all() and torch.equal(got[0, :, 8:], clean[0, :, 8:])
    assert torch.equal(got[3], clean[3])
    sees = torch.arange(300 - new, 300, device="cuda") >= 290
    assert torch.equal(got[1, :, :8], clean[1, :, :8])
    assert torch.isposinf(got[1, sees, 8:, 9]).all()
    keep = torch.ones(256, dtype=torch.bool, device="cuda")
    keep[9] = False
    assert torch.isfinite(got[1, :, 8:][..., keep]).all() and torch.isfinite(got[1, ~sees]).all()
    # +inf: the key has a weight of exp(100) to the others' few: its values; -inf: none
    q0 = c.q.view(4, new, 16, 256)[2, :, :8, 0]
    page, row = at(2, 3)
    value = c.v[page, row, 0].float()
    up = got[2, :, :8][q0 > 0]
    assert len(up) and ((up - value).abs() <= 1e-5 * value.abs() + 1e-30).all()
    assert torch.isfinite(got[2]).all()


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_the_only_key_is_nan(pk, kind):
    for lens, new in (([1, 1], [1, 1]), ([20, 20], [20, 20])):
        c = Case(18, lens, new, 16, 2, 256, kind)
        c.k[int(c.tables[0, 0]), 0, 1, 3] = math.nan
        got = c.run(pk).view(2, -1, 16, 256)
        assert torch.isnan(got[0, :, 8:]).all() and torch.isfinite(got[0, :, :8]).all() and torch.isfinite(got[1]).all()


def test_pages_that_are_none_are_reported(pk):
    for new in (1, 30):
        c = Case(11, [200, 100], [new, new], 16, 2, 256, "f16")
        c.tables[0, 2] = -1
        c.tables[1, 1] = 1 << 20
        c.check(pk)
        assert pk.lib().pkv_device_status() != 0 and b"page" in pk.lib().pkv_last_error()
    assert pk.lib().pkv_device_status() == 0


def test_lengths_and_starts_past_what_is_there(pk):
    """Lengths are taken into the table, starts into the step."""
    c = Case(12, [64, 64], [1, 1], 8, 1, 64, "f16")
    c.tables = c.tables[:, :2].contiguous()
    want = c.run(pk)
    got = pk.attend_pages(c.q, c.k, c.v, c.tables, i32([1 << 30, 64]), c.scale, starts=i32([-5, 1, 9]), out=c.out.clone())
    assert torch.equal(got, want)
    c.lens = [-3, 64]
    got = c.run(pk)
    assert int((got[0] != 0).sum()) == 0 and torch.equal(got[1], want[1])
    pk.attend_pages(c.q, c.k, c.v, c.tables, i32([64, 64]), c.scale, starts=i32([2, 0, 2]))
    # starts that run up and down name more rows than there are: any, but no others
    n = 40
    tables = c.tables[:1].expand(n, 2).contiguous()
    out = torch.full((6, 8, 64), 7.0, device="cuda")
    pk.attend_pages(c.q[:1].expand(6, 8, 64), c.k, c.v, tables, i32([64] * n), c.scale, starts=i32([0, 6] * (n // 2) + [0]), out=out)
    torch.cuda.synchronize()
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("lens,new,window", [([131073], [1], 0), ([40000, 33, 9000], [1, 1, 1], 0), ([16896], [512], 0),
                                             ([70000, 20000], [5, 5], 4096), ([3000], [3000], 0), ([1500, 900], [1500, 900], 500)])
def test_long(pk, kind, lens, new, window):
    say("long", kind, lens, new, window)
    Case(13, lens, new, 16, 2, 256, kind, page=256).check(pk, window, 4)


def test_many_requests(pk):
    r = random.Random(4)
    lens = [r.randint(0, 600) for _ in range(1500)]
    Case(14, lens, [1] * 1500, 2, 1, 64, "bf16").check(pk)
    new = [min(x, r.randint(0, 9)) for x in lens]
    Case(15, lens, new, 2, 1, 64, "f16", pad=5).check(pk, 100, 4)


def test_pages_past_4_gib(pk):
    page, kv, dim = 1 << 14, 2, 256
    n_pages = (1 << 32) // (page * kv * dim * 2) + 2  # 16 MiB a page, 4 GiB and 32 MiB a plane
    k, v = (torch.zeros(n_pages, page, kv, dim, dtype=torch.float16, device="cuda") for _ in range(2))
    g = gen(2)
    ids = [n_pages - 1, 0, n_pages - 2]
    for p in ids:
        k[p].normal_(generator=g)
        v[p].normal_(generator=g)
    tables, lens = i32([ids]), [2 * page + 77]
    for tokens in (1, 40):
        q = torch.randn(tokens, 16, dim, device="cuda", generator=g)
        starts = i32([0, tokens])
        want, bound = attend64(q, k[ids], v[ids], i32([[0, 1, 2]]), lens, 0.0625, starts, 0, 0, torch.zeros_like(q))
        got = pk.attend_pages(q, k, v, tables, i32(lens), 0.0625, starts=starts)
        assert ((got.double() - want).abs() <= bound).all()
    x = torch.randn(2, kv, dim, device="cuda", generator=g)
    slots = torch.tensor([n_pages * page - 1, (n_pages - 2) * page], device="cuda")
    pk.append_pages(x, -x, slots, k, v)
    assert torch.equal(k[-1, -1], x[0].half()) and torch.equal(v[-2, 0], (-x[1]).half())


def test_another_stream_and_a_graph(pk):
    """A captured call with lengths, tables and queries that change between replays, beside
    eager calls; two graphs over the same pages."""
    c = Case(16, [900, 40, 300], [1, 1, 1], 16, 2, 256, "f16")
    d = Case(17, [900, 40, 300], [60, 5, 9], 16, 2, 256, "f16")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        one = c.run(pk)
    side.synchronize()
    assert torch.equal(one, c.run(pk))
    lens, q = i32(c.lens), c.q.clone()
    lens2, q2 = i32(d.lens), d.q.clone()
    graphs, outs = [], []
    for x, n, s in ((q, lens, c), (q2, lens2, d)):
        out = s.out.clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            pk.attend_pages(x, s.k, s.v, s.tables, n, s.scale, starts=s.starts, window=200, sinks=4, out=out)
        graphs.append(g)
        outs.append(out)
    r = random.Random(1)
    for turn in range(4):
        new = [[r.randint(1, x) for x in s.lens] for s in (c, d)]
        for x, n, s, values in ((q, lens, c, new[0]), (q2, lens2, d, new[1])):
            n.copy_(i32(values))
            x.normal_()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        for x, n, s, out in ((q, lens, c, outs[0]), (q2, lens2, d, outs[1])):
            want = pk.attend_pages(x, s.k, s.v, s.tables, n, s.scale, starts=s.starts, window=200, sinks=4, out=s.out.clone())
            assert torch.equal(out, want)


# ------------------------------------------------------------------ drafted tokens
def probs(g, n, rows, vocab, peak=3.0):
    return torch.softmax(peak * torch.randn(n, rows, vocab, device="cuda", generator=g), -1)


@pytest.mark.parametrize("n,k,vocab,sure,ragged", [
    (1, 0, 1000, False, False), (3, 1, 7, False, False), (5, 4, 8192, True, True), (2, 5, 151936, False, False),
    (1, 5, 151936, True, False), (4, 63, 333, False, True), (40, 3, 1, False, False), (200, 2, 50, True, True),
    (2, 3, 100003, False, True),
])
def test_verify(pk, n, k, vocab, sure, ragged):
    say("verify", n, k, vocab, sure, ragged)
    g = gen(n + k)
    for turn in range(4):
        target = probs(g, n, k + 1, vocab)
        draft = None if sure else probs(g, n, k, vocab, 2.0) if turn % 2 else (target[:, :k] * 0.8 + 0.2 * probs(g, n, k, vocab)).contiguous()
        drafts = torch.randint(0, vocab, (n, k), device="cuda", generator=g).to(torch.int32)
        if k and turn != 1:  # likely ones
            drafts = target[:, :k].argmax(-1).to(torch.int32)
        u = torch.rand(n, k + 1, device="cuda", generator=g)
        if turn == 2:
            u[:, -1] = 0.0
        if turn == 3:
            u[:, -1] = 1 - 2.0 ** -24
        counts = torch.randint(-1, k + 3, (n,), device="cuda", generator=g).to(torch.int32) if ragged else None
        tokens, accepted = pk.verify_drafts(target, drafts, u, draft_probs=draft, n_drafts=counts)
        want = verify64(target, drafts, u, draft, counts)
        assert torch.equal(accepted.cpu(), want[1]) and torch.equal(tokens.cpu(), want[0])


def test_verify_at_the_ends(pk):
    """Tokens outside the vocabulary, rows without weight, NaN, and a rest that is nothing."""
    g = gen(3)
    target = probs(g, 6, 3, 4000)
    draft = probs(g, 6, 2, 4000)
    drafts = target[:, :2].argmax(-1).to(torch.int32)
    drafts[0, 0], drafts[1, 1] = -1, 4000
    target[2] = 0.0
    target[3, :, 100:3000] = float("nan")
    draft[4] = target[4, :2]          # the same rows: every draft is accepted
    draft[5] = 2 * target[5, :2]      # nothing is left behind a rejected draft
    u = torch.full((6, 3), 0.7, device="cuda")
    tokens, accepted = pk.verify_drafts(target, drafts, u, draft_probs=draft)
    want = verify64(target, drafts, u, draft, None)
    assert torch.equal(accepted.cpu(), want[1]) and torch.equal(tokens.cpu(), want[0])
    assert accepted[0] == 0 and accepted[4] == 2 and accepted[5] == 0 and tokens[5, 0] >= 0
    assert tokens[2].tolist() == [-1, -1, -1]
    tokens, accepted = pk.verify_drafts(target, drafts, u)
    want = verify64(target, drafts, u, None, None)
    assert torch.equal(accepted.cpu(), want[1]) and torch.equal(tokens.cpu(), want[0])


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_more_tiles_than_shares(pk, kind):
    """Many KV heads of short requests: parts are joined by cut, from the workgroups' own plan and
    from the plan's launch."""
    r = random.Random(4)
    for n, new in ((64, 16), (70, 16), (20, 40)):
        lens = [r.choice([0, 16, 40, 300, 700]) for _ in range(n)]
        say("more tiles", kind, n, new, sum(lens))
        Case(26, lens, [min(new, x) if i % 9 else 0 for i, x in enumerate(lens)], 8, 8, 256, kind).check(pk, 200 if n == 70 else 0, 3)


def test_two_calls_at_once(pk):
    """Calls on two streams, eager and as two graphs that are replayed together, each with a workspace
    of its own."""
    cases = [(Case(27, [9000, 40, 700], [1, 1, 1], 16, 2, 256, "bf16"), 0), (Case(28, [900, 600], [700, 300], 16, 2, 256, "f16"), 256),
             (Case(29, [3000] * 8, [5] * 8, 16, 2, 256, "bf16"), 1000), (Case(30, [2000] * 30, [1] * 30, 32, 8, 128, "f16"), 0)]
    want = [c.run(pk, w, 2) for c, w in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    graphs = [torch.cuda.CUDAGraph() for _ in cases]
    outs = [c.out.clone() for c, _ in cases]
    lens = [i32(c.lens) for c, _ in cases]
    call = lambda i: pk.attend_pages(cases[i][0].q, cases[i][0].k, cases[i][0].v, cases[i][0].tables, lens[i], cases[i][0].scale,  # noqa: E731
                                     starts=cases[i][0].starts, window=cases[i][1], sinks=2, out=outs[i])
    for i, stream in enumerate(streams):
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream), torch.cuda.graph(graphs[i], stream=stream):
            call(i)
    for turn in range(6):
        for x in outs:
            x.fill_(turn)
        torch.cuda.synchronize()
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                call(i) if turn % 2 else graphs[i].replay()
        torch.cuda.synchronize()
        for x, y in zip(outs, want):
            assert torch.equal(x, y)


def test_nothing_to_do(pk):
    c = Case(24, [40], [0], 16, 2, 256, "f16")
    assert c.run(pk).shape == (0, 16, 256)
    pk.append_pages(c.q[:, :2], c.q[:, :2], torch.empty(0, dtype=torch.int64, device="cuda"), c.k, c.v)
    tokens, accepted = pk.verify_drafts(torch.empty(0, 3, 9, device="cuda"), i32([]).view(0, 2), torch.empty(0, 3, device="cuda"))
    assert tokens.shape == (0, 3) and accepted.shape == (0,)


def test_verify_and_map_captured_on_another_stream(pk):
    g = gen(9)
    n, k, vocab = 3, 4, 5000
    target, draft, u = probs(g, n, k + 1, vocab), probs(g, n, k, vocab), torch.rand(n, k + 1, device="cuda", generator=g)
    drafts = draft.argmax(-1).to(torch.int32)
    lens, add = i32([5, 70, 0]), i32([1, 1, 40])
    t = Tables(random.Random(2), n, 8, 32, 12, [5, 70, 0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    start = [x.clone() for x in (t.t, t.h, t.free, t.count)]
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            m = pk.map_pages(lens, add, t.t, t.h, t.free, t.count, 32, 64)
            tokens, accepted = pk.verify_drafts(target, drafts, u, draft_probs=draft)
    for turn in range(4):
        new = [[5 + turn, 70, 31 * turn], [1, turn, 40]]
        with torch.cuda.stream(side):
            for x, y in zip((t.t, t.h, t.free, t.count), start):
                x.copy_(y)
            lens.copy_(i32(new[0]))
            add.copy_(i32(new[1]))
            target.copy_(probs(g, n, k + 1, vocab))
            u.uniform_(generator=g)
            graph.replay()
        side.synchronize()
        want = map_pages64(*new, start[0].tolist(), start[1].tolist(), start[2].tolist()[:start[3].item()], 32, t.capacity, 64)
        assert m.status.tolist() == [want[0]] == [0]
        assert m.slots.tolist() == want[4] and m.starts.tolist() == want[6] and t.h.tolist() == want[2]
        ok = verify64(target, drafts, u, draft, None)
        assert torch.equal(tokens.cpu(), ok[0]) and torch.equal(accepted.cpu(), ok[1])


def test_storage_outlives_the_pool_object(pk):
    pool = pk.PagedKvPool(1, 64, 32, 4, pk.KvCacheQuantization.BF16)
    k, v = pool.storage()
    assert k.shape == (4, 32, 1, 64) and k.dtype is torch.bfloat16 and int((k != 0).sum()) == 0
    ids = pool.take_pages(4)
    assert sorted(ids.tolist()) == [0, 1, 2, 3] and pool.take_pages(0).numel() == 0
    with pytest.raises(pk.KvCacheOverflow):
        pool.take_pages(1)
    with pytest.raises(pk.KvCacheOverflow):
        pool.sequence().append_quantized(torch.zeros(1, 1, 1, 64, device="cuda"), torch.zeros(1, 1, 1, 64, device="cuda"))
    for bad in ([0, 0], [1, 4], [-1]):
        with pytest.raises(pk.KvCacheError, match="not taken"):
            pool.give_pages(torch.tensor(bad, dtype=torch.int32))
    pool.give_pages(ids[:2])
    with pytest.raises(pk.KvCacheError, match="not taken"):
        pool.give_pages(ids[1:3])
    assert pool.free_pages == 2
    del pool
    k.fill_(1)
    torch.cuda.synchronize()
    assert float(k.float().sum()) == 4 * 32 * 64
    with pytest.raises(pk.KvCacheError, match="F16 or BF16"):
        pk.PagedKvPool(2, 256, 32, 2).storage()


# ------------------------------------------------------------------ a step of all of them
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_serving_steps_captured(pk, kind):
    """Prompts, then drafted tokens that are verified and taken back in part, over the pages of
    a pool beside the pool's own sequences: eager and as one captured step, replayed. Every
    step's attention is checked against the tokens that each request really has."""
    g, r = gen(21), random.Random(21)
    n, heads, kv, dim, page, k, vocab = 5, 16, 2, 256, 32, 3, 500
    quant = pk.KvCacheQuantization.F16 if kind == "f16" else pk.KvCacheQuantization.BF16
    pool = pk.PagedKvPool(kv, dim, page, 64, quant)
    seq = pool.sequence()
    sk = torch.randn(1, kv, 70, dim, device="cuda", generator=g)
    seq.append_quantized(sk, -sk)
    before = [x.clone() for x in seq.get_kv()]
    ids = pool.take_pages(50)
    assert pool.free_pages == 64 - 3 - 50
    kp, vp = pool.storage()
    tables = torch.full((n, 12), -1, dtype=torch.int32, device="cuda")
    held, free, count = i32([0] * n), ids.cuda(), i32([50])
    lens = i32([0] * n)
    rows = 128
    history = [[] for _ in range(n)]  # each request's K and V rows, as the cache rounds them

    q, nk, nv = (torch.empty(rows, h, dim, device="cuda") for h in (heads, kv, kv))
    add, target, draft = i32([0] * n), torch.empty(n, k + 1, vocab, device="cuda"), torch.empty(n, k, vocab, device="cuda")
    drafts, u = i32([[0] * k] * n), torch.empty(n, k + 1, device="cuda")
    out = torch.zeros(rows, heads, dim, device="cuda")

    def step():
        m = pk.map_pages(lens, add, tables, held, free, count, page, rows)
        pk.append_pages(nk, nv, m.slots, kp, vp)
        pk.attend_pages(q, kp, vp, tables, m.totals, 0.0625, starts=m.starts, window=64, sinks=4, out=out)
        tokens, accepted = pk.verify_drafts(target, drafts, u, draft_probs=draft)
        return m, tokens, accepted

    def fill(turn):
        for x in (q, nk, nv):
            x.normal_(generator=g)
        target.copy_(probs(g, n, k + 1, vocab))
        draft.copy_(0.5 * target[:, :k] + 0.5 * probs(g, n, k, vocab))
        drafts.copy_(draft.argmax(-1))
        u.uniform_(generator=g)
        new = [r.randint(1, 25) for _ in range(n)] if turn == 0 else [k + 1 if r.random() < 0.9 else 0 for _ in range(n)]
        add.copy_(i32(new))
        return new

    graph, static = None, None
    for turn in range(9):
        new = fill(turn)
        if turn == 3:  # one request ends, another is taken back
            lens[1] = 0
            history[1] = []
            lens[2] = 5
            history[2] = history[2][:5]
        if turn == 5:
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                static = step()
        if graph is not None:
            graph.replay()
            m, tokens, accepted = static
        else:
            m, tokens, accepted = step()
        assert m.status.item() == 0
        had = [len(x) for x in history]
        assert lens.tolist() == had and m.totals.tolist() == [a + b for a, b in zip(had, new)]
        at = 0
        for b in range(n):
            for i in range(new[b]):
                history[b].append((nk[at + i].to(TYPES[kind]), nv[at + i].to(TYPES[kind])))
            at += new[b]
        # the requests' own rows, page by page in order
        width = 12
        ck, cv = (torch.zeros(n * width, page, kv, dim, dtype=TYPES[kind], device="cuda") for _ in range(2))
        for b in range(n):
            for j, (x, y) in enumerate(history[b]):
                ck[b * width + j // page, j % page] = x
                cv[b * width + j // page, j % page] = y
        plain = torch.arange(n * width, dtype=torch.int32, device="cuda").view(n, width)
        want, bound = attend64(q, ck, cv, plain, m.totals.tolist(), 0.0625, m.starts, 64, 4, out)
        assert ((out.double() - want).abs() <= bound)[:at].all()
        ok = verify64(target, drafts, u, draft, None)
        assert torch.equal(tokens.cpu(), ok[0]) and torch.equal(accepted.cpu(), ok[1])
        # drafts that were not accepted leave the cache by a shorter length
        if turn:
            kept = [a + min(x, int(y) + 1) for a, x, y in zip(had, new, accepted.tolist())]
        else:
            kept = m.totals.tolist()
        history = [h[:x] for h, x in zip(history, kept)]
        lens.copy_(i32(kept))
    assert sum(held.tolist()) + count.item() == 50
    for a, b in zip(before, seq.get_kv()):
        assert torch.equal(a, b)
    # the pool's own sequence, named by a table: its attention with a window
    table = seq.page_ids().cuda().view(1, -1)
    qs = torch.randn(1, heads, dim, device="cuda", generator=g)
    whole = pk.attend_pages(qs, kp, vp, table, i32([70]), 0.0625)
    theirs = seq.attend(qs.view(1, 1, heads, dim), 0.0625, 69)
    assert float((whole - theirs[0]).abs().max()) <= 2e-3
    del graph, static
    torch.cuda.synchronize()
    pool.give_pages(ids)
    assert pool.free_pages == 61
