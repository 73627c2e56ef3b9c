"""The attention over pages at the ends of its ranges: values whose sums leave f32 though their means
do not, positions near 2^31, tables as wide as they can be, starts that run backwards, a pool's pages
beside the rows that were appended. Against the plain forms of pages_checks.py in 64 bits."""
import random

import pytest

torch = pytest.importorskip("torch")

from pages_checks import E, attend64  # noqa: E402
from test_gpu_pages import TYPES, Case, Tables, gen, i32, pk, say  # noqa: E402, F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("lens,new", [([3000], [1]), ([3000, 700, 40], [1, 1, 1]), ([3000, 700, 40], [5, 5, 5]),
                                      ([2000, 300], [300, 300]), ([90, 33], [90, 33])])
@pytest.mark.parametrize("mag", [1e36, 1e37, 1e38, 3.38e38])
@pytest.mark.parametrize("signed", [False, True])
def test_means_of_the_largest_values(pk, dim, lens, new, mag, signed):
    """BF16 values up to the type's largest, 3.39e38: a sum of a few of them is past f32, a weighted
    mean never is. Scores stay below a few units, so that keys weigh nearly alike.

    Where a sum passes f32 the row is made again key by key as a running mean, which rounds in half
    steps of f32: the weight 2 and the sum of weights 5 a key, its reciprocal 1 and the two
    products' factors 5, the products and their sum 3: 16 a key at most, on top of the bound for sums."""
    say("means", dim, lens, new, mag, signed)
    c = Case(31, lens, new, 8, 1, dim, "bf16", spread=0.3)
    c.v = (torch.rand(c.v.shape, device="cuda", generator=gen(1)) * (2 if signed else 1) - (1 if signed else 0)).mul(mag).to(torch.bfloat16)
    c.v[:, ::7] = mag
    assert torch.isfinite(c.v).all()
    want, bound = attend64(c.q, c.k, c.v, c.tables, c.lens, c.scale, c.starts, 0, 0, c.out)
    weigh, _ = attend64(c.q, c.k, c.v.abs(), c.tables, c.lens, c.scale, c.starts, 0, 0, c.out)
    got = c.run(pk)
    assert torch.isfinite(got).all()
    assert ((got.double() - want).abs() <= bound + 16 * max(lens) * E * weigh).all()
    few = c.run(pk, 100, 4)
    want, bound = attend64(c.q, c.k, c.v, c.tables, c.lens, c.scale, c.starts, 100, 4, c.out)
    weigh, _ = attend64(c.q, c.k, c.v.abs(), c.tables, c.lens, c.scale, c.starts, 100, 4, c.out)
    assert torch.isfinite(few).all()
    assert ((few.double() - want).abs() <= bound + 16 * 400 * E * weigh).all()


def test_refusals_of_empty_shapes(pk):
    """Slots that are no row of numbers, and pages without heads: the framework's error, and nothing moved."""
    k, v = (torch.zeros(2, 32, 2, 64, dtype=torch.float16, device="cuda") for _ in range(2))
    new = torch.ones(1, 2, 64, device="cuda")
    for slots in (torch.tensor(3, device="cuda"), torch.zeros(1, 1, dtype=torch.int64, device="cuda")):
        with pytest.raises(pk.KvCacheError, match="slots must have shape"):
            pk.append_pages(new, new, slots, k, v)
    none = k[:, :, :0].contiguous()
    with pytest.raises(pk.KvCacheError, match="heads a multiple"):
        pk.attend_pages(torch.zeros(1, 4, 64, device="cuda"), none, none, i32([[0]]), i32([1]), 0.1)
    with pytest.raises(pk.KvCacheError, match="n_kv_heads"):
        pk.append_pages(new[:, :0], new[:, :0], torch.zeros(1, dtype=torch.int64, device="cuda"), none, none)
    assert int((k != 0).sum()) == 0


def holds(got, want, bound):
    assert torch.isfinite(got).all()
    off = (got.double() - want).abs()
    say("   worst share of the bound", round(float((off / bound.clamp(min=1e-30)).max()), 4))
    assert (off <= bound).all()


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("new", [1, 5, 60])
@pytest.mark.parametrize("window,sinks", [(70, 40), (1, 0), (4096, 4)])
def test_positions_near_2_31(pk, kind, new, window, sinks):
    """The longest table there is: 2047 pages of 2^20 tokens, two of them in turn. What the queries see is
    the same as in a short request of the sinks and the window's keys."""
    say("far", kind, new, window, sinks)
    g, page, wide, dim, heads = gen(40 + new), 1 << 20, 2047, 64, 8
    k, v = (torch.randn(2, page, 1, dim, device="cuda", generator=g).to(TYPES[kind]) for _ in range(2))
    tables = (torch.arange(wide, device="cuda") % 2).to(torch.int32).view(1, wide)
    length = wide * page - 5
    q = torch.randn(new, heads, dim, device="cuda", generator=g)
    starts = i32([0, new])
    got = pk.attend_pages(q, k, v, tables, i32([length]), 0.125, starts=starts, window=window, sinks=sinks)
    at = torch.cat([torch.arange(sinks), torch.arange(length - new - window + 1, length)]).cuda()
    rows = tables[0].long()[at // page] * page + at % page
    short = [torch.nn.functional.pad(x.view(-1, 1, dim)[rows], (0, 0, 0, 0, 0, -len(at) % 32)).view(-1, 32, 1, dim) for x in (k, v)]
    few = torch.arange(short[0].shape[0], dtype=torch.int32, device="cuda").view(1, -1)
    want, bound = attend64(q, *short, few, [len(at)], 0.125, starts, window, sinks, torch.zeros_like(q))
    holds(got, want, bound)


@pytest.mark.parametrize("new", [1, 2])
@pytest.mark.parametrize("n", [32, 33])
def test_the_widest_tables(pk, n, new):
    """33 tables of 2047 pages of 2^20 tokens pass the 32 bits in which a workgroup's own plan sums, 32 do not."""
    r, g, page, wide = random.Random(n), gen(n), 1 << 20, 2047
    k, v = (torch.randn(2, page, 1, 64, device="cuda", generator=g).half() for _ in range(2))
    tables = torch.ones(n, wide, dtype=torch.int32, device="cuda")
    tables[:, 0] = 0
    lens = [r.choice([0, 1, 33, 700, r.randint(0, 3000)]) for _ in range(n - 1)] + [page + 70]
    q = torch.randn(n * new, 8, 64, device="cuda", generator=g)
    starts = i32([new * i for i in range(n + 1)])
    got = pk.attend_pages(q, k, v, tables, i32(lens), 0.125, starts=starts)
    want, bound = attend64(q, k, v, tables, lens, 0.125, starts, 0, 0, torch.zeros_like(q))
    holds(got, want, bound)


def test_map_near_2_31(pk):
    """Positions and slots of the longest request, whose slots pass 32 bits."""
    page, wide = 1 << 20, 2047
    t = Tables(random.Random(5), 2, wide, page, 40, [wide * page - 100, 3 * page])
    t.step(pk, [wide * page - 100, 3 * page], [60, 5], 70)
    t.step(pk, [wide * page - 40, 3 * page + 5], [40, 2], 70)
    t.step(pk, [wide * page, 5], [1, 0], 70)  # a page past the table: refused


@pytest.mark.parametrize("heads,kv,dim,kind", [(8, 1, 64, "f16"), (16, 2, 256, "bf16")])
def test_starts_that_run_backwards(pk, heads, kv, dim, kind):
    """Such requests have no rows, the others theirs, and nothing outside of out is written."""
    c = Case(41, [64, 90], [1, 1], heads, kv, dim, kind)
    guard = torch.full((40, heads, dim), 7.0, device="cuda")
    out = guard[16:18]
    pk.attend_pages(c.q, c.k, c.v, c.tables, i32(c.lens), c.scale, starts=i32([2, 0, 2]), out=out)
    want, bound = attend64(c.q, c.k, c.v, c.tables[1:], [90], c.scale, i32([0, 2]), 0, 0, torch.zeros_like(c.q))
    holds(out, want, bound)
    assert (guard[:16] == 7).all() and (guard[18:] == 7).all()
    # 20 requests name the same 6 rows of the same cache, 20 run back: any of the 20, or rows left as they were
    for n, rows in ((40, 6), (4, 20), (70, 6)):
        guard.fill_(7)
        out = guard[10:10 + rows]
        q = c.q[:1].expand(rows, heads, dim)
        tables = c.tables[:1].expand(n, c.tables.shape[1]).contiguous()
        pk.attend_pages(q, c.k, c.v, tables, i32([64] * n), c.scale, starts=i32([0, rows] * (n // 2) + [0]), out=out)
        want, bound = attend64(q, c.k, c.v, c.tables[:1], [64], c.scale, i32([0, rows]), 0, 0, torch.zeros_like(out))
        left = (out == 7).flatten(1).all(1)
        assert not left.all()
        holds(out[~left], want[~left], bound[~left])
        assert (guard[:10] == 7).all() and (guard[10 + rows:] == 7).all()


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("new", [1, 4, 30])
def test_pages_of_a_pool(pk, kind, new):
    """Attention over a pool sequence's own pages, against the rows that were appended to it."""
    g, kv, dim, page, length = gen(42), 2, 256, 32, 170
    pool = pk.PagedKvPool(kv, dim, page, 16, pk.KvCacheQuantization.F16 if kind == "f16" else pk.KvCacheQuantization.BF16)
    other, seq = pool.sequence(), pool.sequence()
    rows = [torch.randn(1, kv, length, dim, device="cuda", generator=g) for _ in range(2)]
    for first, end in ((0, 70), (70, 71), (71, length)):  # its pages lie between another one's
        seq.append_quantized(*(x[:, :, first:end].contiguous() for x in rows))
        other.append_quantized(rows[1][:, :, :40].contiguous(), rows[0][:, :, :40].contiguous())
    q = torch.randn(new, 16, dim, device="cuda", generator=g)
    got = pk.attend_pages(q, *pool.storage(), seq.page_ids().cuda().view(1, -1), i32([length]), 0.0625, starts=i32([0, new]), window=100, sinks=3)
    planes = [torch.nn.functional.pad(x[0].transpose(0, 1).to(TYPES[kind]), (0, 0, 0, 0, 0, -length % page)).reshape(-1, page, kv, dim) for x in rows]
    plain = torch.arange(planes[0].shape[0], dtype=torch.int32, device="cuda").view(1, -1)
    want, bound = attend64(q, *planes, plain, [length], 0.0625, i32([0, new]), 100, 3, torch.zeros_like(q))
    holds(got, want, bound)
