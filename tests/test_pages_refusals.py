"""What the operators over pages on the device refuse, through the C ABI and the Python entry
points, before anything is launched (no GPU: addresses stand for device memory that nothing
touches); and their plain forms in pages_checks.py against cases worked out by hand."""
import ctypes
import math

import pytest

torch = pytest.importorskip("torch")

import paramecia_amd as pk  # noqa: E402
from pages_checks import attend64, map_pages64, verify64  # noqa: E402
from paramecia_amd._lib import ERR_ARG, ERR_OVERFLOW, ERR_UNSUPPORTED, lib  # noqa: E402

A, B, C, D, F, G, H, I, J, K, L = (0x10000000000 * i for i in range(1, 12))  # far from each other


def err():
    return lib().pkv_last_error().decode()


def pages_map(**k):
    a = dict(lens=A, add=B, n=4, tables=C, mp=8, held=D, free=F, count=G, cap=100, page=64, slots=H, pos=I, mt=16,
             starts=J, totals=K, status=L)
    a.update(k)
    return lib().pkv_pages_map(a["lens"], a["add"], a["n"], a["tables"], a["mp"], a["held"], a["free"], a["count"],
                               a["cap"], a["page"], a["slots"], a["pos"], a["mt"], a["starts"], a["totals"], a["status"], None)


@pytest.mark.parametrize("k,code,word", [
    *[({name: None}, ERR_ARG, "null") for name in ("lens", "add", "tables", "held", "free", "count", "slots", "pos", "starts", "totals", "status")],
    (dict(n=0), ERR_ARG, "n, max_pages"), (dict(mp=0), ERR_ARG, "max_pages"), (dict(cap=0), ERR_ARG, "capacity"),
    (dict(page=16), ERR_ARG, "power of two"), (dict(page=96), ERR_ARG, "power of two"), (dict(page=1 << 21), ERR_ARG, "power of two"),
    (dict(mt=-1), ERR_ARG, "max_tokens"), (dict(mt=1 << 31), ERR_ARG, "max_tokens"),
    (dict(mp=1 << 29), ERR_UNSUPPORTED, "2^31 pages"),
    (dict(totals=A), ERR_ARG, "overlap"), (dict(held=C + 4 * 31), ERR_ARG, "overlap"), (dict(pos=H + 120), ERR_ARG, "overlap"),
    (dict(starts=L - 16), ERR_ARG, "overlap"), (dict(count=F + 396), ERR_ARG, "overlap"),
])
def test_map(k, code, word):
    assert pages_map(**k) == code and word in err()


def append(**k):
    a = dict(quant=1, k=A, v=B, ks=512, vs=512, slots=C, n=10, kp=D, vp=F, ns=640, h=2, d=256)
    a.update(k)
    return lib().pkv_pages_append(a["quant"], a["k"], a["v"], a["ks"], a["vs"], a["slots"], a["n"], a["kp"], a["vp"],
                                  a["ns"], a["h"], a["d"], None)


@pytest.mark.parametrize("k,code,word", [
    *[({name: None}, ERR_ARG, "null") for name in ("k", "v", "slots", "kp", "vp")],
    (dict(n=-1), ERR_ARG, "n must"), (dict(ns=0), ERR_ARG, "n_slots"), (dict(h=0), ERR_ARG, "n_kv_heads"), (dict(d=0), ERR_ARG, "head_dim"),
    (dict(quant=3), ERR_UNSUPPORTED, "F16 or BF16"), (dict(quant=4), ERR_UNSUPPORTED, "F16 or BF16"), (dict(quant=9), ERR_UNSUPPORTED, "F16"),
    (dict(ks=511), ERR_ARG, "overlap"), (dict(vs=256), ERR_ARG, "overlap"), (dict(n=1, ks=-1), ERR_ARG, "strides"),
    (dict(n=1 << 22), ERR_UNSUPPORTED, "2^31"), (dict(h=1 << 20, d=1 << 20), ERR_UNSUPPORTED, "2^31"),
    (dict(vp=D + 640 * 1024 - 2), ERR_ARG, "overlap"), (dict(kp=A + 20000), ERR_ARG, "overlap"), (dict(vp=C), ERR_ARG, "overlap"),
])
def test_append(k, code, word):
    assert append(**k) == code and word in err()


def attend(**k):
    a = dict(quant=2, q=A, qt=4096, qh=256, kp=B, vp=C, np=50, page=64, tables=D, mp=10, lens=F, starts=G, n=3, t=20, h=16, kv=2,
             d=256, scale=0.1, w=0, s=0, out=H, ws=I, wb=None)
    a.update(k)
    wb = a["wb"] if a["wb"] is not None else lib().pkv_pages_attend_workspace(a["n"], a["t"], a["h"], a["kv"], a["d"])
    return lib().pkv_pages_attend(a["quant"], a["q"], a["qt"], a["qh"], a["kp"], a["vp"], a["np"], a["page"], a["tables"], a["mp"],
                                  a["lens"], a["starts"], a["n"], a["t"], a["h"], a["kv"], a["d"], a["scale"], a["w"], a["s"],
                                  a["out"], a["ws"], wb, None)


@pytest.mark.parametrize("k,code,word", [
    *[({name: None}, ERR_ARG, "null") for name in ("q", "kp", "vp", "tables", "lens", "out", "ws")],
    (dict(n=0), ERR_ARG, "n and num_heads"), (dict(t=-1), ERR_ARG, "tokens >= 0"), (dict(h=15), ERR_ARG, "multiple"),
    (dict(kv=0), ERR_ARG, "multiple"), (dict(np=0), ERR_ARG, "n_pages"), (dict(mp=0), ERR_ARG, "max_pages"),
    (dict(page=48), ERR_ARG, "power of two"), (dict(mp=1 << 25), ERR_ARG, "2^31 - 64"), (dict(w=-1), ERR_ARG, "window"),
    (dict(s=-1), ERR_ARG, "sinks"), (dict(scale=math.nan), ERR_ARG, "finite"), (dict(scale=math.inf), ERR_ARG, "finite"),
    (dict(starts=None), ERR_ARG, "tokens must be n"), (dict(quant=4), ERR_UNSUPPORTED, "F16 or BF16"),
    (dict(d=80, qh=80), ERR_UNSUPPORTED, "64, 128 or 256"), (dict(d=512, qh=512), ERR_UNSUPPORTED, "64, 128 or 256"),
    (dict(t=1 << 28), ERR_UNSUPPORTED, "2^31"), (dict(n=1 << 24), ERR_UNSUPPORTED, "2^24"),
    (dict(qh=252), ERR_ARG, "overlap"), (dict(qt=4092), ERR_ARG, "overlap"), (dict(qt=4098), ERR_ARG, "multiples of 4"),
    (dict(q=A + 8), ERR_ARG, "16-byte"), (dict(out=H + 4), ERR_ARG, "16-byte"), (dict(kp=B + 2), ERR_ARG, "16-byte"),
    (dict(wb=100), ERR_ARG, "workspace"), (dict(ws=I + 16), ERR_ARG, "256-byte"), (dict(out=A), ERR_ARG, "overlap"),
    (dict(ws=H), ERR_ARG, "overlap"), (dict(out=B), ERR_ARG, "overlap"), (dict(ws=D - 256), ERR_ARG, "overlap"),
])
def test_attend(k, code, word):
    assert attend(**k) == code and word in err()


def test_attend_workspace():
    f = lib().pkv_pages_attend_workspace
    assert f(0, 5, 16, 2, 256) == 0 and f(3, 0, 16, 2, 256) == 0 and f(3, 5, 16, 3, 256) == 0 and f(3, 5, 16, 2, 96) == 0
    assert f(1, 1 << 30, 16, 2, 256) == 0
    assert 0 < f(1, 1, 16, 2, 256) <= 160 << 20 and 0 < f(8, 8001, 16, 2, 256) <= 160 << 20


@pytest.mark.parametrize("heads,kv,dim", [(16, 2, 256), (8, 1, 64), (32, 8, 128), (28, 4, 128), (96, 2, 256), (6, 6, 128), (2, 2, 64)])
def test_attend_workspace_for_the_largest_step_serves_all(heads, kv, dim):
    counts = [1, 2, 3, 4, 6, 7, 9, 16, 24, 33, 64, 65, 100, 144, 300, 1025, 8192, 20000]
    f = lambda n, t: lib().pkv_pages_attend_workspace(n, t, heads, kv, dim)  # noqa: E731
    for n, more in zip(counts, counts[1:] + [100000]):
        for t, longer in zip(counts, counts[1:] + [100000]):
            assert 0 < f(n, t) <= f(n, longer) and f(n, t) <= f(more, t), (n, t)
    # a buffer for 64 requests and 8192 tokens is taken by steps of fewer (that end at the next check)
    for n, t in ((24, 144), (1, 1), (64, 64), (3, 8000)):
        assert attend(n=n, t=t, h=heads, kv=kv, d=dim, qt=heads * dim, qh=dim, wb=f(64, 8192), ws=H) == ERR_ARG and "overlap" in err()


@pytest.mark.parametrize("scale", [2.4e38, -3.4e38, math.inf, -math.inf, math.nan, 1e39])
def test_attend_refuses_scales_whose_product_passes_f32(scale):
    """Scores are held times log2(e): 1.44 scale has to be a number too, or zeros would give NaN."""
    assert attend(scale=scale) == ERR_ARG and "finite" in err()


def test_attend_takes_the_largest_scale():
    for scale in (2.3e38, -2.3e38, 0.0):  # (they end at the next check)
        assert attend(scale=scale, starts=None) == ERR_ARG and "tokens must be n" in err()


def verify(**k):
    a = dict(p=A, ps=1000, q=B, qs=1000, x=C, c=D, u=F, n=3, k=4, v=1000, t=G, acc=H, ws=I, wb=None)
    a.update(k)
    wb = a["wb"] if a["wb"] is not None else lib().pkv_verify_drafts_workspace(a["n"], a["v"])
    return lib().pkv_verify_drafts(a["p"], a["ps"], a["q"], a["qs"], a["x"], a["c"], a["u"], a["n"], a["k"], a["v"],
                                   a["t"], a["acc"], a["ws"], wb, None)


@pytest.mark.parametrize("k,code,word", [
    *[({name: None}, ERR_ARG, "null") for name in ("p", "x", "u", "t", "acc", "ws")],
    (dict(n=-1), ERR_ARG, "n and k"), (dict(k=-1), ERR_ARG, "n and k"), (dict(v=0), ERR_ARG, "vocab"),
    (dict(k=64), ERR_UNSUPPORTED, "63 drafts"), (dict(n=65536), ERR_UNSUPPORTED, "65535"), (dict(ps=999), ERR_ARG, "overlap"),
    (dict(qs=10), ERR_ARG, "overlap"), (dict(wb=0), ERR_ARG, "workspace"), (dict(ws=I + 4), ERR_ARG, "8-byte"),
    (dict(t=A), ERR_ARG, "overlap"), (dict(acc=G + 56), ERR_ARG, "overlap"), (dict(ws=B + 4 * 11992), ERR_ARG, "overlap"),
])
def test_verify(k, code, word):
    assert verify(**k) == code and word in err()


def test_nothing_to_do():
    assert append(n=0) == 0 and attend(t=0) == 0 and verify(n=0) == 0


def test_pool_pages_without_a_pool():
    L_ = lib()
    ids = (ctypes.c_int * 4)()
    assert L_.pkv_pool_take_pages(None, 1, ids) == ERR_ARG and L_.pkv_pool_give_pages(None, 1, ids) == ERR_ARG
    assert L_.pkv_pool_storage(None, None, None, None, None, None) == ERR_ARG
    assert L_.pkv_seq_page_ids(None, ids, 4) == ERR_ARG


def test_python_refuses_host_tensors_and_shapes():
    t = torch.zeros
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    h = lambda *s: torch.zeros(*s, dtype=torch.float16)  # noqa: E731
    with pytest.raises(pk.KvCacheError, match="int32 device tensor"):
        pk.map_pages(i(2), i(2), i(2, 4), i(2), i(8), i(1), 64, 10)
    with pytest.raises(pk.KvCacheError, match="expects lens"):
        pk.map_pages(i(0), i(0), i(0, 4), i(0), i(8), i(1), 64, 10)
    with pytest.raises(pk.KvCacheError, match="float16 or bfloat16"):
        pk.append_pages(t(1, 2, 64), t(1, 2, 64), i(1), t(4, 32, 2, 64), t(4, 32, 2, 64))
    with pytest.raises(pk.KvCacheError, match="device tensor"):
        pk.append_pages(t(1, 2, 64), t(1, 2, 64), i(1), h(4, 32, 2, 64), h(4, 32, 2, 64))
    with pytest.raises(pk.KvCacheError, match="device tensor"):
        pk.attend_pages(t(1, 4, 64), h(4, 32, 2, 64), h(4, 32, 2, 64), i(1, 4), i(1), 0.1)
    with pytest.raises(pk.KvCacheError, match="expects target_probs"):
        pk.verify_drafts(t(1, 9), i(1, 2), t(1, 3))
    with pytest.raises(pk.KvCacheError, match="float32 device tensor"):
        pk.verify_drafts(t(1, 3, 9), i(1, 2), t(1, 3))


@pytest.mark.parametrize("bad", [2 ** 31, 2 ** 32, 2 ** 32 + 64, 2 ** 64 + 64, -2 ** 32, -1])
def test_python_refuses_numbers_past_32_bits(bad):
    """ctypes drops the high bits of a number: what does not fit C's int is refused in front of it."""
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    h = lambda *s: torch.zeros(*s, dtype=torch.float16)  # noqa: E731
    t = torch.zeros
    words = r"must be in \[0, 2\^31\)"
    for page, tokens in ((bad, 10), (64, bad)):
        with pytest.raises(pk.KvCacheError, match=words):
            pk.map_pages(i(2), i(2), i(2, 4), i(2), i(8), i(1), page, tokens)
    for k in (dict(window=bad), dict(sinks=bad), dict(window=5, sinks=bad)):
        with pytest.raises(pk.KvCacheError, match=words):
            pk.attend_pages(t(1, 4, 64), h(4, 32, 2, 64), h(4, 32, 2, 64), i(1, 4), i(1), 0.1, **k)
    pool = object.__new__(pk.PagedKvPool)
    with pytest.raises(pk.KvCacheError, match=words):
        pool.take_pages(bad)
    for at in range(4):
        with pytest.raises(pk.KvCacheError, match=words):
            pk.PagedKvPool(*[bad if j == at else x for j, x in enumerate((2, 64, 32, 4))], pk.KvCacheQuantization.F16, stream=0)


def test_python_refuses_shapes_past_32_bits():
    i = lambda *s: torch.zeros(1, dtype=torch.int32).expand(*s)  # noqa: E731
    h = lambda *s: torch.zeros(1, dtype=torch.float16).expand(*s)  # noqa: E731
    f = lambda *s: torch.zeros(1).expand(*s)  # noqa: E731
    big, words = 2 ** 32 + 2, r"must be in \[0, 2\^31\)"
    with pytest.raises(pk.KvCacheError, match=words):
        pk.map_pages(i(2), i(2), i(2, big), i(2), i(8), i(1), 64, 10)
    with pytest.raises(pk.KvCacheError, match=words):
        pk.map_pages(i(2), i(2), i(2, 4), i(2), i(big), i(1), 64, 10)
    with pytest.raises(pk.KvCacheError, match=words):
        pk.append_pages(f(1, 2, 64), f(1, 2, 64), torch.zeros(1, dtype=torch.int64), h(big, 32, 2, 64), h(big, 32, 2, 64))
    with pytest.raises(pk.KvCacheError, match=words):
        pk.attend_pages(f(1, 4, 64), h(4, 32, 2, 64), h(4, 32, 2, 64), i(1, big), i(1), 0.1)
    with pytest.raises(pk.KvCacheError, match=words):
        pk.verify_drafts(f(1, 3, big), i(1, 2), f(1, 3))


# ------------------------------------------------------------------ the plain forms themselves
def test_plain_map():
    # a request shrinks from three pages to one, one ends, one takes two pages: theirs, last given first
    got = map_pages64([10, 0, 40], [0, 0, 50], [[5, 6, 7, 0], [8, 0, 0, 0], [9, 1, 0, 0]], [3, 1, 2], [4], 32, 10, 60)
    status, tables, held, stack, slots, positions, starts, totals = got
    assert status == 0 and held == [1, 0, 3] and stack == [4, 6, 7] and totals == [10, 0, 90] and starts == [0, 0, 0, 50]
    assert tables[2][:3] == [9, 1, 8]
    assert positions[:2] == [40, 41] and slots[0] == 1 * 32 + 8 and slots[49] == 8 * 32 + 25 and slots[50:] == [-1] * 10
    assert map_pages64([0, 0], [64, 65], [[0] * 4] * 2, [0, 0], [1, 2, 3, 4], 32, 4, 200)[0] == ERR_OVERFLOW
    assert map_pages64([0], [200], [[0] * 4], [0], [1, 2, 3, 4], 32, 4, 300)[0] == ERR_ARG


def test_plain_attention():
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(4, 32, 1, 64, generator=g).half() for _ in range(2))
    tables = torch.tensor([[3, 1, -1]], dtype=torch.int32)
    q = torch.randn(2, 1, 64, generator=g)
    # 40 keys, two queries at 38 and 39, a window of 3 and one sink: keys 0, 36 .. 38 and 0, 37 .. 39
    out, bound = attend64(q, k, v, tables, [40], 0.125, torch.tensor([0, 2]), 3, 1, torch.zeros(2, 1, 64))
    rows_k, rows_v = (torch.cat([x[3, :, 0], x[1, :, 0]]).double() for x in (k, v))
    for i, keys in enumerate(([0, 36, 37, 38], [0, 37, 38, 39])):
        w = torch.softmax(0.125 * rows_k[keys] @ q[i, 0].double(), 0)
        assert torch.allclose(out[i, 0], w @ rows_v[keys], rtol=1e-12, atol=1e-14)
    assert (bound > 0).all() and (bound < 1e-3).all()
    # a page that is none, and a query in front of the first key
    out, _ = attend64(q, k, v, torch.tensor([[9, -1]], dtype=torch.int32), [40], 0.125, torch.tensor([0, 2]), 0, 0, torch.ones(2, 1, 64))
    assert (out == 0).all()
    out, _ = attend64(q, k, v, tables, [1], 0.125, torch.tensor([0, 2]), 0, 0, torch.ones(2, 1, 64))
    assert (out[0] == 0).all() and torch.equal(out[1, 0], rows_v[0])


def test_plain_verify():
    p = torch.tensor([[[0.5, 0.5, 0.0], [0.1, 0.2, 0.7], [0.25, 0.25, 0.5]]])
    q = torch.tensor([[[0.25, 0.75, 0.0], [0.8, 0.1, 0.1]]])
    x = torch.tensor([[0, 0]], dtype=torch.int32)
    # 0.9 * 0.25 < 0.5; 0.5 * 0.8 is not below 0.1; what is left: 0.1 of token 1, 0.6 of token 2
    tokens, accepted = verify64(p, x, torch.tensor([[0.9, 0.5, 0.1]]), q, None)
    assert accepted.tolist() == [1] and tokens.tolist() == [[0, 1, -1]]
    tokens, accepted = verify64(p, x, torch.tensor([[0.9, 0.5, 0.2]]), q, None)
    assert tokens.tolist() == [[0, 2, -1]]
    tokens, accepted = verify64(p, x, torch.tensor([[0.9, 0.1, 0.6]]), q, None)
    assert accepted.tolist() == [2] and tokens.tolist() == [[0, 0, 2]]
    # certain drafts: accepted with p itself; a rejected one is not drawn again
    tokens, accepted = verify64(p, x, torch.tensor([[0.6, 0.1, 0.0]]), None, None)
    assert accepted.tolist() == [0] and tokens.tolist() == [[1, -1, -1]]
    tokens, accepted = verify64(p, x, torch.tensor([[0.6, 0.1, 0.0]]), None, torch.tensor([0]))
    assert accepted.tolist() == [0] and tokens.tolist() == [[0, -1, -1]]
