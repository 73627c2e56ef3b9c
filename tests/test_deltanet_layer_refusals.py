"""What the operators of a Gated-DeltaNet layer refuse, through the C ABI and the Python
entry points, before anything is launched (no GPU: addresses stand for device memory that
nothing touches)."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

import paramecia_amd as pk  # noqa: E402
from paramecia_amd import _lib  # noqa: E402
from paramecia_amd._lib import ERR_ARG, ERR_UNSUPPORTED, lib  # noqa: E402

A, B, C, D, F, G = (0x10000000000 * i for i in range(1, 7))  # far from each other


def err():
    return lib().pkv_last_error().decode()


def conv(**k):
    a = dict(x=A, sb=80 * 64, st=64, w=B, bias=None, state=C, lens=None, out=D, b=2, n=80, ch=64, taps=4)
    a.update(k)
    return lib().pkv_causal_conv(a["x"], a["sb"], a["st"], a["w"], a["bias"], a["state"], a["lens"], a["out"], a["b"],
                                 a["n"], a["ch"], a["taps"], 1, None)


@pytest.mark.parametrize("k,code,word", [
    (dict(x=None), ERR_ARG, "null"), (dict(w=None), ERR_ARG, "null"), (dict(state=None), ERR_ARG, "null"),
    (dict(out=None), ERR_ARG, "null"), (dict(b=0), ERR_ARG, "batch"), (dict(n=-1), ERR_ARG, "n >= 0"),
    (dict(ch=0), ERR_ARG, "channels"), (dict(st=63), ERR_ARG, "overlap"), (dict(sb=-64), ERR_ARG, "overlap"),
    (dict(out=A), ERR_ARG, "overlap"), (dict(out=A + 4 * (2 * 80 * 64 - 1)), ERR_ARG, "overlap"),
    (dict(state=D + 4), ERR_ARG, "overlap"), (dict(taps=1), ERR_UNSUPPORTED, "taps"),
    (dict(taps=5), ERR_UNSUPPORTED, "taps"), (dict(b=70000, sb=80 * 64), ERR_ARG, "65535"),
    (dict(b=1, n=1 << 24), ERR_ARG, "n must be"),
    (dict(b=1, ch=(1 << 24) + 4, st=(1 << 24) + 4, x=A, out=G << 4), ERR_ARG, "2^24 channels"),
])
def test_conv(k, code, word):
    assert conv(**k) == code and word in err()


def test_nothing_to_do():
    assert conv(n=0) == 0 and scan(n=0) == 0 and norm(rows=0) == 0


def scan(**k):
    w = 64 * 128
    a = dict(q=A, k=A + 4 * 2048, v=A + 4 * 4096, st=[80 * w, w] * 3, gate=B, beta=C, state=D, off=None, lens=None,
             out=F, b=2, n=80, hk=16, h=32, d=128, ws=G, wb=1 << 40)
    a.update(k)
    st = (ctypes.c_int64 * 6)(*a["st"])
    return lib().pkv_deltanet_prompt(a["q"], a["k"], a["v"], st, a["gate"], a["beta"], a["state"], a["off"], a["lens"],
                                     a["out"], a["b"], a["n"], a["hk"], a["h"], a["d"], 0.1, 1e-6, a["ws"], a["wb"], None)


@pytest.mark.parametrize("k,code,word", [
    (dict(q=None), ERR_ARG, "null"), (dict(k=None), ERR_ARG, "null"), (dict(v=None), ERR_ARG, "null"),
    (dict(gate=None), ERR_ARG, "null"), (dict(state=None), ERR_ARG, "null"), (dict(out=None), ERR_ARG, "null"),
    (dict(b=0), ERR_ARG, "batch"), (dict(n=-1), ERR_ARG, "n >= 0"), (dict(hk=5), ERR_ARG, "multiple"),
    (dict(hk=0), ERR_ARG, "multiple"), (dict(d=96), ERR_UNSUPPORTED, "64, 128 or 256"),
    (dict(q=A + 4), ERR_ARG, "16-byte"), (dict(state=D + 8), ERR_ARG, "16-byte"),
    (dict(st=[80 * 8194, 8194] + [80 * 8192, 8192] * 2), ERR_ARG, "multiples of 4"),
    (dict(st=[80 * 8192, 1024] + [80 * 8192, 8192] * 2), ERR_ARG, "rows do not overlap"),
    (dict(out=A + 4096), ERR_ARG, "overlap"), (dict(state=A + 64), ERR_ARG, "overlap"),
    (dict(out=D), ERR_ARG, "overlap"), (dict(b=70000), ERR_ARG, "65535"),
    (dict(b=16385, q=A, k=A + (1 << 43), v=A + (1 << 44), gate=1 << 60, beta=1 << 60, state=1 << 61, out=1 << 62), ERR_ARG, "2^26"),
    (dict(b=1, n=(1 << 30) + 1, out=1 << 62, state=1 << 61, ws=1 << 60), ERR_ARG, "2^30"),
])
def test_scan(k, code, word):
    assert scan(**k) == code and word in err()


def test_scan_workspace():
    need = lib().pkv_deltanet_prompt_workspace(2, 80, 16, 32, 128)
    assert lib().pkv_deltanet_prompt_workspace(0, 80, 16, 32, 128) == 0
    if need:
        assert scan(wb=need - 1) == ERR_ARG and "workspace" in err()
        assert scan(ws=None) == ERR_ARG and "workspace" in err()
        assert scan(ws=G + 8) == ERR_ARG
        for at in (A, D, F, A - 16):
            assert scan(ws=at) == ERR_ARG and "overlap" in err()


def norm(**k):
    a = dict(x=A, st=256, res=None, alpha=B, gate=None, out=C, q8=None, rows=9, d=256)
    a.update(k)
    return lib().pkv_rms_norm(a["x"], a["st"], a["res"], a["alpha"], a["gate"], 1e-6, a["out"], a["q8"], a["rows"], a["d"], None)


@pytest.mark.parametrize("k,code,word", [
    (dict(x=None), ERR_ARG, "null"), (dict(alpha=None), ERR_ARG, "null"), (dict(out=None), ERR_ARG, "null"),
    (dict(rows=-1), ERR_ARG, "rows"), (dict(d=0), ERR_ARG, "dim"), (dict(st=255), ERR_ARG, "overlap"),
    (dict(d=32769, st=32769), ERR_UNSUPPORTED, "32768"), (dict(q8=D + 1), ERR_ARG, "2-byte"),
    (dict(out=A + 4), ERR_ARG, "overlap"), (dict(res=A + 1024), ERR_ARG, "overlap"),
    (dict(res=C), ERR_ARG, "overlap"), (dict(out=A, st=260), ERR_ARG, "overlap"), (dict(q8=A), ERR_ARG, "overlap"),
    (dict(gate=F, res=F), ERR_ARG, "overlap"), (dict(q8=C), ERR_ARG, "overlap"),
    (dict(rows=1 << 31, out=1 << 61), ERR_UNSUPPORTED, "rows"), (dict(rows=1 << 25, out=1 << 61), ERR_UNSUPPORTED, "rows"),
    (dict(rows=1 << 21, d=8193, st=8193, out=1 << 61), ERR_UNSUPPORTED, "rows"),
])
def test_norm(k, code, word):
    assert norm(**k) == code and word in err()


def lora(**k):
    a = dict(x=A, g=None, w=B, wt=12, la=C, lb=C + (1 << 30), lt=2, n=3, r=16, s=D, ids=D + 4096, out=F, b=20, i=4096, o=64, ws=G, wb=None)
    a.update(k)
    wb = a["wb"] if a["wb"] is not None else lib().pkv_gated_oproj_lora_workspace(a["wt"], a["b"], a["i"], a["o"], a["r"])
    return lib().pkv_gated_oproj_lora(a["x"], a["g"], a["w"], a["wt"], a["la"], a["lb"], a["lt"], a["n"], a["r"], a["s"],
                                      a["ids"], a["out"], a["b"], a["i"], a["o"], a["ws"], wb, None)


@pytest.mark.parametrize("k,code,word", [
    (dict(x=None), ERR_ARG, "null"), (dict(w=None), ERR_ARG, "null"), (dict(la=None), ERR_ARG, "null"),
    (dict(lb=None), ERR_ARG, "null"), (dict(s=None), ERR_ARG, "null"), (dict(ids=None), ERR_ARG, "null"),
    (dict(ws=None), ERR_ARG, "null"), (dict(b=0), ERR_ARG, "batch"), (dict(n=0), ERR_ARG, "n_adapters"),
    (dict(r=0), ERR_ARG, "rank"), (dict(r=129), ERR_UNSUPPORTED, "rank"), (dict(lt=3), ERR_UNSUPPORTED, "F32, F16"),
    (dict(out=A), ERR_ARG, "overlap"), (dict(g=F), ERR_ARG, "overlap"), (dict(ws=F), ERR_ARG, "overlap"), (dict(ws=A), ERR_ARG, "overlap"),
    (dict(b=65536, wb=1 << 32), ERR_ARG, "65535"),
    (dict(la=C + 8), ERR_ARG, "16-byte"), (dict(wb=0), ERR_ARG, "workspace"), (dict(ws=G + 16), ERR_ARG, "256-byte"),
])
def test_lora(k, code, word):
    assert lora(**k) == code and word in err()


def test_lora_workspace():
    f = lib().pkv_gated_oproj_lora_workspace
    assert f(12, 0, 4096, 64, 16) == 0 and f(12, 65536, 4096, 64, 16) == 0 and f(12, 2**31 - 1, 4096, 64, 16) == 0
    assert f(12, 20, 4096, 64, 16) > 20 * 4096 * 4  # the batched projection's operands and the small product
    assert f(8, 20, 4096, 64, 16) >= 20 * 16 * 4


def test_python_refuses_host_tensors_and_shapes():
    t = torch.zeros
    with pytest.raises(pk.KvCacheError, match="float32 device tensor"):
        pk.causal_conv(t(1, 2, 8), t(8, 4), t(1, 8, 3))
    with pytest.raises(pk.KvCacheError, match="expects q, k"):
        pk.gated_delta_rule(t(1, 2, 4, 64), t(1, 2, 2, 64), t(1, 2, 4, 64), t(1, 2, 4), t(1, 2, 4), t(1, 4, 64, 64), 1.0, 1e-6)
    with pytest.raises(pk.KvCacheError, match="value heads"):
        pk.gated_delta_rule(t(1, 2, 3, 64), t(1, 2, 3, 64), t(1, 2, 4, 64), t(1, 2, 4), t(1, 2, 4), t(1, 4, 64, 64), 1.0, 1e-6)
    with pytest.raises(pk.KvCacheError, match="device tensor"):
        pk.rms_norm(t(2, 8), t(8), 1e-6)
    with pytest.raises(pk.KvCacheError, match="device tensor"):
        pk.gated_o_proj_lora(t(1, 4096), None, t(64, dtype=torch.uint8), 1, t(1, 1, 4096), t(1, 1, 1), t(1), t(1, dtype=torch.int32))
    lin = pk.LinearAttentionState()
    with pytest.raises(pk.KvCacheError, match="conv_dim"):
        lin.causal_conv(t(1, 2, 8), t(8, 4), 2, 64)
    with pytest.raises(pk.KvCacheError, match="expects v"):
        lin.delta_net_chunked(t(1), t(1), t(1), t(1), t(1))
    assert lin.recurrent_state is None


def test_symbols_are_declared():
    for name in ("pkv_causal_conv", "pkv_deltanet_prompt", "pkv_rms_norm", "pkv_gated_oproj_lora"):
        assert name in _lib.SYMBOLS
