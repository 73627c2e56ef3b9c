"""The operators of a Gated-DeltaNet layer around its single-token update, against plain
formulas in 64 bits: the short causal convolution (depthwise_conv1d, paramecia-model/src/
ops.rs:18-20), the gated delta rule over a prompt (delta_net_chunked, qwen3_next.rs:
3506-3731), the RMS norm with residual, gate and Q8_0 rows, and the output projection with
low-rank adapters (models/with_tracing.rs:253-300); and the layer as they make it.

Half a step of f32 is E = 2^-24 relative to the rounded value. Where a tolerance is not
elementwise it bounds the 2-norm of the error over that of the result."""
import sys

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
EPS = 1e-6


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
    g = torch.Generator(device="cuda").manual_seed(seed)
    return lambda *s: torch.randn(s, device="cuda", generator=g)


def rel(got, ref):
    got, ref = got.double(), ref.double()
    assert torch.isfinite(got).all()
    return float((got - ref).norm() / ref.norm().clamp(min=1e-300))


def ends(lens, b, n):
    return [n] * b if lens is None else [min(max(int(x), 0), n) for x in lens]


# ------------------------------------------------------------------ convolution
def conv64(x, w, state, bias, lens, silu, out):
    """(out, state, bound): the formula in 64 bits and what f32 may be off by: K products
    and sums, each half a step of the sum of magnitudes, through an activation of slope at
    most 1.1, whose own exp, sum, quotient and rounding are 8 half steps of its value."""
    out, state = out.double(), state.double()
    bound = torch.zeros_like(out)
    k = w.shape[1]
    for i, end in enumerate(ends(lens, x.shape[0], x.shape[1])):
        rows = torch.cat([state[i].T, x[i, :end].double()])
        if end:
            win = rows.unfold(0, k, 1)
            y, mag = (win * w.double()).sum(-1), (win * w.double()).abs().sum(-1)
            if bias is not None:
                y, mag = y + bias.double(), mag + bias.double().abs()
            err = 1.1 * (k + 1) * E * mag
            if silu:
                y = y * torch.sigmoid(y)
                err = err + 8 * E * y.abs()
            out[i, :end], bound[i, :end] = y, err + 1e-37
        state[i] = rows[len(rows) - (k - 1):].T
    return out, state, bound


@pytest.mark.parametrize("b,n,ch,taps,bias,silu,lens", [
    (1, 1, 8192, 4, False, True, None),          # a token
    (16, 1, 260, 4, True, True, None),           # a batch's token, a last workgroup of few channels
    (2, 2, 64, 4, False, True, None),            # fewer tokens than kept inputs
    (1, 3, 64, 4, False, False, None),
    (3, 5, 1024, 3, True, True, None),           # one more than a short tile
    (2, 16, 132, 2, False, True, None),          # a whole tile
    (2, 33, 67, 4, True, True, None),            # channels no multiple of four
    (1, 1, 1, 4, True, True, None),
    (1, 700, 8192, 4, False, True, None),
    (5, 40, 256, 4, False, True, [40, 0, 1, 17, 2]),
    (6, 4, 128, 4, True, True, [4, 3, 2, 1, 0, -5]),
    (2, 20, 63, 3, False, True, [99, 18]),       # a length past the padding is the padding's
])
def test_conv(pk, b, n, ch, taps, bias, silu, lens):
    say(f"conv b={b} n={n} ch={ch} taps={taps} lens={lens}")
    r = gen(n + ch)
    x, w, state = r(b, n, ch), r(ch, taps), r(b, ch, taps - 1)
    bias = r(ch) if bias else None
    out = r(b, n, ch)
    for i, e in enumerate(ends(lens, b, n)):
        x[i, e:] = float("nan")  # padding is not read
    ref, ref_state, bound = conv64(x, w, state, bias, lens, silu, out)
    dl = None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")
    got = pk.causal_conv(x, w, state, bias=bias, lens=dl, silu=silu, out=out)
    assert got is out
    assert bool(((got.double() - ref).abs() <= bound).all())
    assert torch.equal(state.double(), ref_state)


def test_conv_slices_and_pieces(pk):
    """A slice of a wider projection, and a prompt in pieces, give what a dense prompt does."""
    say("conv: strides and pieces")
    r = gen(3)
    b, n, ch = 2, 50, 256
    wide, w, state = r(b, n, ch + 64), r(ch, 4), r(b, ch, 3)
    x = wide[..., 32:32 + ch]
    s0, s1, s2 = state.clone(), state.clone(), state.clone()
    dense = pk.causal_conv(x.contiguous(), w, s0)
    assert torch.equal(pk.causal_conv(x, w, s1), dense) and torch.equal(s0, s1)
    odd = wide[..., 1:1 + ch]  # rows that are not 16-byte aligned
    s3, s4 = state.clone(), state.clone()
    assert torch.equal(pk.causal_conv(odd, w, s3), pk.causal_conv(odd.contiguous(), w, s4))
    parts = [pk.causal_conv(x[:, a:z], w, s2) for a, z in ((0, 1), (1, 3), (3, 3), (3, 20), (20, 50))]
    assert torch.equal(torch.cat(parts, 1), dense) and torch.equal(s2, s0)


# ------------------------------------------------------------------ gated delta rule
def scan64(q, k, v, gate, beta, state, scale, lens, out, offset):
    """Token by token in 64 bits."""
    b, n, hk, d = q.shape
    h = v.shape[2]
    out, state, offset = out.double(), state.double().clone(), offset.double().clone()
    end = torch.tensor(ends(lens, b, n), device=q.device)
    q, k = q.double(), k.double()
    q = (q * scale / (q.square().sum(-1, keepdim=True) + EPS).sqrt()).repeat_interleave(h // hk, 2)
    k = (k / (k.square().sum(-1, keepdim=True) + EPS).sqrt()).repeat_interleave(h // hk, 2)
    alpha, be = gate.double().exp(), torch.sigmoid(beta.double())
    for t in range(n):
        s = state * alpha[:, t, :, None, None]
        u = be[:, t, :, None] * (v[:, t].double() - (s * k[:, t, :, None]).sum(-1))
        s = s + u[..., None] * k[:, t, :, None]
        o = (s * q[:, t, :, None]).sum(-1)
        on = (t < end)[:, None, None]
        state = torch.where(on[..., None], s, state)
        out[:, t] = torch.where(on, o, out[:, t])
    for i, e in enumerate(end.tolist()):
        offset[i] += gate[i, :e].double().sum(0)
    return out, state, offset


def scan_inputs(r, b, n, hk, h, d, rate=0.5):
    x = r(b, n, (2 * hk + h) * d)
    x = x * torch.sigmoid(x)
    q, k, v = x.split([hk * d, hk * d, h * d], -1)
    gate = -rate * torch.nn.functional.softplus(r(b, n, h))
    return (q.view(b, n, hk, d), k.view(b, n, hk, d), v.view(b, n, h, d), gate, r(b, n, h),
            0.3 * r(b, h, d, d), r(b, h))


def scan_limit(n):
    """A token's norms, dot products and update are some 16 roundings; the state's errors of
    n tokens add up as independent ones (its factors are below one)."""
    return E * (16 + 2 * n ** 0.5)


def check_scan(pk, ins, scale, lens, out):
    q, k, v, gate, beta, state, offset = ins
    ref, ref_state, ref_offset = scan64(q, k, v, gate, beta, state, scale, lens, out, offset)
    dl = None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")
    got = pk.gated_delta_rule(q, k, v, gate, beta, state, scale, EPS, gate_offset=offset, lens=dl, out=out)
    lim = scan_limit(q.shape[1])
    whole = got
    on = (torch.arange(q.shape[1]) < torch.tensor(ends(lens, *q.shape[:2]))[:, None]).cuda()[..., None, None]
    got, ref = torch.where(on, got, 0.0), torch.where(on, ref, 0.0)
    say(f"  out {rel(got, ref):.2e} state {rel(state, ref_state):.2e} limit {lim:.2e}")
    # f32 holds nothing to a relative precision below its smallest normal value
    small = 2.0 ** -126
    for x, y in ((got, ref), (state, ref_state)):
        assert torch.isfinite(x).all()
        assert float((x.double() - y).norm()) <= lim * float(y.norm()) + small * y.numel() ** 0.5
    # no single value is far off: 40 times the mean error, of the largest values' size
    assert float((got.double() - ref).abs().max() / ref.abs().max()) <= 40 * lim
    # the gates' sum is rounded once after its own 64 bits (and once more as the offset's)
    assert float((offset.double() - ref_offset).abs().max()) <= 2 * E * float(ref_offset.abs().max() + 1)
    return whole


@pytest.mark.parametrize("b,n,hk,h,d,lens", [
    (1, 1, 16, 32, 128, None),
    (2, 5, 16, 32, 128, None),
    (1, 16, 2, 2, 128, None),
    (1, 17, 2, 6, 128, None),
    (1, 63, 2, 4, 128, None),
    (1, 64, 2, 4, 128, None),
    (1, 65, 2, 4, 128, None),
    (1, 129, 1, 1, 128, None),
    (1, 300, 16, 32, 128, None),
    (3, 130, 2, 4, 128, [130, 0, 67]),
    (4, 9, 2, 4, 128, [1, 9, -3, 100]),
    (2, 100, 3, 3, 64, [100, 64]),
    (1, 200, 2, 4, 64, None),
    (2, 90, 2, 4, 256, [33, 90]),
    (1, 7, 4, 4, 256, None),
    (1, 1500, 1, 2, 128, None),
    (16, 200, 16, 32, 128, None),
    (16, 700, 16, 32, 128, None),
    (1, 4700, 16, 32, 128, None),                # more than one segment of chunks
    (2, 2400, 16, 32, 128, [2399, 700]),         # the second sequence ends in the first segment
    (1, 2000, 3, 9, 64, None),                   # three value heads over two workgroups
    (9, 333, 16, 32, 128, [333, 0, 48, 47, 200, 256, 257, 1, 128]),
    (1, 130, 3, 15, 64, None),                   # an odd number of value heads per key head
    (2, 70, 8, 8, 256, [70, 65]),
])
def test_scan(pk, b, n, hk, h, d, lens):
    say(f"scan b={b} n={n} hk={hk} h={h} d={d} lens={lens}")
    r = gen(1000 + n + d)
    ins = scan_inputs(r, b, n, hk, h, d)
    for t in ins[:5]:
        for i, e in enumerate(ends(lens, b, n)):
            t[i, e:] = float("nan")  # padding is not read
    out = r(b, n, h, d)
    keep = out.clone()
    got = check_scan(pk, ins, d ** -0.5, lens, out)
    for i, e in enumerate(ends(lens, b, n)):
        assert torch.equal(got[i, e:], keep[i, e:])


@pytest.mark.parametrize("n", [11, 150])
@pytest.mark.parametrize("kind", ["slow", "fast", "mixed", "reset", "same_keys", "zero_rows", "large", "small", "closed", "growing", "huge", "far_apart", "late",
                                  "one_write", "one_write_mild", "few_writes", "tiny_keys", "tiny_queries"])
def test_scan_values(pk, kind, n):
    """Decays from none to whole, keys that all point the same way, zero vectors, magnitudes."""
    say(f"scan values {kind} n={n}")
    r = gen(77 + n)
    b, hk, h, d = 1, 2, 4, 128
    q, k, v, gate, beta, state, offset = scan_inputs(r, b, n, hk, h, d)
    if kind == "slow":
        gate = gate * 1e-4
    elif kind == "fast":
        gate = gate * 20
    elif kind == "mixed":  # far sums of gates beside tokens that forget nothing
        gate = torch.where(torch.rand(gate.shape, device="cuda") < 0.2, -40.0, -1e-3)
    elif kind == "reset":  # exp(gate) = 0: the state in front is gone
        gate[:, n // 2] = float("-inf")
        gate[:, n // 3] = -1e30
    elif kind == "same_keys":
        k[:] = k[:, :1]
        gate = gate * 0.01
        beta = beta + 4
    elif kind == "zero_rows":
        q[:, ::3] = 0
        k[:, 1::4] = 0
        v[:, 2::5] = 0
    elif kind == "large":
        v, state = v * 1e15, state * 1e15
    elif kind == "small":
        v, state = v * 1e-15, state * 1e-15
    elif kind == "growing":  # a positive gate, in one head only
        gate[:, n // 2, 1] = 0.05
    elif kind == "huge":  # past what a state in two fp16 parts is scaled for
        v = v * 1e28
    elif kind == "far_apart":  # value channels of unlike magnitude share a tile
        far = torch.exp2(4.0 * (torch.arange(d, device="cuda") % 16) - 32.0)
        v, state = v * far, state * far[:, None]
    elif kind.startswith("one_write"):  # one token writes, the decay leaves little of it
        beta = torch.where(torch.arange(n, device="cuda")[:, None] == 3, beta, -200.0)
        gate = gate * (2 if kind == "one_write" else 0.4)
    elif kind == "few_writes":  # the first tokens write, the others all but nothing
        beta = torch.where(torch.arange(n, device="cuda")[:, None] < 8, beta, -25.0)
        state = state * 0
    elif kind == "tiny_keys":  # what eps leaves of them is far below one
        k = k * 1e-9
        state = state * 0
    elif kind == "tiny_queries":
        q = q * 1e-9
    elif kind == "late":  # the largest values come last
        v = v * torch.exp2(torch.linspace(-20, 10, n, device="cuda"))[:, None, None]
    elif kind == "closed":  # sigmoid(beta) = 0: nothing is written
        beta = beta * 0 - 200.0
    out = torch.empty_like(v)
    if kind == "reset":
        ref, ref_state, _ = scan64(q, k, v, gate, beta, state, 0.1, None, out, offset)
        got = pk.gated_delta_rule(q, k, v, gate, beta, state, 0.1, EPS)
        assert rel(got, ref) <= scan_limit(n) and rel(state, ref_state) <= scan_limit(n)
        return
    ins = (q, k, v, gate.contiguous(), beta, state, offset)
    ref, ref_state, _ = scan64(*ins[:6], 0.1, None, out, offset)
    got = check_scan(pk, ins, 0.1, None, out)
    # each head and value channel by itself, of the output and of the state
    lim = 4 * scan_limit(n)
    for x, y, over in ((got, ref, 1), (state, ref_state, 3)):
        err, mag = (x.double() - y).norm(dim=over), y.norm(dim=over)
        room = lim * mag + 2.0 ** -126 * x.shape[over] ** 0.5  # f32's smallest normal value
        assert bool((err <= room).all()), float((err / room).max())


def test_scan_pieces_and_tokens(pk):
    """A prompt in pieces and token by token (pkv_deltanet_step) is the prompt at once."""
    say("scan: pieces")
    r = gen(5)
    b, n, hk, h, d = 2, 150, 2, 4, 128
    q, k, v, gate, beta, state, offset = scan_inputs(r, b, n, hk, h, d)
    lin = [pk.LinearAttentionState(conv_dim=(2 * hk + h) * d) for _ in range(3)]
    whole = lin[0].delta_net_chunked(q, k, v, gate, beta)
    cut = [(0, 1), (1, 1), (1, 70), (70, 71), (71, 150)]
    parts = torch.cat([lin[1].delta_net_chunked(*(t[:, a:z] for t in (q, k, v, gate, beta))) for a, z in cut], 1)
    rep = lambda t: t.repeat_interleave(h // hk, 2)  # noqa: E731
    steps = torch.cat([lin[2].delta_net_autoregressive(*(t[:, i:i + 1] for t in (rep(q), rep(k), v, gate, beta)))
                       for i in range(n)], 1)
    for got in (parts, steps):
        assert rel(got, whole) <= 2 * scan_limit(n)
    for other in lin[1:]:
        assert rel(other.recurrent_state.ssm_state, lin[0].recurrent_state.ssm_state) <= 2 * scan_limit(n)
        assert rel(other.recurrent_state.gate_cumsum_offset, lin[0].recurrent_state.gate_cumsum_offset) <= 2 * n * E


def test_scan_is_deterministic(pk):
    say("scan: twice the same")
    r = gen(6)
    ins = scan_inputs(r, 2, 333, 4, 8, 128)
    got = []
    for _ in range(2):
        state = ins[5].clone()
        got.append((pk.gated_delta_rule(*ins[:5], state, 0.1, EPS), state))
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])


def test_scan_token_path_of_some_heads(pk):
    """Heads that cannot go by chunks beside heads that do, 32 value channels a workgroup, over
    several segments, the odd values in the first, a middle and the last one."""
    say("scan: some heads token by token")
    r = gen(14)
    b, n, hk, h, d = 16, 700, 16, 32, 128
    q, k, v, gate, beta, state, offset = scan_inputs(r, b, n, hk, h, d)
    gate[2, 5, 7] = 0.02
    gate[3, 350, 0] = float("-inf")
    k[4, 690, 3] *= 1e-30
    v[5, 300, 9] *= 1e28
    ref, ref_state, ref_offset = scan64(q, k, v, gate, beta, state, 0.1, None, torch.zeros_like(v), offset)
    got = pk.gated_delta_rule(q, k, v, gate, beta, state, 0.1, EPS, gate_offset=offset)
    lim = scan_limit(n)
    err, mag = (got.double() - ref).norm(dim=(1, 3)), ref.norm(dim=(1, 3))
    assert bool((err <= lim * mag).all())
    err, mag = (state.double() - ref_state).norm(dim=(2, 3)), ref_state.norm(dim=(2, 3))
    assert bool((err <= lim * mag).all())
    fin = torch.isfinite(ref_offset)
    assert torch.equal(offset[~fin].double(), ref_offset[~fin])
    # a rounding per segment
    assert bool(((offset.double() - ref_offset)[fin].abs() <= 6 * E * (ref_offset[fin].abs() + 1)).all())


def test_scan_sequences_do_not_touch(pk):
    """A sequence full of NaN leaves the others as they are."""
    say("scan: NaN stays in its sequence")
    r = gen(8)
    ins = scan_inputs(r, 3, 100, 2, 4, 128)
    s0 = ins[5].clone()
    clean = pk.gated_delta_rule(*ins[:5], s0, 0.1, EPS)
    ins[2][1] = float("nan")
    s1 = ins[5].clone()
    got = pk.gated_delta_rule(*ins[:5], s1, 0.1, EPS)
    for i in (0, 2):
        assert torch.equal(got[i], clean[i]) and torch.equal(s1[i], s0[i])
    assert torch.isnan(got[1]).all()


@pytest.mark.parametrize("n,at", [(200, 100), (200, 0), (90, 89), (20, 7)])
@pytest.mark.parametrize("what", ["q", "k", "v", "gate", "beta"])
def test_scan_nan_goes_forward_only(pk, n, at, what):
    """A NaN in one token reaches the tokens behind it, never those in front, and no other
    key head's value heads."""
    say(f"scan: NaN in {what} at {at} of {n}")
    r = gen(9)
    ins = scan_inputs(r, 1, n, 2, 4, 128)
    s0, s1 = ins[5].clone(), ins[5].clone()
    clean = pk.gated_delta_rule(*ins[:5], s0, 0.1, EPS)
    {"q": ins[0], "k": ins[1], "v": ins[2], "gate": ins[3], "beta": ins[4]}[what][0, at, 1] = float("nan")
    got = pk.gated_delta_rule(*ins[:5], s1, 0.1, EPS)
    lim = 2 * scan_limit(n)  # the head with the NaN may go another way
    hit = slice(2, 4) if what in "qk" else slice(1, 2)
    other = [h for h in range(4) if h not in range(4)[hit]]
    assert torch.equal(got[:, :, other], clean[:, :, other]) and torch.equal(s1[:, other], s0[:, other])
    if at:
        assert rel(got[:, :at, hit], clean[:, :at, hit]) <= lim
    assert torch.isnan(got[:, at, hit]).all()
    if what == "q":
        assert rel(s1, s0) <= lim
    elif at + 1 < n:
        assert torch.isnan(got[:, at + 1:, hit]).any()


# ------------------------------------------------------------------ norm
def q8_rows(y):
    """(codes, scales, blocks' bytes) of f32 rows as BlockQ8_0::from_float encodes them."""
    y = y.cpu().numpy()
    rows, d = y.shape
    z = np.zeros((rows, (d + 31) // 32 * 32), np.float32)
    z[:, :d] = y
    z = z.reshape(rows, -1, 32)
    step = (np.nanmax(np.abs(np.where(np.isnan(z), 0, z)), -1, keepdims=True) / np.float32(127)).astype(np.float32)
    with np.errstate(divide="ignore", invalid="ignore"):
        inv = np.where(step != 0, np.float32(1) / step, np.float32(0)).astype(np.float32)
        c = (z * inv).astype(np.float32)
    c = np.where(np.isnan(c), 0, np.clip(np.trunc(c.astype(np.float64) + np.copysign(0.5, c)), -128, 127)).astype(np.int8)
    return np.concatenate([step.astype(np.float16).view(np.uint8).reshape(rows, -1, 2), c.view(np.uint8)], -1)


@pytest.mark.parametrize("rows,d,residual,gate,f32,q8", [
    (1, 2048, True, False, True, False),
    (37, 2048, True, False, True, True),
    (5, 2048, False, False, False, True),
    (130, 128, False, True, True, False),
    (17, 128, False, True, True, True),
    (3, 1, True, False, True, True),
    (9, 33, True, True, True, True),
    (2, 129, False, False, True, True),
    (4, 512, True, False, True, True),
    (4, 515, True, False, True, True),
    (3, 2049, True, True, True, True),
    (2, 8192, True, False, True, True),
    (2, 8196, False, False, True, True),
    (2, 20001, True, True, True, True),
    (1, 32768, True, False, True, True),
])
def test_norm(pk, rows, d, residual, gate, f32, q8):
    say(f"norm rows={rows} d={d} residual={residual} gate={gate} q8={q8}")
    r = gen(rows + d)
    x, alpha = r(rows, d) * 2, 1 + 0.3 * r(d)
    res = r(rows, d) if residual else None
    g = r(rows, d) * 2 if gate else None
    h = x if res is None else res + x
    y, blocks = pk.rms_norm(x, alpha, EPS, residual=res, gate=g, f32_out=f32, q8_0_out=q8)
    if residual:
        assert torch.equal(res, h)
    z = h.double()
    ref = z / (z.square().mean(-1, keepdim=True) + np.float32(EPS)).sqrt() * alpha.double()
    if gate:
        ref = ref * g.double() * torch.sigmoid(g.double())
    if f32:
        # one rounding of 64-bit values; the gate, without 8-bit rows, in 32 bits (8 half steps)
        tol = (1.001 if q8 or not gate else 9) * E
        assert bool(((y.double() - ref).abs() <= tol * ref.abs() + 1e-37).all())
    else:
        assert y is None
    if q8:
        assert blocks.shape == (rows, (d + 31) // 32, 34) and blocks.dtype == torch.uint8
        want = q8_rows(y if f32 else ref.float())
        got = blocks.cpu().numpy()
        if f32:
            assert np.array_equal(got, want)
        else:  # ref.float() may round the other way where 64 bits differ in their last place
            assert np.mean(got != want) < 1e-4
    else:
        assert blocks is None


def test_norm_in_place_and_views(pk):
    say("norm: strides, shapes, zero rows")
    r = gen(12)
    wide, alpha = r(40, 300), r(256)
    dense, _ = pk.rms_norm(wide[:, 20:276].contiguous(), alpha, EPS)
    assert torch.equal(pk.rms_norm(wide[:, 20:276], alpha, EPS)[0], dense)
    odd, _ = pk.rms_norm(wide[:, 21:277].contiguous(), alpha, EPS)
    assert torch.equal(pk.rms_norm(wide[:, 21:277], alpha, EPS)[0], odd)
    four = r(2, 3, 4, 128)
    y, q8 = pk.rms_norm(four, r(128), EPS, q8_0_out=True)
    assert y.shape == four.shape and q8.shape == (2, 3, 4, 4, 34)
    empty, _ = pk.rms_norm(r(0, 256), alpha, EPS)
    assert empty.shape == (0, 256)
    zero, q8 = pk.rms_norm(torch.zeros(3, 256, device="cuda"), alpha, EPS, q8_0_out=True)
    assert not zero.any() and not q8.any()
    from paramecia_amd._lib import lib
    x = r(7, 256)  # out may be x itself
    want, _ = pk.rms_norm(x.clone(), alpha, EPS)
    assert lib().pkv_rms_norm(x.data_ptr(), 256, None, alpha.data_ptr(), None, EPS, x.data_ptr(), None, 7, 256,
                              torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(x, want)


def test_norm_values(pk):
    """A row of infinities or NaN, huge and tiny rows, beside ordinary ones."""
    say("norm: values")
    r = gen(13)
    x, alpha = r(6, 2048), 1 + 0.1 * r(2048)
    clean, cq = pk.rms_norm(x.clone(), alpha, EPS, q8_0_out=True)
    x[1] = float("nan")
    x[2, 5] = float("inf")
    x[3] *= 1e30
    x[4] *= 1e-30
    y, q8 = pk.rms_norm(x, alpha, EPS, q8_0_out=True)
    for i in (0, 5):
        assert torch.equal(y[i], clean[i]) and torch.equal(q8[i], cq[i])
    assert torch.isnan(y[1]).all() and torch.isnan(y[2, 5]) and not y[2, :5].any()
    assert not q8[1].any()  # as the cache encodes a block of NaN
    z = x.double()
    ref = z / (z.square().mean(-1, keepdim=True) + np.float32(EPS)).sqrt() * alpha.double()
    for i in (3, 4):
        assert bool(((y[i].double() - ref[i]).abs() <= 1.001 * E * ref[i].abs() + 1e-45).all())


# ------------------------------------------------------------------ adapters
def lora64(x, g, wdq, a, b, scale, ids, n):
    y = x.double() if g is None else x.double() * torch.sigmoid(g.double())
    out = y @ wdq.T
    base = out.clone()
    for i, s in enumerate(ids):
        if 0 <= s < n:
            out[i] += scale[s].double() * (b[s].double() @ (a[s].double() @ y[i]))
    return out, base


W_BYTES = {8: 34 / 32, 12: 144 / 256, 13: 176 / 256, 14: 210 / 256}


@pytest.mark.parametrize("rows,inner,width,rank,n,dtype,w_type,gated", [
    (1, 4096, 2048, 16, 3, "bfloat16", 12, True),
    (1, 4096, 100, 1, 1, "float32", 12, False),
    (3, 8192, 64, 7, 4, "float16", 12, True),
    (7, 4096, 70, 33, 2, "bfloat16", 14, True),
    (8, 4096, 256, 64, 5, "float16", 12, True),
    (24, 4096, 2048, 32, 9, "float16", 12, True),
    (16, 4096, 130, 17, 6, "float32", 13, True),
    (33, 8192, 72, 128, 3, "bfloat16", 12, False),
    (40, 4096, 96, 5, 40, "bfloat16", 8, True),
    (130, 4096, 300, 20, 4, "float16", 8, True),    # Q8_0 weights, batched
    (70, 8192, 513, 33, 5, "float32", 8, False),
    (13, 4096, 2048, 16, 13, "bfloat16", 8, True),
    (130, 4096, 300, 64, 3, "bfloat16", 12, True),
    (257, 4096, 513, 20, 4, "float16", 14, True),
    (600, 4096, 64, 8, 2, "float32", 12, True),
    (2, 4096, 40, 100, 3, "float16", 14, True),
    (5, 8192, 33, 128, 2, "float32", 8, False),
    (64, 4096, 257, 16, 50, "float16", 12, True),
])
def test_lora(pk, orc, rows, inner, width, rank, n, dtype, w_type, gated):
    from kquant_blocks import random_weight_bytes
    say(f"lora rows={rows} in={inner} out={width} rank={rank} n={n} {dtype} w={w_type}")
    r = gen(rows + width + rank)
    rng = np.random.default_rng(rows + width)
    t = getattr(torch, dtype)
    wb = random_weight_bytes(rng, w_type, width, inner, d_scale=1e-4)
    x, g = r(rows, inner), r(rows, inner) if gated else None
    a, b, scale = (r(n, rank, inner) * inner ** -0.5).to(t), (r(n, width, rank) * rank ** -0.5).to(t), 1 + r(n).abs()
    ids = rng.integers(-1, n, rows)
    ids[0] = n - 1
    if rows > 100:
        ids = np.sort(ids)  # prompts: a request's rows stand together
    wdq = torch.from_numpy(orc.dequantize_weight(wb, w_type, width * inner).reshape(width, inner)).cuda().double()
    ref, base = lora64(x, g, wdq, a, b, scale, ids.tolist(), n)
    got = pk.gated_o_proj_lora(x, g, torch.from_numpy(wb).cuda(), width, a, b, scale,
                               torch.from_numpy(ids.astype(np.int32)).cuda(), w_type=w_type)
    # f32 sums: a chain of m roundings of a growing sum of independent terms is off by about
    # E / 2 * sqrt(m / 2), m at most 4096: 1.4e-6; elementwise, as the projection's own tests
    say(f"  rel {rel(got, ref):.2e}")
    assert rel(got, ref) < 2e-6
    assert float((got.double() - ref).abs().max() / ref.square().mean().sqrt()) < 2e-5
    if rows > 1 and (ids < 0).any():  # rows without an adapter are the projection's
        plain = pk.gated_o_proj(x, g, torch.from_numpy(wb).cuda(), width, w_type=w_type)
        at = torch.from_numpy(ids < 0).cuda()
        if w_type == 8 and rows * inner * width > 3 << 25:  # the projection alone goes token by token
            assert rel(got[at], plain[at]) < 2 * 2e-6
        else:
            assert torch.equal(got[at], plain[at])
    assert pk.lib().pkv_device_status() == 0


def test_lora_ids_and_values(pk, orc):
    """No adapter anywhere, an id past the adapters (reported, no adapter taken), an unused
    adapter full of NaN, twice the same adapter, any order of ids."""
    from kquant_blocks import random_weight_bytes
    say("lora: ids")
    r = gen(99)
    rng = np.random.default_rng(99)
    rows, inner, width, rank, n = 20, 4096, 96, 8, 4
    wb = torch.from_numpy(random_weight_bytes(rng, 12, width, inner, d_scale=1e-4)).cuda()
    x, g = r(rows, inner), r(rows, inner)
    a, b, scale = r(n, rank, inner) * inner ** -0.5, r(n, width, rank), torch.ones(n, device="cuda")
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    run = lambda ids: pk.gated_o_proj_lora(x, g, wb, width, a, b, scale, i32(ids))  # noqa: E731
    plain = pk.gated_o_proj(x, g, wb, width)
    assert torch.equal(run([-1] * rows), plain)
    assert torch.equal(run([-7, -2 ** 31] * (rows // 2)), plain)
    a[2], b[2], scale[2] = float("nan"), float("nan"), float("nan")
    ids = [3, 0, 0, 1, -1, 3, 1, 0, 3, 3] * 2
    first = run(ids)
    assert torch.isfinite(first).all() and not torch.equal(first, plain)
    assert torch.equal(run(ids), first)
    order = torch.randperm(rows, device="cuda")
    mixed = pk.gated_o_proj_lora(x[order], g[order], wb, width, a, b, scale, i32(ids)[order])
    assert rel(mixed, first[order]) < 2e-6
    assert pk.lib().pkv_device_status() == 0
    ids[4] = n
    past = run(ids)
    assert torch.equal(past, first)
    from paramecia_amd._lib import ERR_HIP, lib
    assert lib().pkv_device_status() == ERR_HIP and b"adapter id" in lib().pkv_last_error()
    assert lib().pkv_device_status() == 0
    shaped = pk.gated_o_proj_lora(x.view(2, 10, inner), g.view(2, 10, inner), wb, width, a, b, scale,
                                  i32(ids).view(2, 10))
    assert torch.equal(shaped.view(rows, width), first)
    lib().pkv_device_status()


# ------------------------------------------------------------------ the layer
def layer(pk, lin, x, z, p, ids, lens=None):
    """A Gated-DeltaNet layer from its projections to the next layer's input: convolution,
    state update, norm per head with its gate, projection with adapters, residual and norm."""
    hk, h, d = 16, 32, 128
    b, n, _ = x.shape
    c = lin.causal_conv(x, p["conv"], h, d, lens=lens)
    q, k, v = c.split([hk * d, hk * d, h * d], -1)
    o = lin.delta_net_chunked(q.unflatten(-1, (hk, d)), k.unflatten(-1, (hk, d)), v.unflatten(-1, (h, d)),
                              p["gate"][:, :n], p["beta"][:, :n], lens=lens)
    y, _ = pk.rms_norm(o, p["head_alpha"], EPS, gate=z)
    m = pk.gated_o_proj_lora(y.flatten(2), None, p["wo"], 2048, p["a"], p["b"], p["scale"], ids)
    return pk.rms_norm(m, p["alpha"], EPS, residual=p["stream"], q8_0_out=True)


def layer_inputs(pk, b, n, seed):
    from kquant_blocks import random_weight_bytes
    r = gen(seed)
    p = dict(conv=0.5 * r(8192, 4), gate=-torch.nn.functional.softplus(r(b, n, 32)), beta=r(b, n, 32),
             head_alpha=1 + 0.1 * r(128), alpha=1 + 0.1 * r(2048), stream=r(b, n, 2048),
             a=(r(3, 16, 4096) / 64).bfloat16(), b=(r(3, 2048, 16) / 4).bfloat16(), scale=1 + r(3).abs(),
             wo=torch.from_numpy(random_weight_bytes(np.random.default_rng(seed), 12, 2048, 4096, d_scale=1e-4)).cuda())
    return r(b, n, 8192), r(b, n, 32, 128), p


def test_layer_matches_formulas(pk, orc):
    """A prompt and the token behind it, in a padded batch, against the same in 64 bits."""
    say("layer")
    b, n = 2, 70
    x, z, p = layer_inputs(pk, b, n + 1, 21)
    lens = torch.tensor([70, 33], dtype=torch.int32, device="cuda")
    lin = pk.LinearAttentionState()
    ids = torch.tensor([[1], [-1]], dtype=torch.int32, device="cuda").expand(b, n + 1).contiguous()
    stream0 = p["stream"].clone()
    wdq = torch.from_numpy(orc.dequantize_weight(p["wo"].cpu().numpy(), 12, 2048 * 4096).reshape(2048, 4096)).cuda().double()
    conv_state = torch.zeros(b, 8192, 3, device="cuda").double()
    state, off = torch.zeros(b, 32, 128, 128, device="cuda").double(), torch.zeros(b, 32, device="cuda")

    def ref(xs, zs, gate, beta, stream, ids, lens, conv_state, state):
        m = xs.shape[1]
        zero = torch.zeros(b, m, 8192, device="cuda")
        c, conv_state, _ = conv64(xs, p["conv"], conv_state, None, lens, True, zero)
        q, k, v = c.split([2048, 2048, 4096], -1)
        o, state, _ = scan64(q.unflatten(-1, (16, 128)), k.unflatten(-1, (16, 128)), v.unflatten(-1, (32, 128)),
                             gate, beta, state, 128 ** -0.5, lens, torch.zeros(b, m, 32, 128, device="cuda"), off)
        y = o / (o.square().mean(-1, keepdim=True) + EPS).sqrt() * p["head_alpha"].double()
        y = (y * zs.double() * torch.sigmoid(zs.double())).flatten(2).flatten(0, 1)
        out, _ = lora64(y, None, wdq, p["a"], p["b"], p["scale"], ids.flatten().tolist(), 3)
        hh = stream.double() + out.view(b, m, 2048)
        return hh / (hh.square().mean(-1, keepdim=True) + EPS).sqrt() * p["alpha"].double(), hh, conv_state, state

    p["stream"] = stream0[:, :n].contiguous()
    y, q8 = layer(pk, lin, x[:, :n], z[:, :n].contiguous(), p, ids[:, :n].contiguous(), lens=lens)
    r1, h1, conv_state, state = ref(x[:, :n], z[:, :n], p["gate"][:, :n], p["beta"][:, :n], stream0[:, :n], ids[:, :n],
                                    lens.tolist(), conv_state, state)
    # each stage passes the error in front of it on and adds its own; the norm per head can
    # raise a small head's: ten times the largest of the stages' limits
    lim = 10 * 2e-6
    for i, e in enumerate(lens.tolist()):
        say(f"  y {rel(y[i, :e], r1[i, :e]):.2e} stream {rel(p['stream'][i, :e], h1[i, :e]):.2e}")
        assert rel(y[i, :e], r1[i, :e]) < lim and rel(p["stream"][i, :e], h1[i, :e]) < lim
    assert np.array_equal(q8.cpu().numpy().reshape(b * n, 64, 34), q8_rows(y.view(b * n, 2048)))
    # the token behind the prompt, of each sequence
    p2 = dict(p, gate=p["gate"][:, n:], beta=p["beta"][:, n:], stream=stream0[:, n:].contiguous())
    y2, _ = layer(pk, lin, x[:, n:], z[:, n:].contiguous(), p2, ids[:, n:].contiguous())
    r2, *_ = ref(x[:, n:], z[:, n:], p["gate"][:, n:], p["beta"][:, n:], stream0[:, n:], ids[:, n:], None, conv_state, state)
    assert rel(y2, r2) < lim


@pytest.mark.parametrize("b,n", [(3, 1), (1, 200)])
def test_layer_in_a_graph(pk, b, n):
    """The layer captured once and replayed on new inputs, with eager work of the same layer
    between the replays, gives what eager calls give; two graphs in turn do not disturb each
    other."""
    say(f"layer in a graph b={b} n={n}")
    x, z, p = layer_inputs(pk, b, n, 31)
    ids = torch.zeros(b, n, dtype=torch.int32, device="cuda")
    stream0 = p["stream"].clone()

    def fresh():
        lin = pk.LinearAttentionState()
        lin._state(b, 32, 128, x.device)
        return lin

    def eager(lin, x):
        p["stream"].copy_(stream0)
        y, q8 = layer(pk, lin, x, z, p, ids)
        return y, q8, lin.recurrent_state.ssm_state.clone()

    want_lin = fresh()
    xs = [x * f for f in (1.0, 0.5, -1.0)]
    want = [eager(want_lin, v) for v in xs]
    side = torch.cuda.Stream()
    graphs = []
    for _ in range(2):
        lin, static = fresh(), x.clone()
        with torch.cuda.stream(side):
            eager(fresh(), static)
        side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            p["stream"].copy_(stream0)
            y, q8 = layer(pk, lin, static, z, p, ids)
        lin.recurrent_state.ssm_state.zero_()
        lin.recurrent_state.conv_state.zero_()
        graphs.append((g, lin, static, y, q8))
    for step, v in enumerate(xs):
        for g, lin, static, y, q8 in graphs:
            static.copy_(v)
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, want[step][0]) and torch.equal(q8, want[step][1])
            assert torch.equal(lin.recurrent_state.ssm_state, want[step][2])
            eager(fresh(), v)


def test_two_streams(pk):
    """Two layers' calls on two streams at once are what they are one after the other."""
    say("two streams")
    sets = [layer_inputs(pk, 1, 150, 41 + i) for i in range(2)]
    ids = torch.zeros(1, 150, dtype=torch.int32, device="cuda")
    want = []
    for x, z, p in sets:
        want.append(layer(pk, pk.LinearAttentionState(), x, z, dict(p, stream=p["stream"].clone()), ids)[0])
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in sets], [None, None]
    for _ in range(3):
        for i, (x, z, p) in enumerate(sets):
            with torch.cuda.stream(streams[i]):
                got[i] = layer(pk, pk.LinearAttentionState(), x, z, dict(p, stream=p["stream"].clone()), ids)[0]
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert torch.equal(g, w)


# ------------------------------------------------------------------ offsets past 2^32 bytes
def test_long_prompt(pk):
    """131109 tokens of 8192 channels (4.3 GB): the convolution's last tokens are those of its
    last inputs alone, and the scan over slices of such rows is the scan in two pieces."""
    say("long prompt")
    r = gen(51)
    n, ch, hk, h, d, tail = 131109, 8192, 16, 32, 128, 1000
    x, w = r(1, n, ch), r(ch, 4)
    state = torch.zeros(1, ch, 3, device="cuda")
    y = pk.causal_conv(x, w, state)
    torch.cuda.synchronize()
    at = n - tail
    s = x[:, at - 3:at].transpose(1, 2).contiguous()
    assert torch.equal(pk.causal_conv(x[:, at:], w, s), y[:, at:]) and torch.equal(s, state)
    assert torch.equal(state[0], x[0, -3:].T)
    say("  scan")
    q, k, v = (t.view(1, n, -1, d) for t in (y[..., :2048], y[..., 2048:4096], y[..., 4096:]))
    gate, beta = -0.1 * r(1, n, h).abs(), r(1, n, h)
    s1, s2 = torch.zeros(1, h, d, d, device="cuda"), torch.zeros(1, h, d, d, device="cuda")
    whole = pk.gated_delta_rule(q, k, v, gate, beta, s1, d ** -0.5, EPS)
    parts = [pk.gated_delta_rule(*(t[:, a:z].contiguous() for t in (q, k, v, gate, beta)), s2, d ** -0.5, EPS)
             for a, z in ((0, at), (at, n))]
    # each is off by the errors that the state has kept: those of some 1 / 0.08 tokens, as its
    # gates are -0.08 on average; a hundred are allowed for
    assert rel(whole[:, at:], parts[1]) <= 2 * scan_limit(100) and rel(s1, s2) <= 2 * scan_limit(100)
    assert rel(whole[:, :at], parts[0]) <= 2 * scan_limit(100)


def test_many_rows(pk):
    """600037 rows of 2048 (4.9 GB): the last ones are the norm of these rows alone."""
    say("many rows")
    r = gen(52)
    rows, d = 600037, 2048
    x, res, alpha = r(rows, d), r(rows, d), 1 + 0.1 * r(d)
    xs, rs = x[-50:].clone(), res[-50:].clone()
    y, q8 = pk.rms_norm(x, alpha, EPS, residual=res, q8_0_out=True)
    ys, qs = pk.rms_norm(xs, alpha, EPS, residual=rs, q8_0_out=True)
    assert torch.equal(y[-50:], ys) and torch.equal(q8[-50:], qs) and torch.equal(res[-50:], rs)


@pytest.mark.parametrize("rows", [2, 9])
def test_many_adapters(pk, rows):
    """2200 adapters of rank 128 over 8192 inputs (4.6 GB), the last one beside itself alone."""
    from kquant_blocks import random_weight_bytes
    say(f"many adapters rows={rows}")
    r = gen(53)
    n, rank, inner, width = 2200, 128, 8192, 64
    wb = torch.from_numpy(random_weight_bytes(np.random.default_rng(1), 12, width, inner, d_scale=1e-4)).cuda()
    a = torch.zeros(n, rank, inner, dtype=torch.bfloat16, device="cuda")
    b = torch.zeros(n, width, rank, dtype=torch.bfloat16, device="cuda")
    a[-1], b[-1] = (r(rank, inner) * inner ** -0.5).bfloat16(), (r(width, rank) * rank ** -0.5).bfloat16()
    x, scale = r(rows, inner), torch.ones(n, device="cuda")
    ids = torch.full((rows,), n - 1, dtype=torch.int32, device="cuda")
    many = pk.gated_o_proj_lora(x, None, wb, width, a, b, scale, ids)
    one = pk.gated_o_proj_lora(x, None, wb, width, a[-1:], b[-1:], scale[-1:], torch.zeros_like(ids))
    assert torch.equal(many, one)
    assert float((many - pk.gated_o_proj(x, None, wb, width)).abs().max()) > 0
