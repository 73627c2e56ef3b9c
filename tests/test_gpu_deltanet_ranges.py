"""The gated delta rule over prompts (delta_net_chunked, paramecia-model/src/qwen3_next.rs:
3506-3731) where magnitudes differ: states that decay away, values that fall, rise or jump
within a chunk, masked tokens, eps = 0, infinite states; at every head size, over chunks,
segments and the token-by-token form, each token and value channel held by itself.

A row S_i of the state (value channel i) has a norm of at most
  N_t = exp(gate_t) N_(t-1) + sigmoid(beta_t) |v_ti|,  N_0 = |S_i|
while no gate is positive, as I - sigmoid(beta) k k^T lengthens nothing (|k| <= 1). A token's
step rounds some 16 times, by half a step of f32 (E = 2^-24) of values up to N_t, and what it is
off decays as N_t does; errors of n tokens that add up as independent ones make
E (16 + 2 sqrt(n)) N_t of the row, and scale times that of an output, as |q| <= 1."""
import random
import sys

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
TINY = 2.0 ** -126  # f32's smallest normal value: nothing is held to a relative precision below


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


def formula(q, k, v, gate, beta, state, scale, eps, lens=None):
    """(outputs, state, N of every token, N behind the last) token by token in 64 bits; rows
    behind a sequence's end are zeros."""
    b, n, hk, d = q.shape
    rep = v.shape[2] // hk
    end = torch.full((b,), n) if lens is None else torch.tensor(lens)
    end = end.clamp(0, n).to(q.device)
    q, k, v, gate, beta, s = (t.double() for t in (q, k, v, gate, beta, state))
    q = (q * scale / (q.square().sum(-1, keepdim=True) + eps).sqrt()).repeat_interleave(rep, 2)
    k = (k / (k.square().sum(-1, keepdim=True) + eps).sqrt()).repeat_interleave(rep, 2)
    alpha, be = gate.exp(), torch.sigmoid(beta)
    out, size, norm = torch.zeros_like(v), torch.zeros_like(v), s.norm(dim=-1)
    for t in range(n):
        on = (t < end)[:, None, None]
        old = s * alpha[:, t, :, None, None]
        u = be[:, t, :, None] * (v[:, t] - (old * k[:, t, :, None]).sum(-1))
        new = old + u[..., None] * k[:, t, :, None]
        grown = norm * alpha[:, t, :, None] + be[:, t, :, None] * v[:, t].abs()
        out[:, t] = torch.where(on, (new * q[:, t, :, None]).sum(-1), out[:, t])
        size[:, t] = torch.where(on, grown, size[:, t])
        s, norm = torch.where(on[..., None], new, s), torch.where(on, grown, norm)
    return out, s, size, norm


def inputs(seed, b, n, hk, h, d):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    return (r(b, n, hk, d), r(b, n, hk, d), r(b, n, h, d), -0.5 * torch.nn.functional.softplus(r(b, n, h)),
            r(b, n, h), 0.3 * r(b, h, d, d))


def check(pk, q, k, v, gate, beta, state, eps=1e-6, lens=None, scale=0.1):
    n = q.shape[1]
    want, want_state, size, norm = formula(q, k, v, gate, beta, state, scale, eps, lens)
    out = torch.zeros_like(v)
    dl = None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")
    pk.gated_delta_rule(q, k, v, gate.contiguous(), beta.contiguous(), state, scale, eps, lens=dl, out=out)
    lim = E * (16 + 2 * n ** 0.5)
    assert torch.isfinite(out).all() and torch.isfinite(state).all()
    off = ((out.double() - want).abs() / (scale * (lim * size + TINY))).max()
    # what decays by more than e^-87 within a chunk may be taken for nothing
    off_state = ((state.double() - want_state).norm(dim=-1) / (lim * norm + TINY * state.shape[-1] ** 0.5)).max()
    say(f"  off by {float(off):.2e} of the limit, the state by {float(off_state):.2e}")
    assert off <= 1 and off_state <= 1
    return out


KINDS = ["plain", "silent", "whisper", "falling", "falling_chunk", "early", "late", "jump", "masked_jump", "masked_token",
         "fast", "forgetful", "opened"]


def shaped(kind, q, k, v, gate, beta, state):
    n = q.shape[1]
    t = torch.arange(n, device="cuda")
    ramp = torch.linspace(0, 1, n, device="cuda")[:, None, None]
    if kind in ("silent", "whisper"):  # a decay of e^-31, then values of zero, or next to it
        gate = torch.where(t[:, None] == 3, -30.0, -1e-3).expand_as(gate)
        v = v * (0.0 if kind == "silent" else 1e-20)
    elif kind == "falling":  # values far below the state in front of them, which decays
        gate, v = gate * 0 - 1.0, v * 1e-8
    elif kind == "falling_chunk":  # from one chunk to the next
        gate, v = gate * 0 - 1.0, torch.where((t < 64)[:, None, None], v, v * 1e-6)
        state = state * 0
    elif kind == "early":
        v, state = v * torch.exp2(-60 * ramp), state * 0
    elif kind == "late":
        v, state = v * torch.exp2(60 * ramp - 60), state * 0
    elif kind == "jump":  # one token's values outweigh those in front of it in its chunk
        v, state = torch.where((t % 64 == 50)[:, None, None], v * 2.0 ** 30, v), state * 0
    elif kind == "masked_jump":  # sigmoid(beta) = 0: nothing of them is written
        at = t % 64 == 20
        v, beta = torch.where(at[:, None, None], v * 2.0 ** 40, v), torch.where(at[:, None], -200.0, beta)
    elif kind == "masked_token":  # next to nothing of them is written
        at = t % 64 == 20
        v, beta = torch.where(at[:, None, None], v * 2.0 ** 20, v), torch.where(at[:, None], -25.0, beta)
    elif kind == "fast":
        gate = gate * 0 - 11.0
    elif kind == "forgetful":  # a large state gone at once, small values behind
        gate, v, state = torch.where(t[:, None] % 64 == 7, -60.0, gate), v * 1e-10, state * 1e6
    elif kind == "opened":  # the first tokens write all but nothing
        beta, state = torch.where((t < 40)[:, None], -30.0, beta), state * 0
    return q, k, v, gate, beta, state


def workspace(pk, q, v):
    b, n, hk, d = q.shape
    return pk.lib().pkv_deltanet_prompt_workspace(b, n, hk, v.shape[2], d)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("n", [193, 256, 330])
@pytest.mark.parametrize("kind", KINDS)
def test_magnitudes(pk, kind, n, d):
    say(f"magnitudes {kind} n={n} d={d}")
    ins = shaped(kind, *inputs(n + d, 1, n, 1, 2, d))
    assert workspace(pk, ins[0], ins[2]) > 0  # by chunks
    check(pk, *ins)


@pytest.mark.parametrize("kind", KINDS)
def test_magnitudes_of_few_tokens(pk, kind):
    say(f"magnitudes {kind}, token by token")
    ins = shaped(kind, *inputs(41, 1, 41, 1, 2, 128))
    assert workspace(pk, ins[0], ins[2]) == 0
    check(pk, *ins)


@pytest.mark.parametrize("b,n,hk,h,d,lens", [
    (1, 72, 1, 1, 256, None),
    (2, 130, 2, 4, 256, [130, 65]),
    (1, 300, 2, 2, 256, None),                   # five chunks, an odd number
    (1, 257, 1, 3, 64, None),
    (4, 200, 2, 4, 64, [200, 0, 129, 64]),
    (2, 3100, 8, 16, 256, [3100, 1000]),         # more than one segment
    (4, 2200, 16, 32, 64, [2200, 2100, 5, 2048]),
    (2, 80, 16, 32, 128, [80, 33]),              # a padded batch by chunks
])
def test_sizes_by_chunks(pk, b, n, hk, h, d, lens):
    say(f"sizes b={b} n={n} hk={hk} h={h} d={d} lens={lens}")
    ins = inputs(n + h, b, n, hk, h, d)
    assert workspace(pk, ins[0], ins[2]) > 0
    for i, e in enumerate([n] * b if lens is None else lens):
        for t in ins[:5]:
            t[i, e:] = float("nan")  # padding is not read
    clean = [t.nan_to_num() for t in ins[:5]]
    want, want_state, size, norm = formula(*clean, ins[5], 0.1, 1e-6, lens)
    out, state = torch.zeros_like(ins[2]), ins[5].clone()
    dl = None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")
    pk.gated_delta_rule(*ins[:5], state, 0.1, 1e-6, lens=dl, out=out)
    lim = E * (16 + 2 * n ** 0.5)
    assert bool(((out.double() - want).abs() <= 0.1 * lim * size).all())
    assert bool(((state.double() - want_state).norm(dim=-1) <= lim * norm).all())


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("what", ["gate", "closed_gate", "key", "value"])
def test_heads_token_by_token_beside_chunks(pk, what, d):
    """A head that cannot go by chunks, from its second chunk on, beside one that does."""
    say(f"odd head: {what} d={d}")
    q, k, v, gate, beta, state = inputs(d, 1, 300, 2, 4, d)
    if what == "gate":
        gate[0, 100, 1] = 0.05
    elif what == "closed_gate":
        gate[0, 100, 1] = -20000.0
    elif what == "key":
        k[0, 100, 1] *= 1e-30
    else:
        v[0, 100, 1] *= 1e28
    check(pk, q, k, v, gate, beta, state)


@pytest.mark.parametrize("d", [64, 256])
@pytest.mark.parametrize("at", [0, 130, 299])
def test_nan_goes_forward_only(pk, d, at):
    say(f"NaN at {at} d={d}")
    ins = inputs(d + at, 1, 300, 1, 2, d)
    s0, s1 = ins[5].clone(), ins[5].clone()
    want, _, size, _ = formula(*ins[:5], s0, 0.1, 1e-6)
    clean = pk.gated_delta_rule(*ins[:5], s0, 0.1, 1e-6)
    ins[2][0, at, 1, 5] = float("nan")
    got = pk.gated_delta_rule(*ins[:5], s1, 0.1, 1e-6)
    assert torch.equal(got[:, :, 0], clean[:, :, 0]) and torch.equal(s1[:, 0], s0[:, 0])
    lim = 0.1 * E * (16 + 2 * 300 ** 0.5)
    assert bool(((got[:, :at, 1].double() - want[:, :at, 1]).abs() <= lim * size[:, :at, 1]).all())
    assert torch.isnan(got[0, at:, 1, 5]).all() and torch.isnan(s1[0, 1, 5]).all()
    others = [i for i in range(d) if i != 5]  # a value channel reaches no other
    assert torch.isfinite(got[0, :, 1, others]).all() and torch.isfinite(s1[0, 1, others]).all()


@pytest.mark.parametrize("b,n,d,lens", [(1, 1, 128, None), (2, 5, 64, None), (1, 17, 128, None), (1, 7, 256, None),
                                        (3, 40, 128, [40, 3, 0]), (1, 100, 128, None), (2, 90, 256, [90, 70])])
def test_eps_zero(pk, b, n, d, lens):
    """Without eps every key and query has a norm to divide by; padding has none."""
    say(f"eps=0 b={b} n={n} d={d}")
    check(pk, *inputs(n, b, n, 2, 4, d), eps=0.0, lens=lens)


@pytest.mark.parametrize("b,n,d,lens", [(1, 5, 128, None), (1, 3, 256, None), (2, 40, 64, [40, 19]), (1, 100, 128, None)])
def test_infinite_state_is_kept(pk, b, n, d, lens):
    """The last token writes an infinity: what the slots behind it hold changes nothing."""
    say(f"infinite state b={b} n={n} d={d}")
    ins = inputs(n, b, n, 1, 2, d)
    for i, e in enumerate([n] * b if lens is None else lens):
        ins[2][i, e - 1, 1, 3] = float("inf")
    _, want, _, _ = formula(*ins, 0.1, 1e-6, lens)
    dl = None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")
    pk.gated_delta_rule(*ins, 0.1, 1e-6, lens=dl)
    assert torch.isinf(want[:, 1, 3]).all() and torch.equal(ins[5][:, 1, 3].double(), want[:, 1, 3])
    fine = torch.isfinite(want)
    lim = E * (16 + 2 * n ** 0.5)
    assert bool(((ins[5].double() - want)[fine].abs() <= 40 * lim).all())


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("n", [193, 200, 256, 320])
@pytest.mark.parametrize("kind", ["silent", "whisper"])
def test_vanishing_state_stays_finite(pk, kind, n, d):
    """What is left of a state far below its scale, with no values to hide it."""
    say(f"vanishing state {kind} n={n} d={d}")
    q, k, v, gate, beta, state = shaped(kind, *inputs(n + d, 1, n, 1, 2, d))
    assert workspace(pk, q, v) > 0
    out = pk.gated_delta_rule(q, k, v, gate.contiguous(), beta, state, 0.1, 1e-6)
    assert torch.isfinite(out).all() and torch.isfinite(state).all()
    assert float(state.abs().max()) < 1e-9 and float(out[:, 64:].abs().max()) < 1e-9


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rate", [0.3, 0.97, 1.21])
def test_one_write_ages(pk, rate, d):
    """One token writes, along the only key, and decays by up to e^-77 in its chunk: what is left of it
    is off by the roundings of its tokens' decays."""
    say(f"one write ages rate={rate} d={d}")
    n = 128
    q, k, v, gate, beta, state = inputs(d, 1, n, 1, 2, d)
    k = k[:, :1].expand_as(k).contiguous()
    q, gate, state = k.clone(), gate * 0 - rate, state * 0
    gate[..., 1] *= 1.01
    for at in (0, 64):
        b = torch.where((torch.arange(n, device="cuda") == at)[:, None], 3.0, -200.0).expand_as(beta)
        check(pk, q, k, v, gate, b, state.clone())
        check(pk, *(t[:, :at + 72].contiguous() for t in (q, k, v, gate, b)), state.clone())


@pytest.mark.parametrize("seed", range(32))
def test_mixes(pk, seed):
    """Spans of values over tokens and channels, decays, gates, keys and states, mixed at random."""
    rng = random.Random(seed)
    d, n, hk, b = rng.choice([64, 128, 256]), rng.choice([72, 100, 128, 193, 256, 330]), rng.choice([1, 2]), rng.choice([1, 2])
    h = hk * rng.choice([1, 2, 3])
    q, k, v, _, beta, state = inputs(seed, b, n, hk, h, d)
    rand = lambda *s: torch.rand(s, device="cuda", generator=g)  # noqa: E731
    g = torch.Generator(device="cuda").manual_seed(100 + seed)
    if rng.random() < 0.4:
        k = k[:, :1] + rng.choice([0, 0.01, 0.3]) * k
    v = v * torch.exp2(-rng.choice([0, 5, 20, 40, 60]) * rand(b, n, 1, 1) - rng.choice([0, 10, 40]) * rand(1, 1, h, d))
    v = v * 2.0 ** rng.choice([0, -40, 40, 60])
    if rng.random() < 0.3:
        v = v * (rand(b, n, h, 1) < 0.1)
    gate = -rng.choice([1e-5, 1e-3, 0.1, 1, 5, 20]) * rand(b, n, h) ** rng.choice([1, 4, 16])
    if rng.random() < 0.3:
        gate = torch.where(rand(b, n, h) < 0.03, -rng.choice([20.0, 60.0, 90.0, 300.0, 9000.0]), gate)
    beta = rng.choice([1, 5, 40]) * beta + rng.choice([-5, 0, 5])
    state = state * rng.choice([0, 1, 1e-8, 1e6])
    eps = rng.choice([1e-6, 1e-12, 1.0])
    say(f"mix {seed}: b={b} n={n} hk={hk} h={h} d={d} eps={eps}")
    want, want_state, size, norm = formula(q, k, v, gate, beta, state, 0.1, eps)
    # what decays by more than e^-87 within a chunk is held to 2^-126 of the largest so far
    least = TINY * (1 + float(size.max()) + float(state.norm(dim=-1).max()))
    out = pk.gated_delta_rule(q, k, v, gate, beta, state, 0.1, eps)
    lim = E * (16 + 2 * n ** 0.5)
    assert bool(((out.double() - want).abs() <= 0.1 * (lim * size + least)).all())
    assert bool(((state.double() - want_state).norm(dim=-1) <= lim * norm + least * d ** 0.5).all())
