"""The operators of a Gated-DeltaNet layer around its single-token state update, and of the
layer's end, as cases to be timed.

A model of this framework has 48 layers; 36 of them keep a recurrent state instead of a
cache. From such a layer's projections to the next layer's input a prompt or a token passes

- conv:  the short causal convolution (4 taps, 8192 channels, SiLU) over q, k and v, whose
         last 3 inputs are kept as the sequence's conv state;
- scan:  the gated delta rule over all tokens of a prompt: 16 key heads, 32 value heads of
         128, one 128 x 128 state per value head;
- lora:  the output projection (4096 -> 2048, GGUF weights) with the low-rank adapter that
         each request has chosen, if any;
- norm:  the root-mean-square norm behind the residual's addition, in f32 and in Q8_0 blocks
         for the next projections, and the norm per head with its output gate.

`draw` takes more of each: prompts from one token to 8001, one to 24 sequences, padded
batches of ragged lengths, other head counts, widths, ranks, adapter and weight types.
"""
import math

import torch

own = False

HIDDEN, INNER = 2048, 4096
EPS = 1e-6
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
W_TYPE = {"q8_0": 8, "q4k": 12, "q6k": 14}
W_BLOCK = {"q8_0": (32, 34), "q4k": (256, 144), "q6k": (256, 210)}


def listed():
    return [
        # the next token of 16 conversations: only the newest input and 3 kept ones per channel
        dict(name="conv_token_16", op="conv", batch=16, n=1, channels=8192, taps=4, bias=False, ragged=False),
        # a long prompt of ragged length
        dict(name="conv_prompt_8k", op="conv", batch=1, n=8001, channels=8192, taps=4, bias=False, ragged=False),
        # five drafted tokens that are verified at once
        dict(name="scan_verify_5", op="scan", batch=1, n=5, key_heads=16, heads=32, dim=128, ragged=False),
        # a question: the first prompt of a chat
        dict(name="scan_prompt_509", op="scan", batch=1, n=509, key_heads=16, heads=32, dim=128, ragged=False),
        # seven prompts that a server takes together, padded to the longest
        dict(name="scan_ragged_7x1100", op="scan", batch=7, n=1100, key_heads=16, heads=32, dim=128, ragged=True),
        # a file or a long conversation as one prompt
        dict(name="scan_prompt_8k", op="scan", batch=1, n=8001, key_heads=16, heads=32, dim=128, ragged=False),
        # one user's token with that user's adapter
        dict(name="lora_token", op="lora", rows=1, requests=1, adapters=4, rank=16, type="bf16", weight="q4k", inner=INNER, width=HIDDEN),
        # the next token of 24 conversations that chose among 9 adapters or none
        dict(name="lora_serve_24", op="lora", rows=24, requests=24, adapters=9, rank=32, type="f16", weight="q4k", inner=INNER, width=HIDDEN),
        # three prompts of one batch, an adapter each
        dict(name="lora_prompts_4001", op="lora", rows=4001, requests=3, adapters=6, rank=64, type="bf16", weight="q4k", inner=INNER, width=HIDDEN),
        # one token's residual and norm in front of the experts
        dict(name="norm_token", op="norm", rows=1, width=HIDDEN, residual=True, gate=False, f32=True, q8=False),
        # the same for a long prompt, also in 8 bits for the projections that follow
        dict(name="norm_prompt_q8_8k", op="norm", rows=8001, width=HIDDEN, residual=True, gate=False, f32=True, q8=True),
        # the norm per value head behind the scan, with its output gate: 1021 tokens of 32 heads
        dict(name="norm_heads_gated", op="norm", rows=1021 * 32, width=128, residual=False, gate=True, f32=True, q8=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["conv", "scan", "scan", "lora", "norm"])
    if op == "conv":
        batch = _log(rng, 1, 24)
        n = 1 if rng.random() < 0.25 else _log(rng, 2, 8001 // batch)
        return dict(op=op, batch=batch, n=n, channels=rng.choice([8192, 8192, _log(rng, 64, 8192)]), taps=rng.choice([4, 4, 3, 2]),
                    bias=rng.random() < 0.3, ragged=batch > 1 and n > 1 and rng.random() < 0.5)
    if op == "scan":
        batch = _log(rng, 1, 16)
        key_heads, heads = rng.choice([(16, 32), (16, 32), (4, 4), (2, 6), (8, 16)])
        n = _log(rng, 1, 8001 // batch)
        return dict(op=op, batch=batch, n=n, key_heads=key_heads, heads=heads, dim=rng.choice([128, 128, 128, 64, 256 if heads < 32 else 128]),
                    ragged=batch > 1 and n > 1 and rng.random() < 0.5)
    if op == "lora":
        rows = _log(rng, 1, 4001)
        return dict(op=op, rows=rows, requests=_log(rng, 1, min(rows, 32)), adapters=_log(rng, 1, 40), rank=_log(rng, 1, 64),
                    type=rng.choice(["f16", "bf16", "f32"]), weight=rng.choice(["q4k", "q4k", "q6k", "q8_0"]) if rows < 600 else "q4k",
                    inner=rng.choice([4096, 4096, 8192]) if rows < 1500 else INNER, width=rng.choice([HIDDEN, _log(rng, 64, HIDDEN)]))
    rows, width = _log(rng, 1, 8001), rng.choice([HIDDEN, 128, _log(rng, 32, 8192)])
    while rows * width > 8001 * HIDDEN:
        rows //= 2
    gate = rng.random() < 0.3
    f32 = rng.random() < 0.7
    return dict(op=op, rows=rows, width=width, residual=not gate and rng.random() < 0.8, gate=gate, f32=f32, q8=not f32 or rng.random() < 0.4)


# ---- inputs

class _Draws:
    """Seeded draws on the GPU."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(seed * 1000003 + 17)

    def normal(self, *shape):
        return torch.randn(shape, generator=self.g, device="cuda")

    def uniform(self, *shape):
        return torch.rand(shape, generator=self.g, device="cuda")

    def below(self, most, *shape):
        return torch.randint(0, most, shape, generator=self.g, device="cuda")


def _silu(x):
    return x / (1 + torch.exp(-x))


def _lengths(d, c):
    """The valid tokens of each sequence of a padded batch: the longest fills it, a short one may be empty."""
    if not c["ragged"]:
        return None
    lens = (d.uniform(c["batch"]) * (c["n"] + 1)).to(torch.int32).clamp_(max=c["n"])
    lens[0] = c["n"]
    if c["batch"] > 2:
        lens[1] = 0
    return lens


def _weight_blocks(d, weight, rows, inner):
    """GGUF blocks of a trained matrix's magnitude: random codes, finite f16 scales."""
    elems, size = W_BLOCK[weight]
    blocks = d.below(256, rows * inner // elems, size).to(torch.uint8)
    scale = ((d.uniform(blocks.shape[0], 1) + 0.1) * {"q8_0": 4e-4, "q4k": 1e-4, "q6k": 1e-5}[weight]).half()
    if weight == "q6k":
        blocks[:, 208:210] = scale.view(torch.uint8)
    else:
        blocks[:, 0:2] = scale.view(torch.uint8)
    if weight == "q4k":
        blocks[:, 2:4] = (scale.float() * 7).half().view(torch.uint8)
    return blocks.reshape(-1)


def prepare(case, seed):
    c, d = case, _Draws(seed)
    if c["op"] == "conv":
        b, n, ch = c["batch"], c["n"], c["channels"]
        return dict(c, x=d.normal(b, n, ch), state=d.normal(b, ch, c["taps"] - 1), w=0.5 * d.normal(ch, c["taps"]),
                    b=0.1 * d.normal(ch) if c["bias"] else None, lens=_lengths(d, c), out=torch.zeros(b, n, ch, device="cuda"))
    if c["op"] == "scan":
        b, n, hk, h, dim = c["batch"], c["n"], c["key_heads"], c["heads"], c["dim"]
        # the convolution's output: q, k and v beside each other in a token's row
        x = _silu(d.normal(b, n, (2 * hk + h) * dim))
        q, k, v = x.split([hk * dim, hk * dim, h * dim], -1)
        # heads that forget within a few tokens and heads that hardly forget
        rate = torch.exp(d.uniform(h) * math.log(2000.0)) * 0.002
        gate = -rate * torch.log1p(torch.exp(d.normal(b, n, h)))
        return dict(c, q=q.view(b, n, hk, dim), k=k.view(b, n, hk, dim), v=v.view(b, n, h, dim), gate=gate, beta=d.normal(b, n, h),
                    state=0.3 * d.normal(b, h, dim, dim), offset=d.normal(b, h), lens=_lengths(d, c), scale=dim ** -0.5,
                    out=torch.zeros(b, n, h, dim, device="cuda"))
    if c["op"] == "lora":
        rows, r, t = c["rows"], c["rank"], TYPES[c["type"]]
        a = (d.normal(c["adapters"], r, c["inner"]) * c["inner"] ** -0.5).to(t)
        b = (d.normal(c["adapters"], c["width"], r) * r ** -0.5).to(t)
        # a request's rows stand together; a tenth of the requests have no adapter
        choice = d.below(c["adapters"], c["requests"])
        choice = torch.where(d.uniform(c["requests"]) < 0.1, -1, choice)
        request = torch.sort(torch.cat([torch.arange(c["requests"], device="cuda"), d.below(c["requests"], rows - c["requests"])]))[0]
        return dict(c, x=d.normal(rows, c["inner"]), gate=d.normal(rows, c["inner"]), w=_weight_blocks(d, c["weight"], c["width"], c["inner"]),
                    a=a, b=b, factor=0.5 + 1.5 * d.uniform(c["adapters"]), ids=choice[request].to(torch.int32))
    rows, width = c["rows"], c["width"]
    return dict(c, x=d.normal(rows, width) * torch.exp(d.normal(rows, 1)), residual=3 * d.normal(rows, width) if c["residual"] else None,
                gate=d.normal(rows, width) if c["gate"] else None, alpha=1 + 0.2 * d.normal(width))


# ---- the framework's calls

def _run_own(s):
    import paramecia_amd as pk
    if s["op"] == "conv":
        return pk.causal_conv(s["x"], s["w"], s["state"], bias=s["b"], lens=s["lens"], out=s["out"]), s["state"]
    if s["op"] == "scan":
        out = pk.gated_delta_rule(s["q"], s["k"], s["v"], s["gate"], s["beta"], s["state"], s["scale"], EPS,
                                  gate_offset=s["offset"], lens=s["lens"], out=s["out"])
        return out, s["state"], s["offset"]
    if s["op"] == "lora":
        return pk.gated_o_proj_lora(s["x"], s["gate"], s["w"], s["width"], s["a"], s["b"], s["factor"], s["ids"], w_type=W_TYPE[s["weight"]])
    y, q8 = pk.rms_norm(s["x"], s["alpha"], EPS, residual=s["residual"], gate=s["gate"], f32_out=s["f32"], q8_0_out=s["q8"])
    return _norm_outputs(s, y, None if q8 is None else (q8[..., 2:].view(torch.int8), q8[..., :2].view(torch.float16)))


def _norm_outputs(s, y, q8):
    """The norm's results: the residual stream, the f32 rows, and what the 8-bit rows stand for."""
    got = {} if s["residual"] is None else {"residual": s["residual"]}
    if y is not None:
        got["y"] = y
    if q8 is not None:
        got["q8"] = (q8[0] * q8[1]).flatten(1)[:, :s["width"]]
    return got


# ---- the plain forms

def _conv_plain(s):
    x, k, n = s["x"], s["taps"], s["n"]
    full = torch.cat([s["state"].transpose(1, 2), x], 1)
    y = sum(full[:, j:j + n] * s["w"][:, j] for j in range(k))
    if s["b"] is not None:
        y = y + s["b"]
    y = _silu(y)
    if s["lens"] is None:
        s["out"].copy_(y)
        s["state"].copy_(full[:, n:].transpose(1, 2))
    else:
        at = s["lens"].long()[:, None] + torch.arange(k - 1, device="cuda")
        s["out"].copy_(torch.where((torch.arange(n, device="cuda") < s["lens"][:, None])[..., None], y, s["out"]))
        s["state"].copy_(torch.gather(full, 1, at[..., None].expand(-1, -1, s["channels"])).transpose(1, 2))
    return s["out"], s["state"]


CHUNK = 64


def _unit_lower_inverse(a):
    """(I + a)^-1 of strictly lower triangular a [.., CHUNK, CHUNK], from blocks twice as large each time."""
    x = torch.eye(CHUNK, device=a.device).expand(a.shape).contiguous()
    size = 1
    while size < CHUNK:
        m = CHUNK // (2 * size)
        ab, xb = (t.unflatten(-2, (m, 2, size)).unflatten(-1, (m, 2, size)) for t in (a, x))
        i = torch.arange(m, device=a.device)
        low = ab[..., i, 1, :, i, 0, :]  # [m, .., size, size]
        first, second = xb[..., i, 0, :, i, 0, :], xb[..., i, 1, :, i, 1, :]
        xb[..., i, 1, :, i, 0, :] = -((second.contiguous() @ low.contiguous()) @ first.contiguous())
        x = xb.reshape(a.shape)
        size *= 2
    return x


def _scan_plain(s):
    b, n, h, dim = s["v"].shape
    rep = h // s["key_heads"]
    chunks = -(-n // CHUNK)
    live = torch.ones(b, n, dtype=torch.bool, device="cuda") if s["lens"] is None else torch.arange(n, device="cuda") < s["lens"][:, None]

    def chunked(x):  # [b, n, h, ..] -> [chunks, b, h, CHUNK, ..], zero behind each sequence's end
        x = torch.where(live.reshape(b, n, *[1] * (x.dim() - 2)), x, 0.0)
        x = torch.cat([x, x.new_zeros(b, chunks * CHUNK - n, *x.shape[2:])], 1).unflatten(1, (chunks, CHUNK))
        return x.transpose(2, 3).transpose(0, 1).contiguous()

    q, k, v = s["q"], s["k"], s["v"]
    q = q * (s["scale"] / torch.sqrt((q * q).sum(-1, keepdim=True) + EPS))
    k = k / torch.sqrt((k * k).sum(-1, keepdim=True) + EPS)
    q, k = (chunked(x.repeat_interleave(rep, 2)) for x in (q, k))
    v, beta = chunked(v), chunked(1 / (1 + torch.exp(-s["beta"])))[..., None]
    total = torch.cumsum(chunked(s["gate"]).double(), -1)  # in 64 bits: differences of long sums
    decay = torch.exp(torch.tril(total[..., :, None] - total[..., None, :]).float())
    kt = k.transpose(-1, -2).contiguous()
    inverse = _unit_lower_inverse(torch.tril(beta * (k @ kt) * decay, -1))
    p = torch.tril((q @ kt) * decay)
    grown = torch.exp(total.float())[..., None]
    u0, w = inverse @ (beta * v), inverse @ (beta * grown * k)
    q = q * grown
    last = total[..., -1:]
    kt = kt * torch.exp((last - total).float())[..., None, :]
    last = torch.exp(last.float())[..., None]
    state, outs = s["state"].transpose(-1, -2).contiguous(), []
    for i in range(chunks):  # the recurrence itself
        u = u0[i] - w[i] @ state
        outs.append(q[i] @ state + p[i] @ u)
        state = last[i] * state + kt[i] @ u
    o = torch.stack(outs, 1).transpose(2, 3).flatten(1, 2)[:, :n]
    s["out"].copy_(torch.where(live[..., None, None], o, s["out"]))
    s["state"].copy_(state.transpose(-1, -2))
    s["offset"].copy_((s["offset"].double() + torch.where(live[..., None], s["gate"], 0.0).double().sum(1)).float())
    return s["out"], s["state"], s["offset"]


def _weight_plain(weight, blocks, rows, inner):
    """The f32 matrix that GGUF blocks stand for."""
    elems, size = W_BLOCK[weight]
    b = blocks.view(-1, size)
    half = lambda at: b[:, at:at + 2].contiguous().view(torch.float16).float()  # noqa: E731
    if weight == "q8_0":
        w = half(0) * b[:, 2:].view(torch.int8).float()
    elif weight == "q4k":
        s = b[:, 4:16].int()
        scale = torch.cat([s[:, 0:4] & 63, (s[:, 8:12] & 15) | ((s[:, 0:4] >> 6) << 4)], 1).float()
        least = torch.cat([s[:, 4:8] & 63, (s[:, 8:12] >> 4) | ((s[:, 4:8] >> 6) << 4)], 1).float()
        codes = b[:, 16:].view(-1, 4, 1, 32)
        codes = torch.cat([codes & 15, codes >> 4], 2).view(-1, 8, 32).float()
        w = (half(0) * scale)[..., None] * codes - (half(2) * least)[..., None]
    else:
        low, high = b[:, :128].view(-1, 2, 1, 2, 32), b[:, 128:192].view(-1, 2, 1, 32)
        low = torch.cat([low & 15, low >> 4], 2)  # [.., half, nibble, group, 32]
        high = torch.cat([high & 3, (high >> 2) & 3, (high >> 4) & 3, high >> 6], 2).view(-1, 2, 2, 2, 32)
        codes = (low | (high << 4)).float() - 32
        w = (half(208) * b[:, 192:208].contiguous().view(torch.int8).float())[..., None] * codes.view(-1, 16, 16)
    return w.reshape(rows, inner)


def _lora_plain(s):
    x = s["x"] / (1 + torch.exp(-s["gate"]))
    y = x @ _weight_plain(s["weight"], s["w"], s["width"], s["inner"]).T
    a, b, n, r = s["a"].float(), s["b"].float(), s["adapters"], s["rank"]
    # every adapter's small product for every row, then the row's own one
    t = (x @ a.reshape(n * r, -1).T).view(-1, n, r)
    mine = s["ids"][:, None] == torch.arange(n, device="cuda")
    t = t * (mine * s["factor"])[..., None]
    return y + t.reshape(-1, n * r) @ b.transpose(1, 2).reshape(n * r, -1)


def _norm_plain(s):
    h = s["x"]
    if s["residual"] is not None:
        h = s["residual"].add_(h)
    wide = torch.float64 if s["q8"] else torch.float32  # values next to a code's border: 64 bits up to the rounded row
    y = h.to(wide)
    y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + EPS) * s["alpha"]
    if s["gate"] is not None:
        y = y * _silu(s["gate"].to(wide))
    y = y.float()
    q8 = None
    if s["q8"]:
        z = torch.cat([y, y.new_zeros(y.shape[0], -s["width"] % 32)], 1).unflatten(1, (-1, 32))
        step = z.abs().amax(-1, keepdim=True) / 127
        z = z * torch.where(step > 0, 1 / step, 0.0)
        codes = torch.sign(z) * torch.floor(z.abs().double() + 0.5).float()  # halves go away from zero
        q8 = codes.to(torch.int8), step.half()
    return _norm_outputs(s, y if s["f32"] else None, q8)


def run(state):
    if own:
        return _run_own(state)
    return {"conv": _conv_plain, "scan": _scan_plain, "lora": _lora_plain, "norm": _norm_plain}[state["op"]](state)


def work(case):
    c = case
    if c["op"] == "conv":
        m = c["batch"] * c["n"] * c["channels"]
        kept = c["batch"] * c["channels"] * (c["taps"] - 1)
        return {"bytes": 4 * (2 * m + 2 * kept + c["channels"] * c["taps"]), "flops": (2 * c["taps"] + 4) * m}
    if c["op"] == "scan":
        m, h, dim = c["batch"] * c["n"], c["heads"], c["dim"]
        if c["ragged"]:
            m //= 2  # half of a padded batch is padding
        return {"bytes": 4 * (m * (2 * c["key_heads"] * dim + 2 * h * dim + 2 * h) + 2 * c["batch"] * h * dim * dim), "flops": 6 * m * h * dim * dim}
    if c["op"] == "lora":
        elems, size = W_BLOCK[c["weight"]]
        used = min(c["adapters"], c["requests"])
        wide = c["inner"] + c["width"]
        return {"bytes": c["width"] * c["inner"] // elems * size + used * c["rank"] * wide * TYPES[c["type"]].itemsize + 4 * c["rows"] * (2 * c["inner"] + c["width"]),
                "flops": 2 * c["rows"] * (c["inner"] * c["width"] + c["rank"] * wide)}
    m = c["rows"] * c["width"]
    return {"bytes": m * (4 + 8 * c["residual"] + 4 * c["gate"] + 4 * c["f32"] + 34 / 32 * c["q8"]), "flops": m * (6 + 5 * c["gate"] + 4 * c["q8"])}


# ---- the definitions in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"conv": _conv_exact, "scan": _scan_exact, "lora": _lora_exact, "norm": _norm_exact}[case["op"]](s)


def _ends(s):
    return [s["n"]] * s["batch"] if s["lens"] is None else s["lens"].tolist()


def _conv_exact(s):
    out, state = s["out"].double(), s["state"].double()
    for i, end in enumerate(_ends(s)):
        rows = torch.cat([state[i].T, s["x"][i, :end].double()])  # [taps - 1 + end, channels]
        y = (rows.unfold(0, s["taps"], 1) * s["w"].double()).sum(-1) if end else rows[:0]
        y = y if s["b"] is None else y + s["b"].double()
        out[i, :end] = y * torch.sigmoid(y)
        state[i] = rows[len(rows) - (s["taps"] - 1):].T
    return out, state


def _scan_exact(s):
    rep = s["heads"] // s["key_heads"]
    out, state, offset = s["out"].double(), s["state"].double(), s["offset"].double()
    ends = torch.tensor(_ends(s), device="cuda")
    alpha, beta = torch.exp(s["gate"].double()), torch.sigmoid(s["beta"].double())
    for t in range(s["n"]):
        q, k, v = s["q"][:, t].double(), s["k"][:, t].double(), s["v"][:, t].double()
        q = (q * s["scale"] * torch.rsqrt(q.pow(2).sum(-1, keepdim=True) + EPS)).repeat_interleave(rep, 1)
        k = (k * torch.rsqrt(k.pow(2).sum(-1, keepdim=True) + EPS)).repeat_interleave(rep, 1)
        s1 = state * alpha[:, t, :, None, None]
        u = beta[:, t, :, None] * (v - (s1 * k[:, :, None]).sum(-1))
        s1 = s1 + u[..., None] * k[:, :, None]
        o = (s1 * q[:, :, None]).sum(-1)
        if s["lens"] is None:
            state, out[:, t] = s1, o
        else:
            on = (t < ends)[:, None, None]
            state, out[:, t] = torch.where(on[..., None], s1, state), torch.where(on, o, out[:, t])
    for i, end in enumerate(ends.tolist()):
        offset[i] += s["gate"][i, :end].double().sum(0)
    return out, state, offset


def _weight_exact(weight, blocks, count):
    """Element by element, from the block's layout: GGUF's own numbering of codes and scales."""
    elems, size = W_BLOCK[weight]
    b = blocks.view(-1, size).long()
    e = torch.arange(elems, device=b.device)
    f16 = lambda at: (b[:, at] + 256 * b[:, at + 1]).to(torch.int16).view(torch.float16).double()[:, None]  # noqa: E731
    signed = lambda x: torch.where(x > 127, x - 256, x)  # noqa: E731
    if weight == "q8_0":
        w = f16(0) * signed(b[:, 2 + e])
    elif weight == "q4k":
        sub = e // 32
        code = (b[:, 16 + 32 * (e // 64) + e % 32] >> (4 * (sub % 2))) % 16
        near, far = b[:, 4 + sub % 4], b[:, 8 + sub % 4]
        extra = b[:, 12 + sub % 4]
        scale = torch.where(sub < 4, near % 64, extra % 16 + 16 * (near // 64))
        least = torch.where(sub < 4, far % 64, extra // 16 + 16 * (far // 64))
        w = f16(0) * scale * code - f16(2) * least
    else:
        part, r = e // 128, e % 128
        low = (b[:, 64 * part + r % 64] >> (4 * (r // 64))) % 16
        high = (b[:, 128 + 32 * part + r % 32] >> (2 * (r // 32))) % 4
        w = f16(208) * signed(b[:, 192 + e // 16]) * (low + 16 * high - 32)
    return w.reshape(count, -1)


def _lora_exact(s):
    x = s["x"].double() * torch.sigmoid(s["gate"].double())
    y = x @ _weight_exact(s["weight"], s["w"], s["width"]).T
    for a in range(s["adapters"]):
        at = (s["ids"] == a).nonzero()[:, 0]
        if len(at):
            y[at] += s["factor"][a].double() * ((x[at] @ s["a"][a].double().T) @ s["b"][a].double().T)
    return y


def _norm_exact(s):
    h = s["x"].double()
    got = {}
    if s["residual"] is not None:
        h = s["residual"].double() + h
        got["residual"] = h
    y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS) * s["alpha"].double()
    if s["gate"] is not None:
        y = y * s["gate"].double() * torch.sigmoid(s["gate"].double())
    if s["f32"]:
        got["y"] = y
    if s["q8"]:
        blocks = torch.nn.functional.pad(y, (0, -s["width"] % 32)).unflatten(1, (-1, 32))
        step = blocks.abs().max(-1, keepdim=True)[0] / 127
        code = torch.where(step > 0, blocks / step, 0.0)
        code = torch.trunc(code + 0.5 * torch.sign(code))
        got["q8"] = (code * step.half().double()).flatten(1)[:, :s["width"]]
    return got
