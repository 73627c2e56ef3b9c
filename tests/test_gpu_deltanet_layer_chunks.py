"""A Gated-DeltaNet layer over a padded batch whose state update goes by chunks, from the
convolution to the next layer's input, against the same formulas in 64 bits (LinearAttention,
paramecia-model/src/qwen3_next.rs:2900-4208)."""
import pytest

torch = pytest.importorskip("torch")

from test_gpu_deltanet_layer import EPS, conv64, layer, layer_inputs, lora64, pk, rel, say, scan64  # noqa: E402, F401

pytestmark = pytest.mark.gpu


def test_layer_by_chunks(pk, orc):  # noqa: F811
    say("layer by chunks")
    b, n = 2, 150
    lens = [150, 77]
    assert pk.lib().pkv_deltanet_prompt_workspace(b, n, 16, 32, 128) > 0
    x, z, p = layer_inputs(pk, b, n, 61)
    ids = torch.tensor([[1], [-1]], dtype=torch.int32, device="cuda").expand(b, n).contiguous()
    stream0 = p["stream"].clone()
    dl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    lin = pk.LinearAttentionState()
    y, _ = layer(pk, lin, x, z, p, ids, lens=dl)

    wdq = torch.from_numpy(orc.dequantize_weight(p["wo"].cpu().numpy(), 12, 2048 * 4096).reshape(2048, 4096)).cuda().double()
    zeros = lambda *s: torch.zeros(s, device="cuda")  # noqa: E731
    c, conv_state, _ = conv64(x, p["conv"], zeros(b, 8192, 3).double(), None, lens, True, zeros(b, n, 8192))
    q, k, v = c.split([2048, 2048, 4096], -1)
    o, state, _ = scan64(q.unflatten(-1, (16, 128)), k.unflatten(-1, (16, 128)), v.unflatten(-1, (32, 128)), p["gate"],
                         p["beta"], zeros(b, 32, 128, 128).double(), 128 ** -0.5, lens, zeros(b, n, 32, 128), zeros(b, 32))
    want = o / (o.square().mean(-1, keepdim=True) + EPS).sqrt() * p["head_alpha"].double()
    want = (want * z.double() * torch.sigmoid(z.double())).flatten(2).flatten(0, 1)
    m, _ = lora64(want, None, wdq, p["a"], p["b"], p["scale"], ids.flatten().tolist(), 3)
    h = stream0.double() + m.view(b, n, 2048)
    want = h / (h.square().mean(-1, keepdim=True) + EPS).sqrt() * p["alpha"].double()
    # each stage passes the error in front of it on and adds its own; the norm per head can raise
    # a small head's: ten times the largest of the stages' limits
    lim = 10 * 2e-6
    for i, e in enumerate(lens):
        say(f"  y {rel(y[i, :e], want[i, :e]):.2e} state {rel(lin.recurrent_state.ssm_state[i], state[i]):.2e}")
        assert rel(y[i, :e], want[i, :e]) < lim and rel(p["stream"][i, :e], h[i, :e]) < lim
        assert rel(lin.recurrent_state.ssm_state[i], state[i]) < lim
    assert rel(lin.recurrent_state.conv_state, conv_state) < lim
