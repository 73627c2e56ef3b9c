"""The projection with adapters (forward_with_scales_and_lora, paramecia-model/src/models/
with_tracing.rs:253-300) over rows of very small and very large inputs, each row held by itself."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from test_gpu_deltanet_layer import gen, lora64, pk, say  # noqa: E402, F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("w_type,rows", [(12, 3), (12, 24), (14, 300), (8, 24), (8, 300)])
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_magnitudes(pk, orc, w_type, rows, dtype):  # noqa: F811
    """Rows scaled by powers of two from 2^-113 to 2^100, adapters scaled by 2^-9: the sums' errors scale
    with the row (as in the projection's own tests, 2e-6 of the row's norm)."""
    from kquant_blocks import random_weight_bytes
    say(f"adapter magnitudes w={w_type} rows={rows} {dtype}")
    r = gen(rows)
    inner, width, rank, n = 4096, 300, 16, 3
    wb = random_weight_bytes(np.random.default_rng(rows), w_type, width, inner, d_scale=1e-8)
    wdq = torch.from_numpy(orc.dequantize_weight(wb, w_type, width * inner).reshape(width, inner)).cuda().double()
    t = getattr(torch, dtype)
    x = r(rows, inner) * torch.exp2(torch.tensor([-113.0, -60.0, 0.0, 100.0], device="cuda")[torch.arange(rows) % 4])[:, None]
    a, b = (r(n, rank, inner) * inner ** -0.5).to(t), (16 * r(n, width, rank)).to(t)
    scale = 2.0 ** -9 * (1 + r(n).abs())
    ids = torch.arange(rows, dtype=torch.int32, device="cuda") % n
    ref, base = lora64(x, None, wdq, a, b, scale, ids.tolist(), n)
    got = pk.gated_o_proj_lora(x, None, torch.from_numpy(wb).cuda(), width, a, b, scale, ids, w_type=w_type)
    assert torch.isfinite(got).all()
    err = (got.double() - ref).norm(dim=1) / ref.norm(dim=1)
    low = (ref - base).norm(dim=1) / ref.norm(dim=1)
    say(f"  rel {float(err.max()):.2e}, adapters make {float(low.min()):.2f} of a row")
    assert float(err.max()) < 2e-6
