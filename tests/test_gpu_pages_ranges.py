"""The attention over pages at the ends of its ranges: values whose sums leave f32 though their means
do not. Against the plain forms of pages_checks.py in 64 bits."""
import pytest

torch = pytest.importorskip("torch")

from pages_checks import E, attend64  # noqa: E402
from test_gpu_pages import Case, gen, i32, pk, say  # noqa: E402, F401

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
