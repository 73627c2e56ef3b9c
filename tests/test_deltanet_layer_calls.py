"""Calls of the operators around a Gated-DeltaNet layer's state update that are refused for the right
reason (no GPU: addresses stand for device memory that nothing touches)."""
import pytest

pytest.importorskip("torch")

from paramecia_amd._lib import ERR_ARG  # noqa: E402
from test_deltanet_layer_refusals import G, err, lora  # noqa: E402


def test_lora_rows_past_a_call():
    """More rows than a call takes have no workspace (its size is 0): what is refused is their number."""
    for b in (65536, 1 << 20):
        assert lora(b=b, ws=None) == ERR_ARG and "65535" in err()
        assert lora(b=b, ws=G, wb=0) == ERR_ARG and "65535" in err()
    assert lora(b=65535, ws=None) == ERR_ARG and "null" in err()
