"""Refusals at the edges of what the operators take (the library's own checks, no GPU)."""
import numpy as np
import pytest

from test_cpu_operators import answer, raw_segments
from tts_amd import Adapter


@pytest.mark.parametrize("which,count", [("lora_grad", "adapters"), ("norm_grad", "gains")])
def test_more_gradients_than_a_call_can_have_tokens_are_refused(which, count):
    """Every adapter or gain of a backward call has sums of its own to be written; their numbers stay 32 bits wide."""
    seg = raw_segments([0, 10], [0])
    assert answer(which, seg, **{count: (1 << 24) - 1})[0] >= 0
    for n in (1 << 24, (1 << 31) - 129, (1 << 31) - 1):
        rc, msg = answer(which, seg, **{count: n})
        assert rc == -22 and f"{count} must be" in msg, (n, rc, msg)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("where", ["a", "b", "gain", "offset"])
def test_adapters_that_are_not_numbers_are_refused(where, bad):
    """One such value reaches every duration of its sentence, and a batch with a sentence of no frames fails as a whole."""
    a, b, gain, offset = np.ones((2, 768)), np.ones((768, 2)), np.ones(768), np.ones(768)
    assert Adapter({"key": (a, b)}, 1.0, {"full_norm": (gain, offset)}).rank == 2
    {"a": a, "b": b, "gain": gain, "offset": offset}[where].flat[-1] = bad
    with pytest.raises(ValueError, match="finite"):
        Adapter({"key": (a, b)}, 1.0, {"full_norm": (gain, offset)})
