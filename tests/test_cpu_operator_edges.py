"""Refusals at the edges of what the operators take (the library's own checks, no GPU)."""
import pytest

from test_cpu_operators import answer, raw_segments


@pytest.mark.parametrize("which,count", [("lora_grad", "adapters"), ("norm_grad", "gains")])
def test_more_gradients_than_a_call_can_have_tokens_are_refused(which, count):
    """Every adapter or gain of a backward call has sums of its own to be written; their numbers stay 32 bits wide."""
    seg = raw_segments([0, 10], [0])
    assert answer(which, seg, **{count: (1 << 24) - 1})[0] >= 0
    for n in (1 << 24, (1 << 31) - 129, (1 << 31) - 1):
        rc, msg = answer(which, seg, **{count: n})
        assert rc == -22 and f"{count} must be" in msg, (n, rc, msg)
