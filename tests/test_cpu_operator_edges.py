"""Refusals at the edges of what the operators take (the library's own checks, no GPU)."""
import ctypes as C

import numpy as np
import pytest
import torch

from test_cpu_operators import answer, lora, raw_segments
from tts_amd import Adapter, Operators, _lib


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


def test_a_closed_handle_is_named_as_the_reason():
    """Not the text of whatever failed before it."""
    lib = _lib.load()
    assert answer("lora", act=7)[0] == -22 and b"act" in lib.k82_last_error(None)
    assert lib.k82_op_lora(None, lora(), raw_segments([0, 10], [0]), None) == -22
    assert b"handle" in lib.k82_last_error(None)
    ops = object.__new__(Operators)
    ops.device, ops.h, ops.lib, ops._stream = -1, C.c_void_p(), lib, lambda: 1
    x, gain = torch.zeros(4, 8), torch.ones(1, 8)
    with pytest.raises(ValueError, match="handle"):
        ops.op_layernorm(x, gain, gain)
