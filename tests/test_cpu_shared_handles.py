"""One handle and several threads: what the Python faces of the library promise to threads that share an engine.  No GPU: the
library is a stub, or is never reached."""
import threading

import numpy as np
import pytest

from tts_amd import Adapter, Engine


class WatchedLock:
    """An RLock that says when a thread other than its maker asks for it."""

    def __init__(self):
        self.lock, self.maker, self.asked = threading.RLock(), threading.get_ident(), threading.Event()

    def __enter__(self):
        if threading.get_ident() != self.maker:
            self.asked.set()
        self.lock.acquire()
        return self

    def __exit__(self, *exc):
        self.lock.release()


class Library:
    """k82_set_adapters and k82_fork by what they leave: a table of scales, which a fork inherits as it is at its call."""

    def __init__(self):
        self.table, self.forked = [], []

    def k82_set_adapters(self, h, table, n):
        self.table = [table[i].scale for i in range(n)]
        return 0

    def k82_fork(self, h, out):
        self.forked.append(list(self.table))
        return 0

    def k82_destroy(self, h):
        return 0


def stub_engine():
    import ctypes as C
    e = object.__new__(Engine)
    e.lib, e.h, e._lock, e._forks, e._parent = Library(), C.c_void_p(), WatchedLock(), [], None
    e.config, e.device, e.precision, e._pending = {}, 0, "fp32", None
    return e


@pytest.mark.parametrize("then", [{"y": 2.0, "x": 1.0}, {"y": 2.0}, {}, {"z": 3.0, "y": 2.0, "x": 1.0}])
def test_a_fork_takes_names_and_table_of_one_moment(then):
    """Another thread replaces the set while fork() waits for the engine: the fork's names mean the table that it inherits."""
    scales = {"x": 1.0, "y": 2.0}
    e = stub_engine()
    e.set_adapters({n: Adapter(scale=s) for n, s in scales.items()})
    made = []
    t = threading.Thread(target=lambda: made.append(e.fork()))
    with e._lock:
        t.start()
        assert e._lock.asked.wait(60)
        e.set_adapters({n: Adapter(scale=s) for n, s in then.items()})
    t.join(60)
    (child,), (table,) = made, e.lib.forked
    assert table == list(then.values())
    assert {n: table[i] for n, i in child._adapters.items()} == then
    for n in scales:
        if n in then:
            assert table[child._adapter_indices([n], 1)[0]] == scales[n]
        else:
            with pytest.raises(KeyError, match="not found"):
                child._adapter_indices([n], 1)
    assert np.array_equal(child._adapter_indices([None], 1), [-1])


@pytest.mark.parametrize("call", ["op_lora", "op_lora_grad", "op_layernorm", "op_layernorm_grad"])
def test_a_first_call_beside_a_first_call(call):
    """Whatever of a fresh handle the first call has set up so far, another thread's call goes through to the library (which
    refuses it here: there is no handle behind this face)."""
    import ctypes as C

    import torch

    from tts_amd import Operators, _lib
    x, norm, one = torch.zeros(4, 8), torch.ones(1, 8), torch.ones(4)
    a, b, scale, h, dy = torch.zeros(1, 2, 8), torch.zeros(1, 6, 2), torch.ones(1), torch.zeros(4, 2), torch.zeros(4, 6)
    args = {"op_lora": (x, a, b, scale), "op_lora_grad": (x, dy, h, a, b, scale), "op_layernorm": (x, norm, norm),
            "op_layernorm_grad": (x, x, norm, one, one)}[call]
    said = []

    def other(face):
        try:
            getattr(face, call)(*args)
        except Exception as e:
            said.append(repr(e))

    class Face(Operators):
        watched = threading.get_ident()

        def _stream(self):                                       # (torch has none to name without a GPU)
            return 1

        def __setattr__(self, name, value):
            super().__setattr__(name, value)
            if threading.get_ident() == self.watched and name not in ("device", "h", "lib"):
                t = threading.Thread(target=other, args=(self,))
                t.start()
                t.join(60)

    face = Face.__new__(Face)
    face.device, face.h, face.lib = -1, C.c_void_p(), _lib.load()
    other(face)
    assert len(said) > 1 and all("k82 error -22" in s for s in said), said
