"""Refusals of the operators on caller-owned tensors (include/k82.h): the library's own checks need no GPU, and the Python
face refuses before it reaches the library."""
import ctypes as C

import numpy as np
import pytest
import torch

from tts_amd import Operators, Segments, _lib

P = 1 << 20                      # pointers that nothing reads


def lora(**kw):
    d = dict(dtype=0, layout=0, act=0, cin=16, cout=24, rank=4, adapters=2, tokens=10, x=P, ldx=16, base=None, ldbase=0,
             y=2 * P, ldy=24, a=3 * P, b=4 * P, scale=5 * P, h=None)
    return _lib.K82Lora(**{**d, **kw})


def lora_grad(**kw):
    d = dict(dtype=0, cin=16, cout=24, rank=4, adapters=2, tokens=10, x=P, ldx=16, dy=2 * P, lddy=24, h=3 * P, dx_base=None,
             lddx_base=0, dx=4 * P, lddx=16, a=5 * P, b=6 * P, scale=7 * P, da=8 * P, db=9 * P)
    return _lib.K82LoraGrad(**{**d, **kw})


def norm(**kw):
    d = dict(dtype=0, layout=0, c=16, gains=2, eps=1e-5, tokens=10, x=P, ldx=16, res=None, ldres=0, y=2 * P, ldy=16,
             gain=3 * P, offset=4 * P, mean=None, rstd=None)
    return _lib.K82Layernorm(**{**d, **kw})


def norm_grad(**kw):
    d = dict(dtype=0, c=16, gains=2, tokens=10, x=P, ldx=16, res=None, ldres=0, dy=2 * P, lddy=16, dx=3 * P, lddx=16,
             gain=4 * P, mean=5 * P, rstd=6 * P, dgain=7 * P, doffset=8 * P)
    return _lib.K82LayernormGrad(**{**d, **kw})


def raw_segments(off, index):
    """A k82_segments of unchecked values (the arrays stay alive through the returned object)."""
    o, i = np.array(off, np.int64), np.array(index, np.int32)
    s = _lib.K82Segments(off=o.ctypes.data, index=i.ctypes.data, n=i.size)
    s.keep = (o, i)
    return s


FUNCTIONS = {"lora": (lora, "k82_op_lora_check"), "lora_grad": (lora_grad, "k82_op_lora_grad_workspace"),
             "norm": (norm, "k82_op_layernorm_check"), "norm_grad": (norm_grad, "k82_op_layernorm_grad_workspace")}


def answer(which, seg=None, **kw):
    lib = _lib.load()
    make, name = FUNCTIONS[which]
    rc = getattr(lib, name)(make(**kw), seg if seg is not None else raw_segments([0, 4, 10], [0, 1]))
    return rc, lib.k82_last_error(None).decode() if rc < 0 else ""


@pytest.mark.parametrize("which", FUNCTIONS)
def test_ordinary_arguments_are_accepted(which):
    for kw in ({}, {"tokens": 0, "x": None}, {"dtype": 1}):
        seg = raw_segments([0], []) if kw.get("tokens") == 0 else None
        assert answer(which, seg, **kw)[0] >= 0, kw
    # empty segments, an index that comes twice, rows that no segment holds
    assert answer(which, raw_segments([2, 2, 5, 5, 9], [0, 1, 1, 0]))[0] >= 0


@pytest.mark.parametrize("which,kw,word", [
    ("lora", dict(dtype=2), "dtype"), ("lora", dict(layout=2), "layout"), ("lora", dict(layout=1, dtype=1), "K82_F32 only"),
    ("lora", dict(act=7), "act"), ("lora", dict(rank=0), "rank"), ("lora", dict(rank=129), "rank"),
    ("lora", dict(cin=0), "channel"), ("lora", dict(cout=-1), "channel"), ("lora", dict(tokens=-1), "tokens"),
    ("lora", dict(tokens=1 << 31), "tokens"), ("lora", dict(x=None), "x must not"), ("lora", dict(y=None), "y must not"),
    ("lora", dict(a=None), "a, b and scale"), ("lora", dict(scale=None), "a, b and scale"),
    ("lora", dict(adapters=-1), "adapters"), ("lora", dict(ldx=15), "ld of x"), ("lora", dict(ldy=0), "ld of y"),
    ("lora", dict(base=6 * P, ldbase=23), "ld of base"), ("lora", dict(x=P + 2), "aligned"),
    ("lora", dict(y=P), "overlap"), ("lora", dict(y=P + 8 * 4), "overlap"), ("lora", dict(base=2 * P + 4, ldbase=24), "overlap"),
    ("lora", dict(base=2 * P, ldbase=25, ldy=24), "overlap"), ("lora", dict(h=2 * P), "overlaps"),
    ("lora", dict(layout=1, ldx=9, ldy=10), "ld of x"), ("lora", dict(ldx=(1 << 25) + 1), "2^25"), ("lora", dict(a=3 * P + 1), "aligned"),
    ("lora", dict(h=9 * P + 2), "aligned"), ("lora_grad", dict(da=8 * P + 1), "aligned"), ("norm", dict(gain=3 * P + 2), "aligned"),
    ("norm_grad", dict(rstd=6 * P + 1), "aligned"), ("lora", dict(tokens=1 << 24), "tokens"),
    ("lora_grad", dict(dtype=3), "dtype"), ("lora_grad", dict(rank=200), "rank"), ("lora_grad", dict(h=None), "h must not"),
    ("lora_grad", dict(da=None), "da and db"), ("lora_grad", dict(dx=P), "overlaps"), ("lora_grad", dict(dx=2 * P), "overlaps"),
    ("lora_grad", dict(dx_base=4 * P + 4, lddx_base=16), "without being one"), ("lora_grad", dict(lddy=23), "ld of dy"),
    ("norm", dict(c=0), "channel"), ("norm", dict(gains=0), "gain"), ("norm", dict(gain=None), "gain"),
    ("norm", dict(eps=-1.0), "eps"), ("norm", dict(eps=float("nan")), "eps"), ("norm", dict(mean=6 * P), "come together"),
    ("norm", dict(layout=1, dtype=1), "K82_F32 only"), ("norm", dict(y=P + 4), "overlap"), ("norm", dict(ldx=15), "ld of x"),
    ("norm", dict(mean=2 * P, rstd=9 * P), "overlaps"),
    ("norm_grad", dict(mean=None), "mean and rstd"), ("norm_grad", dict(dgain=None), "dgain"),
    ("norm_grad", dict(dx=P + 4), "overlaps"), ("norm_grad", dict(dx=5 * P), "overlaps mean"), ("norm_grad", dict(dy=None), "dy must not"),
])
def test_bad_arguments_are_refused(which, kw, word):
    rc, msg = answer(which, **kw)
    assert rc == -22 and word in msg, (rc, msg)


@pytest.mark.parametrize("which", FUNCTIONS)
@pytest.mark.parametrize("off,index,word", [
    ([0, 5, 4], [0, 1], "decrease"), ([-1, 4, 10], [0, 1], "negative"), ([0, 4, 11], [0, 1], "10 tokens"),
    ([0, 4, 10], [0, 2], "index 2"), ([0, 4, 10], [-3, 1], "index -3"),
])
def test_bad_segments_are_refused(which, off, index, word):
    rc, msg = answer(which, raw_segments(off, index))
    assert rc == -22 and word in msg, (rc, msg)


def test_no_adapter_is_for_adapters_only():
    for which in ("lora", "lora_grad"):
        assert answer(which, raw_segments([0, 10], [-1]))[0] >= 0
        assert answer(which, raw_segments([0, 10], [-1]), adapters=0, a=None, b=None, scale=None)[0] >= 0
    for which in ("norm", "norm_grad"):
        assert answer(which, raw_segments([0, 10], [-1]))[0] == -22


def test_shared_buffers_that_do_not_overlap_are_accepted():
    # x and y are column ranges of one buffer; base is y; dx is dx_base; the norm works in place
    assert answer("lora", x=P, ldx=40, y=P + 16 * 4, ldy=40)[0] == 0
    assert answer("lora", x=P, ldx=40, y=P + 15 * 4, ldy=40)[0] == -22
    assert answer("lora", base=2 * P, ldbase=24)[0] == 0
    assert answer("lora", layout=1, x=P, ldx=32, y=P + 16 * 32 * 4, ldy=32)[0] == 0
    assert answer("lora_grad", dx_base=4 * P, lddx_base=16)[0] >= 0
    assert answer("norm", y=P, ldy=16)[0] == 0
    for d in (P, 2 * P):
        assert answer("norm_grad", dx=d)[0] >= 0


def test_null_arguments_are_refused():
    lib = _lib.load()
    seg = raw_segments([0, 10], [0])
    assert lib.k82_op_lora_check(None, seg) == -22 and lib.k82_op_layernorm_check(None, seg) == -22
    assert lib.k82_op_lora_grad_workspace(None, seg) == -22 and lib.k82_op_layernorm_grad_workspace(None, seg) == -22
    assert lib.k82_op_lora_check(lora(), None) == -22
    bad = _lib.K82Segments(off=None, index=None, n=2)
    assert lib.k82_op_lora_check(lora(), bad) == -22
    assert lib.k82_op_lora_check(lora(), _lib.K82Segments(off=None, index=None, n=-1)) == -22
    assert lib.k82_op_lora(None, lora(), seg, None) == -22        # no handle


def test_segments_class_refuses_what_is_not_a_cut():
    s = Segments.of_lengths([3, 0, 4], [1, 0, -1])
    assert s.offsets.tolist() == [0, 3, 3, 7] and (s.lo, s.hi) == (0, 7)
    for off, index in (([0, 2], [0, 1]), ([0, 3, 2], [0, 1]), ([-1, 3], [0]), ([[0, 1]], [0])):
        with pytest.raises(ValueError):
            Segments(off, index)
    for off, index, word in (([0.0, 2.5], [0], "whole numbers"), ([0, 2], [0.5], "whole numbers"), ([0, 2], [1 << 32], "32 bits")):
        with pytest.raises(ValueError, match=word):
            Segments(off, index)
    with pytest.raises(ValueError):
        s.offsets[0] = 5                                        # the library reads this memory
    mine = np.array([0, 4], np.int64)
    s = Segments(mine, np.array([0], np.int32))
    mine[1] = 99
    assert s.offsets.tolist() == [0, 4]


def test_padded_batches_are_cut_into_sentences_and_padding():
    s = Segments.of_padded([3, 0, 5], [1, 0, -1], 5)
    assert s.offsets.tolist() == [0, 3, 5, 5, 10, 15, 15] and s.index.tolist() == [1, -2, 0, -2, -1, -2]
    assert not s.covers(15) and Segments([0, 15], [0]).covers(15) and not Segments([0, 14], [0]).covers(15)
    for which in FUNCTIONS:
        rc, msg = answer(which, raw_segments([0, 3, 5, 10], [1, -2, 0]))
        assert rc >= 0, msg
    for lengths, index in (([6], [0]), ([-1], [0]), ([1, 2], [0])):
        with pytest.raises(ValueError):
            Segments.of_padded(lengths, index, 5)


def test_python_face_refuses_before_the_library():
    ops = object.__new__(Operators)                              # no GPU here: a face without a handle
    ops.device, ops.h, ops.lib = 0, C.c_void_p(), _lib.load()
    ops._bind()
    x, a, b, s = torch.zeros(4, 8), torch.zeros(1, 2, 8), torch.zeros(1, 6, 2), torch.ones(1)
    with pytest.raises(ValueError, match="must be on cuda:0"):
        ops.op_lora(x, a, b, s)
    with pytest.raises(TypeError, match="torch tensor"):
        ops.op_lora(x.numpy(), a, b, s)
    with pytest.raises(ValueError, match="must be on cuda:0"):
        ops.op_layernorm(x, torch.ones(1, 8), torch.ones(1, 8))
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        ops.op_lora(x.half(), a, b, s)
    ops.device = -1                                              # (what get_device() says of this machine's tensors)
    with pytest.raises(TypeError, match="b is torch.bfloat16"):
        ops.op_lora(x, a, b.bfloat16(), s)
    with pytest.raises(TypeError, match="scale is torch.float64"):
        ops.op_lora(x, a, b, s.double())
    with pytest.raises(TypeError, match="a must be a torch tensor"):
        ops.op_lora(x, a.numpy(), b, s)
    with pytest.raises(ValueError, match="act must be one of"):
        ops.op_lora(x, a, b, s, act="relu")
    with pytest.raises(ValueError, match="two dimensions"):
        ops.op_lora(x[None], a, b, s)
    with pytest.raises(ValueError, match="share one layout"):
        ops.op_lora(x, a, b, s, base=torch.zeros(6, 4).t())      # rows beside channel-first
    with pytest.raises(ValueError, match="share one layout"):
        ops.op_lora(torch.zeros(1, 8).expand(4, 8), a, b, s)     # rows that lie on each other
    with pytest.raises(ValueError, match="share one layout"):
        ops.op_lora_grad(torch.zeros(8, 4).t(), torch.zeros(4, 6), torch.zeros(4, 2), a, b, s)       # the backward pass takes rows
    with pytest.raises(ValueError, match="scale has shape"):
        ops.op_lora(x, a, b, torch.ones(2))
    with pytest.raises(ValueError, match="b has shape"):
        ops.op_lora(x, a, torch.zeros(1, 6, 3), s)
    with pytest.raises(ValueError, match="x has shape"):
        ops.op_lora(torch.zeros(4, 7), a, b, s)
    with pytest.raises(ValueError, match="base has shape"):
        ops.op_lora(x, a, b, s, base=torch.zeros(4, 7))
    with pytest.raises(ValueError, match="contiguous"):
        ops.op_lora(x, torch.zeros(1, 8, 2).transpose(1, 2), b, s)
    with pytest.raises(ValueError, match="end at token 5"):
        ops.op_lora(x, a, b, s, Segments([0, 5], [0]))
    with pytest.raises(TypeError, match="Segments"):
        ops.op_lora(x, a, b, s, [0, 4])
    with pytest.raises(ValueError, match="h has shape"):
        ops.op_lora_grad(x, torch.zeros(4, 6), torch.zeros(4, 3), a, b, s)
    with pytest.raises(ValueError, match="gain has shape"):
        ops.op_layernorm(x, torch.ones(1, 7), torch.ones(1, 8))
    with pytest.raises(ValueError, match="mean has shape"):
        ops.op_layernorm_grad(x, x, torch.ones(1, 8), torch.ones(3), torch.ones(4))
    # the library's own refusal comes through with its reason
    with pytest.raises(ValueError, match="index 1 of segment 0"):
        ops.op_lora_grad(x, torch.zeros(4, 6), torch.zeros(4, 2), a, b, s, Segments([0, 4], [1]))


@pytest.mark.parametrize("call,wrong", [("op_lora", "x a b scale"), ("op_lora_grad", "x dy h a b scale"),
                                        ("op_layernorm", "x gain offset"), ("op_layernorm_grad", "x dy gain mean rstd")])
def test_python_face_names_what_is_missing(call, wrong):
    ops = object.__new__(Operators)
    ops.device, ops.h, ops.lib = -1, C.c_void_p(), _lib.load()
    given = dict(x=torch.zeros(4, 8), a=torch.zeros(1, 2, 8), b=torch.zeros(1, 6, 2), scale=torch.ones(1), h=torch.zeros(4, 2),
                 dy=torch.zeros(4, 6 if "lora" in call else 8), gain=torch.ones(1, 8), offset=torch.ones(1, 8),
                 mean=torch.ones(4), rstd=torch.ones(4))
    names = wrong.split()
    for name in names:
        with pytest.raises(TypeError, match=f"^{name} must be a torch tensor"):
            getattr(ops, call)(**{**{n: given[n] for n in names}, name: None})
        with pytest.raises(ValueError):
            getattr(ops, call)(**{**{n: given[n] for n in names}, name: torch.tensor(1.0)})


def test_python_face_refuses_numbers_that_do_not_fit():
    ops = object.__new__(Operators)
    ops.device, ops.h, ops.lib = -1, C.c_void_p(), _lib.load()
    x, gain = torch.zeros(4, 8), torch.ones(1, 8)
    for eps in (None, "1e-5"):
        with pytest.raises(ValueError, match="does not fit"):
            ops.op_layernorm(x, gain, gain, eps=eps)
    wide = torch.empty(0, 1 << 31)                               # no memory behind it
    with pytest.raises(ValueError, match="does not fit"):
        ops.op_layernorm(wide, wide, wide, Segments([0], []))


def test_packed_arguments_are_the_structs():
    from tts_amd import operators as O
    for packed, c in ((O._LORA, _lib.K82Lora), (O._LORA_GRAD, _lib.K82LoraGrad), (O._NORM, _lib.K82Layernorm), (O._NORM_GRAD, _lib.K82LayernormGrad)):
        assert packed.size == C.sizeof(c)
        fields = [n for n, _ in c._fields_]
        values = list(range(1, len(fields) + 1))
        s = c.from_buffer_copy(packed.pack(*values))
        assert [int(getattr(s, n)) for n in fields] == values


def test_layouts_of_single_tokens_and_channels_are_taken_either_way():
    def layout(*t, rows_only=False):
        return Operators._layout(rows_only, [("t", v, None) for v in t])
    one = torch.zeros(32, 32).t()[:1, :8]                        # one token, channel-first
    assert layout(one) == (1, [32])
    assert layout(one, torch.zeros(1, 6)) == (1, [32, 1])
    assert layout(torch.zeros(1, 8)) == (0, [8])
    assert layout(torch.zeros(5, 9)[:, 1:], None) == (0, [9, 0])
    assert layout(torch.zeros(9, 32).t()[:5]) == (1, [32])
    assert layout(torch.zeros(7, 3)[:, :1]) == (0, [3])


# ---------------------------------------------------------------------------------------------- adapters of voices
def small_adapter(rank=4, parts=("query", "ffn"), norms=("full_norm",), seed=0, scale=0.5):
    from tts_amd import Adapter
    from tts_amd.adapters import part_shape
    r = np.random.default_rng(seed)
    f = {p: (r.standard_normal((rank, part_shape(p)[0])), r.standard_normal((part_shape(p)[1], rank))) for p in parts}
    return Adapter(f, scale, {m: (r.standard_normal(768), r.standard_normal(768)) for m in norms})


def test_adapter_files_come_back_as_they_went(tmp_path):
    from tts_amd import Adapter
    a = small_adapter()
    a.save(tmp_path / "voice.npz")
    b = Adapter.load(tmp_path / "voice.npz")
    assert (b.rank, b.scale, set(b.factors), set(b.norms)) == (4, 0.5, {"query", "ffn"}, {"full_norm"})
    for part in a.factors:
        for x, y in zip(a.factors[part], b.factors[part]):
            assert x.dtype == np.float32 and np.array_equal(x, y)
    s = b.c_struct()
    assert s.rank == 4 and s.a[0] and s.b[0] and not s.a[1] and s.a[4] and s.gain[1] and not s.gain[0]
    np.savez(tmp_path / "odd.npz", **{"query.a": a.factors["query"][0], "query.b": a.factors["query"][1], "else": np.zeros(3)})
    with pytest.raises(ValueError, match="unexpected arrays"):
        Adapter.load(tmp_path / "odd.npz")
    np.savez(tmp_path / "half.npz", **{"query.a": a.factors["query"][0]})
    with pytest.raises(KeyError):
        Adapter.load(tmp_path / "half.npz")


def test_adapters_that_do_not_fit_are_refused():
    from tts_amd import Adapter
    z = np.zeros
    for factors, norms, word in (
            ({"nose": (z((2, 768)), z((768, 2)))}, {}, "unknown part"), ({"ffn": (z((2, 768)), z((768, 2)))}, {}, "ffn needs"),
            ({"query": (z((129, 768)), z((768, 129)))}, {}, "rank 1 to 128"), ({"query": (z((2, 768)), z((768, 3)))}, {}, "query needs"),
            ({"query": (z((0, 768)), z((768, 0)))}, {}, "rank 1 to 128"),
            ({"query": (z((2, 768)), z((768, 2))), "key": (z((3, 768)), z((768, 3)))}, {}, "one rank"),
            ({}, {"full_norm": (z(768), z(767))}, "gain and an offset"), ({}, {"norm": (z(768), z(768))}, "unknown norm")):
        with pytest.raises(ValueError, match=word):
            Adapter(factors, 1.0, norms)
    with pytest.raises(ValueError, match="finite"):
        Adapter({}, float("inf"))


def test_names_of_adapters_are_resolved_for_the_batch():
    from tts_amd import Engine
    e = object.__new__(Engine)
    e.h = C.c_void_p()
    e._adapters = {"x": 0, "y": 1}
    assert e._adapter_indices(None, 3) is None
    assert e._adapter_indices(["y", None, "x"], 3).tolist() == [1, -1, 0]
    with pytest.raises(ValueError, match="2 sentences, the batch has 3"):
        e._adapter_indices(["x", "y"], 3)
    with pytest.raises(KeyError, match="'z' not found"):
        e._adapter_indices(["z"], 1)
    with pytest.raises(TypeError, match="not a tts_amd.Adapter"):
        e.set_adapters({"x": 3})


def test_the_scheduler_hands_adapters_to_their_sentences():
    from tts_amd.scheduler import BatchSynthesizer
    seen = {}

    class Fake:
        device = 0

        def pack(self, id_lists):
            lens = np.array([len(x) + 2 for x in id_lists], np.int32)
            self.now = [tuple(x) for x in id_lists]
            return np.zeros((len(id_lists), lens.max()), np.int64), lens

        def session(self):
            import contextlib
            return contextlib.nullcontext(self)

        def durations(self, ids, lens, refs, speed=None, **more):
            for k, x in enumerate(self.now):
                seen.setdefault(x, []).append(more["adapters"][k] if more else "none given")
            self.n = np.array([1 if x[0] != 9 else 50 for x in self.now], np.int64)      # ragged: the batch is split and run again
            return np.ones((len(lens), lens.max()), np.int32), self.n

        def decode(self, seeds=None):
            off = np.concatenate([[0], np.cumsum(600 * self.n)])
            return np.zeros(off[-1], np.float32), off

    ids = [[1], [2, 2], [9, 9, 9], [4, 4]]
    names = ["a", None, "b", "a"]
    s = BatchSynthesizer(Fake(), frame_pad_limit=1.5)
    assert len(s.synthesize(ids, [np.zeros(256, np.float32)] * 4, adapters=names)) == 4
    assert s.stats["rebucketed"] >= 1
    for x, n in zip(ids, names):
        assert set(seen[tuple(x)]) == {n}
    seen.clear()
    s.synthesize(ids, [np.zeros(256, np.float32)] * 4)
    assert {v for w in seen.values() for v in w} == {"none given"}
    with pytest.raises(ValueError, match="adapters names 3 sentences, there are 4"):
        s.synthesize(ids, [np.zeros(256, np.float32)] * 4, adapters=names[:3])
