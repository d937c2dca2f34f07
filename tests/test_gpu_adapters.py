"""Adapters of tuned voices through the engine: a sentence with an adapter against the oracle with the adapter's factors
multiplied into its weights (W + scale B A, the same function), and the bits of sentences that share a batch."""
import warnings

import numpy as np
import pytest
import torch

import helpers as H
from tts_amd import Adapter, spec
from tts_amd.adapters import NORMS, PARTS, part_shape

pytestmark = pytest.mark.gpu

KEYS = {"query": "attention.query", "key": "attention.key", "value": "attention.value", "dense": "attention.dense", "ffn": "ffn",
        "ffn_output": "ffn_output", "attention_norm": "attention.LayerNorm", "full_norm": "full_layer_layer_norm"}


def make_adapter(rank, parts=PARTS, norms=NORMS, seed=0, scale=0.7, size=0.05):
    r = np.random.default_rng(seed)
    f = {p: (r.standard_normal((rank, part_shape(p)[0])) / np.sqrt(part_shape(p)[0]), size * r.standard_normal((part_shape(p)[1], rank)))
         for p in parts}
    return Adapter(f, scale, {m: (1 + 0.05 * r.standard_normal(768), 0.02 * r.standard_normal(768)) for m in norms})


def merged(sds, adapter):
    """The state dicts with the adapter multiplied in (the products in 64 bits)."""
    out = {k: dict(v) for k, v in sds.items()}
    bert = out["bert"]

    def key(part, what):
        end = f"albert_layers.0.{KEYS[part]}.{what}"
        (name,) = [k for k in bert if k.endswith(end)]
        return name

    for part, (a, b) in adapter.factors.items():
        w = np.asarray(bert[key(part, "weight")], dtype=np.float64)
        bert[key(part, "weight")] = (w + adapter.scale * (b.astype(np.float64) @ a.astype(np.float64))).astype(np.float32)
    for norm, (gain, offset) in adapter.norms.items():
        bert[key(norm, "weight")], bert[key(norm, "bias")] = gain, offset
    return out


@pytest.fixture(scope="module")
def adapted(synthetic_sds):
    from tts_amd.engine import Engine
    e = Engine(synthetic_sds)
    yield e
    e.close()


def run(e, id_lists, ref_s, adapters=None):
    ids, lens = e.pack(id_lists)
    with e.session():
        e.debug_enable(True)
        try:
            pred, nfr = e.durations(ids, lens, ref_s, adapters=adapters)
            bert = e.debug_get("bert_out")
        finally:
            e.debug_enable(False)
        audio, off = e.decode(seeds=np.arange(len(id_lists), dtype=np.uint64))
    return [(pred[b, :lens[b]].copy(), bert[b, :, :lens[b]].copy(), audio[off[b]:off[b + 1]].copy()) for b in range(len(id_lists))]


def test_adapted_sentences_match_the_oracle_with_merged_weights(adapted, synthetic_sds):
    warnings.filterwarnings("ignore")
    from oracle import kokoro_ref as R
    voices = {"all": make_adapter(7, seed=1), "factors": make_adapter(16, norms=(), seed=2), "norms": make_adapter(1, parts=(), seed=3),
              "query": make_adapter(33, parts=("query",), norms=("attention_norm",), seed=4)}
    adapted.set_adapters(voices)
    names = [None, "all", "factors", "norms", "query", "all"]
    id_lists, ref_s = H.make_batch(31, [20, 9, 57, 33, 40, 70])
    got = run(adapted, id_lists, ref_s, names)
    models = {n: R.build(spec.DEFAULT_CONFIG, merged(synthetic_sds, v)) for n, v in voices.items()}
    models[None] = R.build(spec.DEFAULT_CONFIG, synthetic_sds)
    plain = run(adapted, id_lists, ref_s)
    for b, n in enumerate(names):
        taps = {}
        ids = torch.tensor([[0] + id_lists[b] + [0]])
        noise = torch.zeros(1, 600 * int(got[b][0].sum()), 9)
        _, pd = models[n].forward_with_tokens(ids, torch.from_numpy(ref_s[b:b + 1].copy()), 1.0, noise=noise, taps=taps)
        want = H.to_bct("bert_out", taps["bert_out"])
        # twelve layers of Linears over 768 / 2048 channels in 32 bits on either side: the stage's own bar in the parity suite
        assert np.abs(got[b][1] - want).max() <= 5e-4 * max(1.0, np.abs(want).max()), (n, np.abs(got[b][1] - want).max())
        if n is None:
            assert np.array_equal(got[b][0], pd.numpy())
        else:
            assert np.abs(got[b][1] - plain[b][1]).max() > 1e-2, n       # the adapter does something


def test_bits_do_not_depend_on_the_batch(adapted):
    voices = {"x": make_adapter(8, seed=5), "y": make_adapter(3, parts=("ffn", "value"), norms=("full_norm",), seed=6)}
    adapted.set_adapters(voices)
    id_lists, ref_s = H.make_batch(32, [12, 45, 3, 66, 31, 8])
    names = ["x", None, "y", None, "x", "y"]
    mixed = run(adapted, id_lists, ref_s, names)
    plain = run(adapted, id_lists, ref_s)
    for b, n in enumerate(names):
        alone = run(adapted, id_lists[b:b + 1], ref_s[b:b + 1], [n])[0]
        for what, u, v in zip(("durations", "bert_out"), mixed[b], alone):
            assert np.array_equal(u, v), (b, n, what)
        if n is None:
            for what, u, v in zip(("durations", "bert_out", "audio"), mixed[b], plain[b]):
                assert np.array_equal(u, v), (b, what)


def test_an_adapter_of_zeros_changes_no_bit(adapted):
    zero = make_adapter(5, norms=(), seed=7, size=0.0)
    adapted.set_adapters({"zero": zero})
    id_lists, ref_s = H.make_batch(33, [25, 14])
    for u, v in zip(run(adapted, id_lists, ref_s, ["zero", None]), run(adapted, id_lists, ref_s)):
        for a, b in zip(u, v):
            assert np.array_equal(a, b)


def test_forks_inherit_and_protect_adapters(adapted):
    adapted.set_adapters({"x": make_adapter(8, seed=5)})
    id_lists, ref_s = H.make_batch(34, [25, 14])
    want = run(adapted, id_lists, ref_s, ["x", None])
    f = adapted.fork()
    try:
        for u, v in zip(run(f, id_lists, ref_s, ["x", None]), want):
            for a, b in zip(u, v):
                assert np.array_equal(a, b)
        with pytest.raises(RuntimeError, match="forks"):
            adapted.set_adapters({})
        with pytest.raises(RuntimeError, match="forks"):
            f.set_adapters({})
    finally:
        f.close()
    adapted.set_adapters({})
    with pytest.raises(KeyError):
        adapted.durations(*adapted.pack(id_lists), ref_s, adapters=["x", None])


def test_indices_outside_are_refused_by_the_library(adapted):
    import ctypes as C
    adapted.set_adapters({"x": make_adapter(8, seed=5)})
    id_lists, ref_s = H.make_batch(35, [5])
    ids, lens = adapted.pack(id_lists)
    for bad in (1, -2):
        k = np.array([bad], np.int32)
        rc = adapted.lib.k82_durations_adapted(adapted.h, ids.ctypes.data, lens.ctypes.data, 1, ids.shape[1], ref_s.ctypes.data, None,
                                               None, k.ctypes.data, None, None, None)
        assert rc == -22 and b"outside [-1, 1)" in adapted.lib.k82_last_error(adapted.h)
    from tts_amd import _lib
    bad = _lib.K82Adapter(rank=0, scale=1.0)
    bad.a[0] = bad.b[0] = ids.ctypes.data
    assert adapted.lib.k82_set_adapters(adapted.h, C.byref(bad), 1) == -22
    bad = _lib.K82Adapter(rank=4, scale=1.0)
    bad.a[0] = ids.ctypes.data
    assert adapted.lib.k82_set_adapters(adapted.h, C.byref(bad), 1) == -22
    assert adapted.lib.k82_set_adapters(adapted.h, None, 2) == -22


def test_the_front_door_takes_an_adapter():
    from tts_amd import Kokoro
    k = Kokoro("synthetic", None)
    k.engine.set_adapters({"voice": make_adapter(8, seed=9)})
    try:
        text = "abc def"
        plain, _ = k.create(text, "af_synthetic", is_phonemes=True, trim=False)
        tuned, _ = k.create(text, "af_synthetic", is_phonemes=True, trim=False, adapter="voice")
        assert plain.shape != tuned.shape or not np.array_equal(plain, tuned)
        both = k.create_batch([text, text], "af_synthetic", is_phonemes=True, trim=False, adapter=[None, "voice"])
        assert np.array_equal(both[0][0], plain) and both[1][0].shape == tuned.shape
        with pytest.raises(KeyError):
            k.create(text, "af_synthetic", is_phonemes=True, adapter="nobody")
        with pytest.raises(ValueError):
            k.create_batch([text, text], "af_synthetic", is_phonemes=True, adapter=["voice"])
    finally:
        k.engine.set_adapters({})
