"""What sentences with adapters say: durations and samples against the oracle with the adapters multiplied into its weights, and
their bits alone and in a batch, samples included.  Bars: the parity suite's (test_gpu_parity.py), 2e-3 for a duration before it
is rounded, 1e-3 for a sample with F0, N and the source's transform taken from the engine; the adapter is one more product of
768 or 2048 terms beside each Linear, in the same 32 bits."""
import warnings

import numpy as np
import pytest
import torch

import helpers as H
from oracle import kokoro_ref as R
from test_gpu_adapters import adapted, make_adapter, merged  # noqa: F401
from tts_amd import spec

pytestmark = pytest.mark.gpu

VOICES = {"all": dict(rank=7, seed=1), "factors": dict(rank=16, norms=(), seed=2), "norms": dict(rank=1, parts=(), seed=3),
          "ffn": dict(rank=33, parts=("ffn", "dense"), norms=("full_norm",), seed=4)}


def test_durations_and_samples_of_adapted_sentences(adapted, synthetic_sds):  # noqa: F811
    warnings.filterwarnings("ignore")
    voices = {n: make_adapter(**v) for n, v in VOICES.items()}
    adapted.set_adapters(voices)
    models = {n: R.build(spec.DEFAULT_CONFIG, merged(synthetic_sds, v)) for n, v in voices.items()}
    models[None] = R.build(spec.DEFAULT_CONFIG, synthetic_sds)
    names = ["all", None, "norms", "factors", "ffn", None, "all"]
    id_lists, ref_s = H.make_batch(41, [12, 5, 30, 21, 9, 16, 2])
    ids, lens = adapted.pack(id_lists)
    forced = np.zeros(ids.shape, np.int32)
    with adapted.session():
        adapted.debug_enable(True)
        try:
            pred, _ = adapted.durations(ids, lens, ref_s, adapters=names)
            raw = adapted.debug_get("duration")[:, 0, :]
            for b, n in enumerate(names):
                t = torch.tensor([[0] + id_lists[b] + [0]])
                pd, _, want = models[n].durations(t, torch.from_numpy(ref_s[b:b + 1].copy()), 1.0)
                want = want.numpy().reshape(-1)
                assert np.abs(raw[b, :lens[b]] - want).max() <= 2e-3, (b, n, np.abs(raw[b, :lens[b]] - want).max())
                sure = (np.abs(want % 1.0 - 0.5) > 2e-3) | (want < 1.0)              # not at a border of the rounding
                assert np.array_equal(pred[b, :lens[b]][sure], pd.numpy()[sure]), (b, n)
                forced[b, :lens[b]] = pd.numpy()
            _, nfr = adapted.durations(ids, lens, ref_s, forced_dur=forced, adapters=names)
            noise = np.concatenate([R.counter_noise(b, int(f) * 600) for b, f in enumerate(nfr)])
            audio, off = adapted.decode(noise=noise)
            f0, n_curve, har = (adapted.debug_get(k) for k in ("F0", "N", "har"))
        finally:
            adapted.debug_enable(False)
    for b, n in enumerate(names):
        F = int(nfr[b])
        a_ref, _ = H.oracle_run(models[n], id_lists[b], ref_s[b], 1.0, noise.reshape(-1, 9)[off[b]:off[b + 1]], forced=forced[b, :lens[b]],
                                f0=f0[b, 0, :2 * F], n=n_curve[b, 0, :2 * F], har=har[b][:22, :120 * F + 1])
        assert np.abs(audio[off[b]:off[b + 1]] - a_ref).max() <= 1e-3, (b, n)


def test_samples_do_not_depend_on_the_batch(adapted):  # noqa: F811
    """Every second sentence with norms or factors of its own, more pieces than one launch's table holds."""
    adapted.set_adapters({n: make_adapter(**v) for n, v in VOICES.items()})
    some = list(VOICES)
    names = [some[(i // 2) % 4] if i % 2 else None for i in range(140)]
    id_lists, ref_s = H.make_batch(42, [1 + (5 * i) % 7 for i in range(140)])
    seeds = np.arange(140, dtype=np.uint64) + 50

    def run(which, names):
        ids, lens = adapted.pack([id_lists[i] for i in which])
        with adapted.session():
            pred, _ = adapted.durations(ids, lens, ref_s[which], adapters=names)
            audio, off = adapted.decode(seeds=seeds[which])
        return [(pred[k, :lens[k]].copy(), audio[off[k]:off[k + 1]].copy()) for k in range(len(which))]

    batch = run(list(range(140)), names)
    for i in (0, 1, 2, 3, 5, 7, 63, 127, 128, 129, 138, 139):
        for got, want in zip(batch[i], run([i], [names[i]])[0]):
            assert np.array_equal(got, want), (i, names[i])
    for i, (got, want) in enumerate(zip(batch, run(list(range(140)), None))):
        if names[i] is None:
            assert all(np.array_equal(u, v) for u, v in zip(got, want)), i


def test_adapters_that_are_not_numbers_are_refused_by_the_library(adapted):  # noqa: F811
    voice = make_adapter(rank=3, seed=5)
    adapted.set_adapters({"x": voice})
    for values in (*voice.factors["ffn_output"], *voice.norms["attention_norm"]):
        kept, values.flat[-1] = float(values.flat[-1]), float("nan")
        with pytest.raises(ValueError, match="must be finite"):
            adapted.set_adapters({"y": voice})
        values.flat[-1] = kept
    assert adapted._adapter_indices(["x"], 1).tolist() == [0]                         # the set is what it was
    adapted.set_adapters({"y": voice})
