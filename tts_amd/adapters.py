"""Adapters of tuned voices: what a voice carries beyond its style vector (include/k82.h, k82_set_adapters).

An adapter holds low-rank factors for some of the Linears of the ALBERT encoder -- ``y += scale * (x @ a.T) @ b.T`` beside the
shared projection, at each of its layers (they share weights) -- and / or a gain and an offset in the place of its layer
norms.  Sentences of one batch may each have their own (``Engine.durations(adapters=...)``, ``Kokoro.create(adapter=...)``).
On disk: an ``.npz`` of ``<part>.a`` f32[rank, in], ``<part>.b`` f32[out, rank], ``scale``, ``<norm>.gain`` and
``<norm>.offset`` f32[768].
"""
from __future__ import annotations

import numpy as np

from . import _lib, spec

PARTS = ("query", "key", "value", "dense", "ffn", "ffn_output")      # K82_ADAPTER_*
NORMS = ("attention_norm", "full_norm")


def part_shape(part, config=None):
    """(in features, out features) of a part's Linear."""
    pl = (config or spec.DEFAULT_CONFIG)["plbert"]
    d, i = pl["hidden_size"], pl["intermediate_size"]
    return {"ffn": (d, i), "ffn_output": (i, d)}.get(part, (d, d))


class Adapter:
    """``factors``: {part: (a, b)}; ``norms``: {norm: (gain, offset)}; one rank and one scale for all parts."""

    def __init__(self, factors=None, scale=1.0, norms=None, config=None):
        d = (config or spec.DEFAULT_CONFIG)["plbert"]["hidden_size"]
        self.scale = float(scale)
        if not np.isfinite(self.scale):
            raise ValueError("Adapter: scale must be finite")
        self.rank, self.factors, self.norms = 0, {}, {}
        for part, (a, b) in (factors or {}).items():
            if part not in PARTS:
                raise ValueError(f"Adapter: unknown part {part!r}, there are {PARTS}")
            a, b = (np.ascontiguousarray(v, dtype=np.float32) for v in (a, b))
            cin, cout = part_shape(part, config)
            rank = a.shape[0] if a.ndim == 2 else 0
            if a.shape != (rank, cin) or b.shape != (cout, rank) or not 1 <= rank <= 128:
                raise ValueError(f"Adapter: {part} needs a [rank, {cin}] and b [{cout}, rank] with rank 1 to 128, "
                                 f"got {a.shape} and {b.shape}")
            if not (np.isfinite(a).all() and np.isfinite(b).all()):
                raise ValueError(f"Adapter: the factors of {part} must be finite")
            if self.rank not in (0, rank):
                raise ValueError(f"Adapter: one rank for all parts, got {self.rank} and {rank}")
            self.rank = rank
            self.factors[part] = (a, b)
        for norm, pair in (norms or {}).items():
            if norm not in NORMS:
                raise ValueError(f"Adapter: unknown norm {norm!r}, there are {NORMS}")
            gain, offset = (np.ascontiguousarray(v, dtype=np.float32) for v in pair)
            if gain.shape != (d,) or offset.shape != (d,):
                raise ValueError(f"Adapter: {norm} needs a gain and an offset of {d} values")
            if not (np.isfinite(gain).all() and np.isfinite(offset).all()):
                raise ValueError(f"Adapter: gain and offset of {norm} must be finite")
            self.norms[norm] = (gain, offset)

    @classmethod
    def load(cls, path, config=None):
        with np.load(path, allow_pickle=False) as z:
            names = set(z.files)
            parts = {p: (z[p + ".a"], z[p + ".b"]) for p in PARTS if p + ".a" in names or p + ".b" in names}
            norms = {m: (z[m + ".gain"], z[m + ".offset"]) for m in NORMS if m + ".gain" in names or m + ".offset" in names}
            known = {f"{p}.{x}" for p in parts for x in "ab"} | {f"{m}.{x}" for m in norms for x in ("gain", "offset")} | {"scale"}
            if names - known:
                raise ValueError(f"{path}: unexpected arrays {sorted(names - known)[:5]}")
            return cls(parts, float(z["scale"]) if "scale" in names else 1.0, norms, config)

    def save(self, path):
        arrays = {"scale": np.float32(self.scale)}
        for part, (a, b) in self.factors.items():
            arrays.update({part + ".a": a, part + ".b": b})
        for norm, (gain, offset) in self.norms.items():
            arrays.update({norm + ".gain": gain, norm + ".offset": offset})
        with open(path, "wb") as f:
            np.savez(f, **arrays)

    def c_struct(self):
        """The k82_adapter of this adapter; it reads the arrays that this object holds."""
        s = _lib.K82Adapter(rank=self.rank, scale=self.scale)
        for i, part in enumerate(PARTS):
            if part in self.factors:
                s.a[i], s.b[i] = (v.ctypes.data for v in self.factors[part])
        for i, norm in enumerate(NORMS):
            if norm in self.norms:
                s.gain[i], s.offset[i] = (v.ctypes.data for v in self.norms[norm])
        return s
