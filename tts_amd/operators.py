"""Operators on the caller's own GPU tensors (include/k82.h): per-request weights beside the model's shared ones.

``Operators`` is a handle without model weights; ``Engine`` is one with them and has the same methods.  Tensors are torch
tensors on the handle's GPU -- the buffers, nothing else: every number is computed in libk82.so.  A call enqueues on
torch's current stream and returns at once; outputs and workspaces come from torch's allocator, so a call may be captured
into a graph.  There is no autograd: gradients are calls of their own (``op_*_grad``).  Refused arguments raise ``ValueError`` / ``TypeError`` before anything is enqueued.

Tensors are ``[tokens, channels]``, rows (unit stride along the channels) or, float32 forward only, channel-first (unit
stride along the tokens: ``buffer[channels, pitch].t()``, the engine's own layout).
"""
from __future__ import annotations

import ctypes as C
import struct

import numpy as np

from . import _lib, spec

ACTS = {"none": 0, "gelu_new": 1}

# The argument structs of include/k82.h as native byte strings (a small call is bound by the host: 0.6 us where filling a
# ctypes.Structure takes 2); the ctypes forms in _lib.py have the same sizes.
_LORA = struct.Struct("@7i4xqPqPqPqPPPP")
_LORA_GRAD = struct.Struct("@5i4xqPqPqPPqPqPPPPP")
_NORM = struct.Struct("@4if4xqPqPqPqPPPP")
_NORM_GRAD = struct.Struct("@3i4xqPqPqPqPqPPPPP")


def _cfg_struct(config):
    pl = config["plbert"]
    return _lib.K82Config(
        n_token=config["n_token"], hidden_dim=config["hidden_dim"], style_dim=config["style_dim"],
        n_layer=config["n_layer"], max_dur=config["max_dur"], text_kernel=config["text_encoder_kernel_size"],
        bert_hidden=pl["hidden_size"], bert_heads=pl["num_attention_heads"], bert_inter=pl["intermediate_size"],
        bert_layers=pl["num_hidden_layers"], bert_max_pos=pl["max_position_embeddings"],
        bert_embed=spec.ALBERT_EMBED)


class Segments:
    """The cut of a packed token axis: segment ``s`` holds the tokens ``offsets[s]:offsets[s + 1]`` and uses adapter (or
    gain) ``index[s]``; -1 is a sentence without an adapter, ``Segments.SKIP`` tokens that belong to nobody (padding).  Host
    data; keep it for as many calls as the batch makes."""

    SKIP = -2
    __slots__ = ("offsets", "index", "c", "address", "lo", "hi", "whole")

    def __init__(self, offsets, index):
        offsets, index = np.asarray(offsets), np.asarray(index)
        if (offsets.size and offsets.dtype.kind not in "iu") or (index.size and index.dtype.kind not in "iu"):
            raise ValueError("Segments: offsets and index are whole numbers")
        if index.size and (index.min() < -(1 << 31) or index.max() >= 1 << 31):
            raise ValueError("Segments: an index does not fit 32 bits")
        self.offsets = offsets.astype(np.int64)                  # copies: nobody else writes what the library reads
        self.index = index.astype(np.int32)
        if self.offsets.ndim != 1 or self.index.ndim != 1 or self.offsets.size != self.index.size + 1:
            raise ValueError("Segments: offsets holds one value more than index")
        if self.offsets[0] < 0 or (self.offsets[1:] < self.offsets[:-1]).any():
            raise ValueError("Segments: offsets must not be negative and must not decrease")
        self.offsets.flags.writeable = self.index.flags.writeable = False
        self.lo, self.hi = int(self.offsets[0]), int(self.offsets[-1])
        self.whole = not (self.index == self.SKIP).any()         # every token from lo to hi is somebody's
        self.c = _lib.K82Segments(off=self.offsets.ctypes.data, index=self.index.ctypes.data, n=self.index.size)
        self.address = C.addressof(self.c)

    @classmethod
    def of_lengths(cls, lengths, index):
        return cls(np.concatenate([[0], np.cumsum(np.asarray(lengths, dtype=np.int64))]).astype(np.int64), index)

    @classmethod
    def of_padded(cls, lengths, index, pitch):
        """A padded batch ``[len(lengths) * pitch, channels]``: sentence ``s`` in the first ``lengths[s]`` of its rows."""
        lengths, index = np.asarray(lengths, dtype=np.int64), np.asarray(index, dtype=np.int64)
        if lengths.shape != index.shape or lengths.ndim != 1 or (lengths < 0).any() or (lengths > pitch).any():
            raise ValueError(f"Segments: a length in [0, {pitch}] and an index for each sentence")
        start = np.arange(lengths.size, dtype=np.int64) * pitch
        off = np.stack([start, start + lengths], 1).reshape(-1)
        return cls(np.append(off, lengths.size * pitch), np.stack([index, np.full_like(index, cls.SKIP)], 1).reshape(-1))

    def covers(self, tokens):
        """Whether every one of ``tokens`` tokens is somebody's."""
        return self.whole and self.lo == 0 and self.hi == tokens


class Operators:
    """A handle of libk82.so for the operators alone (``k82_create`` without weights)."""

    _torch = None

    def __init__(self, device=0):
        self.device = device
        self._open(spec.DEFAULT_CONFIG)

    def _open(self, config):
        self.lib = _lib.load()
        self.h = C.c_void_p()
        cfg = _cfg_struct(config)
        rc = self.lib.k82_create(C.byref(cfg), self.device, C.byref(self.h))
        if rc != 0:
            raise RuntimeError(f"k82_create failed ({rc}): {self.lib.k82_last_error(None).decode()}")

    def _check(self, rc):
        if rc != 0:
            msg = self.lib.k82_last_error(self.h).decode()
            if rc in (-22, -28):
                raise ValueError(f"k82 error {rc}: {msg}")
            raise RuntimeError(f"k82 error {rc}: {msg}")

    def close(self):
        if getattr(self, "h", None) and self.h.value:
            self.lib.k82_destroy(self.h)
            self.h = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    # ------------------------------------------------------------------ arguments
    def _bind(self):
        """What every call needs: torch (never imported before a handle is) and the entry points for packed arguments."""
        import torch
        # the handle alone where torch offers it: a Stream object costs a microsecond
        self._raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda d: torch.cuda.current_stream(d).cuda_stream)
        self._codes = {torch.float32: 0, torch.bfloat16: 1}
        vp, i64 = C.c_void_p, C.c_int64
        forward, backward = C.CFUNCTYPE(C.c_int, vp, C.c_char_p, vp, vp), C.CFUNCTYPE(C.c_int, vp, C.c_char_p, vp, vp, i64, vp)
        size = C.CFUNCTYPE(i64, C.c_char_p, vp)
        fn = {}
        for op in ("lora", "layernorm"):
            fn[op] = forward((f"k82_op_{op}", self.lib))
            fn[op + "_grad"] = (backward((f"k82_op_{op}_grad", self.lib)), size((f"k82_op_{op}_grad_workspace", self.lib)))
        self._fn = fn
        self._torch = torch                                      # last: a thread that finds it set finds the rest
        return torch

    def _stream(self):
        # torch's default stream is handle 0, which the library takes for "the handle's own": name it hipStreamLegacy (1)
        return self._raw_stream(self.device) or 1

    def _placed(self, dtype, named, optional=()):
        """Every tensor is one of this GPU and of ``dtype``; those of ``optional`` may be None."""
        dev = self.device
        for some, needed in ((named, True), (optional, False)):
            for name, t in some:
                if t is None and not needed:
                    continue
                try:
                    at, dt = t.get_device(), t.dtype
                except AttributeError:
                    raise TypeError(f"{name} must be a torch tensor on the GPU") from None
                if at != dev:
                    raise ValueError(f"{name} must be on cuda:{dev}, it is on {t.device}")
                if dt is not dtype:
                    raise TypeError(f"{name} is {dt}, {dtype} is needed")

    def _code(self, x):
        code = self._codes.get(getattr(x, "dtype", None))
        if code is None:
            if not hasattr(x, "data_ptr"):
                raise TypeError("x must be a torch tensor on the GPU")
            raise TypeError(f"float32 or bfloat16 tensors are needed, x is {x.dtype}")
        return code

    @staticmethod
    def _layout(rows_only, shapes):
        """-> (layout, [ld of each]) of [tokens, channels] tensors that share one layout; shapes: (name, tensor or None,
        wanted shape or None)."""
        rows, cols, found, plain = True, not rows_only, [], True
        for name, t, want in shapes:
            if t is None:
                continue
            shape = t.shape
            if len(shape) != 2:
                raise ValueError(f"{name} must have two dimensions [tokens, channels], it has {len(shape)}")
            if want is not None and shape != want:
                raise ValueError(f"{name} has shape {tuple(shape)}, {tuple(want)} is needed")
            plain = plain and t.is_contiguous()
        if plain:                                                # the common case in half the time
            return 0, [0 if t is None else t.shape[1] or 1 for _, t, _ in shapes]
        for name, t, want in shapes:
            if t is None:
                found.append(None)
                continue
            n, c = t.shape
            sn, sc = t.stride()
            rows = rows and (sc == 1 or c == 1) and (n <= 1 or sn >= c)
            cols = cols and (sn == 1 or n == 1) and (c <= 1 or sc >= n)
            found.append((n, c, sn, sc))
        if rows:
            return 0, [0 if v is None else v[2] if v[0] > 1 else max(1, v[1]) for v in found]
        if cols:
            return 1, [0 if v is None else v[3] if v[1] > 1 else max(1, v[0]) for v in found]
        raise ValueError("tensors must share one layout: unit stride along the channels" + (
            "" if rows_only else " (or along the tokens: channel-first)") + " and rows that do not overlap")

    @staticmethod
    def _packed(form, *values):
        try:
            return form.pack(*values)
        except struct.error as e:
            raise ValueError(f"an argument does not fit the library's: {e}") from None

    @staticmethod
    def _need(name, t, shape):
        if t.shape != shape:
            raise ValueError(f"{name} has shape {tuple(t.shape)}, {shape} is needed")
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")

    def _out(self, x, n, channels, cols, full):
        """A new [tokens, channels] tensor in the layout of x and its ld; zero where no segment will write."""
        ld = max(32, (n + 31) // 32 * 32) if cols else channels
        out = x.new_empty_strided((n, channels), (1, ld)) if cols else x.new_empty((n, channels))
        return out if full else out.zero_(), ld

    @staticmethod
    def _segments(seg, n):
        if seg is None:
            return Segments([0, n], [0])
        if not isinstance(seg, Segments):
            raise TypeError("seg must be a Segments (or None: every token uses index 0)")
        if seg.hi > n:
            raise ValueError(f"the segments end at token {seg.hi}, the tensors hold {n}")
        return seg

    def _factors(self, a, b, scale):
        of_a, of_b = a.shape, b.shape
        if len(of_a) != 3 or len(of_b) != 3:
            raise ValueError("a is [adapters, rank, cin] and b [adapters, cout, rank]")
        n, rank, cin = of_a
        cout = of_b[1]
        self._need("b", b, (n, cout, rank))
        self._need("scale", scale, (n,))
        if not a.is_contiguous():
            raise ValueError("a must be contiguous")
        return n, rank, cin, cout

    # ------------------------------------------------------------------ low-rank adapters
    def op_lora(self, x, a, b, scale, seg=None, base=None, act="none", out=None, keep=False):
        """k82_op_lora: ``act(base + scale[k] * (x @ a[k].T) @ b[k].T)`` with ``k`` the adapter of the token's segment
        (-1: ``act(base)``).  ``a`` [adapters, rank, cin], ``b`` [adapters, cout, rank], ``scale`` float32 [adapters].
        ``base``: the shared projection's output, which ``out`` may be.  ``keep``: returns ``(y, h)`` with
        ``h = x @ a[k].T`` in float32, which ``op_lora_grad`` takes."""
        torch = self._torch or self._bind()
        code, dt, f32 = self._code(x), x.dtype, torch.float32
        self._placed(dt, (("x", x), ("a", a), ("b", b)), (("base", base), ("out", out)))
        self._placed(f32, (("scale", scale),))
        if act not in ACTS:
            raise ValueError(f"act must be one of {sorted(ACTS)}, not {act!r}")
        n, rank, cin, cout = self._factors(a, b, scale)
        tokens = x.shape[0] if x.dim() else 0
        of_y = (tokens, cout)
        layout, (ldx, ldbase, ldy) = self._layout(False, (("x", x, (tokens, cin)), ("base", base, of_y), ("out", out, of_y)))
        seg = self._segments(seg, tokens)
        full = seg.covers(tokens)
        if out is None:
            out, ldy = self._out(x, tokens, cout, layout, full)
        h = scale.new_empty((tokens, rank)) if keep else None
        if keep and not full:
            h.zero_()
        p = self._packed(_LORA, code, layout, ACTS[act], cin, cout, rank, n, tokens, x.data_ptr(), ldx, 0 if base is None else base.data_ptr(),
                         ldbase, out.data_ptr(), ldy, a.data_ptr(), b.data_ptr(), scale.data_ptr(), 0 if h is None else h.data_ptr())
        rc = self._fn["lora"](self.h, p, seg.address, self._stream())
        if rc:
            self._check(rc)
        return (out, h) if keep else out

    def op_lora_grad(self, x, dy, h, a, b, scale, seg=None, dx_base=None, dx=None):
        """k82_op_lora_grad -> ``(dx, da, db)``; ``dy`` is the gradient in front of the activation, ``h`` what
        ``op_lora(keep=True)`` returned, ``dx_base`` the shared projection's gradient (which ``dx`` may be).  ``da`` and
        ``db`` are float32 sums over the tokens in a fixed order, zero for an adapter without tokens."""
        torch = self._torch or self._bind()
        code, dt, f32 = self._code(x), x.dtype, torch.float32
        self._placed(dt, (("x", x), ("dy", dy), ("a", a), ("b", b)), (("dx_base", dx_base), ("dx", dx)))
        self._placed(f32, (("h", h), ("scale", scale)))
        n, rank, cin, cout = self._factors(a, b, scale)
        tokens = x.shape[0] if x.dim() else 0
        of_x = (tokens, cin)
        _, (ldx, lddy, ldbase, lddx) = self._layout(True, (("x", x, of_x), ("dy", dy, (tokens, cout)), ("dx_base", dx_base, of_x),
                                                           ("dx", dx, of_x)))
        self._need("h", h, (tokens, rank))
        seg = self._segments(seg, tokens)
        if dx is None:
            dx, lddx = self._out(x, tokens, cin, 0, seg.covers(tokens))
        da, db = scale.new_empty((n, rank, cin)), scale.new_empty((n, cout, rank))
        p = self._packed(_LORA_GRAD, code, cin, cout, rank, n, tokens, x.data_ptr(), ldx, dy.data_ptr(), lddy, h.data_ptr(),
                         0 if dx_base is None else dx_base.data_ptr(), ldbase, dx.data_ptr(), lddx, a.data_ptr(),
                         b.data_ptr(), scale.data_ptr(), da.data_ptr(), db.data_ptr())
        self._with_workspace("lora_grad", p, seg, x)
        return dx, da, db

    # ------------------------------------------------------------------ layer norm
    def op_layernorm(self, x, gain, offset, seg=None, res=None, eps=1e-12, out=None, stats=False):
        """k82_op_layernorm: ``(z - mean) * rstd * gain[k] + offset[k]`` over the channels of ``z = x + res``, ``gain`` and
        ``offset`` ``[gains, channels]``, ``k`` the index of the token's segment.  ``out`` may be ``x`` or ``res``.
        ``stats``: returns ``(y, mean, rstd)`` (float32), which ``op_layernorm_grad`` takes."""
        torch = self._torch or self._bind()
        code = self._code(x)
        self._placed(x.dtype, (("x", x), ("gain", gain), ("offset", offset)), (("res", res), ("out", out)))
        shape = x.shape
        layout, (ldx, ldres, ldy) = self._layout(False, (("x", x, None), ("res", res, shape), ("out", out, shape)))
        tokens, c = shape
        gains = gain.shape[0] if gain.dim() else 0
        self._need("gain", gain, (gains, c))
        self._need("offset", offset, (gains, c))
        seg = self._segments(seg, tokens)
        full = seg.covers(tokens)
        if out is None:
            out, ldy = self._out(x, tokens, c, layout, full)
        mean = rstd = None
        if stats:
            new = torch.empty if full else torch.zeros
            mean, rstd = (new((tokens,), dtype=torch.float32, device=x.device) for _ in range(2))
        p = self._packed(_NORM, code, layout, c, gains, eps, tokens, x.data_ptr(), ldx, 0 if res is None else res.data_ptr(), ldres,
                         out.data_ptr(), ldy, gain.data_ptr(), offset.data_ptr(), 0 if mean is None else mean.data_ptr(),
                         0 if rstd is None else rstd.data_ptr())
        rc = self._fn["layernorm"](self.h, p, seg.address, self._stream())
        if rc:
            self._check(rc)
        return (out, mean, rstd) if stats else out

    def op_layernorm_grad(self, x, dy, gain, mean, rstd, seg=None, res=None, dx=None):
        """k82_op_layernorm_grad -> ``(dx, dgain, doffset)``: ``dx`` is the gradient of ``x`` and of ``res`` alike and may be
        ``dy``, ``x`` or ``res`` itself; ``dgain`` and ``doffset`` are float32 sums over the tokens in a fixed order."""
        torch = self._torch or self._bind()
        code, f32 = self._code(x), torch.float32
        self._placed(x.dtype, (("x", x), ("dy", dy), ("gain", gain)), (("res", res), ("dx", dx)))
        self._placed(f32, (("mean", mean), ("rstd", rstd)))
        shape = x.shape
        _, (ldx, ldres, lddy, lddx) = self._layout(True, (("x", x, None), ("res", res, shape), ("dy", dy, shape), ("dx", dx, shape)))
        tokens, c = shape
        gains = gain.shape[0] if gain.dim() else 0
        self._need("gain", gain, (gains, c))
        self._need("mean", mean, (tokens,))
        self._need("rstd", rstd, (tokens,))
        seg = self._segments(seg, tokens)
        if dx is None:
            dx, lddx = self._out(x, tokens, c, 0, seg.covers(tokens))
        dgain, doffset = mean.new_empty((gains, c)), mean.new_empty((gains, c))
        p = self._packed(_NORM_GRAD, code, c, gains, tokens, x.data_ptr(), ldx, 0 if res is None else res.data_ptr(), ldres,
                         dy.data_ptr(), lddy, dx.data_ptr(), lddx, gain.data_ptr(), mean.data_ptr(), rstd.data_ptr(),
                         dgain.data_ptr(), doffset.data_ptr())
        self._with_workspace("layernorm_grad", p, seg, x)
        return dx, dgain, doffset

    def _with_workspace(self, op, p, seg, x):
        call, size = self._fn[op]
        need = size(p, seg.address)
        if need < 0:
            raise ValueError(f"k82 error {need}: {self.lib.k82_last_error(None).decode()}")
        ws = self._torch.empty((need,), dtype=self._torch.uint8, device=x.device) if need else None
        rc = call(self.h, p, seg.address, None if ws is None else ws.data_ptr(), need, self._stream())
        if rc:
            self._check(rc)
