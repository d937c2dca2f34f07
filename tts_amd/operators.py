"""Operators on the caller's own GPU tensors (include/k82.h): per-request weights beside the model's shared ones.

``Operators`` is a handle without model weights; ``Engine`` is one with them and has the same methods.  Tensors are torch
tensors on the handle's GPU -- the buffers, nothing else: every number is computed in libk82.so.  A call enqueues on
torch's current stream and returns at once; outputs and workspaces come from torch's allocator, so a call may be captured
into a graph.  Refused arguments raise ``ValueError`` / ``TypeError`` before anything is enqueued.

Tensors are ``[tokens, channels]``, rows (unit stride along the channels) or, float32 forward only, channel-first (unit
stride along the tokens: ``buffer[channels, pitch].t()``, the engine's own layout).
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from . import _lib, spec

ACTS = {"none": 0, "gelu_new": 1}


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
    gain) ``index[s]``; -1 is a sentence without an adapter.  Host data; keep it for as many calls as the batch makes."""

    __slots__ = ("offsets", "index", "c", "lo", "hi")

    def __init__(self, offsets, index):
        self.offsets = np.array(offsets, dtype=np.int64)
        self.index = np.array(index, dtype=np.int32)
        if self.offsets.ndim != 1 or self.index.ndim != 1 or self.offsets.size != self.index.size + 1:
            raise ValueError("Segments: offsets holds one value more than index")
        if (np.diff(self.offsets) < 0).any() or self.offsets[0] < 0:
            raise ValueError("Segments: offsets must not be negative and must not decrease")
        self.offsets.flags.writeable = self.index.flags.writeable = False
        self.lo, self.hi = int(self.offsets[0]), int(self.offsets[-1])
        self.c = _lib.K82Segments(off=self.offsets.ctypes.data, index=self.index.ctypes.data, n=self.index.size)

    @classmethod
    def of_lengths(cls, lengths, index):
        return cls(np.concatenate([[0], np.cumsum(np.asarray(lengths, dtype=np.int64))]), index)


class Operators:
    """A handle of libk82.so for the operators alone (``k82_create`` without weights)."""

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
    def _stream(self):
        import torch
        # torch's default stream is handle 0, which the library takes for "the handle's own": name it hipStreamLegacy (1)
        return torch.cuda.current_stream(self.device).cuda_stream or 1

    def _on_gpu(self, **tensors):
        for name, t in tensors.items():
            if t is None:
                continue
            if not hasattr(t, "data_ptr"):
                raise TypeError(f"{name} must be a torch tensor on the GPU")
            if not t.is_cuda or t.get_device() != self.device:
                raise ValueError(f"{name} must be on cuda:{self.device}, it is on {t.device}")

    @staticmethod
    def _dtype(x, **others):
        import torch
        code = {torch.float32: 0, torch.bfloat16: 1}.get(x.dtype)
        if code is None:
            raise TypeError(f"float32 or bfloat16 tensors are needed, x is {x.dtype}")
        for name, t in others.items():
            if t is not None and t.dtype != x.dtype:
                raise TypeError(f"{name} is {t.dtype}, x is {x.dtype}")
        return code

    @staticmethod
    def _layout(rows_only=False, **tensors):
        """-> (layout, [ld of each tensor]) of [tokens, channels] tensors that share one layout."""
        rows, cols, lds = True, not rows_only, []
        for name, t in tensors.items():
            if t is None:
                continue
            if t.dim() != 2:
                raise ValueError(f"{name} must have two dimensions [tokens, channels], it has {t.dim()}")
            (n, c), (sn, sc) = t.shape, t.stride()
            rows &= (sc == 1 or c == 1) and (n <= 1 or sn >= c)
            cols &= (sn == 1 or n == 1) and (c <= 1 or sc >= n)
        if not rows and not cols:
            raise ValueError("tensors must share one layout: unit stride along the channels" + (
                "" if rows_only else " (or along the tokens: channel-first)") + " and rows that do not overlap")
        for t in tensors.values():
            if t is None:
                lds.append(0)
            elif rows:
                lds.append(t.stride(0) if t.shape[0] > 1 else max(1, t.shape[1]))
            else:
                lds.append(t.stride(1) if t.shape[1] > 1 else max(1, t.shape[0]))
        return (0 if rows else 1), lds

    @staticmethod
    def _like(name, t, shape):
        if t is not None and tuple(t.shape) != tuple(shape):
            raise ValueError(f"{name} has shape {tuple(t.shape)}, {tuple(shape)} is needed")

    @staticmethod
    def _contiguous(**tensors):
        for name, t in tensors.items():
            if t is not None and not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous")

    @staticmethod
    def _out(x, channels, cols, seg):
        """A new [tokens, channels] tensor in the layout of x; zero where no segment will write."""
        import torch
        n = x.shape[0]
        new = torch.empty if seg.lo == 0 and seg.hi == n else torch.zeros
        if cols:
            return new((channels, max(1, (n + 31) // 32 * 32)), dtype=x.dtype, device=x.device).t()[:n]
        return new((n, channels), dtype=x.dtype, device=x.device)

    @staticmethod
    def _segments(seg, n):
        if seg is None:
            seg = Segments([0, n], [0])
        elif not isinstance(seg, Segments):
            raise TypeError("seg must be a Segments (or None: every token uses index 0)")
        if seg.hi > n:
            raise ValueError(f"the segments end at token {seg.hi}, the tensors hold {n}")
        return seg

    def _factors(self, x, a, b, scale):
        import torch
        if a.dim() != 3 or b.dim() != 3:
            raise ValueError("a is [adapters, rank, cin] and b [adapters, cout, rank]")
        n, rank, cin = a.shape
        cout = b.shape[1]
        self._like("b", b, (n, cout, rank))
        self._like("scale", scale, (n,))
        if scale.dtype != torch.float32:
            raise TypeError(f"scale must be float32, it is {scale.dtype}")
        self._contiguous(a=a, b=b, scale=scale)
        self._like("x", x, (x.shape[0], cin))
        return n, rank, cin, cout

    # ------------------------------------------------------------------ low-rank adapters
    def op_lora(self, x, a, b, scale, seg=None, base=None, act="none", out=None, keep=False):
        """k82_op_lora: ``act(base + scale[k] * (x @ a[k].T) @ b[k].T)`` with ``k`` the adapter of the token's segment
        (-1: ``act(base)``).  ``base``: the shared projection's output, which ``out`` may be.  ``keep``: returns
        ``(y, h)`` with ``h = x @ a[k].T`` in float32, which ``op_lora_grad`` takes."""
        import torch
        self._on_gpu(x=x, a=a, b=b, scale=scale, base=base, out=out)
        if act not in ACTS:
            raise ValueError(f"act must be one of {sorted(ACTS)}, not {act!r}")
        dtype = self._dtype(x, a=a, b=b, base=base, out=out)
        layout, (ldx, ldbase, ldy) = self._layout(x=x, base=base, out=out)
        n, rank, cin, cout = self._factors(x, a, b, scale)
        tokens = x.shape[0]
        self._like("base", base, (tokens, cout))
        self._like("out", out, (tokens, cout))
        seg = self._segments(seg, tokens)
        if out is None:
            out = self._out(x, cout, layout, seg)
            ldy = out.stride(layout) if out.shape[layout] > 1 else max(1, out.shape[1 - layout])
        full = seg.lo == 0 and seg.hi == tokens
        h = (torch.empty if full else torch.zeros)((tokens, rank), dtype=torch.float32, device=x.device) if keep else None
        p = _lib.K82Lora(dtype, layout, ACTS[act], cin, cout, rank, n, tokens, x.data_ptr(), ldx,
                         None if base is None else base.data_ptr(), ldbase, out.data_ptr(), ldy, a.data_ptr(), b.data_ptr(),
                         scale.data_ptr(), None if h is None else h.data_ptr())
        self._check(self.lib.k82_op_lora(self.h, p, seg.c, self._stream()))
        return (out, h) if keep else out

    def op_lora_grad(self, x, dy, h, a, b, scale, seg=None, dx_base=None, dx=None):
        """k82_op_lora_grad -> ``(dx, da, db)``; ``dy`` is the gradient in front of the activation, ``h`` what
        ``op_lora(keep=True)`` returned, ``dx_base`` the shared projection's gradient (which ``dx`` may be).  ``da`` and
        ``db`` are float32 sums over the tokens in a fixed order, zero for an adapter without tokens."""
        import torch
        self._on_gpu(x=x, dy=dy, h=h, a=a, b=b, scale=scale, dx_base=dx_base, dx=dx)
        dtype = self._dtype(x, dy=dy, a=a, b=b, dx_base=dx_base, dx=dx)
        _, (ldx, lddy, ldbase, lddx) = self._layout(True, x=x, dy=dy, dx_base=dx_base, dx=dx)
        n, rank, cin, cout = self._factors(x, a, b, scale)
        tokens = x.shape[0]
        self._like("dy", dy, (tokens, cout))
        self._like("h", h, (tokens, rank))
        if h.dtype != torch.float32:
            raise TypeError(f"h must be float32, it is {h.dtype}")
        self._contiguous(h=h)
        self._like("dx_base", dx_base, (tokens, cin))
        self._like("dx", dx, (tokens, cin))
        seg = self._segments(seg, tokens)
        if dx is None:
            dx = self._out(x, cin, 0, seg)
            lddx = cin
        da = torch.empty((n, rank, cin), dtype=torch.float32, device=x.device)
        db = torch.empty((n, cout, rank), dtype=torch.float32, device=x.device)
        p = _lib.K82LoraGrad(dtype, cin, cout, rank, n, tokens, x.data_ptr(), ldx, dy.data_ptr(), lddy, h.data_ptr(),
                             None if dx_base is None else dx_base.data_ptr(), ldbase, dx.data_ptr(), lddx, a.data_ptr(),
                             b.data_ptr(), scale.data_ptr(), da.data_ptr(), db.data_ptr())
        self._with_workspace(self.lib.k82_op_lora_grad, self.lib.k82_op_lora_grad_workspace, p, seg, x)
        return dx, da, db

    # ------------------------------------------------------------------ layer norm
    def op_layernorm(self, x, gain, offset, seg=None, res=None, eps=1e-12, out=None, stats=False):
        """k82_op_layernorm: ``(z - mean) * rstd * gain[k] + offset[k]`` over the channels of ``z = x + res``, ``gain`` and
        ``offset`` ``[gains, channels]``, ``k`` the index of the token's segment.  ``out`` may be ``x`` or ``res``.
        ``stats``: returns ``(y, mean, rstd)`` (float32), which ``op_layernorm_grad`` takes."""
        import torch
        self._on_gpu(x=x, gain=gain, offset=offset, res=res, out=out)
        dtype = self._dtype(x, gain=gain, offset=offset, res=res, out=out)
        layout, (ldx, ldres, ldy) = self._layout(x=x, res=res, out=out)
        tokens, c = x.shape
        gains = gain.shape[0]
        self._like("gain", gain, (gains, c))
        self._like("offset", offset, (gains, c))
        self._contiguous(gain=gain, offset=offset)
        self._like("res", res, (tokens, c))
        self._like("out", out, (tokens, c))
        seg = self._segments(seg, tokens)
        if out is None:
            out = self._out(x, c, layout, seg)
            ldy = out.stride(layout) if out.shape[layout] > 1 else max(1, out.shape[1 - layout])
        mean = rstd = None
        if stats:
            new = torch.empty if seg.lo == 0 and seg.hi == tokens else torch.zeros
            mean, rstd = (new((tokens,), dtype=torch.float32, device=x.device) for _ in range(2))
        p = _lib.K82Layernorm(dtype, layout, c, gains, eps, tokens, x.data_ptr(), ldx,
                              None if res is None else res.data_ptr(), ldres, out.data_ptr(), ldy, gain.data_ptr(),
                              offset.data_ptr(), None if mean is None else mean.data_ptr(),
                              None if rstd is None else rstd.data_ptr())
        self._check(self.lib.k82_op_layernorm(self.h, p, seg.c, self._stream()))
        return (out, mean, rstd) if stats else out

    def op_layernorm_grad(self, x, dy, gain, mean, rstd, seg=None, res=None, dx=None):
        """k82_op_layernorm_grad -> ``(dx, dgain, doffset)``: ``dx`` is the gradient of ``x`` and of ``res`` alike and may be
        ``dy``, ``x`` or ``res`` itself; ``dgain`` and ``doffset`` are float32 sums over the tokens in a fixed order."""
        import torch
        self._on_gpu(x=x, dy=dy, gain=gain, mean=mean, rstd=rstd, res=res, dx=dx)
        dtype = self._dtype(x, dy=dy, gain=gain, res=res, dx=dx)
        _, (ldx, ldres, lddy, lddx) = self._layout(True, x=x, res=res, dy=dy, dx=dx)
        tokens, c = x.shape
        gains = gain.shape[0]
        self._like("gain", gain, (gains, c))
        self._like("dy", dy, (tokens, c))
        self._like("res", res, (tokens, c))
        self._like("dx", dx, (tokens, c))
        for name, t in (("mean", mean), ("rstd", rstd)):
            self._like(name, t, (tokens,))
            if t.dtype != torch.float32:
                raise TypeError(f"{name} must be float32, it is {t.dtype}")
        self._contiguous(gain=gain, mean=mean, rstd=rstd)
        seg = self._segments(seg, tokens)
        if dx is None:
            dx = self._out(x, c, 0, seg)
            lddx = c
        dgain = torch.empty((gains, c), dtype=torch.float32, device=x.device)
        doffset = torch.empty((gains, c), dtype=torch.float32, device=x.device)
        p = _lib.K82LayernormGrad(dtype, c, gains, tokens, x.data_ptr(), ldx, None if res is None else res.data_ptr(), ldres,
                                  dy.data_ptr(), lddy, dx.data_ptr(), lddx, gain.data_ptr(), mean.data_ptr(),
                                  rstd.data_ptr(), dgain.data_ptr(), doffset.data_ptr())
        self._with_workspace(self.lib.k82_op_layernorm_grad, self.lib.k82_op_layernorm_grad_workspace, p, seg, x)
        return dx, dgain, doffset

    def _with_workspace(self, call, size, p, seg, x):
        import torch
        need = size(p, seg.c)
        if need < 0:
            raise ValueError(f"k82 error {need}: {self.lib.k82_last_error(None).decode()}")
        ws = torch.empty((need,), dtype=torch.uint8, device=x.device) if need else None
        self._check(call(self.h, p, seg.c, None if ws is None else ws.data_ptr(), need, self._stream()))
