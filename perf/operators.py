"""Cases of the per-request operators: low-rank adapters beside a shared projection and layer norm with a gain and an
offset per request, forward and backward.

A batch is a packed axis of tokens cut into segments (one per sentence); ``index[s]`` names the adapter (or the pair of
gain and offset) of segment ``s``, -1 a sentence without an adapter.  ``own`` selects the framework's kernels."""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
_handles = {}


def listed():
    return [
        # the first token of a request that is alone on the GPU: nothing but latency
        {"name": "lora_token", "op": "lora", "dtype": "bf16", "layout": "rows", "tokens": 1, "segs": 1, "adapters": 1,
         "none": False, "cin": 768, "cout": 768, "rank": 8, "base": True, "act": "none", "keep": False},
        # one sentence in the engine's own layout (channels first), the feed-forward projection with its activation
        {"name": "lora_sentence", "op": "lora", "dtype": "f32", "layout": "cols", "tokens": 57, "segs": 1, "adapters": 1,
         "none": False, "cin": 768, "cout": 2048, "rank": 16, "base": True, "act": "gelu_new", "keep": False},
        # a scheduled batch of 64 sentences in the engine's layout, seven voices and sentences without an adapter
        {"name": "lora_batch_cols", "op": "lora", "dtype": "f32", "layout": "cols", "tokens": 16411, "segs": 64,
         "adapters": 7, "none": True, "cin": 768, "cout": 768, "rank": 16, "base": True, "act": "none", "keep": False},
        # the same batch as a training program holds it: token rows in 16 bits, and h kept for the backward pass
        {"name": "lora_batch_rows", "op": "lora", "dtype": "bf16", "layout": "rows", "tokens": 16411, "segs": 64,
         "adapters": 7, "none": True, "cin": 768, "cout": 2048, "rank": 16, "base": True, "act": "none", "keep": True},
        # a book's worth of sentences with large adapters
        {"name": "lora_book", "op": "lora", "dtype": "bf16", "layout": "rows", "tokens": 65536, "segs": 128, "adapters": 8,
         "none": False, "cin": 2048, "cout": 768, "rank": 64, "base": True, "act": "none", "keep": False},
        # a training step on one short sentence, an odd rank
        {"name": "lora_grad_sentence", "op": "lora_grad", "dtype": "f32", "layout": "rows", "tokens": 211, "segs": 1,
         "adapters": 1, "none": False, "cin": 768, "cout": 768, "rank": 7, "base": True},
        # a training step on a book's worth of sentences, eight adapters at once
        {"name": "lora_grad_book", "op": "lora_grad", "dtype": "bf16", "layout": "rows", "tokens": 65536, "segs": 128,
         "adapters": 8, "none": False, "cin": 768, "cout": 2048, "rank": 16, "base": True},
        # one token: latency
        {"name": "layernorm_token", "op": "layernorm", "dtype": "f32", "layout": "rows", "tokens": 1, "segs": 1, "gains": 1,
         "c": 768, "res": True, "stats": False},
        # the scheduled batch in the engine's layout, each sentence with its voice's gain and offset
        {"name": "layernorm_batch_cols", "op": "layernorm", "dtype": "f32", "layout": "cols", "tokens": 16411, "segs": 64,
         "gains": 8, "c": 768, "res": True, "stats": False},
        # a training forward pass over a book's worth of sentences
        {"name": "layernorm_book", "op": "layernorm", "dtype": "bf16", "layout": "rows", "tokens": 131072, "segs": 128,
         "gains": 8, "c": 768, "res": True, "stats": True},
        # a training step on one short sentence, an odd width
        {"name": "layernorm_grad_sentence", "op": "layernorm_grad", "dtype": "f32", "layout": "rows", "tokens": 97,
         "segs": 1, "gains": 1, "c": 513, "res": False},
        # the backward pass of the book
        {"name": "layernorm_grad_book", "op": "layernorm_grad", "dtype": "bf16", "layout": "rows", "tokens": 131072,
         "segs": 128, "gains": 8, "c": 768, "res": True},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["lora", "lora", "lora_grad", "layernorm", "layernorm_grad"])
    case = {"op": op, "dtype": rng.choice(["f32", "bf16"]), "layout": "rows"}
    if op in ("lora", "layernorm") and case["dtype"] == "f32" and rng.random() < 0.5:
        case["layout"] = "cols"
    size = 4 if case["dtype"] == "f32" else 2
    if op.startswith("lora"):
        cin, cout, rank = _log_int(rng, 64, 2560), _log_int(rng, 64, 2560), _log_int(rng, 1, 64)
        most = int(min(2.4e8 / (size * (cin + 2 * cout)), 5.0e9 / (rank * (cin + cout))))
        tokens = _log_int(rng, 1, max(16, min(65536, most)))
        case.update(tokens=tokens, segs=_log_int(rng, 1, min(128, tokens)), adapters=rng.randint(1, 8),
                    none=rng.random() < 0.4, cin=cin, cout=cout, rank=rank, base=rng.random() < 0.8)
        if op == "lora":
            case.update(act=rng.choice(["none", "none", "gelu_new"]), keep=rng.random() < 0.3)
    else:
        c = _log_int(rng, 64, 4096)
        tokens = _log_int(rng, 1, max(16, min(131072, int(2.0e8 / (size * c)))))
        case.update(tokens=tokens, segs=_log_int(rng, 1, min(128, tokens)), gains=rng.randint(1, 8), c=c,
                    res=rng.random() < 0.6)
        if op == "layernorm":
            case.update(stats=rng.random() < 0.5)
    return case


def _segments(case):
    """(offsets int64[segs + 1], index int32[segs]) of a case, the same for every seed: ragged sentences."""
    r = np.random.RandomState(case["tokens"] * 131 + case["segs"])
    weight = np.exp(0.6 * r.standard_normal(case["segs"]))
    ends = np.floor(np.cumsum(weight) / weight.sum() * case["tokens"]).astype(np.int64)
    ends[-1] = case["tokens"]
    off = np.concatenate([[0], ends]).astype(np.int64)
    if case["op"].startswith("lora"):
        lo = -1 if case["none"] and case["segs"] > 1 else 0
        index = (lo + np.arange(case["segs"]) % (case["adapters"] - lo)).astype(np.int32)
    else:
        index = (np.arange(case["segs"]) % case["gains"]).astype(np.int32)
    return off, index


def _tensors(case, seed):
    """The inputs alone, on the GPU, from the seed."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 7919 + 17)
    dt = DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def tokens_by(n, spread=1.0, centre=0.0, shift=0.0):
        # activations of unit variance with a few loud channels; centre: a mean of its own for each channel
        loud = torch.where(torch.rand(n, generator=g, device="cuda") < 0.02, 4.0, 1.0)
        v = randn(case["tokens"], n) * (loud * spread) + centre * randn(n) + shift
        if case["layout"] == "cols":  # channels first, rows padded to 32 positions
            pitch = (case["tokens"] + 31) // 32 * 32
            buf = torch.zeros(n, pitch, device="cuda", dtype=dt)
            buf[:, :case["tokens"]] = v.t()
            return buf.t()[:case["tokens"]]
        return v.to(dt)

    off, index = _segments(case)
    t = {"of_token": torch.from_numpy(np.repeat(index, np.diff(off)).astype(np.int64)).cuda()}
    if case["op"].startswith("lora"):
        n, r, cin, cout = case["adapters"], case["rank"], case["cin"], case["cout"]
        t["x"] = tokens_by(cin)
        t["a"] = ((torch.rand(n, r, cin, generator=g, device="cuda") * 2 - 1) * math.sqrt(3.0 / cin)).to(dt)
        t["b"] = (randn(n, cout, r) * (0.5 / math.sqrt(r))).to(dt)
        t["scale"] = 0.5 + 1.5 * torch.rand(n, generator=g, device="cuda")
        if case["op"] == "lora":
            t["base"] = tokens_by(cout) if case["base"] else None
        else:
            t["dy"] = tokens_by(cout, 1e-2)
            t["dx_base"] = tokens_by(cin, 1e-2) if case["base"] else None
            # what the forward pass kept
            t["h"] = _select(dict(case, **t), t["x"].float() @ _flat_a(dict(case, **t)).t()).sum(1)
    else:
        n, c = case["gains"], case["c"]
        t["x"] = tokens_by(c, 1.0, 0.5, 0.25)
        t["res"] = tokens_by(c, 1.0, 0.5) if case["res"] else None
        t["gain"] = (1.0 + 0.2 * randn(n, c)).to(dt)
        t["offset"] = (0.1 * randn(n, c)).to(dt)
        if case["op"] == "layernorm_grad":
            t["dy"] = tokens_by(c, 1e-2)
            t["mean"], t["rstd"] = _moments(dict(case, **t))[1:]
    return t


def _eps(case):
    return 1e-12 if case["dtype"] == "f32" else 1e-5


def prepare(case, seed):
    state = dict(case, **_tensors(case, seed))
    if own:
        from tts_amd import Operators, Segments
        if "ops" not in _handles:
            _handles["ops"] = Operators(device=0)
        state["ops"] = _handles["ops"]
        state["seg"] = Segments(*_segments(case))
    return state


def run(state):
    return _own(state) if own else _plain(state)


def _own(s):
    ops = s["ops"]
    if s["op"] == "lora":
        r = ops.op_lora(s["x"], s["a"], s["b"], s["scale"], s["seg"], base=s["base"], act=s["act"], keep=s["keep"])
        return list(r) if s["keep"] else [r]
    if s["op"] == "lora_grad":
        return list(ops.op_lora_grad(s["x"], s["dy"], s["h"], s["a"], s["b"], s["scale"], s["seg"], dx_base=s["dx_base"]))
    if s["op"] == "layernorm":
        r = ops.op_layernorm(s["x"], s["gain"], s["offset"], s["seg"], res=s["res"], eps=_eps(s), stats=s["stats"])
        return list(r) if s["stats"] else [r]
    return list(ops.op_layernorm_grad(s["x"], s["dy"], s["gain"], s["mean"], s["rstd"], s["seg"], res=s["res"]))


def _flat_a(s):
    return s["a"].float().reshape(-1, s["cin"])


def _flat_b(s):
    return s["b"].float().transpose(1, 2).reshape(-1, s["cout"])


def _select(s, v):
    """[tokens, adapters * rank] -> [tokens, adapters, rank] with everything but the token's own adapter at zero."""
    mine = s["of_token"][:, None] == torch.arange(s["adapters"], device=v.device)
    return v.view(-1, s["adapters"], s["rank"]) * mine[:, :, None]


def _moments(s):
    z = s["x"].float()
    if s["res"] is not None:
        z = z + s["res"].float()
    mean = z.mean(1)
    d = z - mean[:, None]
    return d, mean, (d.square().mean(1) + _eps(s)).rsqrt()


def _plain(s):
    dt = DTYPES[s["dtype"]]
    if s["op"] == "lora":
        h = _select(s, s["x"].float() @ _flat_a(s).t())
        y = (h * s["scale"][:, None]).reshape(s["tokens"], -1) @ _flat_b(s)
        if s["base"] is not None:
            y = y + s["base"].float()
        if s["act"] == "gelu_new":
            y = 0.5 * y * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (y + 0.044715 * y * y * y)))
        return [y.to(dt), h.sum(1)] if s["keep"] else [y.to(dt)]
    if s["op"] == "lora_grad":
        n, r = s["adapters"], s["rank"]
        dy = s["dy"].float()
        g = (_select(s, dy @ _flat_b(s).t()) * s["scale"][:, None]).reshape(s["tokens"], -1)
        dx = g @ _flat_a(s)
        if s["dx_base"] is not None:
            dx = dx + s["dx_base"].float()
        h = (_select(s, s["h"].repeat(1, n)) * s["scale"][:, None]).reshape(s["tokens"], -1)
        da = (g.t() @ s["x"].float()).view(n, r, -1)
        db = (dy.t() @ h).view(-1, n, r).transpose(0, 1).contiguous()
        return [dx.to(dt), da, db]
    if s["op"] == "layernorm":
        d, mean, rstd = _moments(s)
        gain, offset = s["gain"].float()[s["of_token"]], s["offset"].float()[s["of_token"]]
        y = (d * rstd[:, None] * gain + offset).to(dt)
        return [y, mean, rstd] if s["stats"] else [y]
    z, dy = s["x"].float(), s["dy"].float()
    if s["res"] is not None:
        z = z + s["res"].float()
    xh = (z - s["mean"][:, None]) * s["rstd"][:, None]
    u = dy * s["gain"].float()[s["of_token"]]
    dx = s["rstd"][:, None] * (u - u.mean(1, keepdim=True) - xh * (u * xh).mean(1, keepdim=True))
    mine = (s["of_token"][None, :] == torch.arange(s["gains"], device=z.device)[:, None]).float()
    return [dx.to(dt), mine @ (dy * xh), mine @ dy]


def work(case):
    off, index = _segments(case)
    size = 4 if case["dtype"] == "f32" else 2
    tokens = case["tokens"]
    length = np.diff(off)
    if case["op"].startswith("lora"):
        with_one = int(length[index >= 0].sum())
        used = len(set(index[(index >= 0) & (length > 0)].tolist()))
        r, cin, cout = case["rank"], case["cin"], case["cout"]
        factors = used * r * (cin + cout)
        if case["op"] == "lora":
            nbytes = size * (with_one * cin + tokens * cout * (2 if case["base"] else 1) + factors)
            nbytes += 4 * tokens * r if case["keep"] else 0
            return {"bytes": nbytes, "flops": 2 * with_one * r * (cin + cout)}
        nbytes = size * (with_one * (cin + cout) + tokens * cin * (2 if case["base"] else 1) + factors)
        return {"bytes": nbytes + 4 * (with_one * r + case["adapters"] * r * (cin + cout)),
                "flops": 4 * with_one * r * (cin + cout)}
    c, used = case["c"], len(set(index[length > 0].tolist()))
    if case["op"] == "layernorm":
        nbytes = size * (tokens * c * (3 if case["res"] else 2) + 2 * used * c) + (8 * tokens if case["stats"] else 0)
        return {"bytes": nbytes, "flops": 8 * tokens * c}
    nbytes = size * (tokens * c * (4 if case["res"] else 3) + used * c) + 8 * tokens + 8 * case["gains"] * c
    return {"bytes": nbytes, "flops": 14 * tokens * c}


def exact(case, seed):
    """The definition in 64 bits, segment by segment."""
    t = {k: v.double() if v is not None else None for k, v in _tensors(case, seed).items() if k != "of_token"}
    off, index = _segments(case)
    spans = [(int(off[i]), int(off[i + 1]), int(k)) for i, k in enumerate(index)]
    x = t["x"]
    if case["op"] == "lora":
        y = t["base"].clone() if t["base"] is not None else x.new_zeros(case["tokens"], case["cout"])
        kept = x.new_zeros(case["tokens"], case["rank"])
        for lo, hi, k in spans:
            if k >= 0:
                kept[lo:hi] = torch.mm(x[lo:hi].contiguous(), t["a"][k].t().contiguous())
                y[lo:hi] += t["scale"][k] * torch.mm(kept[lo:hi], t["b"][k].t().contiguous())
        if case["act"] == "gelu_new":
            y = y / (1.0 + torch.exp(-2.0 * math.sqrt(2.0 / math.pi) * (y + 0.044715 * y ** 3)))
        return [y, kept] if case["keep"] else [y]
    if case["op"] == "lora_grad":
        dy = t["dy"]
        dx = t["dx_base"].clone() if t["dx_base"] is not None else torch.zeros_like(x)
        da, db = torch.zeros_like(t["a"]), torch.zeros_like(t["b"])
        for lo, hi, k in spans:
            if k >= 0:
                g = t["scale"][k] * torch.mm(dy[lo:hi], t["b"][k])
                dx[lo:hi] += torch.mm(g, t["a"][k])
                da[k] += torch.mm(g.t().contiguous(), x[lo:hi])
                db[k] += t["scale"][k] * torch.mm(dy[lo:hi].t().contiguous(), t["h"][lo:hi])
        return [dx, da, db]
    z = x if t["res"] is None else x + t["res"]
    if case["op"] == "layernorm":
        mean = z.sum(1) / case["c"]
        rstd = 1.0 / torch.sqrt(((z - mean[:, None]) ** 2).sum(1) / case["c"] + _eps(case))
    else:
        mean, rstd = t["mean"], t["rstd"]
    xh = (z - mean[:, None]) * rstd[:, None]
    if case["op"] == "layernorm":
        y = torch.empty_like(z)
        for lo, hi, k in spans:
            y[lo:hi] = xh[lo:hi] * t["gain"][k] + t["offset"][k]
        return [y, mean, rstd] if case["stats"] else [y]
    dy = t["dy"]
    dx, dgain, doffset = torch.empty_like(z), torch.zeros_like(t["gain"]), torch.zeros_like(t["offset"])
    for lo, hi, k in spans:
        u = dy[lo:hi] * t["gain"][k]
        inner = (u * xh[lo:hi]).sum(1, keepdim=True) / case["c"]
        dx[lo:hi] = rstd[lo:hi, None] * (u - u.sum(1, keepdim=True) / case["c"] - xh[lo:hi] * inner)
        dgain[k] += (dy[lo:hi] * xh[lo:hi]).sum(0)
        doffset[k] += dy[lo:hi].sum(0)
    return [dx, dgain, doffset]
