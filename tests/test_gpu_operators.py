"""The operators on caller-owned tensors against their definitions in 64 bits.

Tolerances are sums of roundings.  u = 2^-23 bounds one 32-bit operation (a matrix instruction's internal addition may
truncate, hence a whole step and not half of one); a sum of n terms in any order is off by at most n u times the sum of the
terms' magnitudes.  A 16-bit result adds half a step, 2^-8 of its value.  What feeds a matrix product in two 16-bit parts is
off by 2^-8 * 2^-8 = 2^-16 of its value, in three by 2^-24."""
import threading

import numpy as np
import pytest
import torch

from tts_amd import Operators, Segments

pytestmark = pytest.mark.gpu

U = 2.0 ** -23
SPLIT = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -16}
STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
TYPES = [torch.float32, torch.bfloat16]
SENTINEL = 7.25


@pytest.fixture(scope="module")
def ops():
    o = Operators()
    yield o
    o.close()
    torch.cuda.empty_cache()                                 # later tests reserve most of the GPU for the engine


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return lambda *s: torch.randn(*s, generator=g, device="cuda")


def tensor(randn, tokens, c, dt, kind="dense", scale=1.0):
    """[tokens, c]: dense rows, a column range of wider rows at an odd place, or channel-first with padded rows."""
    v = (randn(tokens, c) * scale).to(dt)
    if kind == "slice":
        buf = torch.full((tokens, c + 5), float("nan"), device="cuda", dtype=dt)
        buf[:, 3:3 + c] = v
        return buf[:, 3:3 + c]
    if kind == "cols":
        buf = torch.full((c, (tokens + 31) // 32 * 32 + 1), float("nan"), device="cuda", dtype=dt)
        buf[:, 1:1 + tokens] = v.t()
        return buf.t()[1:1 + tokens]
    return v


def like(t):
    """An output of t's shape and strides, every element (also between the rows) a sentinel."""
    if t.stride(1) == 1:
        ld = max(t.stride(0), t.shape[1]) if t.shape[0] > 1 else t.shape[1]
        buf = torch.full((t.shape[0] + 1, ld), SENTINEL, device="cuda", dtype=t.dtype)
        return buf[:t.shape[0], :t.shape[1]], buf
    buf = torch.full((t.shape[1] + 1, t.stride(1)), SENTINEL, device="cuda", dtype=t.dtype)
    return buf.t()[:t.shape[0], :t.shape[1]], buf


def untouched(buf, view):
    """Nothing of buf outside view was written."""
    probe = buf.clone()
    probe.as_strided(view.shape, view.stride(), view.storage_offset()).fill_(SENTINEL)
    assert (probe == SENTINEL).all()


def spans(seg):
    return [(int(a), int(b), int(k)) for a, b, k in zip(seg.offsets[:-1], seg.offsets[1:], seg.index) if b > a]


def cut(tokens, n, adapters, seed=0, none=False, lo=0, hi=None):
    r = np.random.default_rng(seed)
    hi = tokens if hi is None else hi
    inner = np.sort(r.integers(lo, hi + 1, n - 1)) if n > 1 else np.zeros(0, np.int64)
    return Segments(np.concatenate([[lo], inner, [hi]]), r.integers(-1 if none else 0, adapters, n))


def within(got, want, bound, what):
    got, want, bound = got.double(), want.double(), bound.double()
    assert torch.isfinite(got).all(), what
    bad = (got - want).abs() - bound
    assert bad.max() <= 0, (what, float((got - want).abs().max()), float(bad.max()), int((bad > 0).sum()))


def poison(nbytes):
    """Leaves NaN in the allocator's block of this size: what a workspace is made of holds no zeros by luck."""
    t = torch.full((max(1, nbytes // 4 + 64),), float("nan"), device="cuda")
    del t


# ---------------------------------------------------------------------------------------------- low-rank adapters
def lora_case(tokens, cin, cout, rank, adapters, dt, kind, seed):
    randn = gen(seed)
    x = tensor(randn, tokens, cin, dt, kind)
    base = tensor(randn, tokens, cout, dt, kind)
    a = (randn(adapters, rank, cin) / max(1, cin) ** 0.5).to(dt)
    b = (randn(adapters, cout, rank) / rank ** 0.5).to(dt)
    scale = 0.5 + torch.rand(adapters, device="cuda")
    return x, base, a, b, scale


def lora_want(x, base, a, b, scale, seg, act):
    """(y, bound of y, h, bound of h) in 64 bits."""
    dt, (tokens, cin), cout, rank = x.dtype, x.shape, b.shape[1], a.shape[1]
    x, a, b, s = x.double(), a.double(), b.double(), scale.double()
    y = torch.zeros(tokens, cout, device="cuda", dtype=torch.float64) if base is None else base.double().clone()
    mag = y.abs()
    h, hm = (torch.zeros(tokens, rank, device="cuda", dtype=torch.float64) for _ in range(2))
    for lo, hi, k in spans(seg):
        if k >= 0:
            h[lo:hi], hm[lo:hi] = x[lo:hi] @ a[k].t(), x[lo:hi].abs() @ a[k].abs().t()
            y[lo:hi] += s[k] * (h[lo:hi] @ b[k].t())
            mag[lo:hi] += s[k] * (hm[lo:hi] @ b[k].abs().t())
    bound = ((cin + rank + 8) * U + SPLIT[dt]) * mag
    if act == "gelu_new":
        # |gelu'| < 1.2; the tanh and the four operations around it: a few units of the argument's magnitude
        bound = 1.2 * bound + 8 * U * y.abs()
        y = 0.5 * y * (1 + torch.tanh((2 / np.pi) ** 0.5 * (y + 0.044715 * y ** 3)))
    return y, bound * (1 + STEP[dt]) + STEP[dt] * y.abs() + 1e-38, h, (cin + 4) * U * hm


def check_lora(ops, tokens, cin, cout, rank, adapters, dt, kind, seg, act="none", with_base=True, keep=True, seed=1):
    x, base, a, b, scale = lora_case(tokens, cin, cout, rank, adapters, dt, kind, seed)
    want, bound, h_want, h_bound = lora_want(x, base if with_base else None, a, b, scale, seg, act)
    out, buf = like(base)
    r = ops.op_lora(x, a, b, scale, seg, base=base if with_base else None, act=act, out=out, keep=keep)
    y, h = r if keep else (r, None)
    assert y.data_ptr() == out.data_ptr()
    lo, hi = seg.lo, seg.hi
    what = (tokens, cin, cout, rank, adapters, dt, kind, act)
    if hi > lo:
        within(y[lo:hi], want[lo:hi], bound[lo:hi], what)
        if keep:
            within(h[lo:hi], h_want[lo:hi], h_bound[lo:hi] + 1e-38, what)
    untouched(buf, out[lo:hi])
    return y


@pytest.mark.parametrize("dt,kind", [(torch.float32, "dense"), (torch.float32, "slice"), (torch.float32, "cols"),
                                     (torch.bfloat16, "dense"), (torch.bfloat16, "slice")])
@pytest.mark.parametrize("tokens,cin,cout,rank,adapters,segs", [
    (1, 1, 1, 1, 1, 1), (1, 768, 768, 8, 1, 1), (2, 5, 3, 3, 2, 2), (17, 33, 130, 16, 3, 4), (63, 129, 65, 17, 2, 3),
    (64, 64, 64, 64, 1, 1), (65, 768, 2048, 16, 4, 7), (257, 200, 96, 128, 2, 5), (100, 31, 700, 5, 5, 40),
    (300, 96, 40, 7, 6, 290), (1500, 260, 513, 33, 3, 11), (5000, 64, 100, 4, 2, 3),
])
def test_lora_forward(ops, dt, kind, tokens, cin, cout, rank, adapters, segs):
    seg = cut(tokens, segs, adapters, seed=tokens, none=segs > 1)
    check_lora(ops, tokens, cin, cout, rank, adapters, dt, kind, seg, act="gelu_new" if cin % 2 else "none")


@pytest.mark.parametrize("dt,kind", [(torch.float32, "dense"), (torch.float32, "cols"), (torch.bfloat16, "dense")])
def test_lora_rows_without_a_segment_stay_as_they_were(ops, dt, kind):
    for lo, hi in ((0, 50), (7, 61), (64, 64), (0, 0), (33, 64)):
        seg = cut(64, 4, 2, seed=lo, none=True, lo=lo, hi=hi)
        check_lora(ops, 64, 48, 80, 8, 2, dt, kind, seg, keep=False)
    check_lora(ops, 64, 48, 80, 8, 2, dt, kind, Segments([0], []), keep=False)
    # the same adapter named again and again, empty segments between, no base, no adapter at all
    seg = Segments([0, 9, 9, 20, 20, 21, 64], [1, 0, 1, 1, -1, 1])
    check_lora(ops, 64, 48, 80, 8, 2, dt, kind, seg, with_base=False)
    check_lora(ops, 64, 48, 80, 8, 2, dt, kind, Segments([0, 64], [-1]), act="gelu_new")
    check_lora(ops, 64, 48, 80, 8, 2, dt, kind, Segments([0, 64], [-1]), with_base=False)


@pytest.mark.parametrize("dt,kind", [(torch.float32, "dense"), (torch.float32, "cols"), (torch.bfloat16, "dense")])
def test_lora_values_that_are_not_numbers_stay_in_their_token(ops, dt, kind):
    x, base, a, b, scale = lora_case(70, 40, 50, 6, 2, dt, kind, 3)
    seg = Segments([0, 21, 50, 66], [0, -1, 1])
    clean = ops.op_lora(x, a, b, scale, seg, base=base).clone()
    for t, v in ((5, float("nan")), (30, float("inf")), (60, -float("inf")), (68, float("nan"))):
        x[t] = v
    a_other = a.clone()
    got = ops.op_lora(x, a_other, b, scale, seg, base=base)
    hit = torch.zeros(70, dtype=torch.bool, device="cuda")
    hit[[5, 60]] = True                       # token 30 has no adapter: its x is not looked at; 68 is in no segment
    assert torch.equal(got[:66][~hit[:66]], clean[:66][~hit[:66]])
    assert not torch.isfinite(got[5]).any() and not torch.isfinite(got[60]).any()
    assert (got[66:] == 0).all()
    # an adapter that nobody uses may hold anything
    a_other[1] = float("nan")
    only = Segments([0, 5], [0])
    assert torch.equal(ops.op_lora(x, a_other, b, scale, only, base=base)[:5], clean[:5])


@pytest.mark.parametrize("dt,kind", [(torch.float32, "dense"), (torch.float32, "cols"), (torch.bfloat16, "dense")])
def test_infinities_come_through(ops, dt, kind):
    """One rank, so no two infinities meet: the result is the definition's, sign by sign, and the gradient's too.

    A factor's gradient in bf16 takes g and h in three parts.  An infinity of x or dy times parts of both signs is
    inf - inf, so there, and there alone, a NaN may stand for the infinity; it is never a finite number."""
    x, base, a, b, scale = lora_case(37, 64, 72, 1, 2, dt, kind, 91)
    x[5, 9], x[20, 40] = float("inf"), -float("inf")
    base[7, 3] = float("inf")
    seg = Segments([0, 18, 37], [1, 0])
    want = lora_want(x, base, a, b, scale, seg, "none")[0]
    y, h = ops.op_lora(x, a, b, scale, seg, base=base, keep=True)
    bad = ~torch.isfinite(want)
    assert bad[5].all() and bad[20].all() and torch.equal(bad, ~torch.isfinite(y)) and torch.equal(y[bad].double(), want[bad])
    if kind == "cols":
        return
    x, dy, a, b, scale = lora_case(37, 64, 72, 1, 2, dt, kind, 92)
    _, h = ops.op_lora(x, a, b, scale, seg, keep=True)
    dy[5, 9], h[30] = float("inf"), -float("inf")
    got = ops.op_lora_grad(x, dy, h, a, b, scale, seg)
    for name, g, (w, _) in zip(("dx", "da", "db"), got, lora_grad_want(x, dy, h, None, a, b, scale, seg)):
        bad = ~torch.isfinite(w)
        assert bad.any() and torch.equal(bad, ~torch.isfinite(g))
        if dt == torch.bfloat16 and name == "db":
            bad[1, 9] = False
        assert torch.equal(g[bad].double().nan_to_num(nan=7.0), w[bad].nan_to_num(nan=7.0))


@pytest.mark.parametrize("dt", TYPES)
def test_lora_into_the_shared_projections_own_buffer(ops, dt):
    x, base, a, b, scale = lora_case(90, 72, 136, 12, 3, dt, "dense", 4)
    seg = cut(90, 6, 3, 5, none=True)
    want = ops.op_lora(x, a, b, scale, seg, base=base)
    y = base.clone()
    assert ops.op_lora(x, a, b, scale, seg, base=y, out=y) is y
    assert torch.equal(y, want)
    # x and y as column ranges of one buffer
    buf = torch.cat([x, base], 1)
    ops.op_lora(buf[:, :72], a, b, scale, seg, base=buf[:, 72:], out=buf[:, 72:])
    assert torch.equal(buf[:, 72:], want) and torch.equal(buf[:, :72], x)
    with pytest.raises(ValueError, match="overlap"):
        ops.op_lora(x, a, b[:, :72].contiguous(), scale, seg, base=x, out=x)


def test_lora_of_a_token_does_not_depend_on_its_batch(ops):
    """A sentence alone and among others: the same bits (the engine promises that of its batches)."""
    for dt, kind in ((torch.float32, "cols"), (torch.float32, "dense"), (torch.bfloat16, "dense")):
        x, base, a, b, scale = lora_case(400, 768, 256, 16, 4, dt, kind, 6)
        seg = Segments([0, 57, 190, 230, 400], [2, 0, -1, 3])
        whole = ops.op_lora(x, a, b, scale, seg, base=base)
        alone = ops.op_lora(x[57:190], a, b, scale, Segments([0, 133], [0]), base=base[57:190])
        assert torch.equal(whole[57:190], alone)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("rank,cin,cout", [(33, 72, 40), (64, 64, 136), (128, 200, 24), (100, 37, 51)])
def test_lora_of_many_tokens_takes_larger_tiles(ops, dt, rank, cin, cout):
    """From 32768 tokens on: the definition, and the bits of the same tokens in a small call."""
    tokens, seg = 33001, Segments([0, 5, 100, 20063, 33001], [2, 0, -1, 1])
    check_lora(ops, tokens, cin, cout, rank, 3, dt, "dense", seg, seed=rank)
    x, base, a, b, scale = lora_case(tokens, cin, cout, rank, 3, dt, "dense", 17)
    y, h = ops.op_lora(x, a, b, scale, seg, base=base, keep=True)
    for lo, hi, k in ((5, 100, 0), (20063, 20200, 1), (32950, 33001, 1)):
        alone = ops.op_lora(x[lo:hi], a, b, scale, Segments([0, hi - lo], [k]), base=base[lo:hi], keep=True)
        assert torch.equal(alone[0], y[lo:hi]) and torch.equal(alone[1], h[lo:hi])


def lora_grad_want(x, dy, h, dx_base, a, b, scale, seg):
    dt = x.dtype
    (tokens, cin), cout, rank = x.shape, dy.shape[1], a.shape[1]
    x, dy, h, a, b, s = x.double(), dy.double(), h.double(), a.double(), b.double(), scale.double()
    dx = torch.zeros_like(x) if dx_base is None else dx_base.double().clone()
    dxm, da, dam, db, dbm = dx.abs(), *(torch.zeros_like(v) for v in (a, a, b, b))
    count = torch.zeros(a.shape[0], device="cuda", dtype=torch.float64)
    for lo, hi, k in spans(seg):
        if k < 0:
            continue
        g, gm = s[k] * (dy[lo:hi] @ b[k]), s[k] * (dy[lo:hi].abs() @ b[k].abs())
        dx[lo:hi] += g @ a[k]
        dxm[lo:hi] += gm @ a[k].abs()
        da[k] += g.t() @ x[lo:hi]
        dam[k] += gm.t() @ x[lo:hi].abs()
        db[k] += s[k] * (dy[lo:hi].t() @ h[lo:hi])
        dbm[k] += s[k] * (dy[lo:hi].abs().t() @ h[lo:hi].abs())
        count[k] += hi - lo
    n = count[:, None, None]
    split3 = 2.0 ** -24 if dt == torch.bfloat16 else 0.0
    return [(dx, ((cout + rank + 8) * U + SPLIT[dt]) * dxm * (1 + STEP[dt]) + STEP[dt] * dx.abs() + 1e-38),
            (da, ((n + cout + 8) * U + split3) * dam), (db, ((n + 8) * U + split3) * dbm)]


@pytest.mark.parametrize("dt,kind", [(torch.float32, "dense"), (torch.float32, "slice"), (torch.bfloat16, "dense"), (torch.bfloat16, "slice")])
@pytest.mark.parametrize("tokens,cin,cout,rank,adapters,segs", [
    (1, 1, 1, 1, 1, 1), (2, 5, 3, 3, 2, 2), (17, 33, 130, 16, 3, 4), (63, 129, 65, 17, 2, 3), (64, 64, 64, 64, 1, 1),
    (211, 768, 768, 7, 1, 1), (257, 200, 96, 128, 2, 5), (300, 96, 40, 7, 6, 290), (3000, 260, 513, 33, 3, 11),
    (9000, 64, 100, 4, 2, 3), (700, 140, 70, 8, 400, 500),
])
def test_lora_backward(ops, dt, kind, tokens, cin, cout, rank, adapters, segs):
    x, dy, a, b, scale = lora_case(tokens, cin, cout, rank, adapters, dt, kind, tokens + 1)
    randn = gen(9)
    seg = cut(tokens, segs, adapters, seed=tokens, none=segs > 1)
    _, h = ops.op_lora(x, a, b, scale, seg, keep=True)
    for base in (None, tensor(randn, tokens, cin, dt, kind)):
        dx, buf = like(x)
        poison(tokens * rank * 16)
        got = ops.op_lora_grad(x, dy, h, a, b, scale, seg, dx_base=base, dx=dx)
        for g, (w, bound), name in zip(got, lora_grad_want(x, dy, h, base, a, b, scale, seg), ("dx", "da", "db")):
            within(g, w, bound + 1e-38, (name, tokens, cin, cout, rank, dt, kind))
        untouched(buf, dx)
        again = ops.op_lora_grad(x, dy, h, a, b, scale, seg, dx_base=base)
        for g, w in zip(got, again):
            assert torch.equal(g, w)                         # fixed order of every sum


@pytest.mark.parametrize("dt", TYPES)
def test_lora_backward_leaves_and_zeroes_what_it_should(ops, dt):
    x, dy, a, b, scale = lora_case(60, 40, 50, 6, 4, dt, "dense", 11)
    seg = Segments([5, 20, 20, 33, 44], [2, 3, -1, 2])
    # NaN and infinities in rows that no segment holds, in h of sentences without an adapter, in unused adapters
    _, h = ops.op_lora(x, a, b, scale, seg, keep=True)
    want = lora_grad_want(x, dy, h, None, a, b, scale, seg)
    for t in (0, 4, 25, 44, 59):
        x[t] = float("nan")
        dy[t] = float("inf")
        h[t] = float("nan")
    a[0], b[1], scale[3] = float("nan"), float("nan"), float("inf")
    dx = torch.full_like(x, SENTINEL)
    _, da, db = ops.op_lora_grad(x, dy, h, a, b, scale, seg, dx=dx)
    within(dx[5:44], want[0][0][5:44], want[0][1][5:44], "dx")
    assert (dx[:5] == SENTINEL).all() and (dx[44:] == SENTINEL).all() and (dx[20:33] == 0).all()
    within(da[2], want[1][0][2], want[1][1][2] + 1e-38, "da")
    within(db[2], want[2][0][2], want[2][1][2] + 1e-38, "db")
    for k in (0, 1, 3):
        assert (da[k] == 0).all() and (db[k] == 0).all()
    # no segments at all
    dx, da, db = ops.op_lora_grad(x, dy, h, a, b, scale, Segments([0], []))
    assert (da == 0).all() and (db == 0).all()


def test_lora_gradients_against_differences(ops):
    """The forward pass is linear in x, in a and in b: differences over a whole step are exact up to rounding."""
    x, dy, a, b, scale = lora_case(130, 48, 56, 5, 3, torch.float32, "dense", 12)
    seg = cut(130, 5, 3, 2, none=True)
    _, h = ops.op_lora(x, a, b, scale, seg, keep=True)
    grads = ops.op_lora_grad(x, dy, h, a, b, scale, seg)
    randn = gen(13)
    for i, (g, v) in enumerate(zip(grads, (x, a, b))):
        d = randn(*v.shape) * 0.1
        plus, minus = [x, a, b], [x, a, b]
        plus[i], minus[i] = v + d, v - d
        yp, ym = (ops.op_lora(p[0], p[1], p[2], scale, seg).double() for p in (plus, minus))
        diff = float(((yp - ym) / 2 * dy.double()).sum())
        along = float((g.double() * d.double()).sum())
        # both sides: at most (130 + 48 + 56 + ...) roundings of sums of magnitudes; v +- d itself is rounded
        mag = float((yp.abs() + ym.abs()).mul(dy.double().abs()).sum()) + float((g.double() * d.double()).abs().sum())
        assert abs(diff - along) <= 300 * U * 8 * mag, (i, diff, along)


# ---------------------------------------------------------------------------------------------- layer norm
def norm_want(x, res, gain, offset, seg, eps):
    """(y, bound, mean, bound, rstd, bound) with first-order propagation of the roundings."""
    dt, c = x.dtype, x.shape[1]
    z = x.double() if res is None else x.double() + res.double()
    zm = x.double().abs() if res is None else x.double().abs() + res.double().abs()
    mean = z.mean(1, keepdim=True)
    d = z - mean
    e_mean = (c + 2) * U * zm.mean(1, keepdim=True)
    e_d = e_mean + 2 * U * (zm + mean.abs())
    var = d.square().mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    # d var: the errors of d, then c + 2 roundings of the sum; rstd moves by half of it, sqrt and division by a step each
    e_var = (2 * d.abs() * e_d + e_d.square()).mean(1, keepdim=True) + (c + 4) * U * var
    e_rstd = rstd * (0.5 * e_var / (var + eps) + 4 * U)
    k = torch.zeros(x.shape[0], dtype=torch.long, device="cuda")
    for lo, hi, i in spans(seg):
        k[lo:hi] = i
    g, o = gain.double()[k], offset.double()[k]
    y = d * rstd * g + o
    bound = g.abs() * (e_d * rstd + d.abs() * e_rstd + e_d * e_rstd + 3 * U * (d * rstd).abs()) + 2 * U * (y.abs() + o.abs())
    return y, bound * (1 + STEP[dt]) + STEP[dt] * y.abs() + 1e-38, mean[:, 0], e_mean[:, 0] + 1e-38, rstd[:, 0], e_rstd[:, 0]


def norm_case(tokens, c, gains, dt, kind, seed):
    randn = gen(seed)
    x = tensor(randn, tokens, c, dt, kind)
    x += 0.5
    return x, tensor(randn, tokens, c, dt, kind), (1 + 0.3 * randn(gains, c)).to(dt), (0.2 * randn(gains, c)).to(dt)


@pytest.mark.parametrize("dt,kind", [(torch.float32, "dense"), (torch.float32, "slice"), (torch.float32, "cols"),
                                     (torch.bfloat16, "dense"), (torch.bfloat16, "slice")])
@pytest.mark.parametrize("tokens,c,gains,segs", [
    (1, 1, 1, 1), (1, 768, 2, 1), (3, 2, 2, 2), (17, 63, 1, 1), (64, 512, 3, 4), (65, 768, 4, 9), (50, 513, 2, 3), (300, 130, 5, 290),
    (130, 1000, 2, 3), (20, 4096, 1, 2), (9, 5000, 2, 2), (6, 20011, 1, 1), (3, 70001, 1, 1), (4000, 96, 3, 8),
])
def test_layernorm_forward(ops, dt, kind, tokens, c, gains, segs):
    x, r, gain, offset = norm_case(tokens, c, gains, dt, kind, tokens + c)
    seg = cut(tokens, segs, gains, seed=c)
    eps = 1e-12 if dt == torch.float32 else 1e-5
    for res in (None, r):
        want = norm_want(x, res, gain, offset, seg, eps)
        out, buf = like(x)
        y, mean, rstd = ops.op_layernorm(x, gain, offset, seg, res=res, eps=eps, out=out, stats=True)
        for got, w, bound, name in ((y, want[0], want[1], "y"), (mean, want[2], want[3], "mean"), (rstd, want[4], want[5], "rstd")):
            if c > 1 or name == "mean":                    # one channel: the variance is the rounding of the mean alone
                within(got, w, bound, (name, tokens, c, dt, kind, res is not None))
        if c == 1:
            within(y, want[0], want[1] + (0.02 if dt == torch.float32 else 0), "one channel")
        untouched(buf, out)
        assert torch.equal(ops.op_layernorm(x, gain, offset, seg, res=res, eps=eps), y)


@pytest.mark.parametrize("dt,kind", [(torch.float32, "dense"), (torch.float32, "cols"), (torch.bfloat16, "dense")])
def test_layernorm_special_rows(ops, dt, kind):
    x, res, gain, offset = norm_case(40, 768, 2, dt, kind, 21)
    x[3] = 0.0                                              # no variance: the offset alone
    res[3] = 0.0
    x[4], res[4] = 2.0, 0.0                                 # a constant that sums exactly
    x[5] = 1e4                                              # large mean: the second pass is centred
    x[9, 7], x[11, 3] = float("nan"), float("inf")
    seg = Segments([2, 8, 8, 30], [1, 0, 0])
    eps = 1e-12 if dt == torch.float32 else 1e-5
    out = torch.full_like(x, SENTINEL)
    ops.op_layernorm(x, gain, offset, seg, res=res, eps=eps, out=out)
    assert (out[:2] == SENTINEL).all() and (out[30:] == SENTINEL).all()
    for t in (3, 4):
        assert torch.equal(out[t], offset[1])
    assert torch.isnan(out[9]).all() and torch.isnan(out[11]).all()
    want = norm_want(x, res, gain, offset, seg, eps)
    rows = [2, 5, 6, 7, 8, 10] + list(range(12, 30))
    within(out[rows], want[0][rows], want[1][rows], "rows beside them")


@pytest.mark.parametrize("dt,kind", [(torch.float32, "dense"), (torch.float32, "cols"), (torch.bfloat16, "dense")])
def test_layernorm_in_place(ops, dt, kind):
    for c in (768, 513, 9000):
        x, res, gain, offset = norm_case(33, c, 2, dt, kind, 22)
        seg = cut(33, 3, 2, 1)
        want = ops.op_layernorm(x, gain, offset, seg, res=res)
        y = x.clone(memory_format=torch.preserve_format)
        r = res.clone(memory_format=torch.preserve_format)
        assert torch.equal(ops.op_layernorm(y, gain, offset, seg, res=res, out=y), want)
        assert torch.equal(ops.op_layernorm(x, gain, offset, seg, res=r, out=r), want)


def norm_grad_want(x, res, dy, gain, mean, rstd, seg):
    dt, c = x.dtype, x.shape[1]
    z = x.double() if res is None else x.double() + res.double()
    zm = x.double().abs() if res is None else x.double().abs() + res.double().abs()
    dy, m, r = dy.double(), mean.double()[:, None], rstd.double()[:, None]
    k = torch.zeros(x.shape[0], dtype=torch.long, device="cuda")
    for lo, hi, i in spans(seg):
        k[lo:hi] = i
    g = gain.double()[k]
    xh = (z - m) * r
    e_xh = 3 * U * r * (zm + m.abs())                        # z, its difference to the mean, the product
    u = dy * g
    mu, mux = u.mean(1, keepdim=True), (u * xh).mean(1, keepdim=True)
    dx = r * (u - mu - xh * mux)
    e_mu = (c + 2) * U * u.abs().mean(1, keepdim=True)
    e_mux = (c + 3) * U * (u * xh).abs().mean(1, keepdim=True) + (u.abs() * e_xh).mean(1, keepdim=True)
    e_dx = r * (4 * U * (u.abs() + mu.abs() + (xh * mux).abs()) + e_mu + xh.abs() * e_mux + e_xh * mux.abs() + e_xh * e_mux)
    dg, db, e_g, e_b = (torch.zeros_like(gain, dtype=torch.float64) for _ in range(4))
    for lo, hi, i in spans(seg):
        dg[i] += (dy * xh)[lo:hi].sum(0)
        db[i] += dy[lo:hi].sum(0)
        n = x.shape[0] + 4
        e_g[i] += n * U * (dy * xh)[lo:hi].abs().sum(0) + (dy.abs() * e_xh)[lo:hi].sum(0)
        e_b[i] += n * U * dy[lo:hi].abs().sum(0)
    return [(dx, e_dx * (1 + STEP[dt]) + STEP[dt] * dx.abs() + 1e-38), (dg, e_g + 1e-38), (db, e_b + 1e-38)]


@pytest.mark.parametrize("dt,kind", [(torch.float32, "dense"), (torch.float32, "slice"), (torch.bfloat16, "dense"), (torch.bfloat16, "slice")])
@pytest.mark.parametrize("tokens,c,gains,segs", [
    (1, 1, 1, 1), (1, 768, 2, 1), (3, 2, 2, 2), (17, 63, 1, 1), (97, 513, 1, 1), (65, 768, 4, 9), (300, 130, 5, 290),
    (130, 1000, 2, 3), (9, 5000, 2, 2), (6, 20011, 1, 1), (3, 70001, 1, 1), (4000, 96, 3, 8), (600, 40, 300, 400),
])
def test_layernorm_backward(ops, dt, kind, tokens, c, gains, segs):
    x, r, gain, offset = norm_case(tokens, c, gains, dt, kind, tokens + c)
    dy = tensor(gen(5), tokens, c, dt, kind, 0.1)
    seg = cut(tokens, segs, gains, seed=c)
    for res in (None, r):
        _, mean, rstd = ops.op_layernorm(x, gain, offset, seg, res=res, eps=1e-5, stats=True)
        dx, buf = like(x)
        poison(tokens * c // 8)
        got = ops.op_layernorm_grad(x, dy, gain, mean, rstd, seg, res=res, dx=dx)
        for g, (w, bound), name in zip(got, norm_grad_want(x, res, dy, gain, mean, rstd, seg), ("dx", "dgain", "doffset")):
            within(g, w, bound, (name, tokens, c, dt, kind, res is not None))
        untouched(buf, dx)
        # in place of an input, and the same bits
        for i, t in enumerate((dy, x) if res is None else (dy, x, res)):
            v = [dy, x, res]
            v[i] = t.clone(memory_format=torch.preserve_format)
            again = ops.op_layernorm_grad(v[1], v[0], gain, mean, rstd, seg, res=v[2], dx=v[i])
            for g, w in zip(again, got):
                assert torch.equal(g, w)


@pytest.mark.parametrize("dt", TYPES)
def test_layernorm_backward_leaves_and_zeroes_what_it_should(ops, dt):
    x, res, gain, offset = norm_case(60, 200, 4, dt, "dense", 31)
    dy = tensor(gen(6), 60, 200, dt)
    seg = Segments([5, 20, 20, 33, 44], [2, 3, 1, 2])
    _, mean, rstd = ops.op_layernorm(x, gain, offset, seg, res=res, eps=1e-5, stats=True)
    want = norm_grad_want(x, res, dy, gain, mean, rstd, seg)
    for t in (0, 4, 44, 59):
        x[t] = float("nan")
        dy[t] = float("inf")
        mean[t] = float("nan")
    gain[0] = float("nan")
    dx = torch.full_like(x, SENTINEL)
    _, dg, db = ops.op_layernorm_grad(x, dy, gain, mean, rstd, seg, res=res, dx=dx)
    within(dx[5:44], want[0][0][5:44], want[0][1][5:44], "dx")
    assert (dx[:5] == SENTINEL).all() and (dx[44:] == SENTINEL).all()
    for k in (1, 2):
        within(dg[k], want[1][0][k], want[1][1][k], "dgain")
        within(db[k], want[2][0][k], want[2][1][k], "doffset")
    for k in (0, 3):
        assert (dg[k] == 0).all() and (db[k] == 0).all()
    _, dg, db = ops.op_layernorm_grad(x, dy, gain, mean, rstd, Segments([0], []), res=res)
    assert (dg == 0).all() and (db == 0).all()


@pytest.mark.parametrize("c,dt", [(300, torch.float32), (768, torch.bfloat16), (1100, torch.bfloat16), (5000, torch.float32)])
def test_layernorm_backward_of_a_large_constant_row(ops, c, dt):
    """Every sum of it is exact, so its variance is 0; mean * rstd = 2^110 * 1e6 is an infinity that no channel has."""
    x, _, gain, offset = norm_case(9, c, 2, dt, "dense", 61)
    dy = tensor(gen(62), 9, c, dt)
    x[4] = 2.0 ** 110
    seg = Segments([0, 6, 9], [1, 0])
    _, mean, rstd = ops.op_layernorm(x, gain, offset, seg, stats=True)
    assert mean[4] == 2.0 ** 110 and abs(float(rstd[4]) - 1e6) <= 1e6 * 4 * U
    got = ops.op_layernorm_grad(x, dy, gain, mean, rstd, seg)
    for what, g, (w, bound) in zip(("dx", "dgain", "doffset"), got, norm_grad_want(x, None, dy, gain, mean, rstd, seg)):
        assert torch.isfinite(g).all()
        within(g, w, bound, what)


def test_layernorm_gradients_against_differences(ops):
    """Central differences of the definition in 64 bits: step 1e-5, so 1e-10 of truncation and 1e-11 of rounding."""
    x, res, gain, offset = norm_case(40, 96, 2, torch.float32, "dense", 33)
    dy = tensor(gen(7), 40, 96, torch.float32)
    seg = Segments([0, 17, 40], [1, 0])
    _, mean, rstd = ops.op_layernorm(x, gain, offset, seg, res=res, eps=1e-5, stats=True)
    grads = ops.op_layernorm_grad(x, dy, gain, mean, rstd, seg, res=res)
    bounds = [b for _, b in norm_grad_want(x, res, dy, gain, mean, rstd, seg)]
    randn = gen(8)

    def loss(x, gain, offset):
        return (_norm64(x, res.double(), gain, offset, seg) * dy.double()).sum()

    for i, g in enumerate(grads):
        v = [x.double(), gain.double(), offset.double()]
        d = randn(*v[i].shape).double()
        p, m = list(v), list(v)
        p[i], m[i] = v[i] + 1e-5 * d, v[i] - 1e-5 * d
        diff = float((loss(*p) - loss(*m)) / 2e-5)
        along = float((g.double() * d).sum())
        # mean and rstd are the forward pass's 32-bit ones: c + 8 roundings of theirs on top of the backward's own
        slack = 2 * float((bounds[i] * d.abs()).sum()) + 110 * U * float((g.double() * d).abs().sum())
        assert abs(diff - along) <= slack + 1e-6 * abs(diff), (i, diff, along, slack)


def _norm64(x, res, gain, offset, seg):
    z = x + res
    d = z - z.mean(1, keepdim=True)
    xh = d / torch.sqrt(d.square().mean(1, keepdim=True) + 1e-5)
    return torch.cat([xh[lo:hi] * gain[k] + offset[k] for lo, hi, k in spans(seg)])


# ---------------------------------------------------------------------------------------------- padded batches
@pytest.mark.parametrize("dt,kind", [(torch.float32, "dense"), (torch.float32, "cols"), (torch.bfloat16, "dense")])
@pytest.mark.parametrize("pitch,lengths", [(40, [13, 40, 0, 1, 33]), (7, [3] * 150), (64, [64, 64, 5])])
def test_padding_is_left_alone_and_reaches_nothing(ops, dt, kind, pitch, lengths):
    n, c = len(lengths), 72
    tokens = n * pitch
    index = [i % 3 for i in range(n)]
    padded, packed = Segments.of_padded(lengths, index, pitch), Segments.of_lengths(lengths, index)
    rows = torch.cat([torch.arange(b * pitch, b * pitch + m) for b, m in enumerate(lengths)]).cuda()
    pad = torch.ones(tokens, dtype=torch.bool, device="cuda")
    pad[rows] = False
    x, base, a, b, scale = lora_case(tokens, c, c, 6, 3, dt, kind, 81)
    gain, offset = (1 + 0.1 * gen(82)(3, c)).to(dt), gen(83)(3, c).to(dt)
    x[pad], base[pad] = float("nan"), float("inf")

    def pack(t):
        v = t[rows].contiguous()
        return v.t().contiguous().t() if kind == "cols" else v

    def same(got, want):
        assert torch.equal(got[rows], want)
        assert (got[pad] == 0).all()                             # (outputs of the call's own making)

    y, h = ops.op_lora(x, a, b, scale, padded, base=base, keep=True)
    yp, hp = ops.op_lora(pack(x), a, b, scale, packed, base=pack(base), keep=True)
    same(y, yp)
    same(h, hp)
    out = torch.full_like(x, SENTINEL)
    z, mean, rstd = ops.op_layernorm(x, gain, offset, padded, res=base, out=out, stats=True)
    zp, mp, rp = ops.op_layernorm(pack(x), gain, offset, packed, res=pack(base), stats=True)
    assert torch.equal(z[rows], zp) and (out[pad] == SENTINEL).all()
    same(mean, mp)
    same(rstd, rp)
    if kind == "cols":
        return
    mean[pad], rstd[pad], h[pad] = float("nan"), float("inf"), float("nan")
    got = ops.op_layernorm_grad(x, base, gain, mean, rstd, padded)
    same(got[0], ops.op_layernorm_grad(pack(x), pack(base), gain, mp, rp, packed)[0])
    for g, (w, bound) in zip(got[1:], norm_grad_want(pack(x), None, pack(base), gain, mp, rp, packed)[1:]):
        within(g, w, bound, "gain")
    got = ops.op_lora_grad(x, base, h, a, b, scale, padded)
    same(got[0], ops.op_lora_grad(pack(x), pack(base), hp, a, b, scale, packed)[0])
    for g, (w, bound) in zip(got[1:], lora_grad_want(pack(x), pack(base), hp, None, a, b, scale, packed)[1:]):
        within(g, w, bound + 1e-38, "factors")


# ---------------------------------------------------------------------------------------------- as they are used
def sublayer(ops, x, w, a, b, scale, gain, offset, seg, eps=1e-5):
    """A projection with adapters, the residual and the norm: forward."""
    y, h = ops.op_lora(x, a, b, scale, seg, base=x @ w.t(), keep=True)
    out, mean, rstd = ops.op_layernorm(y, gain, offset, seg, res=x, eps=eps, stats=True)
    return out, (y, h, mean, rstd)


def sublayer_grad(ops, dout, x, w, a, b, scale, gain, seg, kept):
    y, h, mean, rstd = kept
    dz, dgain, doffset = ops.op_layernorm_grad(y, dout, gain, mean, rstd, seg, res=x)
    dx, da, db = ops.op_lora_grad(x, dz, h, a, b, scale, seg, dx_base=dz @ w + dz)
    return dx, da, db, dgain, doffset


def sublayer_case(tokens, c, rank, n, seed):
    randn = gen(seed)
    x = randn(tokens, c)
    w = randn(c, c) / c ** 0.5
    return (x, w, randn(n, rank, c) / c ** 0.5, randn(n, c, rank) * 0.3, 0.5 + torch.rand(n, device="cuda"),
            1 + 0.2 * randn(n, c), 0.1 * randn(n, c), randn(tokens, c))


def test_a_sublayer_forward_and_backward_together(ops):
    x, w, a, b, scale, gain, offset, dout = sublayer_case(150, 96, 8, 3, 41)
    seg = cut(150, 6, 3, 4)
    out, kept = sublayer(ops, x, w, a, b, scale, gain, offset, seg)
    got = sublayer_grad(ops, dout, x, w, a, b, scale, gain, seg, kept)
    # torch's own differentiation of the definition in 64 bits
    leaf = [t.double().cpu().requires_grad_() for t in (x, a, b, gain, offset)]
    xx, aa, bb, gg, oo = leaf
    rows = []
    for lo, hi, k in spans(seg):
        v = xx[lo:hi]
        z = v @ w.double().cpu().t() + float(scale[k]) * (v @ aa[k].t()) @ bb[k].t() + v
        d = z - z.mean(1, keepdim=True)
        rows.append(d / torch.sqrt(d.square().mean(1, keepdim=True) + 1e-5) * gg[k] + oo[k])
    ref = torch.cat(rows)
    (ref * dout.double().cpu()).sum().backward()
    for g, t, name in zip((out, *got), (ref.detach(), *(t.grad for t in leaf)), ("out", "dx", "da", "db", "dgain", "doffset")):
        # a chain of products over 96 channels and sums over 150 tokens in 32 bits: 500 roundings, relative to the largest value
        assert (g.double().cpu() - t).abs().max() <= 500 * U * t.abs().max(), name


def test_captured_beside_eager_and_replayed(ops):
    """Two graphs and eager calls on the same tensors, in turn: each replay gives the eager bits for the inputs it sees."""
    x, w, a, b, scale, gain, offset, dout = sublayer_case(333, 128, 16, 4, 42)
    seg = cut(333, 9, 4, 5)

    def step():
        y, h = ops.op_lora(x, a, b, scale, seg, base=x, keep=True)
        out, mean, rstd = ops.op_layernorm(y, gain, offset, seg, res=x, eps=1e-5, stats=True)
        dz, dgain, doffset = ops.op_layernorm_grad(y, dout, gain, mean, rstd, seg, res=x)
        return (out, dgain, doffset, *ops.op_lora_grad(x, dz, h, a, b, scale, seg, dx_base=dz))

    eager = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    graphs, outs = [], []
    for _ in range(2):
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            outs.append(step())
        graphs.append(g)
    randn = gen(43)
    for i in range(4):
        if i:
            x.copy_(randn(*x.shape))
            dout.copy_(randn(*x.shape))
            eager = [t.clone() for t in step()]
        for g, o in zip(graphs, outs):
            for t in o:
                t.fill_(float("nan"))
            g.replay()
            torch.cuda.synchronize()
            for got, want in zip(o, eager):
                assert torch.equal(got, want), i
    # both graphs at once on two streams
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for g, s in zip(graphs, streams):
        with torch.cuda.stream(s):
            g.replay()
    torch.cuda.synchronize()
    for o in outs:
        for got, want in zip(o, eager):
            assert torch.equal(got, want)


def test_calls_follow_the_current_stream(ops):
    x, w, a, b, scale, gain, offset, dout = sublayer_case(2000, 256, 16, 2, 44)
    seg = cut(2000, 5, 2, 6)
    want = ops.op_layernorm(ops.op_lora(x, a, b, scale, seg, base=x), gain, offset, seg)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        late = torch.zeros_like(x)
        torch.cuda._sleep(20_000_000)
        late.copy_(x)                                       # not there yet when the calls are enqueued
        got = ops.op_layernorm(ops.op_lora(late, a, b, scale, seg, base=late), gain, offset, seg)
    side.synchronize()
    assert torch.equal(got, want)


def test_two_threads_on_one_handle(ops):
    x, w, a, b, scale, gain, offset, dout = sublayer_case(700, 192, 8, 3, 45)
    seg = cut(700, 8, 3, 7)
    want_out, kept = sublayer(ops, x, w, a, b, scale, gain, offset, seg)
    want = [t.clone() for t in sublayer_grad(ops, dout, x, w, a, b, scale, gain, seg, kept)]
    torch.cuda.synchronize()
    bad = []

    def work():
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(10):
                out, k = sublayer(ops, x, w, a, b, scale, gain, offset, seg)
                got = sublayer_grad(ops, dout, x, w, a, b, scale, gain, seg, k)
                torch.cuda.current_stream().synchronize()
                if not torch.equal(out, want_out) or not all(torch.equal(g, t) for g, t in zip(got, want)):
                    bad.append(1)

    threads = [threading.Thread(target=work) for _ in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_the_handles_own_stream_waits(ops):
    """stream NULL through the C-ABI: the result is there when the call returns."""
    from tts_amd import _lib
    x, res, gain, offset = norm_case(50, 128, 1, torch.float32, "dense", 51)
    y = torch.zeros_like(x)
    torch.cuda.synchronize()
    p = _lib.K82Layernorm(0, 0, 128, 1, 1e-12, 50, x.data_ptr(), 128, None, 0, y.data_ptr(), 128, gain.data_ptr(),
                          offset.data_ptr(), None, None)
    seg = Segments([0, 50], [0])
    assert ops.lib.k82_op_layernorm(ops.h, p, seg.c, None) == 0
    host = torch.empty(50, 128)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        host.copy_(y)
    assert torch.equal(host, ops.op_layernorm(x, gain, offset).cpu())


def test_an_engine_has_the_same_operators(engine, ops):
    x, base, a, b, scale = lora_case(40, 64, 64, 8, 2, torch.float32, "dense", 61)
    assert torch.equal(engine.op_lora(x, a, b, scale, base=base), ops.op_lora(x, a, b, scale, base=base))


@pytest.mark.parametrize("dt,kind", [(torch.bfloat16, "rows"), (torch.float32, "cols")])
def test_tokens_behind_two_to_the_31_elements(ops, dt, kind):
    c = 1100
    tokens = 2_000_000
    if kind == "rows":
        buf = torch.empty(tokens, c, dtype=dt, device="cuda")
        view = buf
    else:
        buf = torch.empty(c, tokens, dtype=dt, device="cuda")
        view = buf.t()
    randn = gen(71)
    lo = tokens - 100
    tail = randn(100, c).to(dt)
    view[lo:] = tail
    a, b, scale = (randn(1, 4, c) / 33).to(dt), randn(1, c, 4).to(dt), torch.ones(1, device="cuda")
    gain, offset = (1 + 0.1 * randn(1, c)).to(dt), randn(1, c).to(dt)
    seg, small = Segments([lo, tokens], [0]), Segments([0, 100], [0])
    x = tail if kind == "rows" else tail.t().contiguous().t()
    out = torch.empty_strided(view.shape, view.stride(), dtype=dt, device="cuda")
    ops.op_lora(view, a, b, scale, seg, base=view, out=out)
    assert torch.equal(out[lo:], ops.op_lora(x, a, b, scale, small, base=x))
    y, mean, rstd = ops.op_layernorm(view, gain, offset, seg, out=out, stats=True)
    want, m, r = ops.op_layernorm(x, gain, offset, small, stats=True)
    assert torch.equal(y[lo:], want) and torch.equal(mean[lo:], m) and torch.equal(rstd[lo:], r)
    if kind == "rows":
        h = torch.zeros(tokens, 4, device="cuda")
        h[lo:] = randn(100, 4)
        got = ops.op_lora_grad(view, view, h, a, b, scale, seg, dx=out)
        want = ops.op_lora_grad(x, x, h[lo:], a, b, scale, small)
        assert torch.equal(got[0][lo:], want[0])
        for g, w in zip(got[1:], want[1:]):
            assert torch.equal(g, w)
        got = ops.op_layernorm_grad(view, view, gain, mean, rstd, seg, dx=out)
        want = ops.op_layernorm_grad(x, x, gain, m, r, small)
        assert torch.equal(got[0][lo:], want[0]) and torch.equal(got[1], want[1]) and torch.equal(got[2], want[2])
