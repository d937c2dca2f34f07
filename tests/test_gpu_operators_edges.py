"""The operators at the edges of what their arguments allow.  Tolerances: the bounds of test_gpu_operators.py, sums of
roundings."""
import ctypes as C
import threading

import pytest
import torch

from test_gpu_operators import (TYPES, cut, gen, lora_case, lora_grad_want, lora_want, norm_case, norm_grad_want, ops,  # noqa: F401
                                tensor, within)
from tts_amd import Segments, _lib

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------------------------- values next to the largest
def near_largest(dt, tokens, width):
    """[tokens, width] and weights [1, width] of dt whose product is 2^127 (255/128 + 3/512) = 3.40e38, every term of it exact:
    finite in 32 bits, half a step and more above the largest finite bf16 (255/128 2^127)."""
    v, w = torch.zeros(tokens, width, device="cuda", dtype=dt), torch.zeros(1, width, device="cuda", dtype=dt)
    v[:, 0], v[:, width - 1] = 2.0 ** 127, 2.0 ** 119
    w[0, 0], w[0, width - 1] = 255 / 128, 1.5
    v[1::2] *= -1
    return v, w


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("rank", [1, 7, 17, 40, 65])
def test_a_large_finite_h_stays_finite(ops, dt, rank):
    tokens, cin, cout = 37, 64, 72
    x, w = near_largest(dt, tokens, cin)
    _, base, _, b, _ = lora_case(tokens, cin, cout, rank, 2, dt, "dense", 5)
    a = torch.zeros(2, rank, cin, device="cuda", dtype=dt)
    a[:, rank - 1] = w
    b = (b.float() * 2.0 ** -100).to(dt)
    scale, seg = torch.ones(2, device="cuda"), Segments([0, 20, 37], [1, 0])
    y, h = ops.op_lora(x, a, b, scale, seg, base=base, keep=True)
    want, bound, h_want, h_bound = lora_want(x, base, a, b, scale, seg, "none")
    assert h_want.abs().max() > torch.finfo(torch.bfloat16).max * 1.0015 and h_want.abs().max() < torch.finfo(torch.float32).max
    within(h, h_want, h_bound + 1e-38, "h")
    within(y, want, bound, "y")
    assert want.abs().max() > 2.0 ** 14


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("rank", [1, 7, 17, 40, 65])
def test_large_finite_gradients_stay_finite(ops, dt, rank):
    """dy B_k, and h, as the parts of the two products they enter: dx and da, and db."""
    tokens, cin, cout = 37, 64, 72
    seg = Segments([0, 20, 37], [1, 0])
    scale = torch.ones(2, device="cuda")
    x, _, a, _, _ = lora_case(tokens, cin, cout, rank, 2, dt, "dense", 6)
    dy, w = near_largest(dt, tokens, cout)
    b = torch.zeros(2, cout, rank, device="cuda", dtype=dt)
    b[:, :, rank - 1] = w
    x, a = (x.float() * 2.0 ** -100).to(dt), (a.float() * 2.0 ** -100).to(dt)
    h = gen(7)(tokens, rank) * 2.0 ** -100
    got = ops.op_lora_grad(x, dy, h, a, b, scale, seg)
    for g, (want, bound), name in zip(got, lora_grad_want(x, dy, h, None, a, b, scale, seg), ("dx", "da", "db")):
        within(g, want, bound + 1e-38, name)
        assert want.abs().max() > 2.0 ** 10
    # h next to the largest, dy small
    x, dy, a, b, _ = lora_case(tokens, cin, cout, rank, 2, dt, "dense", 8)
    dy = (dy.float() * 2.0 ** -100).to(dt)
    h = torch.full((tokens, rank), (255 / 128 + 3 / 512) * 2.0 ** 127, device="cuda")
    h[::3] *= -1
    got = ops.op_lora_grad(x, dy, h, a, b, scale, seg)
    for g, (want, bound), name in zip(got, lora_grad_want(x, dy, h, None, a, b, scale, seg), ("dx", "da", "db")):
        within(g, want, bound + 1e-38, name)


# ---------------------------------------------------------------------------------------------- refusals on several threads
def norm_args(eps):
    x, gain, offset = (torch.ones(1, 8, device="cuda") for _ in range(3))
    return _lib.K82Layernorm(0, 0, 8, 1, eps, 1, x.data_ptr(), 8, None, 0, x.data_ptr(), 8, gain.data_ptr(), offset.data_ptr(), None,
                             None), (x, gain, offset)


def test_a_refusal_keeps_its_reason_beside_another_threads(ops):
    """The text of a thread's own last failed call on the handle; a thread that had none reads the handle's last."""
    lib, seg, (bad, keep) = ops.lib, Segments([0, 1], [0]), norm_args(-1.0)
    read = []

    def other():
        read.append(lib.k82_last_error(ops.h))
        assert lib.k82_op_layernorm(ops.h, norm_args(1.0)[0], Segments([0, 1], [7]).c, None) == -22
        read.append(lib.k82_last_error(ops.h))

    assert lib.k82_op_layernorm(ops.h, bad, seg.c, None) == -22
    t = threading.Thread(target=other)
    t.start()
    t.join(60)
    assert b"eps" in lib.k82_last_error(ops.h)
    assert b"eps" in read[0] and b"index 7" in read[1]
    late = []
    t = threading.Thread(target=lambda: late.append(lib.k82_last_error(ops.h)))
    t.start()
    t.join(60)
    assert b"index 7" in late[0]


def test_refusals_of_many_threads_at_once(ops):
    wrong = []

    def work(k):
        for _ in range(300):
            x = torch.ones(1, 8, device="cuda")
            try:
                ops.op_layernorm(x, x, x, Segments([0, 1], [100 + k]))
                wrong.append("accepted")
            except ValueError as e:
                if f"index {100 + k} " not in str(e):
                    wrong.append(str(e))

    threads = [threading.Thread(target=work, args=(k,)) for k in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong[:3]


# ---------------------------------------------------------------------------------------------- the largest launches
def test_layernorm_of_as_many_wide_rows_as_a_call_holds(ops):
    """2^24 - 1 rows of 1024 threads each: equal rows give equal results, the first and the last of every part among them."""
    tokens, c = (1 << 24) - 1, 4097
    torch.cuda.empty_cache()
    free, _ = torch.cuda.mem_get_info()
    if free < 2 * tokens * c + (16 << 30):
        pytest.skip(f"{free >> 30} GiB are free, 137 GB of rows and room to compare are needed")
    row, _, gain, offset = norm_case(1, c, 1, torch.bfloat16, "dense", 3)
    want = ops.op_layernorm(row, gain, offset)
    assert not torch.equal(want, row)
    x = torch.empty(tokens, c, device="cuda", dtype=torch.bfloat16)
    try:
        x.copy_(row.expand(tokens, c))
        assert ops.op_layernorm(x, gain, offset, out=x) is x
        for i in range(0, tokens, 1 << 20):
            assert (x[i:i + (1 << 20)] == want).all(), i
    finally:
        del x
        torch.cuda.empty_cache()


# ---------------------------------------------------------------------------------------------- workspaces
def in_poisoned_workspace(ops, op, p, seg):
    """The C entry point with a workspace of exactly the bytes it asks for, every one 0xff (NaN in either type), and a guard
    behind it that stays as it was."""
    need = getattr(ops.lib, f"k82_op_{op}_workspace")(p, seg.c)
    assert need > 0
    ws = torch.full((need + 4096,), 0xff, device="cuda", dtype=torch.uint8)
    guard = torch.arange(4096, device="cuda").to(torch.uint8)
    ws[need:] = guard
    assert ws.data_ptr() % 256 == 0
    stream = C.c_void_p(torch.cuda.current_stream().cuda_stream or 1)
    call = getattr(ops.lib, f"k82_op_{op}")
    assert call(ops.h, p, seg.c, ws.data_ptr(), need - 1, stream) == -28
    assert call(ops.h, p, seg.c, ws.data_ptr(), need, stream) == 0, ops.lib.k82_last_error(ops.h)
    assert torch.equal(ws[need:], guard)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("tokens,cin,cout,rank,adapters,segs", [
    (1, 1, 1, 1, 1, 1), (2, 5, 3, 3, 2, 2), (63, 129, 65, 17, 2, 3), (64, 64, 64, 64, 1, 1), (211, 768, 768, 7, 1, 1),
    (257, 200, 96, 128, 2, 5), (300, 96, 40, 7, 6, 290), (3000, 260, 513, 33, 3, 11), (700, 140, 70, 8, 400, 500),
    (9000, 64, 100, 4, 2, 3), (34000, 136, 72, 40, 3, 7), (260, 24, 16, 4, 2, 258),
])
def test_lora_backward_writes_all_it_reads_of_its_workspace(ops, dt, tokens, cin, cout, rank, adapters, segs):
    x, dy, a, b, scale = lora_case(tokens, cin, cout, rank, adapters, dt, "dense", tokens + 1)
    seg = cut(tokens, segs, adapters, seed=tokens, none=segs > 1)
    h = gen(3)(tokens, rank)
    dx, da, db = (torch.full(s, float("nan"), device="cuda", dtype=t) for s, t in (((tokens, cin), dt), (a.shape, torch.float32),
                                                                                  (b.shape, torch.float32)))
    p = _lib.K82LoraGrad(TYPES.index(dt), cin, cout, rank, adapters, tokens, x.data_ptr(), cin, dy.data_ptr(), cout, h.data_ptr(),
                         None, 0, dx.data_ptr(), cin, a.data_ptr(), b.data_ptr(), scale.data_ptr(), da.data_ptr(), db.data_ptr())
    in_poisoned_workspace(ops, "lora_grad", p, seg)
    for g, (want, bound), name in zip((dx, da, db), lora_grad_want(x, dy, h, None, a, b, scale, seg), ("dx", "da", "db")):
        within(g, want, bound + 1e-38, name)
    for g, again in zip((dx, da, db), ops.op_lora_grad(x, dy, h, a, b, scale, seg)):
        assert torch.equal(g, again)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("tokens,c,gains,segs", [
    (1, 1, 1, 1), (1, 768, 2, 1), (3, 2, 2, 2), (97, 513, 1, 1), (65, 768, 4, 9), (300, 130, 5, 290), (130, 1000, 2, 3), (9, 5000, 2, 2),
    (6, 20011, 1, 1), (300, 9000, 3, 40), (4000, 96, 3, 8), (600, 40, 300, 400), (40000, 64, 2, 5),
])
def test_layernorm_backward_writes_all_it_reads_of_its_workspace(ops, dt, tokens, c, gains, segs):
    x, res, gain, offset = norm_case(tokens, c, gains, dt, "dense", tokens + c)
    dy = tensor(gen(5), tokens, c, dt, scale=0.1)
    seg = cut(tokens, segs, gains, seed=c)
    _, mean, rstd = ops.op_layernorm(x, gain, offset, seg, res=res, eps=1e-5, stats=True)
    dx = torch.full((tokens, c), float("nan"), device="cuda", dtype=dt)
    dgain, doffset = (torch.full((gains, c), float("nan"), device="cuda") for _ in range(2))
    p = _lib.K82LayernormGrad(TYPES.index(dt), c, gains, tokens, x.data_ptr(), c, res.data_ptr(), c, dy.data_ptr(), c, dx.data_ptr(), c,
                              gain.data_ptr(), mean.data_ptr(), rstd.data_ptr(), dgain.data_ptr(), doffset.data_ptr())
    in_poisoned_workspace(ops, "layernorm_grad", p, seg)
    for g, (want, bound), name in zip((dx, dgain, doffset), norm_grad_want(x, res, dy, gain, mean, rstd, seg), ("dx", "dgain", "doffset")):
        within(g, want, bound, name)
    for g, again in zip((dx, dgain, doffset), ops.op_layernorm_grad(x, dy, gain, mean, rstd, seg, res=res)):
        assert torch.equal(g, again)


def test_a_workspace_that_covers_tokens_of_nobody(ops):
    """The sizes go by the cut's ends, the sums by what lies between: padding, sentences without an adapter, unused ones."""
    tokens, c, rank = 4000, 72, 9
    x, dy, a, b, scale = lora_case(tokens, c, c, rank, 200, torch.bfloat16, "dense", 4)
    seg = Segments.of_padded([(7 * i) % 41 for i in range(100)], [(3 * i) % 200 if i % 5 else -1 for i in range(100)], 40)
    h = gen(4)(tokens, rank)
    dx = torch.full((tokens, c), float("nan"), device="cuda", dtype=torch.bfloat16)
    da, db = torch.full(a.shape, float("nan"), device="cuda"), torch.full(b.shape, float("nan"), device="cuda")
    p = _lib.K82LoraGrad(1, c, c, rank, 200, tokens, x.data_ptr(), c, dy.data_ptr(), c, h.data_ptr(), None, 0, dx.data_ptr(), c,
                         a.data_ptr(), b.data_ptr(), scale.data_ptr(), da.data_ptr(), db.data_ptr())
    in_poisoned_workspace(ops, "lora_grad", p, seg)
    rows = torch.cat([torch.arange(int(lo), int(hi)) for lo, hi, k in zip(seg.offsets[:-1], seg.offsets[1:], seg.index) if k >= -1]).cuda()
    want = lora_grad_want(x, dy, h, None, a, b, scale, seg)
    within(dx[rows], want[0][0][rows], want[0][1][rows], "dx")
    within(da, want[1][0], want[1][1] + 1e-38, "da")
    within(db, want[2][0], want[2][1] + 1e-38, "db")
    left = torch.ones(tokens, dtype=torch.bool, device="cuda")
    left[rows] = False
    assert torch.isnan(dx[left].float()).all()
