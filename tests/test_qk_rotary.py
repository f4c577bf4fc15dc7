"""Rotary positions with several axes and norms of queries and keys with the rotation: against the formulas in 64 bits.

Error bounds, before the type of the result rounds (u = 2^-24): the angle's fraction of a turn is exact to 2^-32 and rounded to
fp32 once (3.2 u rad at half a turn), sine and cosine are good to 2 u, the turn itself rounds three times: 8 u (|a| + |b|) for a
pair (a, b).  A row's 1 / rms is good to 10 u (13 roundings of its sum of squares count half, 3 for the rest).  Results of
16 bits are then half a step off."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

import hyperkernels_b200 as hk

U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = {"f32": F32, "bf16": BF16, "f16": F16}


def half_step(t, y):
    return y.abs() * (torch.finfo(t).eps / 2) + (2.0 ** -25 if t == F16 else 0.0)


def angles(positions, sections, base=10000.0, frequencies=None):
    """[B, 1, T, 32] in 64 bits"""
    n = sum(sections)
    f = frequencies if frequencies is not None else [base ** (-p / 32) for p in range(n)]
    a = torch.zeros((*positions.shape[1:], 32), dtype=torch.float64, device=positions.device)
    p = 0
    for axis, m in enumerate(sections):
        for _ in range(m):
            a[..., p] = positions[axis].double() * f[p]
            p += 1
    return a[:, None]


def pairs(x, interleaved):
    return (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :32], x[..., 32:])


def join(a, b, interleaved):
    return torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)


def turned(x, angle, interleaved):
    a, b = pairs(x, interleaved)
    return join(a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos(), interleaved)


def size_of_pairs(x, interleaved):
    """|a| + |b| of its pair at every element"""
    a, b = pairs(x.abs(), interleaved)
    return join(a + b, a + b, interleaved)


def normed(x, w, eps):
    x = x.double()
    return x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()


def inputs(seed, B, H, Hk, T, dtype, layout, sigma=1.0, device="cuda"):
    g = torch.Generator(device=device).manual_seed(seed)
    if layout == "packed":
        x = (torch.randn((B, T, H + 2 * Hk, 64), generator=g, device=device) * sigma).to(dtype)
        return x[:, :, :H].transpose(1, 2), x[:, :, H:H + Hk].transpose(1, 2)
    if layout == "wide":  # rows 128 elements apart, head by head
        x = (torch.randn((H + Hk, B, T, 128), generator=g, device=device) * sigma).to(dtype)[..., 64:]
        return x[:H].transpose(0, 1), x[H:].transpose(0, 1)
    q, k = ((torch.randn((B, n, T, 64), generator=g, device=device) * sigma).to(dtype) for n in (H, Hk))
    return q, k


def close(got, want, bound, what=""):
    d = (got.double() - want).abs()
    assert bool((d <= bound).all()), (what, float((d - bound).max()), float(d.max()))


SHAPES = [(1, 1, 1, 1), (2, 3, 1, 5), (3, 12, 4, 33), (1, 25, 25, 130), (64, 8, 8, 1), (2, 4, 0, 1027)]


@pytest.mark.gpu
@pytest.mark.parametrize("B,H,Hk,T", SHAPES)
@pytest.mark.parametrize("xt,yt", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("bf16", "f32"), ("f16", "f32"), ("f32", "bf16"), ("f32", "f16")])
@pytest.mark.parametrize("sections,interleaved,layout", [((32,), False, "bhtd"), ((8, 12, 12), False, "packed"), ((5, 9, 2, 9), True, "wide"), ((16, 16), True, "packed")])
def test_rotation_and_back(B, H, Hk, T, xt, yt, sections, interleaved, layout):
    q, k = inputs(B + T, B, H, Hk, T, TYPES[xt], layout)
    k = k if Hk else None
    g = torch.Generator(device="cuda").manual_seed(7)
    pos = torch.randint(-5, 200000, (len(sections), B, T), generator=g, device="cuda", dtype=torch.int32 if T % 2 else torch.int64)
    angle = angles(pos, sections)
    for call, sign in ((hk.rotary_forward, 1), (hk.rotary_backward, -1)):
        got = call(q, k, pos, sections, interleaved=interleaved, out_dtype=TYPES[yt])
        assert (got[1] is None) == (k is None)
        for x, y in zip((q, k), got):
            if x is None:
                continue
            assert y.dtype == TYPES[yt] and y.shape == x.shape
            want = turned(x.double(), sign * angle, interleaved)
            # the definition's own angle: a product in 64 bits, off by 2^-53 of itself
            close(y, want, size_of_pairs(x.double(), interleaved) * (8 * U + 2 ** -52 * 2e5) + half_step(TYPES[yt], want) * (yt != "f32"))


@pytest.mark.gpu
def test_far_positions_and_frequencies_of_ones_own():
    q, _ = inputs(1, 1, 2, 0, 64, F32, "bhtd")
    pos = (torch.arange(64, device="cuda", dtype=torch.int64) * 33554393 + 2 ** 30)[None, None]
    f = [1.0, 0.5, 0.3, 2 * math.pi, 7.25, 1e-9] + [0.01] * 26
    got, none = hk.rotary_forward(q, None, pos, (32,), frequencies=f)
    # exact angles: the fraction of a turn in Python integers (2^-120 of a turn)
    turns = [int(np.longdouble(x) / (2 * np.longdouble(math.pi) + np.longdouble(2.4492935982947064e-16)) * np.longdouble(2.0) ** 64) for x in f]
    a = torch.tensor([[(int(p) * t % 2 ** 64) / 2 ** 64 * 2 * math.pi for t in turns] for p in pos.flatten().tolist()], dtype=torch.float64, device="cuda")
    want = turned(q.double(), a[None, None], False)
    close(got, want, size_of_pairs(q.double(), False) * (8 * U + 2.0 ** 32 * 2 ** -62 * 2 * math.pi))
    assert none is None


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_pairs_behind_the_sections_and_position_zero_keep_their_bits(dtype):
    q, _ = inputs(2, 2, 3, 0, 9, TYPES[dtype], "packed")
    q = q.clone()
    q[0, 0, :, 20] = math.inf
    q[0, 1, :, 31] = math.nan
    pos = torch.arange(9, device="cuda", dtype=torch.int32).expand(1, 2, 9)
    y, _ = hk.rotary_forward(q, None, pos, (8,))
    still = [i for i in range(64) if i % 32 >= 8]
    as_int = torch.int32 if dtype == "f32" else torch.int16
    assert torch.equal(y[..., still].view(as_int), q[..., still].view(as_int))
    assert torch.equal(y[:, :, 0].view(as_int), q[:, :, 0].view(as_int))


@pytest.mark.gpu
@pytest.mark.parametrize("B,H,Hk,T", SHAPES)
@pytest.mark.parametrize("xt,yt,wt", [("f32", "f32", "f32"), ("bf16", "bf16", "bf16"), ("f16", "f32", "f32"), ("bf16", "f32", None), ("f16", "f16", "f16")])
@pytest.mark.parametrize("sections,interleaved,layout", [((32,), False, "bhtd"), ((8, 12, 12), True, "packed"), ((10, 11), False, "wide")])
def test_norm_and_rotation(B, H, Hk, T, xt, yt, wt, sections, interleaved, layout):
    q, k = inputs(B * T, B, H, Hk, T, TYPES[xt], layout, 1.5)
    k = k if Hk else None
    g = torch.Generator(device="cuda").manual_seed(8)
    w = [None, None] if wt is None else [(1 + 0.3 * torch.randn(64, generator=g, device="cuda")).to(TYPES[wt]) for _ in range(2)]
    pos = torch.randint(0, 5000, (len(sections), 1, T), generator=g, device="cuda", dtype=torch.int32).expand(len(sections), B, T)
    angle, eps = angles(pos, sections), 1e-5
    got = hk.qk_norm_rotary_forward(q, k, *w, pos, sections, eps=eps, interleaved=interleaved, out_dtype=TYPES[yt])
    dy = [None if x is None else (torch.randn(x.shape, generator=g, device="cuda") * 0.5).to(TYPES[yt]) for x in (q, k)]
    grads = hk.qk_norm_rotary_backward(q, k, *dy, *w, pos, sections, eps=eps, interleaved=interleaved)
    again = hk.qk_norm_rotary_backward(q, k, *dy, *w, pos, sections, eps=eps, interleaved=interleaved)
    for a, b in zip(grads, again):
        assert (a is None and b is None) or torch.equal(a, b)
    for i, x in enumerate((q, k)):
        if x is None:
            assert got[1] is None and grads[1] is None and grads[3] is None
            continue
        one = torch.ones(64, device="cuda", dtype=torch.float64) if w[i] is None else w[i].double()
        n = normed(x, one, eps)
        want = turned(n, angle, interleaved)
        assert got[i].dtype == TYPES[yt]
        close(got[i], want, size_of_pairs(n, interleaved) * 20 * U + half_step(TYPES[yt], want) * (yt != "f32"), "forward")
        # backward: z = the gradient turned back, n = x / rms
        z = turned(dy[i].double(), -angle, interleaved)
        inv = 1 / (x.double().square().mean(-1, keepdim=True) + eps).sqrt()
        n = x.double() * inv
        want = inv * (one * z - n * (one * z * n).mean(-1, keepdim=True))
        zs = size_of_pairs(dy[i].double(), interleaved)  # bounds |z|; z is 8 u of it off, one * z 9, the mean 9 + 11 + 11
        bound = inv * (zs * one.abs() * 22 * U + n.abs() * (zs * one.abs() * n.abs()).mean(-1, keepdim=True) * 55 * U)
        assert grads[i].dtype == x.dtype
        close(grads[i], want, bound + half_step(x.dtype, want) * (xt != "f32"), "backward")
        if w[i] is None:
            assert grads[2 + i] is None
            continue
        # the longest chain of additions: a lane's rows, the CTA's 32 lanes, sixteen and sixteen CTAs
        terms = (zs * n.abs()).sum((0, 1, 2))
        rows = B * (H + Hk) * T
        assert grads[2 + i].dtype == F32
        close(grads[2 + i], (z * n).sum((0, 1, 2)), terms * (20 + 64 + 40 + rows / 8) * U, "weight")


@pytest.mark.gpu
@pytest.mark.parametrize("B,H,Hk,T", [(3, 4, 2, 1027), (1, 9, 1, 6001), (2600, 3, 3, 1), (5, 32, 8, 700)])
@pytest.mark.parametrize("xt,yt", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f32")])
@pytest.mark.parametrize("layout,grads", [("bhtd", "bhtd"), ("packed", "bhtd"), ("bhtd", "packed"), ("wide", "wide")])
def test_many_tokens(B, H, Hk, T, xt, yt, layout, grads):
    """Enough tokens for warps that go from one to the next, by heads and by tokens."""
    sections, eps = (8, 12, 12), 1e-6
    q, k = inputs(B + T, B, H, Hk, T, TYPES[xt], layout, 1.2)
    dq, dk = inputs(B * T + 1, B, H, Hk, T, TYPES[yt], grads, 0.7)
    g = torch.Generator(device="cuda").manual_seed(3)
    w = [1 + 0.3 * torch.randn(64, generator=g, device="cuda") for _ in range(2)]
    pos = torch.randint(0, 3000, (3, B, T), generator=g, device="cuda")
    angle = angles(pos, sections)
    turn = hk.rotary_forward(q, k, pos, sections, out_dtype=TYPES[yt])
    back = hk.rotary_backward(dq, dk, pos, sections, out_dtype=TYPES[xt])
    norm = hk.qk_norm_rotary_forward(q, k, *w, pos, sections, eps=eps, out_dtype=TYPES[yt])
    grad = hk.qk_norm_rotary_backward(q, k, dq, dk, *w, pos, sections, eps=eps)
    for i, (x, dy) in enumerate(((q, dq), (k, dk))):
        want = turned(x.double(), angle, False)
        close(turn[i], want, size_of_pairs(x.double(), False) * 8.01 * U + half_step(TYPES[yt], want) * (yt != "f32"), "turn")
        want = turned(dy.double(), -angle, False)
        zs = size_of_pairs(dy.double(), False)
        close(back[i], want, zs * 8.01 * U + half_step(TYPES[xt], want) * (xt != "f32"), "back")
        n, one = normed(x, w[i], eps), w[i].double()
        want = turned(n, angle, False)
        close(norm[i], want, size_of_pairs(n, False) * 20 * U + half_step(TYPES[yt], want) * (yt != "f32"), "norm")
        z = turned(dy.double(), -angle, False)
        inv = 1 / (x.double().square().mean(-1, keepdim=True) + eps).sqrt()
        n = x.double() * inv
        want = inv * (one * z - n * (one * z * n).mean(-1, keepdim=True))
        bound = inv * (zs * one.abs() * 22 * U + n.abs() * (zs * one.abs() * n.abs()).mean(-1, keepdim=True) * 55 * U)
        close(grad[i], want, bound + half_step(TYPES[xt], want) * (xt != "f32"), "norm back")
        # a lane's rows: those of its warp, eight lanes a row; then 32 lanes of a CTA, three CTAs, 64 threads
        rows = B * T * x.shape[1] / (148 * 8 * 4) * 3 + 8
        close(grad[2 + i], (z * n).sum((0, 1, 2)), (zs * n.abs()).sum((0, 1, 2)) * (20 + rows + 32 + 3 + 64) * U, "weight")


@pytest.mark.gpu
def test_gradients_against_differences():
    """Directional derivatives of the definition in 64 bits (central differences, step 1e-5: error of the order 1e-10)."""
    sections = (8, 12, 12)
    q, k = inputs(11, 2, 3, 2, 7, F32, "packed", 1.3)
    g = torch.Generator(device="cuda").manual_seed(12)
    wq, wk = (1 + 0.3 * torch.randn(64, generator=g, device="cuda") for _ in range(2))
    pos = torch.randint(0, 999, (3, 2, 7), generator=g, device="cuda", dtype=torch.int32)
    angle = angles(pos, sections)
    dq, dk = torch.randn_like(q), torch.randn_like(k)
    grads = hk.qk_norm_rotary_backward(q, k, dq, dk, wq, wk, pos, sections)

    def loss(q, k, wq, wk):
        return (turned(normed(q, wq, 1e-6), angle, False) * dq.double()).sum() + (turned(normed(k, wk, 1e-6), angle, False) * dk.double()).sum()

    at = [x.double() for x in (q, k, wq, wk)]
    for i in range(4):
        u = torch.randn(at[i].shape, generator=g, device="cuda", dtype=torch.float64)
        step = [x + 1e-5 * u * (j == i) if j == i else x for j, x in enumerate(at)], [x - 1e-5 * u if j == i else x for j, x in enumerate(at)]
        want = float((loss(*step[0]) - loss(*step[1])) / 2e-5)
        got = float((grads[i].double() * u).sum())
        size = float((grads[i].double() * u).abs().sum())
        assert abs(got - want) <= 1e-6 * size, (i, got, want)
    r = hk.rotary_backward(dq, dk, pos, sections)
    u = torch.randn(q.shape, generator=g, device="cuda", dtype=torch.float64)
    want = float((turned(u, angle, False) * dq.double()).sum())  # linear: its own derivative
    assert abs(float((r[0].double() * u).sum()) - want) <= 1e-6 * float((r[0].double() * u).abs().sum())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_results_in_place_and_in_given_tensors(dtype):
    q, k = inputs(3, 2, 5, 5, 37, TYPES[dtype], "packed")
    pos = torch.arange(37, device="cuda", dtype=torch.int32).expand(1, 2, 37)
    w = torch.rand(64, device="cuda")
    for call in (lambda **kw: hk.rotary_forward(q, k, pos, (32,), **kw), lambda **kw: hk.qk_norm_rotary_forward(q, k, w, w, pos, (32,), **kw)):
        base = q._base.clone()
        want = call()
        room = torch.full((2, 40, 12, 64), 7.0, device="cuda", dtype=q.dtype)
        oq, ok = room[:, 1:38, 1:6].transpose(1, 2), room[:, 1:38, 6:11].transpose(1, 2)
        got = call(out_q=oq, out_k=ok)
        assert got[0].data_ptr() == oq.data_ptr() and torch.equal(oq, want[0]) and torch.equal(ok, want[1])
        room[:, 1:38, 1:11] = 7.0
        assert bool((room == 7.0).all())  # nothing else was written
        call(out_q=q, out_k=k)
        assert torch.equal(q, want[0]) and torch.equal(k, want[1])
        q._base.copy_(base)


@pytest.mark.gpu
def test_captured_replayed_and_on_other_streams():
    q, k = inputs(4, 3, 4, 4, 100, F32, "bhtd")
    dq, dk = torch.randn_like(q), torch.randn_like(k)
    w = torch.rand(64, device="cuda")
    pos = torch.arange(100, device="cuda", dtype=torch.int32).expand(1, 3, 100)

    def both():
        return *hk.qk_norm_rotary_forward(q, k, w, w, pos, (32,)), *hk.qk_norm_rotary_backward(q, k, dq, dk, w, w, pos, (32,))

    want = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    for _ in range(2):  # two graphs at once, each with its own workspace
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = both()
        graphs.append((g, got, torch.cuda.Stream()))
    for g, got, s in graphs:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            for _ in range(3):
                g.replay()
    with torch.cuda.stream(side):
        on_side = both()
    given = hk.qk_norm_rotary_backward(q, k, dq, dk, w, w, pos, (32,), stream=side)
    torch.cuda.synchronize()
    for got in [x[1] for x in graphs] + [on_side]:
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert all(torch.equal(a, b) for a, b in zip(given, want[2:]))


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """A view whose last row starts 2^32 bytes and more behind its first."""
    x = torch.empty((2, 1 << 24, 2, 64), device="cuda", dtype=BF16)  # 8.6 GB
    T = 5
    q = x[:, -T:].transpose(1, 2)
    q.copy_(torch.randn(q.shape, device="cuda"))
    pos = torch.arange(T, device="cuda", dtype=torch.int32).expand(1, 2, T)
    want = hk.rotary_forward(q.contiguous(), None, pos, (32,))[0]
    assert torch.equal(hk.rotary_forward(q, None, pos, (32,))[0], want)
    hk.rotary_forward(q, None, pos, (32,), out_q=q)
    assert torch.equal(q, want)


@pytest.mark.gpu
def test_together_with_the_attention_in_training():
    """Norm and rotation, attention, and both backward passes, against autograd of the whole in 64 bits (the attention's own
    gate: its products are TF32)."""
    B, H, T, sections = 2, 3, 200, (8, 12, 12)
    q, k = inputs(5, B, H, H, T, F32, "packed", 1.2)
    g = torch.Generator(device="cuda").manual_seed(6)
    v, dO = (torch.randn((B, H, T, 64), generator=g, device="cuda") for _ in range(2))
    wq, wk = (1 + 0.2 * torch.randn(64, generator=g, device="cuda") for _ in range(2))
    pos = torch.randint(0, 300, (3, B, T), generator=g, device="cuda", dtype=torch.int32)
    qr, kr = hk.qk_norm_rotary_forward(q, k, wq, wk, pos, sections)
    O, LSE = hk.attention_forward(qr, kr, v, 0.125, True)
    dqr, dkr, dV, _ = hk.attention_backward(qr, kr, v, O, dO, LSE, 0.125, True)
    got = hk.qk_norm_rotary_backward(q, k, dqr, dkr, wq, wk, pos, sections)
    leaf = [x.double().requires_grad_() for x in (q, k, wq, wk, v)]
    angle = angles(pos, sections)
    s = turned(normed(leaf[0], leaf[2], 1e-6), angle, False) @ turned(normed(leaf[1], leaf[3], 1e-6), angle, False).transpose(2, 3) * 0.125
    s = s.masked_fill(torch.ones(T, T, device="cuda").triu(1).bool(), -math.inf)
    want_O = torch.softmax(s, -1) @ leaf[4]
    want_O.backward(dO.double())
    assert hk.last_device_status() == 0
    for a, b in [(O, want_O), (dV, leaf[4].grad), *zip(got, (x.grad for x in leaf[:4]))]:
        assert float((a.double() - b.detach()).norm() / b.detach().norm()) <= 1e-3


# ---- what is refused: none of these gets as far as a launch --------------------------------------------------------------------
def test_plan():
    p = hk.rotary_plan((3, 2), base=100.0)
    assert list(p.axis) == [0, 0, 0, 1, 1] + [255] * 27 and p.n_axes == 2 and p.interleaved == 0
    for i in range(5):
        assert abs(p.turn[i] / 2 ** 64 - 100.0 ** (-i / 32) / (2 * math.pi)) < 1e-15
    assert hk.rotary_plan((1,), frequencies=[2 * math.pi * 3.25], interleaved=True).turn[0] / 2 ** 64 == pytest.approx(0.25, abs=1e-14)
    assert hk.rotary_plan((1,), frequencies=[-1.0]).turn[0] / 2 ** 64 == pytest.approx(1 - 1 / (2 * math.pi), abs=1e-15)
    for bad in (dict(sections=(33,)), dict(sections=(16, 17)), dict(sections=(-1, 2)), dict(sections=()), dict(sections=(4,), base=0.0),
                dict(sections=(4,), base=math.nan), dict(sections=(2,), frequencies=[1.0, math.inf])):
        with pytest.raises(hk.HKError):
            hk.rotary_plan(**bad)
    with pytest.raises(ValueError):
        hk.rotary_plan((2,), frequencies=[1.0])


def _host():
    return torch.zeros(2, 3, 5, 64), torch.zeros(2, 1, 5, 64), torch.zeros(1, 2, 5, dtype=torch.int32), torch.zeros(64)


@pytest.mark.parametrize("name,wrong", [
    ("Q", torch.zeros(2, 3, 5, 32)), ("Q", torch.zeros(3, 5, 64)), ("Q", torch.zeros(2, 3, 5, 64, dtype=torch.float64)),
    ("Q", torch.zeros(2, 3, 64, 5).transpose(2, 3)), ("K", torch.zeros(1, 1, 5, 64)), ("K", torch.zeros(2, 1, 4, 64)),
    ("K", torch.zeros(2, 1, 5, 64, dtype=BF16)), ("dQ", torch.zeros(2, 2, 5, 64)), ("dK", torch.zeros(2, 1, 5, 64, dtype=F16)), ("dK", None),
    ("w_q", torch.zeros(32)), ("w_q", torch.zeros(128)[::2]), ("w_k", torch.zeros(64, dtype=BF16)), ("w_q", torch.zeros(64, dtype=torch.float64)),
    ("positions", torch.zeros(2, 5, dtype=torch.int32)), ("positions", torch.zeros(2, 2, 5, dtype=torch.int32)), ("positions", torch.zeros(1, 2, 5)),
    ("positions", torch.zeros(1, 1, 5, dtype=torch.int32)), ("out_q", torch.zeros(2, 3, 5, 64, dtype=BF16)), ("out_k", torch.zeros(2, 3, 5, 64))])
def test_arguments_that_do_not_fit_are_refused(name, wrong):
    q, k, pos, w = _host()
    args = dict(Q=q, K=k, dQ=q, dK=k, w_q=w, w_k=w, positions=pos, sections=(32,))
    args[name] = wrong
    with pytest.raises(AssertionError, match="^" + name if wrong is not None else None):
        hk.qk_norm_rotary_backward(**args)


@pytest.mark.parametrize("name", ["Q", "K", "w_q", "positions", "out_q"])
@pytest.mark.parametrize("wrong", [[1.0], 4096, False])
def test_what_is_no_tensor_is_refused(name, wrong):
    q, k, pos, w = _host()
    args = dict(Q=q, K=k, w_q=w, w_k=w, positions=pos, sections=(32,))
    args[name] = wrong
    with pytest.raises(TypeError, match=f"^{name}: expected a tensor"):
        hk.qk_norm_rotary_forward(**args)


def test_host_tensors_and_other_types_are_refused():
    q, k, pos, w = _host()
    with pytest.raises(AssertionError, match="CUDA"):
        hk.rotary_forward(q, k, pos, (32,))
    with pytest.raises(AssertionError, match="out_k"):
        hk.rotary_forward(q, None, pos, (32,), out_k=k)
    with pytest.raises(TypeError, match="out_dtype"):
        hk.rotary_forward(q, k, pos, (32,), out_dtype=torch.int32)
    with pytest.raises(TypeError):
        hk.rotary_backward(None, None, pos, (32,))


class _View(C.Structure):
    _fields_ = [("ptr", C.c_void_p), ("sB", C.c_int64), ("sM", C.c_int64), ("sH", C.c_int64)]


class _Block(C.Structure):
    _fields_ = [(n, _View) for n in ("q", "k", "q_out", "k_out", "dq_out", "dk_out", "dq", "dk")] + [
        ("q_weight", C.c_void_p), ("k_weight", C.c_void_p), ("dq_weight", C.c_void_p), ("dk_weight", C.c_void_p), ("positions", C.c_void_p),
        ("pos_strideA", C.c_int64), ("pos_strideB", C.c_int64), ("pos_strideT", C.c_int64), ("B", C.c_int), ("nh", C.c_int), ("nh_k", C.c_int),
        ("pos_bits", C.c_int), ("T", C.c_int64), ("dtype", C.c_int), ("out_dtype", C.c_int), ("weight_dtype", C.c_int), ("eps", C.c_float),
        ("plan", hk.RotaryPlan), ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t)]


def _block():
    b = _Block(B=2, nh=3, nh_k=1, T=5, pos_bits=32, positions=0x1000, eps=1e-6, plan=hk.rotary_plan((32,)), workspace=0x1000, workspace_bytes=1 << 24)
    for n in ("q", "k", "q_out", "k_out", "dq_out", "dk_out", "dq", "dk"):
        setattr(b, n, _View(0x1000, 15 * 64, 64, 5 * 64))
    return b


def _set(b, path, value):
    *head, last = path.split(".")
    for x in head:
        b = getattr(b, x)
    setattr(b, last, value)


@pytest.mark.parametrize("call,path,value,status", [
    ("rotary_forward", "q.ptr", None, -1), ("rotary_forward", "q_out.ptr", None, -1), ("rotary_backward", "dq_out.ptr", None, -1), ("rotary_backward", "dk.ptr", None, -1),
    ("qk_norm_rotary_backward", "dk_out.ptr", None, -1), ("qk_norm_rotary_backward", "k.ptr", None, -1), ("rotary_forward", "positions", None, -1),
    ("rotary_forward", "B", 0, -2), ("rotary_forward", "T", 0, -2), ("rotary_forward", "T", (1 << 30) + 1, -2), ("rotary_forward", "nh", 0, -2),
    ("rotary_forward", "nh_k", -1, -2), ("qk_norm_rotary_forward", "eps", -1.0, -2), ("qk_norm_rotary_forward", "eps", math.nan, -2), ("rotary_forward", "plan.n_axes", 0, -2),
    ("rotary_forward", "q.ptr", 0x1008, -3), ("rotary_forward", "q.sM", 66, -3), ("rotary_forward", "k_out.sB", 15 * 64 + 2, -3), ("rotary_forward", "positions", 0x1002, -3),
    ("qk_norm_rotary_forward", "q_weight", 0x1002, -3), ("qk_norm_rotary_backward", "dq_weight", 0x1002, -3), ("rotary_forward", "q.sH", -320, -3),
    ("rotary_forward", "q_out.sH", 0, -6), ("rotary_forward", "q_out.sM", 32, -6), ("rotary_forward", "dtype", 3, -6), ("rotary_forward", "out_dtype", -1, -6), ("rotary_forward", "pos_bits", 16, -6),
    ("qk_norm_rotary_backward", "workspace", None, -5), ("qk_norm_rotary_backward", "workspace_bytes", 100, -5), ("qk_norm_rotary_backward", "workspace", 0x1004, -5)])
def test_blocks_that_are_refused(call, path, value, status):
    b = _block()
    _set(b, path, value)
    f = getattr(hk.lib(), "hk_" + call)
    f.argtypes = [C.c_void_p, C.c_void_p]
    assert f(C.byref(b), None) == status
    assert f(None, None) == -1


def test_mixed_types_are_refused():
    for call, x, y, w in (("rotary_forward", 1, 2, 0), ("qk_norm_rotary_forward", 0, 1, 0), ("qk_norm_rotary_forward", 1, 2, 0), ("qk_norm_rotary_forward", 1, 1, 2)):
        b = _block()
        b.dtype, b.out_dtype, b.weight_dtype = x, y, w
        b.q_weight = 0x1000
        f = getattr(hk.lib(), "hk_" + call)
        f.argtypes = [C.c_void_p, C.c_void_p]
        assert f(C.byref(b), None) == -6, (call, x, y, w)


@pytest.mark.gpu
def test_small_results_are_tensors_of_their_own():
    """They may share an allocation, but no element, and what is done to one, or its end, leaves the others alone."""
    q, k = inputs(8, 3, 4, 2, 5, BF16, "packed")
    pos = torch.arange(5, device="cuda").expand(1, 3, 5)
    w = torch.ones(64, device="cuda", dtype=BF16)
    first = hk.qk_norm_rotary_backward(q, k, q, k, w, w, pos, (32,))
    want = [x.clone() for x in first]
    assert all(x.is_contiguous() and x.data_ptr() % 256 == 0 for x in first)
    spans = sorted((x.data_ptr(), x.data_ptr() + x.numel() * x.element_size()) for x in first)
    assert all(a[1] <= b[0] for a, b in zip(spans, spans[1:]))
    kept = first[3]
    for x in first[:3]:
        x.fill_(7.0)
    assert torch.equal(kept, want[3]) and kept._version == 0 and kept._base is None
    del first, x
    others = [hk.qk_norm_rotary_backward(q, k, q, k, w, w, pos, (32,)) for _ in range(20)]
    assert torch.equal(kept, want[3]) and all(torch.equal(a, b) for o in others for a, b in zip(o, want))
    with torch.inference_mode():
        assert torch.equal(hk.rotary_forward(q, None, pos, (32,))[0], hk.rotary_forward(q, None, pos, (32,))[0])
    leaf = hk.rotary_forward(q, None, pos, (32,), out_dtype=F32)[0].requires_grad_()  # as any tensor: autograd takes it for a leaf
    (leaf * 2.0).sum().backward()
    assert bool((leaf.grad == 2.0).all())
    huge = torch.zeros((1, 1, 1, 64), device="cuda").expand(1 << 20, 1 << 10, 1 << 20, 64)  # 2^58 bytes
    with pytest.raises((hk.HKError, RuntimeError)):
        hk.rotary_forward(huge, None, pos[:, :1, :1].expand(1, 1 << 20, 1 << 20), (32,))


# ---- results that lie on top of each other: B = 2, 3 heads of queries, 1 of keys, 5 tokens -------------------------------------------
@pytest.mark.parametrize("call,view", [("rotary_forward", "q_out"), ("rotary_backward", "dq"), ("qk_norm_rotary_forward", "q_out"), ("qk_norm_rotary_backward", "dq")])
@pytest.mark.parametrize("strides", [(64, 64, 64), (320, 320, 320), (960, 64, 64), (960, 128, 64), (640, 64, 256), (256, 64, 640), (64, 64, 1 << 40)])
def test_results_on_top_of_each_other_are_refused(call, view, strides):
    b = _block()
    v = getattr(b, view)
    v.sB, v.sM, v.sH = strides
    b.k_out.ptr = b.dk.ptr = 0x100000
    f = getattr(hk.lib(), "hk_" + call)
    f.argtypes = [C.c_void_p, C.c_void_p]
    assert f(C.byref(b), None) == -6


def test_results_that_lie_apart_get_past_that():
    f = hk.lib().hk_qk_norm_rotary_backward
    f.argtypes = [C.c_void_p, C.c_void_p]
    for strides in ((960, 64, 320), (960, 192, 64), (64, 384, 128), (320, 64, 640), (1 << 60, 1 << 40, 1 << 50)):
        b = _block()
        b.dq.sB, b.dq.sM, b.dq.sH = strides
        b.dk.ptr, b.workspace = 0x100000, None
        assert f(C.byref(b), None) == -5, strides
    for call, q, k in (("rotary_forward", "q_out", "k_out"), ("rotary_backward", "dq", "dk"), ("qk_norm_rotary_forward", "q_out", "k_out"), ("qk_norm_rotary_backward", "dq", "dk")):
        b = _block()  # the same memory for both
        assert getattr(b, q).ptr == getattr(b, k).ptr
        f = getattr(hk.lib(), "hk_" + call)
        f.argtypes = [C.c_void_p, C.c_void_p]
        assert f(C.byref(b), None) == -6


@pytest.mark.parametrize("base", [1.0, 100.0, 10000.0, 500000.0, 2.5e6, 1e30, 0.5, 1e-3])
@pytest.mark.parametrize("given", [False, True])
def test_fractions_of_a_turn_to_the_last_bits(base, given):
    """Against 50 decimal digits.  Numbers of 64 bits: the power is a step off (2^-63 of itself), 2 pi and the quotient half of one each, and
    the fraction is rounded to 2^-64: half a unit of that and four for every turn per position."""
    import decimal

    with decimal.localcontext() as c:
        c.prec = 50
        two_pi = 2 * decimal.Decimal("3.14159265358979323846264338327950288419716939937511")
        exact = [(decimal.Decimal(base).ln() * -p / 32).exp() for p in range(32)]
        plan = hk.rotary_plan((32,), frequencies=[float(x) for x in exact]) if given else hk.rotary_plan((32,), base=base)
        for p in range(32):
            turns = (decimal.Decimal(float(exact[p])) if given else exact[p]) / two_pi
            off = abs(plan.turn[p] - turns * 2 ** 64) % 2 ** 64
            assert min(off, 2 ** 64 - off) <= decimal.Decimal(0.5) + 4 * turns, p


@pytest.mark.gpu
def test_each_result_has_memory_of_its_own():
    """What keeps, shares or writes out one of them has nothing of the others."""
    import io

    q, k = inputs(8, 3, 4, 2, 5, BF16, "packed")
    pos, w = torch.arange(5, device="cuda").expand(1, 3, 5), torch.ones(64, device="cuda", dtype=BF16)
    lens = torch.full((3,), 5, device="cuda", dtype=torch.int32)
    for results in (hk.rotary_forward(q, k, pos, (32,)), hk.rotary_backward(q, k, pos, (32,)), hk.qk_norm_rotary_forward(q, k, w, w, pos, (32,)),
                    hk.qk_norm_rotary_backward(q, k, q, k, w, w, pos, (32,)), hk.shared_prefix_attention(q, k[0], k[0], k, k, lens, 0.125)):
        assert len({x.untyped_storage().data_ptr() for x in results}) == len(results)
        for x in results:
            assert x.storage_offset() == 0 and x.untyped_storage().nbytes() == x.numel() * x.element_size()
            file = io.BytesIO()
            torch.save(x, file)
            assert file.tell() < x.numel() * x.element_size() + 4096
