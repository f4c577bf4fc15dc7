"""Attention of a batch that shares a prefix, against the definition in 64 bits, request by request.

Error bounds (u = 2^-24).  A score in fp32 is a sum of 64 products: 80 u of the sum of the products' sizes, whatever the order;
so its exponential is off by that much of itself (D), and O, a weighted mean, by 2 D of the mean of |v| plus the roundings of
sums over the keys, taken by blocks of at most 128 keys and 64 blocks in a row: 200 u.  The exponential's own error (2 u) and the
argument's rounding (u times its size, below 64 in log2 units here) are 70 u.  Sixteen-bit types round each weight and the result
by half a step; their products are exact in fp32."""
import ctypes as C
import math

import pytest
import torch

import hyperkernels_b200 as hk

U = 2.0 ** -24
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SCALE = 0.125


def make(seed, B, H, Hk, T, P, S, dtype, layout="bhtd", lengths=None, junk=math.nan, sigma=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = TYPES[dtype]

    def rand(*shape):
        return (torch.randn(shape, generator=g, device="cuda") * sigma).to(t)

    if layout == "bthd":
        q = rand(B, T, H, 64).transpose(1, 2)
        kp, vp = (rand(P, Hk, 64).transpose(0, 1) for _ in range(2))
        k, v = (rand(B, S, Hk, 64).transpose(1, 2) for _ in range(2))
    elif layout == "wide":  # rows of a fused cache: keys and values side by side, with room between heads
        q = rand(B, H, T, 192)[..., 64:128]
        kp, vp = (lambda x: (x[..., :64], x[..., 64:]))(rand(Hk, P + 3, 128)[:, :P])
        k, v = (lambda x: (x[..., :64], x[..., 64:]))(rand(B, Hk, S + 5, 128)[:, :, :S])
    else:
        q = rand(B, H, T, 64)
        kp, vp = (rand(Hk, P, 64) for _ in range(2))
        k, v = (rand(B, Hk, S, 64) for _ in range(2))
    if lengths is None:
        lengths = [(7 * b + 3) % (S + 1) for b in range(B)]
    for b, n in enumerate(lengths):  # what is behind a request's last key must not matter
        k[b, :, max(0, n):], v[b, :, max(0, n):] = junk, junk
    return q, kp, vp, k, v, torch.tensor(lengths, device="cuda", dtype=torch.int32)


def definition(q, kp, vp, k, v, lens, causal, scale=SCALE):
    """O, LSE, and for the bounds the mean of |v| under the softmax and the largest sum of products' sizes of a row"""
    B, H, T, _ = q.shape
    G, P = H // k.shape[1], kp.shape[-2]
    O, LSE, mean, size = (torch.zeros((B, H, T, n), device="cuda", dtype=torch.float64) for n in (64, 1, 64, 1))
    for b in range(B):
        n = min(max(int(lens[b]), 0), k.shape[2])
        kk = torch.cat([kp, k[b, :, :n]], 1).double().repeat_interleave(G, 0)
        vv = torch.cat([vp, v[b, :, :n]], 1).double().repeat_interleave(G, 0)
        x = q[b].double() @ kk.transpose(1, 2) * scale
        if causal:
            own = torch.arange(P + n, device="cuda") - P
            x = x.masked_fill((own >= 0) & (own > n - T + torch.arange(T, device="cuda")[:, None]), -math.inf)
        if P + n == 0:
            LSE[b] = -math.inf
            continue
        w = torch.nan_to_num(torch.softmax(x, -1))  # rows that see nothing
        O[b], mean[b], LSE[b, ..., 0] = w @ vv, w @ vv.abs(), torch.logsumexp(x, -1)
        size[b] = (q[b].double().abs() @ kk.abs().transpose(1, 2) * abs(scale)).amax(-1, keepdim=True)
    return O, LSE[..., 0], mean, size[..., 0]


def check(got, want, dtype, what=""):
    (o, lse), (O, LSE, mean, size) = got, want
    step = torch.finfo(TYPES[dtype]).eps / 2 if dtype != "f32" else 0.0
    d = (80 * size + 70) * U
    bound = (2 * d[..., None] + 200 * U + step) * mean + step * O.abs() + (2.0 ** -25 if dtype == "f16" else 1e-30)
    off = (o.double() - O).abs()
    assert o.dtype == TYPES[dtype] and lse.dtype == torch.float32
    assert bool((off <= bound).all()), (what, float((off - bound).max()), float(off.max()))
    seen = LSE > -math.inf
    assert torch.equal(lse > -math.inf, seen), what
    assert bool((o[~seen] == 0).all()), what
    assert bool(((lse.double() - LSE).abs()[seen] <= (d + 200 * U + 4 * U * LSE.abs())[seen]).all()), what
    if dtype == "f32" and bool(seen.any()):  # fp32 throughout: roundings that do not add up all one way
        assert float((o.double() - O).norm() / O.norm()) <= 1e-5, what


# (B, H, Hk, T, P, S): one token to long, odd sizes, groups, empty parts, tiles' borders
SIZES = [
    (1, 1, 1, 1, 1, 1), (1, 1, 1, 1, 0, 5), (2, 2, 1, 1, 7, 0), (4, 12, 12, 1, 333, 64), (3, 6, 2, 1, 130, 257), (16, 4, 4, 1, 1000, 65),
    (64, 8, 2, 1, 515, 100), (5, 3, 3, 2, 128, 128), (2, 8, 1, 3, 64, 33), (9, 8, 2, 5, 129, 300), (3, 4, 4, 17, 127, 63), (2, 4, 2, 77, 500, 333),
    (2, 3, 3, 128, 256, 128), (1, 2, 1, 200, 100, 450), (2, 2, 2, 300, 0, 300), (70, 1, 1, 1, 40, 9), (1, 16, 1, 9, 2000, 0), (1, 1, 1, 130, 5, 131),
    (33, 5, 5, 4, 65, 20), (1, 32, 8, 1, 5000, 700)]


@pytest.mark.gpu
@pytest.mark.parametrize("B,H,Hk,T,P,S", SIZES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("layout", ["bhtd", "bthd", "wide"])
def test_against_the_definition(B, H, Hk, T, P, S, dtype, causal, layout):
    x = make(B + P, B, H, Hk, T, P, S, dtype, layout)
    got = hk.shared_prefix_attention(*x, SCALE, causal)
    check(got, definition(*x, causal), dtype)
    assert hk.last_device_status() == 0
    again = hk.shared_prefix_attention(*x, SCALE, causal)
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])


# sizes for each way of cutting the work: few rows and many, the prefix in runs and in one go with the requests' own keys, blocks of
# rows in parts of their keys
WAYS = [
    (4, 12, 12, 1, 333, 64, "f32"), (64, 8, 2, 1, 515, 100, "f16"), (5, 6, 6, 2, 130, 70, "f32"), (3, 4, 4, 9, 90, 61, "f32"),
    (1, 2, 1, 1, 9000, 500, "f32"), (2, 1, 1, 1, 9001, 500, "f32"), (1, 4, 4, 2, 9000, 513, "f32"), (16, 4, 4, 1, 4000, 300, "f32"),
    (8, 4, 2, 1, 4000, 700, "f32"), (4, 12, 4, 1, 3000, 400, "f32"), (20, 8, 2, 1, 3001, 400, "bf16"), (1, 2, 2, 24, 20000, 100, "f16"),
    (4, 4, 4, 1, 3000, 0, "bf16"), (40, 8, 2, 1, 3000, 0, "f32"), (9, 4, 4, 1, 0, 4000, "f32"), (300, 4, 2, 1, 0, 400, "f16"),
    (64, 32, 8, 1, 8192, 1000, "bf16"), (64, 32, 8, 1, 4100, 1000, "f32"), (16, 8, 2, 20, 2500, 300, "bf16"),
    (16, 4, 4, 40, 2500, 300, "f32"), (16, 4, 4, 77, 4097, 333, "f16"), (700, 8, 1, 1, 3000, 0, "bf16"), (700, 8, 1, 1, 3001, 0, "f32"),
    (40, 4, 4, 260, 300, 300, "bf16"), (37, 4, 2, 129, 301, 300, "f16"), (3, 4, 4, 300, 900, 400, "f32"), (3, 8, 2, 301, 901, 403, "bf16"),
    (40, 4, 4, 130, 300, 140, "f32"), (2, 4, 4, 700, 0, 700, "bf16"), (2, 4, 4, 700, 0, 701, "f32"), (5, 8, 2, 512, 3001, 700, "f16"),
    (37, 4, 4, 100, 1, 129, "bf16"), (37, 4, 4, 100, 64, 65, "f32"), (1, 3000, 3000, 1, 70, 0, "f32"), (3, 2400, 2400, 1, 33, 0, "bf16"),
    (1, 5000, 2500, 3, 40, 9, "f16")]


def test_the_sizes_take_every_way():
    """On the 148 SMs that the library takes where there is no device."""
    f = hk.lib().hk_shared_prefix_plan
    f.argtypes = [C.c_void_p, C.POINTER(C.c_int)]
    seen = set()
    for B, H, Hk, T, P, S, dtype in WAYS:
        b = _block()
        b.B, b.nh, b.nh_kv, b.T, b.prefix_len, b.kv_len, b.dtype = B, H, Hk, T, P, S, list(TYPES).index(dtype)
        plan = (C.c_int * 6)()
        assert f(C.byref(b), plan) == 0
        prefix_many, own_many, whole, runs, own_runs, slots = plan
        assert slots == (slots if whole else runs + own_runs) and slots >= 1 and (runs > 0 or whole or P == 0) and (own_runs > 0 or S == 0)
        kind = ("f32" if dtype == "f32" else "16", "many" if own_many else "few")
        seen.add(kind + (("whole", slots > 1) if whole else ("many" if prefix_many else "few" if runs else "no prefix", own_runs > 0)))
    for d in ("f32", "16"):
        assert {(d, "few", "whole", False), (d, "few", "few", True), (d, "few", "few", False), (d, "few", "many", True), (d, "many", "many", True),
                (d, "many", "whole", True), (d, "many", "whole", False)} <= seen, sorted(x for x in seen if x[0] == d)
    assert {("f32", "few", "no prefix", True), ("16", "few", "many", False)} <= seen, sorted(seen)


@pytest.mark.gpu
@pytest.mark.parametrize("B,H,Hk,T,P,S,dtype", WAYS)
@pytest.mark.parametrize("causal,layout", [(True, "bhtd"), (True, "wide"), (False, "bthd")])
def test_every_way_of_cutting_the_work(B, H, Hk, T, P, S, dtype, causal, layout):
    x = make(B + T, B, H, Hk, T, P, S, dtype, layout, junk=math.nan if layout == "bhtd" else math.inf)
    got = hk.shared_prefix_attention(*x, SCALE, causal)
    check(got, definition(*x, causal), dtype)
    again = hk.shared_prefix_attention(*x, SCALE, causal)
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])
    assert hk.last_device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("B,H,Hk,T,P,S,dtype", [
    (64, 32, 8, 1, 4100, 1000, "f32"), (3, 4, 4, 300, 900, 400, "f32"), (8, 12, 12, 77, 4096, 333, "f32"), (64, 32, 8, 1, 8192, 1000, "bf16"),
    (5, 8, 2, 512, 3001, 700, "f16"), (16, 12, 12, 1, 2047, 512, "f32")])
def test_the_same_bits_however_late_the_keys_come(B, H, Hk, T, P, S, dtype):
    """Every other call finds its keys in the L2, the others in memory: tiles land in other orders and at other times."""
    x = make(B + T, B, H, Hk, T, P, S, dtype, "bthd")
    want = hk.shared_prefix_attention(*x, SCALE)
    check(want, definition(*x, True), dtype)
    room = torch.empty(1 << 28, device="cuda", dtype=torch.uint8)
    different = torch.zeros((), device="cuda", dtype=torch.int64)
    for i in range(400):
        if i % 2:
            room.fill_(i & 255)
        o, lse = hk.shared_prefix_attention(*x, SCALE)
        different += (o != want[0]).any() | (lse != want[1]).any()
    assert int(different) == 0 and hk.last_device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T", [1, 3, 40, 150, 400])
@pytest.mark.parametrize("P", [0, 70, 2600])
def test_lengths_at_borders_and_outside(dtype, T, P):
    """Empty, one, tiles' ends and the rows next to them, full, and lengths that the cache does not have (taken into it)."""
    lengths = [0, 1, 2, 63, 64, 65, 127, 128, 129, 191, 192, 193, 255, 256, 300, -4, 1000000]
    x = make(T, len(lengths), 4, 2, T, P, 300, dtype, lengths=lengths)
    for junk in (math.nan, math.inf, 60000.0):
        for b, n in enumerate(lengths):
            x[3][b, :, max(0, n):], x[4][b, :, max(0, n):] = junk, junk
        for causal in (True, False):
            check(hk.shared_prefix_attention(*x, SCALE, causal), definition(*x, causal), dtype, (junk, causal))
    assert hk.last_device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T", [1, 6, 130])
def test_no_lengths_means_all(dtype, T):
    x = list(make(1, 3, 4, 4, T, 90, 200, dtype, lengths=[200] * 3))
    full = hk.shared_prefix_attention(*x, SCALE)
    x[5] = None
    none = hk.shared_prefix_attention(*x, SCALE)
    assert torch.equal(full[0], none[0]) and torch.equal(full[1], none[1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,P,S", [(1, 4000, 60), (3, 4000, 0), (150, 4000, 200), (700, 2000, 700), (140, 0, 300)])
def test_many_small_weights_beside_a_large_one(dtype, T, P, S):
    """The first key takes nearly all, and its value is 0: the result is what the others give, each 2^-26 of the first.

    A weight of 2^-26.1 or more (26 ln 2 rounds to within 0.1), lifted by seven binary places in fp16, is rounded there to a multiple of
    2^-24: by 2^-25 in 2^-19.1 at most; in the other types by half a step.  The score of the first key is 26 ln 2 more than that of the others, which is 0; a score's error of
    d = 80 u * 26 + 70 u moves all weights by less than 2 d, and a rounding of the result to fp16 is 2^-25 at most below 2^-14."""
    t = TYPES[dtype]
    q = torch.zeros((2, 2, T, 64), device="cuda", dtype=t)
    q[..., 0] = 26.0 * math.log(2.0)
    kp, vp = (torch.full((2, P, 64), x, device="cuda", dtype=t) for x in (0.0, 1.0))
    k, v = (torch.full((2, 2, S, 64), x, device="cuda", dtype=t) for x in (0.0, 1.0))
    first = (kp[:, 0], vp[:, 0]) if P else (k[:, :, 0], v[:, :, 0])
    first[0][..., 0], first[1][:] = 1.0, 0.0
    lens = torch.full((2,), S, device="cuda", dtype=torch.int32)
    o, lse = hk.shared_prefix_attention(q, kp, vp, k, v, lens, 1.0, True)
    O, LSE, _, _ = definition(q, kp, vp, k, v, lens, True, 1.0)
    d = (80 * 26 + 70) * U
    step = torch.finfo(t).eps / 2 if dtype != "f32" else 0.0
    weight = 2.0 ** -5.9 if dtype == "f16" else step
    assert bool(((o.double() - O).abs() <= (2 * d + 200 * U + weight + step) * O + (2.0 ** -25 if dtype == "f16" else 0.0)).all())
    assert bool(((lse.double() - LSE).abs() <= d + 200 * U + 4 * U * LSE.abs()).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,P,S", [(140, 390, 0), (300, 0, 300), (3, 390, 5)])
@pytest.mark.parametrize("height", [4.0, 30.0, 90.0, 1000.0, 40000.0])
def test_one_late_key_that_takes_all(height, T, P, S, dtype):
    """Scores of about 1, and in each column of the second and third tile, in turn, one key of `height` (16-bit types hold all five)."""
    t = TYPES[dtype]
    x = list(make(9, 1, 1, 1, T, P, S, dtype, lengths=[S], sigma=0.3))
    x[0][..., 0] = 1.0
    keys, values, n = (x[1], x[2], P) if P else (x[3][:, 0], x[4][:, 0], S)
    keys[..., 0] = 0.0
    step = torch.finfo(t).eps / 2 if dtype != "f32" else 0.0
    for at in range(128, min(n, 384), 1 if height == 90.0 else 7):
        keys[0, at, 0] = height
        O, LSE, mean, size = definition(*x, P > 0, 1.0)
        o, lse = hk.shared_prefix_attention(*x, 1.0, P > 0)
        keys[0, at, 0] = 0.0
        d = (80 * size + 3 * size.clamp(min=1) * 1.45 + 70) * U
        bound = (2 * d[..., None] + 200 * U + step) * mean + step * O.abs() + (2.0 ** -25 if dtype == "f16" else 1e-30)
        assert bool(((o.double() - O).abs() <= bound).all()), at
        assert bool(((lse.double() - LSE).abs() <= d + 200 * U + 4 * U * LSE.abs()).all()), at
    assert hk.last_device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,T,P,S", [(2, 1, 300, 40), (2, 3, 0, 200), (2, 140, 300, 300), (2, 300, 1000, 300), (8, 40, 1500, 100), (2, 140, 0, 300)])
def test_scores_that_are_no_numbers(H, T, P, S, dtype):
    """Scores that are NaN, in any column of a tile, make NaN of the rows that see them; the others stay as they were."""
    x = make(5, 2, H, 2, T, P, S, dtype, lengths=[S, S - 3])
    want = definition(*x, True)
    plain = hk.shared_prefix_attention(*x, SCALE)
    check(plain, want, dtype)
    first = (S - 3) - T  # keys that all rows of request 1 see, with one more for each row
    for at in list(range(3)) + list(range(60, 70)) + [127, 128, 129] + list(range(134, 140)) + [188, 255]:
        for bad in (math.nan, math.inf):
            for where in ("prefix", "own"):
                if at >= (P if where == "prefix" else first):
                    continue
                k, rows = (x[1][0], slice(None)) if where == "prefix" else (x[3][1, 0], slice(1, 2))
                keep = k[at].clone()
                k[at] = bad  # infinities of both signs meet in a score
                o, lse = hk.shared_prefix_attention(*x, SCALE)
                k[at] = keep
                hit, G = torch.zeros_like(lse, dtype=torch.bool), H // 2
                hit[rows, :G] = True
                assert bool(o[hit].isnan().all()) and bool(lse[hit].isnan().all()), (at, bad, where)
                assert torch.equal(o[~hit], plain[0][~hit]) and torch.equal(lse[~hit], plain[1][~hit]), (at, bad, where)
    assert hk.last_device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T", [1, 20, 140])
def test_large_scores_and_other_scales(dtype, T):
    """Scores of +-200: one key takes almost everything, the maximum moves late, masked keys would be the largest."""
    x = make(3, 3, 4, 2, T, 200, 150, dtype, lengths=[100, 150, 0], sigma=1.0)
    x[1][:, 150:] *= 3.0
    x[3][:, :, :100] *= 3.0
    for scale in (1.0, -0.7, 1e-3):
        O, LSE, mean, size = definition(*x, True, scale)
        o, lse = hk.shared_prefix_attention(*x, scale, True)
        d = (80 * size + 3 * size.clamp(min=1) * 1.45 + 70) * U  # the exponent's argument in log2 units is as large as the scores
        step = torch.finfo(TYPES[dtype]).eps / 2 if dtype != "f32" else 0.0
        bound = (2 * d[..., None] + 200 * U + step) * mean + step * O.abs() + (2.0 ** -25 if dtype == "f16" else 1e-30)
        assert bool(((o.double() - O).abs() <= bound).all()), scale
        assert bool(((lse.double() - LSE).abs() <= d + 200 * U + 4 * U * LSE.abs()).all()), scale
    assert hk.last_device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 5, 150])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_given_tensors_graphs_and_streams(dtype, T):
    x = make(5, 4, 8, 2, T, 700, 260, dtype, lengths=[260, 200, 151, 160])
    want = hk.shared_prefix_attention(*x, SCALE)
    room = torch.full((4, T + 2, 9, 64), 7.0, device="cuda", dtype=TYPES[dtype])
    out = room[:, 1:T + 1, :8].transpose(1, 2)
    lse_room = torch.full((4, 8, T + 3), 7.0, device="cuda")
    got = hk.shared_prefix_attention(*x, SCALE, out=out, lse=lse_room[..., :T])
    assert got[0].data_ptr() == out.data_ptr() and torch.equal(out, want[0]) and torch.equal(lse_room[..., :T], want[1])
    room[:, 1:T + 1, :8] = 7.0
    assert bool((room == 7.0).all()) and bool((lse_room[..., T:] == 7.0).all())
    # two graphs, each with a workspace of its own, replayed side by side; lengths are read at replay
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            r = hk.shared_prefix_attention(*x, SCALE)
        graphs.append((g, r, torch.cuda.Stream()))
    for lens in ([260, 200, 151, 160], [150, 260, 0, 1]):
        x[5].copy_(torch.tensor(lens, dtype=torch.int32))
        for b, n in enumerate(lens):
            x[3][b, :, :n] = torch.nan_to_num(x[3][b, :, :n], 0.25)
            x[4][b, :, :n] = torch.nan_to_num(x[4][b, :, :n], 0.5)
        want = hk.shared_prefix_attention(*x, SCALE)
        torch.cuda.synchronize()
        for _ in range(3):
            for g, _, s in graphs:
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for _, r, _ in graphs:
            assert torch.equal(r[0], want[0]) and torch.equal(r[1], want[1])
        check(want, definition(*x, True), dtype)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(50_000_000)
    r = hk.shared_prefix_attention(*x, SCALE, stream=side)  # its workspace is given back before the kernels have begun
    others = [torch.full((1 << 22,), 3.0, device="cuda") for _ in range(4)]
    torch.cuda.synchronize()
    assert torch.equal(r[0], want[0]) and torch.equal(r[1], want[1]) and all(bool((t == 3.0).all()) for t in others)
    assert hk.last_device_status() == 0


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """A cache whose last request starts more than 2^32 elements behind the first."""
    B, Hk, S = 3, 2, 1 << 24
    cache = torch.empty((B, Hk, S, 64), device="cuda", dtype=torch.bfloat16)  # 12.9 GB
    x = list(make(6, B, 4, Hk, 1, 100, 500, "bf16"))
    want = hk.shared_prefix_attention(*x, SCALE)
    cache[:, :, :500] = x[3]
    values = x[4]
    x[3] = cache
    big = torch.empty((B, Hk, S, 64), device="cuda", dtype=torch.bfloat16)
    big[:, :, :500] = values
    x[4] = big
    got = hk.shared_prefix_attention(*x, SCALE)
    # the work may be cut otherwise: the sums' order differs, a result by a step of its type
    assert torch.allclose(got[0].float(), want[0].float(), rtol=2.0 ** -7, atol=2.0 ** -9) and torch.allclose(got[1], want[1], atol=1e-5)


@pytest.mark.gpu
def test_views_that_a_tensor_map_cannot_describe_are_refused():
    """A stride of 0 over heads or requests, as attention_forward refuses it; queries may be broadcast."""
    x = list(make(7, 3, 4, 2, 1, 60, 50, "f32"))
    want = hk.shared_prefix_attention(*x, SCALE)
    one = x[0][:, :1].expand(3, 4, 1, 64)
    same = hk.shared_prefix_attention(one, *x[1:], SCALE)
    copy = hk.shared_prefix_attention(one.contiguous(), *x[1:], SCALE)
    assert torch.equal(same[0], copy[0])
    for i in (1, 2):
        y = list(x)
        y[i] = y[i][:1].expand(2, 60, 64)
        with pytest.raises(hk.HKError, match="unsupported"):
            hk.shared_prefix_attention(*y, SCALE)
    for i in (3, 4):
        y = list(x)
        y[i] = y[i][:1].expand(3, 2, 50, 64)
        with pytest.raises(hk.HKError, match="unsupported"):
            hk.shared_prefix_attention(*y, SCALE)
    assert torch.equal(hk.shared_prefix_attention(*x, SCALE)[0], want[0])


@pytest.mark.gpu
def test_two_threads_on_streams_of_their_own():
    import threading

    cases = [make(i, 16, 8, 2, T, 3000, 300, "bf16") for i, T in enumerate((1, 20))]
    want = [hk.shared_prefix_attention(*x, SCALE) for x in cases]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(50):
                got = hk.shared_prefix_attention(*cases[i], SCALE)
                s.synchronize()
                if not (torch.equal(got[0], want[i][0]) and torch.equal(got[1], want[i][1])):
                    bad.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad and hk.last_device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_serving_loop(dtype):
    """A prompt's common part goes into the prefix once; then requests of different lengths take a first chunk and decode: norm and
    rotation, append, attention.  Every step against the whole computed again in 64 bits."""
    t, B, H, Hk, P, S = TYPES[dtype], 5, 6, 3, 150, 40
    g = torch.Generator(device="cuda").manual_seed(9)
    w = [(1 + 0.2 * torch.randn(64, generator=g, device="cuda")) for _ in range(2)]

    def project(batch, T):
        return [torch.randn((batch, n, T, 64), generator=g, device="cuda").to(t) for n in (H, Hk, Hk)]

    _, k, v = project(1, P)
    pos = torch.arange(P, device="cuda", dtype=torch.int32)[None, None]
    kp, vp = hk.qk_norm_rotary_forward(k, None, w[1], None, pos, (32,))[0][0], v[0]
    K, V = (torch.full((B, Hk, S, 64), math.nan, device="cuda", dtype=t) for _ in range(2))
    lens = torch.zeros(B, device="cuda", dtype=torch.int32)
    for step, new in enumerate([7, 1, 1, 1, 3, 1]):
        q, k, v = project(B, new)
        start = lens.clone()
        if step == 0:
            start += torch.arange(B, device="cuda", dtype=torch.int32)  # requests that are some tokens in already
            K[:, :, :B], V[:, :, :B] = 0.5, -0.25
        lens = start + new
        pos = (P + start[:, None] + torch.arange(new, device="cuda"))[None].to(torch.int32)
        q, k = hk.qk_norm_rotary_forward(q, k, *w, pos, (32,))
        rows = (start[:, None] + torch.arange(new, device="cuda"))[:, None, :, None].expand(B, Hk, new, 64)
        K.scatter_(2, rows, k)
        V.scatter_(2, rows, v)
        got = hk.shared_prefix_attention(q, kp, vp, K, V, lens, SCALE)
        check(got, definition(q, kp, vp, K, V, lens, True), dtype, step)


# ---- what is refused: none of these gets as far as a launch --------------------------------------------------------------------
def _host():
    return dict(Q=torch.zeros(2, 4, 3, 64), K_prefix=torch.zeros(2, 9, 64), V_prefix=torch.zeros(2, 9, 64), K=torch.zeros(2, 2, 8, 64),
                V=torch.zeros(2, 2, 8, 64), lengths=torch.zeros(2, dtype=torch.int32), scale=SCALE)


@pytest.mark.parametrize("name,wrong", [
    ("Q", torch.zeros(2, 4, 3, 32)), ("Q", torch.zeros(2, 4, 3, 64, dtype=torch.float64)), ("K", torch.zeros(3, 2, 8, 64)), ("K", torch.zeros(2, 2, 64, 8).transpose(2, 3)),
    ("V", torch.zeros(2, 2, 7, 64)), ("V", torch.zeros(2, 2, 8, 64, dtype=torch.bfloat16)), ("K_prefix", torch.zeros(3, 9, 64)), ("K_prefix", torch.zeros(2, 2, 9, 64)),
    ("K_prefix", torch.zeros(9, 64)), ("V_prefix", torch.zeros(2, 8, 64)), ("lengths", torch.zeros(3, dtype=torch.int32)), ("lengths", torch.zeros(2, dtype=torch.int64)),
    ("lengths", torch.zeros(4, dtype=torch.int32)[::2]), ("out", torch.zeros(2, 4, 3, 64, dtype=torch.float16)), ("out", torch.zeros(2, 4, 2, 64)),
    ("lse", torch.zeros(2, 4, 4)), ("lse", torch.zeros(2, 4, 3, dtype=torch.float64))])
def test_arguments_that_do_not_fit_are_refused(name, wrong):
    with pytest.raises(AssertionError, match="^" + name):
        hk.shared_prefix_attention(**{**_host(), name: wrong})


@pytest.mark.parametrize("name", ["Q", "K_prefix", "V_prefix", "K", "V", "lengths", "workspace", "out", "lse"])
@pytest.mark.parametrize("wrong", [[1.0], 4096, False])
def test_what_is_no_tensor_is_refused(name, wrong):
    with pytest.raises(TypeError, match=f"^{name}: expected a tensor"):
        hk.shared_prefix_attention(**{**_host(), name: wrong})


def test_host_tensors_are_refused():
    with pytest.raises(AssertionError, match="CUDA"):
        hk.shared_prefix_attention(**_host())


class _View(C.Structure):
    _fields_ = [("ptr", C.c_void_p), ("sB", C.c_int64), ("sM", C.c_int64), ("sH", C.c_int64)]


class _Block(C.Structure):
    _fields_ = [(n, _View) for n in ("Q", "Kp", "Vp", "K", "V", "O")] + [
        ("LSE", C.c_void_p), ("lse_sB", C.c_int64), ("lse_sH", C.c_int64), ("lengths", C.c_void_p), ("B", C.c_int), ("nh", C.c_int), ("nh_kv", C.c_int),
        ("dtype", C.c_int), ("T", C.c_int64), ("prefix_len", C.c_int64), ("kv_len", C.c_int64), ("scale", C.c_float), ("is_causal", C.c_bool),
        ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t)]


def _block():
    b = _Block(LSE=0x1000, lse_sB=12, lse_sH=3, lengths=0x1000, B=2, nh=4, nh_kv=2, T=3, prefix_len=9, kv_len=8, scale=SCALE, workspace=0x1000, workspace_bytes=1 << 30)
    for n, rows, heads in (("Q", 3, 4), ("Kp", 9, 2), ("Vp", 9, 2), ("K", 8, 2), ("V", 8, 2), ("O", 3, 4)):
        setattr(b, n, _View(0x1000, heads * rows * 64, 64, rows * 64))
    return b


@pytest.mark.parametrize("path,value,status", [
    ("Q.ptr", None, -1), ("Kp.ptr", None, -1), ("V.ptr", None, -1), ("O.ptr", None, -1), ("LSE", None, -1), ("B", 0, -2), ("nh", 0, -2), ("nh_kv", 0, -2), ("nh_kv", 3, -2),
    ("T", 0, -2), ("T", (1 << 30) + 1, -2), ("prefix_len", -1, -2), ("kv_len", -1, -2), ("kv_len", (1 << 30) + 1, -2), ("scale", 0.0, -2), ("scale", math.inf, -2), ("scale", math.nan, -2),
    ("Q.ptr", 0x1004, -3), ("K.sM", 66, -3), ("Vp.sH", 9 * 64 + 2, -3), ("K.sB", -1024, -3), ("lengths", 0x1002, -3), ("LSE", 0x1002, -3),
    ("lse_sB", 2, -6), ("lse_sH", 0, -6), ("O.sM", 0, -6), ("O.sH", 32, -6), ("Kp.sH", 0, -6), ("K.sB", 0, -6), ("V.sM", 0, -6), ("dtype", 3, -6), ("dtype", -1, -6)])
def test_blocks_that_are_refused(path, value, status):
    b = _block()
    *head, last = path.split(".")
    x = b
    for n in head:
        x = getattr(x, n)
    setattr(x, last, value)
    f = hk.lib().hk_shared_prefix_attention
    f.argtypes = [C.c_void_p, C.c_void_p]
    assert f(C.byref(b), None) == status
    assert f(None, None) == -1


# ---- calls behind other launches -----------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("B,H,Hk,T,P,S,dtype", [
    (4, 12, 12, 1, 333, 64, "f32"), (16, 12, 12, 1, 2047, 512, "f32"), (2, 1, 1, 1, 9001, 500, "f32"), (4, 12, 4, 1, 3000, 400, "f32"), (64, 32, 8, 1, 8192, 1000, "bf16"),
    (64, 8, 2, 1, 515, 100, "f16"), (300, 4, 2, 1, 0, 400, "f16"), (16, 8, 2, 20, 2500, 300, "bf16"), (16, 4, 4, 77, 4097, 333, "f32"), (37, 4, 4, 100, 1, 160, "bf16")])
@pytest.mark.parametrize("last", ["lengths", "queries"])
def test_lengths_and_queries_written_by_the_launch_before(B, H, Hk, T, P, S, dtype, last):
    """A decoding loop without a synchronisation: each step's queries and lengths come from the launches right before the call, in the
    memory that the step before used.  Every step has the bits of the same call on inputs that were there long before."""
    steps, t = 24, TYPES[dtype]
    _, kp, vp, k, v, _ = make(B + T, B, H, Hk, T, P, S, dtype, lengths=[S] * B)
    g = torch.Generator(device="cuda").manual_seed(4)
    rows = torch.randn((steps, B, H, T, 64), generator=g, device="cuda").to(t)
    pos = torch.randint(0, 9000, (1, B, T), generator=g, device="cuda", dtype=torch.int32)
    first = (torch.arange(B, device="cuda") % (S - T - steps) + T).to(torch.int32)
    q, lens, got = torch.zeros((B, H, T, 64), device="cuda", dtype=t), first.clone(), []
    torch.cuda.synchronize()
    torch.cuda._sleep(20_000_000)  # all steps are in the queue before the first one runs
    for i in range(steps):
        if last == "queries":
            lens.add_(1)
        hk.rotary_forward(rows[i], None, pos, (32,), out_q=q)
        if last == "lengths":
            lens.add_(1)
        got.append(hk.shared_prefix_attention(q, kp, vp, k, v, lens, SCALE))
    torch.cuda.synchronize()
    for i, (o, lse) in enumerate(got):
        q, lens = hk.rotary_forward(rows[i], None, pos, (32,))[0], first + (i + 1)
        torch.cuda.synchronize()
        O, LSE = hk.shared_prefix_attention(q, kp, vp, k, v, lens, SCALE)
        torch.cuda.synchronize()
        assert torch.equal(o, O) and torch.equal(lse, LSE), i
    check((O, LSE), definition(q, kp, vp, k, v, lens, True), dtype)
    assert hk.last_device_status() == 0


# ---- results that lie on top of each other: B = 2, 4 heads, 3 tokens ----------------------------------------------------------------
@pytest.mark.parametrize("o", [(64, 64, 64), (64, 256, 64), (192, 192, 384), (256, 64, 128), (768, 64, 128), (384, 64, 192), (512, 256, 64), (128, 256, 64), (192, 768, 384), (64, 64, 1 << 40)])
def test_rows_of_o_on_top_of_each_other_are_refused(o):
    b = _block()
    b.O.sB, b.O.sM, b.O.sH = o
    f = hk.lib().hk_shared_prefix_attention
    f.argtypes = [C.c_void_p, C.c_void_p]
    assert f(C.byref(b), None) == -6


@pytest.mark.parametrize("sB,sH", [(3, 3), (3, 5), (4, 4), (100, 100), (11, 3), (4, 6), (1 << 40, 2)])
def test_rows_of_lse_on_top_of_each_other_are_refused(sB, sH):
    b = _block()
    b.lse_sB, b.lse_sH = sB, sH
    f = hk.lib().hk_shared_prefix_attention
    f.argtypes = [C.c_void_p, C.c_void_p]
    assert f(C.byref(b), None) == -6


def test_results_that_lie_apart_get_past_that():
    """In any order of dimensions, with room between, however far: what is refused is the check behind it."""
    f = hk.lib().hk_shared_prefix_attention
    f.argtypes = [C.c_void_p, C.c_void_p]
    for o in ((768, 64, 192), (768, 256, 64), (192, 384 * 4, 384), (64, 512, 128), (64, 128, 384), (880, 72, 224), (1 << 50, 1 << 40, 1 << 30), (1 << 62, 1 << 60, 1 << 58)):
        b = _block()
        b.O.sB, b.O.sM, b.O.sH = o
        b.LSE = None
        assert f(C.byref(b), None) == -1, o
    for sB, sH in ((12, 3), (3, 6), (4, 7), (3, 11), (1 << 60, 1 << 50)):
        b = _block()
        b.lse_sB, b.lse_sH, b.LSE = sB, sH, 0x1002
        assert f(C.byref(b), None) == -3, (sB, sH)
    b = _block()  # strides of dimensions of one are not used
    b.B, b.nh, b.nh_kv, b.T, b.lse_sB, b.lse_sH, b.LSE = 1, 1, 1, 1, 0, 0, 0x1002
    b.O.sB = b.O.sM = b.O.sH = 0
    assert f(C.byref(b), None) == -3


# ---- workspaces that the caller brings -------------------------------------------------------------------------------------------------
def _tensors_of(B, H, Hk, T, P, S, dtype):
    one = torch.zeros(1, 1, 1, 64, dtype=TYPES[dtype])
    return one.expand(B, H, T, 64), one[0].expand(Hk, P, 64), one.expand(B, Hk, S, 64)


def test_the_size_of_a_workspace():
    """On the 148 SMs that the library takes where there is no device."""
    f = hk.lib().hk_shared_prefix_workspace_bytes
    f.restype, f.argtypes = C.c_size_t, [C.c_void_p]
    seen = set()
    for B, H, Hk, T, P, S, dtype in WAYS:
        b = _block()
        b.B, b.nh, b.nh_kv, b.T, b.prefix_len, b.kv_len, b.dtype = B, H, Hk, T, P, S, list(TYPES).index(dtype)
        need, got = f(C.byref(b)), hk.shared_prefix_workspace_bytes(*_tensors_of(B, H, Hk, T, P, S, dtype))
        assert got == (need + 256 if need else 0)
        seen.add(need > 0)
    assert seen == {False, True}
    q, kp, k = _tensors_of(2, 4, 2, 3, 9, 8, "f32")
    for name, args in (("Q", (q[0], kp, k)), ("K_prefix", (q, kp[:1], k)), ("K", (q, kp, k[:1])), ("K", (q, kp, k.half()))):
        with pytest.raises(AssertionError, match="^" + name):
            hk.shared_prefix_workspace_bytes(*args)
    with pytest.raises(TypeError, match="^K_prefix: expected a tensor"):
        hk.shared_prefix_workspace_bytes(q, None, k)


@pytest.mark.gpu
@pytest.mark.parametrize("B,H,Hk,T,P,S,dtype", [(16, 12, 12, 1, 2047, 512, "f32"), (64, 32, 8, 1, 8192, 1000, "bf16"), (16, 4, 4, 77, 4097, 333, "f16"), (3, 4, 4, 300, 900, 400, "f32"),
                                                (4, 12, 12, 1, 333, 64, "f32")])
def test_a_workspace_of_ones_own(B, H, Hk, T, P, S, dtype):
    """Whatever it holds and wherever it starts, the call has the bits of one that allocates it, and stays inside."""
    x = make(B + T, B, H, Hk, T, P, S, dtype)
    want = hk.shared_prefix_attention(*x, SCALE)
    need = hk.shared_prefix_workspace_bytes(x[0], x[1], x[3])
    room = torch.full((need + 1024,), 0xFF, device="cuda", dtype=torch.uint8)
    for at in (0, 1, 255):
        room.fill_(0xFF)
        got = hk.shared_prefix_attention(*x, SCALE, workspace=room[at:at + need])
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        assert bool((room[:at] == 0xFF).all()) and bool((room[at + need:] == 0xFF).all())
    wide = torch.full((need // 4 + 1,), float("nan"), device="cuda")
    for _ in range(3):  # one after the other in the same memory
        got = hk.shared_prefix_attention(*x, SCALE, workspace=wide)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    if need:
        with pytest.raises(AssertionError, match="too small"):
            hk.shared_prefix_attention(*x, SCALE, workspace=room[:need - 256 - 1])
        with pytest.raises(AssertionError, match="contiguous"):
            hk.shared_prefix_attention(*x, SCALE, workspace=room[:1].expand(need))
    assert hk.last_device_status() == 0


# ---- both kinds of keys in one go --------------------------------------------------------------------------------------------------------
def _plan_of(B, H, Hk, T, P, S, dtype):
    f = hk.lib().hk_shared_prefix_plan
    f.argtypes = [C.c_void_p, C.POINTER(C.c_int)]
    b, plan = _block(), (C.c_int * 6)()
    b.B, b.nh, b.nh_kv, b.T, b.prefix_len, b.kv_len, b.dtype = B, H, Hk, T, P, S, list(TYPES).index(dtype)
    assert f(C.byref(b), plan) == 0
    return tuple(plan)


def test_parts_of_blocks_in_one_go():
    """No runs of the prefix beside it, one of the own keys; few rows in one part, many in up to 16 of their last blocks, never in more than
    two thirds of their tiles; a workspace for exactly those blocks."""
    import random

    g, parts = random.Random(5), set()
    for _ in range(4000):
        Hk = g.choice([1, 2, 4, 8])
        case = (g.randint(1, 48), Hk * g.choice([1, 2, 4]), Hk, g.choice([1, 3, 17, 80, 300, 700]), g.choice([0, 1, 70, 500, 2000]), g.choice([0, 9, 130, 700, 1500]), g.choice(["f32", "bf16"]))
        B, H, _, T, P, S, dtype = case
        prefix_many, own_many, whole, runs, own_runs, slots = _plan_of(*case)
        if not whole:
            assert slots == runs + own_runs, case
            continue
        assert not prefix_many and runs == 0 and own_runs == 1 and 1 <= slots <= 16, case
        assert own_many or slots == 1, case
        rows, keys = (128, 64) if dtype == "f32" else (256, 128)
        blocks = B * Hk * -(-T * (H // Hk) // rows)
        if slots > 1:
            assert blocks % 148 and 1.5 * slots <= -(-P // keys) + -(-S // keys), case
        need = hk.shared_prefix_workspace_bytes(*_tensors_of(*case))
        assert need == (slots * (blocks % 148) * rows * (64 + 2) * 4 + 256 if slots > 1 else 0), case
        parts.add(slots)
    assert {1, 2, 3, 4} <= parts and max(parts) >= 10, parts


@pytest.mark.gpu
@pytest.mark.parametrize("B,H,Hk,T,P,S,dtype", [(2, 4, 4, 700, 0, 1500, "f32"), (2, 4, 4, 700, 0, 1500, "bf16"), (5, 4, 2, 300, 0, 1500, "f16"), (3, 4, 4, 300, 70, 1500, "f32"),
                                                (3, 8, 2, 301, 1, 1500, "bf16")])
@pytest.mark.parametrize("causal", [True, False])
def test_parts_without_keys(B, H, Hk, T, P, S, dtype, causal):
    """Requests with fewer tiles of keys than their blocks have parts: parts without a tile, rows without a key, next to full ones."""
    slots = _plan_of(B, H, Hk, T, P, S, dtype)
    assert slots[1] and slots[2] and slots[5] > 2, slots
    tile = 64 if dtype == "f32" else 128
    for lengths in ([0] * B, [1] * B, [0, 1, tile, tile + 1, S][-B:], [S, 1, 0, tile, 2 * tile + 1][:B], [2] + [0] * (B - 1)):
        x = make(B + T, B, H, Hk, T, P, S, dtype, lengths=lengths)
        room = torch.full((hk.shared_prefix_workspace_bytes(x[0], x[1], x[3]),), 0xFF, device="cuda", dtype=torch.uint8)  # NaN in every slot
        got = hk.shared_prefix_attention(*x, SCALE, causal, workspace=room)
        check(got, definition(*x, causal), dtype, lengths)
    assert hk.last_device_status() == 0
