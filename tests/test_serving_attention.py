"""Attention within packed prompts and of new tokens against a cache of pages, against the definition in 64 bits, request by request.

Error bounds (u = 2^-24).  A score in fp32 is a sum of 64 products: 80 u of the sum of the products' sizes, whatever the order; so its
exponential is off by that much of itself (D), and O, a weighted mean, by 2 D of the mean of |v| plus the roundings of sums over the
keys, taken by blocks of at most 128 keys and up to 64 blocks in a row, and over the parts that the keys are cut in: 200 u.  The exponential's own
error (2 u) and the argument's rounding (u times its size, below 64 in log2 units here) are 70 u.  Sixteen-bit types round each weight and
the result by half a step; their products are exact in fp32; a weight may come from a polynomial that is 2.7e-6 of it off, 45 u, and so
may those of the sum it is divided by."""
import ctypes as C
import math
import random

import pytest
import torch

import hyperkernels_b200 as hk

U = 2.0 ** -24
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SCALE = 0.125


def cdiv(a, b):
    return -(-a // b)


def ints(x):
    return torch.tensor(x, device="cuda", dtype=torch.int32)


def attend(q, k, v, seen, scale):
    """O, LSE, mean |v| under the softmax, largest sum of products' sizes, of rows q [H, T, 64] against k, v [H, n, 64]"""
    q, k, v = q.double(), k.double(), v.double()
    if k.shape[1] == 0:
        return torch.zeros_like(q), q.new_full(q.shape[:2], -math.inf), torch.zeros_like(q), q.new_zeros(q.shape[:2])
    x = (q @ k.transpose(1, 2) * scale).masked_fill(~seen, -math.inf)
    w = torch.nan_to_num(torch.softmax(x, -1))
    size = (q.abs() @ k.abs().transpose(1, 2) * abs(scale)).masked_fill(~seen, 0.0).amax(-1)
    return w @ v, torch.logsumexp(x, -1), w @ v.abs(), size


def check(got, want, dtype, what=""):
    (o, lse), (O, LSE, mean, size) = got, want
    step = torch.finfo(TYPES[dtype]).eps / 2 if dtype != "f32" else 0.0
    d = (80 * size + 3 * (size - 40).clamp(min=0) + 70) * U  # arguments beyond 64 round by more
    poly = 45 * U if dtype != "f32" else 0.0
    bound = (2 * d[..., None] + 200 * U + 2 * poly + step) * mean + step * O.abs() + (2.0 ** -25 if dtype == "f16" else 1e-30)
    off = (o.double() - O).abs()
    assert o.dtype == TYPES[dtype] and lse.dtype == torch.float32
    assert bool((off <= bound).all()), (what, float((off - bound).max()), float(off.max()))
    seen = LSE > -math.inf
    assert torch.equal(lse > -math.inf, seen), what
    assert bool((o[~seen] == 0).all()), what
    assert bool(((lse.double() - LSE).abs()[seen] <= (d + 200 * U + poly + 4 * U * LSE.abs())[seen]).all()), what
    if dtype == "f32" and bool(seen.any()):  # fp32 throughout: roundings that do not add up all one way
        assert float((o.double() - O).norm()) <= 1e-5 * float(O.norm()), what


PIECE = {"f16": 1 << 15, "bf16": 1 << 18}  # keys whose values are summed up at once


def check_long(got, want, dtype, n, what=""):
    """check(), for rows of n keys, whose sums are longer: n / 64 roundings (fp32) of u each in the sum of the weights and in O, which is added up tile by tile.
    16-bit types sum O up in the tensor core, which cuts off less than the last place, 2 u, of the sum there is for every 16 keys, in pieces of PIECE keys (and up to a
    tile), and the weights' sum rounds as above.  Pieces and parts that are added up round by 4 u each."""
    (o, lse), (O, LSE, mean, size) = got, want
    step = torch.finfo(TYPES[dtype]).eps / 2 if dtype != "f32" else 0.0
    poly = 45 * U if dtype != "f32" else 0.0
    d = (80 * size + 3 * (size - 40).clamp(min=0) + 70) * U
    P = min(n, PIECE.get(dtype, n) + 128)
    weights = (P / 64 + 4 * (n // P + 1) + 200) * U
    values = weights if dtype == "f32" else weights + P / 16 * 2 * U
    bound = (2 * d[..., None] + weights + values + 2 * poly + step) * mean + step * O.abs() + (2.0 ** -25 if dtype == "f16" else 1e-30)
    off = (o.double() - O).abs()
    assert bool((off <= bound).all()), (what, float((off / bound).max()), float(off.max()))
    seen = LSE > -math.inf
    assert torch.equal(lse > -math.inf, seen) and bool((o[~seen] == 0).all()), what
    assert bool(((lse.double() - LSE).abs()[seen] <= (d + weights + poly + 4 * U * LSE.abs())[seen]).all()), what


# ---- packed prompts -------------------------------------------------------------------------------------------------------------------
def make_prompts(seed, lens, H, Hk, dtype, layout="packed", before=0, after=0, sigma=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    N, t = before + sum(lens) + after, TYPES[dtype]

    def rand(*shape):
        return (torch.randn(shape, generator=g, device="cuda") * sigma).to(t)

    if layout == "packed":
        x = rand(N, H + 2 * Hk, 64)
        q, k, v = x[:, :H], x[:, H:H + Hk], x[:, H + Hk:]
    elif layout == "heads":  # head by head
        q, k, v = rand(H, N, 64).transpose(0, 1), rand(Hk, N, 64).transpose(0, 1), rand(Hk, N, 64).transpose(0, 1)
    else:  # keys and values side by side, with room between
        q = rand(N, H, 192)[..., 64:128]
        k, v = (lambda x: (x[:, :Hk, :64], x[:, :Hk, 64:]))(rand(N, Hk + 1, 128))
    starts = [before]
    for n in lens:
        starts.append(starts[-1] + n)
    for x in (k, v):
        x[:before], x[before + sum(lens):] = math.nan, math.nan
    return q, k, v, ints(starts)


def prompts(q, k, v, starts, causal, scale=SCALE):
    N, H, _ = q.shape
    G = H // k.shape[1]
    O, LSE, mean, size = (torch.zeros((H, N, n), device="cuda", dtype=torch.float64) for n in (64, 1, 64, 1))
    edges = [min(max(x, 0), N) for x in starts.tolist()]
    for a, b in zip(edges, edges[1:]):
        if b <= a:
            continue
        i = torch.arange(b - a, device="cuda")
        seen = (i <= i[:, None]) | (not causal)
        kk, vv = (x[a:b].transpose(0, 1).repeat_interleave(G, 0) for x in (k, v))
        r = attend(q[a:b].transpose(0, 1), kk, vv, seen, scale)
        O[:, a:b], LSE[:, a:b, 0], mean[:, a:b], size[:, a:b, 0] = r
    return O.transpose(0, 1), LSE[..., 0], mean.transpose(0, 1), size[..., 0]


def check_prompts(got, want, dtype, rows, what=""):
    (o, lse), (O, LSE, mean, size) = got, want
    check((o[rows].transpose(0, 1), lse[:, rows]), (O[rows].transpose(0, 1), LSE[:, rows], mean[rows].transpose(0, 1), size[:, rows]), dtype, what)


LENGTHS = [[1], [5], [0, 3, 0, 0, 2], [64], [65], [127], [128], [129], [255, 1, 256, 257], [1, 77, 0, 128, 300, 2], [700, 13], [1500], [2] * 70, [0] * 5 + [200],
           [1000, 30, 400, 0, 129], [63, 1] * 40]
HEADS = [(1, 1), (4, 4), (6, 2), (8, 1), (12, 12), (7, 1), (10, 2), (32, 8)]


@pytest.mark.gpu
@pytest.mark.parametrize("lens", LENGTHS, ids=lambda x: f"{len(x)}x{max(x)}")
@pytest.mark.parametrize("H,Hk", HEADS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal,layout", [(True, "packed"), (False, "heads"), (True, "wide")])
def test_prompts(lens, H, Hk, dtype, causal, layout):
    x = make_prompts(sum(lens) + H, lens, H, Hk, dtype, layout)
    got = hk.prompt_attention(*x, SCALE, causal)
    check_prompts(got, prompts(*x, causal), dtype, slice(None))
    again = hk.prompt_attention(*x, SCALE, causal)
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])
    assert hk.last_device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("lens,H,Hk", [([4000], 2, 2), ([3001, 5, 900], 4, 1), ([6000, 0, 2000, 1000, 500, 250, 125], 8, 8), ([300] * 30, 8, 2), ([8000, 1], 1, 1), ([500], 64, 64), ([20] * 200, 3, 1),
                                       ([2100], 20, 1), ([900, 2000], 130, 1), ([100, 300], 300, 1)])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [True, False])
def test_long_prompts_and_many(lens, H, Hk, dtype, causal):
    x = make_prompts(len(lens), lens, H, Hk, dtype)
    got = hk.prompt_attention(*x, SCALE, causal)
    check_prompts(got, prompts(*x, causal), dtype, slice(None))
    assert hk.last_device_status() == 0


DEALT = [  # so many blocks that they are dealt out whole (up to 128 prompts), and some just below
    ([1] * 92, 8, 8), ([1] * 93, 8, 8), ([0, 1, 400, 65, 0, 130, 7, 33] * 16, 32, 8), ([0, 1, 400, 65, 0, 130, 7, 33] * 16 + [90], 32, 8),
    ([300, 0, 2, 129] * 8, 64, 64), ([6000], 32, 32), ([0] * 127 + [4000], 24, 12), ([4000] + [0] * 127, 24, 12), ([700, 300], 260, 2), ([5, 900, 40] * 5, 300, 1)]


@pytest.mark.gpu
@pytest.mark.parametrize("lens,H,Hk", DEALT, ids=lambda x: f"{len(x)}x{max(x)}" if isinstance(x, list) else None)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [True, False])
def test_many_blocks(lens, H, Hk, dtype, causal):
    x = make_prompts(len(lens), lens, H, Hk, dtype)
    got = hk.prompt_attention(*x, SCALE, causal)
    check_prompts(got, prompts(*x, causal), dtype, slice(None))
    again = hk.prompt_attention(*x, SCALE, causal)
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])
    assert hk.last_device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_one_graph_for_few_blocks_and_many(dtype):
    """Where the work is cut changes with what `starts` holds when the graph runs."""
    N, H, Hk = 3000, 32, 8
    q, k, v, _ = make_prompts(7, [N], H, Hk, dtype)
    starts = ints([0] * 65)
    out, lse = torch.empty(N, H, 64, device="cuda", dtype=TYPES[dtype]), torch.empty(H, N, device="cuda")
    workspace = torch.empty(hk.prompt_workspace_bytes(q, k, starts), dtype=torch.uint8, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        hk.prompt_attention(q, k, v, starts, SCALE, workspace=workspace, out=out, lse=lse)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        hk.prompt_attention(q, k, v, starts, SCALE, workspace=workspace, out=out, lse=lse)
    for lens in ([N] + [0] * 63, [40] * 64, [0] * 63 + [64], [2] * 64, [0] * 64, [N - 640] + [0, 20] * 31 + [20]):
        edges = [0]
        for n in lens:
            edges.append(edges[-1] + n)
        starts.copy_(ints(edges))
        out.fill_(5.0), lse.fill_(5.0)
        graph.replay()
        n = edges[-1]
        check_prompts((out, lse), prompts(q, k, v, starts, True), dtype, slice(0, n))
        assert bool((out[n:] == 5.0).all()) and bool((lse[:, n:] == 5.0).all())
    assert hk.last_device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens", [[3, 0, 200, 17], [300, 129, 1], [0, 0]])
@pytest.mark.parametrize("before,after", [(0, 5), (130, 0), (1, 300)])
def test_rows_of_no_prompt_stay(dtype, lens, before, after):
    """And what stands in them, or in another prompt, does not matter."""
    x = make_prompts(1, lens, 4, 2, dtype, before=before, after=after)
    N, mine = x[0].shape[0], slice(before, before + sum(lens))
    room = torch.full((N + 2, 5, 64), 7.0, device="cuda", dtype=TYPES[dtype])
    lse_room = torch.full((4, N + 3), 7.0, device="cuda")
    got = hk.prompt_attention(*x, SCALE, True, out=room[1:-1, :4], lse=lse_room[:, :N])
    want = prompts(*x, True)
    assert got[0].data_ptr() == room[1:-1].data_ptr()
    check_prompts(got, want, dtype, mine)
    inside = torch.zeros((N + 2, 5, 64), device="cuda", dtype=torch.bool)
    inside[1:-1, :4][mine] = True
    assert bool((room[~inside] == 7.0).all())
    lse_inside = torch.zeros((4, N + 3), device="cuda", dtype=torch.bool)
    lse_inside[:, mine] = True
    assert bool((lse_room[~lse_inside] == 7.0).all())
    # a prompt of NaN between others
    if sum(lens) > 200:
        a, b = x[3][2 if lens[0] < 300 else 1:][:2].tolist()
        for bad in (math.nan, math.inf):
            for t in x[:3]:
                t[a:b] = bad
            again = hk.prompt_attention(*x, SCALE, True)
            others = torch.ones(N, device="cuda", dtype=torch.bool)
            others[a:b], others[:before], others[before + sum(lens):] = False, False, False
            assert torch.equal(again[0][others], got[0][others]) and torch.equal(again[1][:, others], got[1][:, others])
            assert bool(again[0][a:b].isnan().all())
    assert hk.last_device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_starts_are_taken_into_the_tensor(dtype):
    x = list(make_prompts(1, [50, 200], 2, 2, dtype))
    want = hk.prompt_attention(*x, SCALE)
    x[3] = ints([-7, 50, 100000])
    got = hk.prompt_attention(*x, SCALE)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    for starts in ([2 ** 31 - 1] * 3, [-2 ** 31] * 3, [200, 100, 50], [250, 0, 250]):  # none, or not ascending: no fault, nothing elsewhere
        x[3] = ints(starts)
        room = torch.full((256, 2, 64), 7.0, device="cuda", dtype=TYPES[dtype])
        hk.prompt_attention(*x, SCALE, True, out=room[3:253])
        assert bool((room[:3] == 7.0).all()) and bool((room[253:] == 7.0).all())
    assert hk.last_device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens", [[40], [150, 3], [400], [1100]])
def test_large_scores_and_other_scales(dtype, lens):
    """Scores of +-200: one key takes almost everything, the maximum moves late."""
    x = make_prompts(3, lens, 4, 2, dtype)
    x[1].mul_(torch.linspace(0.2, 3.0, x[1].shape[0], device="cuda")[:, None, None].to(x[1].dtype))
    for scale in (1.0, -0.7, 1e-3):
        for causal in (True, False):
            check_prompts(hk.prompt_attention(*x, scale, causal), prompts(*x, causal, scale), dtype, slice(None), (scale, causal))
    assert hk.last_device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("height", [4.0, 30.0, 90.0, 1000.0, 40000.0])
def test_one_late_key_that_takes_all(height, dtype):
    """Scores of about 1, and in each column of the second and third tile, in turn, one key of `height` (16-bit types hold all five)."""
    x = make_prompts(9, [500], 2, 2, dtype, sigma=0.3)
    x[0][..., 0] = 1.0
    x[1][..., 0] = 0.0
    for at in range(128, 384, 1 if height == 90.0 else 7):
        x[1][at, :, 0] = height
        check_prompts(hk.prompt_attention(*x, 1.0), prompts(*x, True, 1.0), dtype, slice(None), at)
        x[1][at, :, 0] = 0.0
    assert hk.last_device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T", [40, 300, 700])
def test_scores_that_are_no_numbers(dtype, T):
    """A NaN score makes NaN of the rows that see it, in any column; the rows before it stay as they were."""
    x = make_prompts(5, [T, 30], 2, 2, dtype)
    plain = hk.prompt_attention(*x, SCALE)
    for at in [0, 1, 2, 39, 63, 64, 65, 127, 128, 129] + list(range(134, 140)) + [188, 255, 256, 399]:
        if at >= T:
            continue
        for bad in (math.nan, math.inf):
            keep = x[1][at].clone()
            x[1][at] = bad  # infinities of both signs meet in a score
            o, lse = hk.prompt_attention(*x, SCALE)
            x[1][at] = keep
            assert bool(o[at:T].isnan().all()) and bool(lse[:, at:T].isnan().all()), (at, bad)
            for a, b in ((0, at), (T, T + 30)):
                assert torch.equal(o[a:b], plain[0][a:b]) and torch.equal(lse[:, a:b], plain[1][:, a:b]), (at, bad)
    assert hk.last_device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T", [300, 4000])
def test_many_small_weights_beside_a_large_one(dtype, T):
    """The first key takes nearly all, and its value is 0: the result is what the others give, each 2^-26 of the first.

    A weight of 2^-26.1 or more (26 ln 2 rounds to within 0.1), lifted by seven binary places in fp16, is rounded there to a multiple of
    2^-24: by 2^-25 in 2^-19.1 at most; in the other types by half a step."""
    t = TYPES[dtype]
    q = torch.zeros((T, 2, 64), device="cuda", dtype=t)
    q[..., 0] = 26.0 * math.log(2.0)
    k, v = (torch.full((T, 2, 64), x, device="cuda", dtype=t) for x in (0.0, 1.0))
    k[0, :, 0], v[0] = 1.0, 0.0
    starts = ints([0, T])
    for causal in (True, False):
        o, lse = hk.prompt_attention(q, k, v, starts, 1.0, causal)
        O, LSE, _, _ = prompts(q, k, v, starts, causal, 1.0)
        d = (80 * 26 + 70) * U
        step = torch.finfo(t).eps / 2 if dtype != "f32" else 0.0
        weight = 2.0 ** -5.9 if dtype == "f16" else step
        assert bool(((o.double() - O).abs() <= (2 * d + 290 * U + weight + step) * O + (2.0 ** -25 if dtype == "f16" else 0.0)).all())
        assert bool(((lse.double() - LSE).abs() <= d + 245 * U + 4 * U * LSE.abs()).all())


@pytest.mark.gpu
@pytest.mark.parametrize("lens,times,H,Hk", [([1], 1 << 17, 16, 16), ([1, 16, 2, 40, 5], 1 << 14, 8, 8), ([3, 700, 0, 9], 100, 64, 8)], ids=lambda x: str(len(x)) if isinstance(x, list) else None)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [True, False])
def test_very_many_prompts(lens, times, H, Hk, dtype, causal):
    """So many that a short one is little of a unit of the line they make: none may get lost, the first and the last among them."""
    x = q, k, v, starts = make_prompts(len(lens), lens * times, H, Hk, dtype)
    N, G = q.shape[0], H // Hk
    out, lse = torch.full((N, H, 64), math.nan, device="cuda", dtype=TYPES[dtype]), torch.full((H, N), math.nan, device="cuda")
    got = hk.prompt_attention(*x, SCALE, causal, out=out, lse=lse)
    again = hk.prompt_attention(*x, SCALE, causal)
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])
    for c, n in enumerate(lens):  # all of one length at once
        if n == 0:
            continue
        i = torch.arange(n, device="cuda")
        rows = starts[:-1].long()[c::len(lens), None] + i
        for part in rows.split(max(1, (1 << 18) // (n * H))):
            qq, kk, vv, oo = (t[part].transpose(1, 2) for t in (q, k.repeat_interleave(G, 1) if G > 1 else k, v.repeat_interleave(G, 1) if G > 1 else v, out))
            want = attend(qq.reshape(-1, n, 64), kk.reshape(-1, n, 64), vv.reshape(-1, n, 64), (i <= i[:, None]) | (not causal), SCALE)
            check((oo.reshape(-1, n, 64), lse[:, part].transpose(0, 1).reshape(-1, n)), want, dtype, (n, part[0]))
    assert hk.last_device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("N,H", [(700, 2), (3000, 40), (9000, 1)])
def test_the_division_and_the_logarithm_of_fp32(N, H):
    """Keys that all weigh the same, values that are whole numbers: every sum is exact, and what is left are a division, rounded, times the sum (2 u), and
    log2 of the sum (an ulp, 2 u of it) times ln 2 (rounded, and its product: 2 u), whether a block was cut in parts or not."""
    q, k, v = (torch.zeros((N, H, 64), device="cuda") for _ in range(3))
    v[:] = torch.arange(1, 65, device="cuda")
    n = torch.arange(1, N + 1, device="cuda", dtype=torch.float64)
    o, lse = hk.prompt_attention(q, k, v, ints([0, N]), SCALE)
    assert bool(((o.double() / v.double() - 1).abs() <= 2.001 * U).all())
    assert bool(((lse.double() - n.log()).abs() <= 4.001 * U * n.log()).all())


# ---- new tokens against the pages -----------------------------------------------------------------------------------------------------
def make_tree(seed, lens, T, H, Hk, page, dtype, layout="hpd", tree="random", junk=math.nan, sigma=1.0, spare=2):
    """Pages in any order; what is behind a request's last key, and in pages of nobody, is junk"""
    g, rng = torch.Generator(device="cuda").manual_seed(seed), random.Random(seed)
    B, t = len(lens), TYPES[dtype]

    def rand(*shape):
        return (torch.randn(shape, generator=g, device="cuda") * sigma).to(t)

    counts = [cdiv(max(n, 0), page) for n in lens]
    width, P = max(counts) + 1, sum(counts) + spare
    order = list(range(P))
    rng.shuffle(order)
    rows = []
    for n in counts:
        row = [order.pop() for _ in range(n)]
        rows.append(row + [rng.choice([-1, P, -2 ** 31, 2 ** 31 - 1]) for _ in range(width - n)])
    if layout == "phd":
        kp, vp = (rand(P, page, Hk, 64).transpose(1, 2) for _ in range(2))
        q = rand(B, T, H, 64).transpose(1, 2)
        k, v = (rand(B, T, Hk, 64).transpose(1, 2) for _ in range(2))
    elif layout == "wide":
        kp, vp = (lambda x: (x[:, :, :page, :64], x[:, :, :page, 64:]))(rand(P, Hk, page + 3, 128))
        q = rand(B, H, T, 192)[..., 64:128]
        k, v = (lambda x: (x[..., :64], x[..., 64:]))(rand(B, Hk, T, 128))
    else:
        kp, vp = rand(P, Hk, page, 64), rand(P, Hk, page, 64)
        q, k, v = rand(B, H, T, 64), rand(B, Hk, T, 64), rand(B, Hk, T, 64)
    free = set(range(P)) - {p for row, n in zip(rows, counts) for p in row[:n]}
    for x in (kp, vp):
        for p in free:
            x[p] = junk
        for row, n in zip(rows, lens):
            if n > 0 and n % page:
                x[row[n // page], :, n % page:] = junk
    if tree == "random":
        bits = []
        for b in range(B):
            r = []
            for i in range(T):
                parent = rng.randrange(-1, i) if i else -1
                r.append((r[parent] if parent >= 0 else 0) | 1 << i)
            if b % 3 == 2:
                r[-1] = 0  # a place without a draft: sees the cache alone
            bits.append([x - (1 << 64) if x >> 63 else x for x in r])
        tree = torch.tensor(bits, device="cuda")
    return q, k, v, kp, vp, ints(rows), ints(lens), SCALE, tree


def trees(q, k, v, kp, vp, pages, lens, scale, tree):
    B, H, T, _ = q.shape
    G, P, page = H // k.shape[1], kp.shape[0], kp.shape[2]
    out = []
    for b in range(B):
        n = min(max(int(lens[b]), 0), pages.shape[1] * page)
        ids = pages[b, :cdiv(n, page)].tolist()
        old = []
        for x in (kp, vp):
            got = [x[i] if 0 <= i < P else torch.zeros_like(x[0]) for i in ids]
            old.append(torch.cat(got, 1)[:, :n] if got else x[0][:, :0])
        kk, vv = (torch.cat([o, x[b]], 1).repeat_interleave(G, 0) for o, x in zip(old, (k, v)))
        j = torch.arange(T, device="cuda")
        new = (tree[b][:, None] >> j & 1).bool() if tree is not None else j <= j[:, None]
        out.append(attend(q[b], kk, vv, torch.cat([torch.ones((T, n), device="cuda", dtype=torch.bool), new], 1), scale))
    return tuple(torch.stack(x) for x in zip(*out))


CACHES = [  # lens, T, H, Hk, page
    ([0], 1, 1, 1, 16), ([1], 1, 1, 1, 16), ([5, 0, 16, 17, 300], 1, 4, 4, 16), ([333, 64, 65, 0, 1000], 1, 12, 12, 16), ([129, 500, 1, 31], 1, 8, 2, 64), ([700] * 20, 1, 7, 1, 48),
    ([100, 0, 257], 2, 3, 3, 32), ([5, 300], 3, 8, 1, 64), ([128, 127, 0], 5, 6, 2, 128), ([250, 31, 64, 1], 17, 4, 1, 16), ([400, 0], 16, 32, 8, 64), ([90, 1000], 64, 4, 4, 32),
    ([300, 511, 512, 513], 64, 8, 1, 256), ([33, 70], 63, 9, 3, 80), ([1, 2, 3], 33, 2, 1, 1024), ([2000, 10], 8, 16, 2, 112), ([600], 64, 10, 1, 64), ([77] * 9, 4, 5, 1, 16)]


@pytest.mark.gpu
@pytest.mark.parametrize("lens,T,H,Hk,page", CACHES, ids=lambda x: f"{len(x)}x{max(x)}" if isinstance(x, list) else None)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["hpd", "phd", "wide"])
@pytest.mark.parametrize("tree", ["random", None])
def test_trees(lens, T, H, Hk, page, dtype, layout, tree):
    x = make_tree(sum(lens) + T, lens, T, H, Hk, page, dtype, layout, tree)
    got = hk.tree_attention(*x)
    check(got, trees(*x), dtype)
    again = hk.tree_attention(*x)
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])
    assert hk.last_device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("lens,T,H,Hk,page", [
    ([9000], 1, 2, 1, 64), ([9000, 1, 500], 1, 1, 1, 16), ([4000] * 3, 4, 4, 4, 32), (list(range(0, 2000, 61)), 1, 12, 12, 16), (list(range(0, 6000, 190)), 1, 32, 8, 64), ([30] * 300, 1, 4, 2, 16),
    (list(range(0, 3000, 200)), 16, 32, 8, 64), ([5000, 0, 800], 64, 8, 2, 128), ([10000], 40, 16, 16, 48), ([15000, 3], 2, 64, 1, 16), ([100] * 60 + [7000], 6, 6, 3, 64), ([0] * 40, 1, 8, 8, 16),
    ([3000] * 8, 64, 64, 8, 64), ([1200, 50], 64, 96, 3, 32), ([2500] * 2, 1, 300, 1, 64), ([40000], 1, 1, 1, 64)])
@pytest.mark.parametrize("dtype", TYPES)
def test_long_caches_and_many(lens, T, H, Hk, page, dtype):
    x = make_tree(len(lens) + T, lens, T, H, Hk, page, dtype, "phd" if T == 1 else "hpd")
    got = hk.tree_attention(*x)
    check(got, trees(*x), dtype)
    again = hk.tree_attention(*x)
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])
    assert hk.last_device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("T,H,Hk", [(1, 8, 4), (3, 8, 4), (4, 16, 4), (8, 8, 8), (2, 24, 12), (16, 4, 4), (5, 12, 4), (1, 64, 4)])
@pytest.mark.parametrize("lens,page", [(list(range(0, 2000, 61)), 16), ([700, 0, 33], 64), ([300] * 50, 48), ([6000, 5], 32)], ids=lambda x: f"{len(x)}x{max(x)}" if isinstance(x, list) else None)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["hpd", "phd"])
def test_key_heads_in_fours(T, H, Hk, lens, page, dtype, layout):
    """Where four key heads are taken side by side, and where there are too few of them for that."""
    x = make_tree(len(lens) + T, lens, T, H, Hk, page, dtype, layout)
    got = hk.tree_attention(*x)
    check(got, trees(*x), dtype)
    again = hk.tree_attention(*x)
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])
    assert hk.last_device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,G", [(1, 1), (1, 4), (3, 1), (9, 2), (40, 4)])
@pytest.mark.parametrize("junk", [math.nan, math.inf, 60000.0])
def test_lengths_at_borders_and_outside(dtype, T, G, junk):
    lens = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 191, 192, 193, 255, 256, 300, -4]
    x = list(make_tree(T, lens, T, 2 * G, 2, 32, dtype, junk=junk))
    check(hk.tree_attention(*x), trees(*x), dtype)
    full = cdiv(300, 32) + 1  # longer than the table: all of it, where entries without a page are zeros
    x[6][-2], x[6][4] = 1000000, 2 ** 31 - 1
    for p in (3, 4):
        x[p].nan_to_num_(0.5, 0.5, 0.5).clamp_(-5, 5)
    assert x[5].shape[1] == full
    check(hk.tree_attention(*x), trees(*x), dtype)
    assert hk.last_device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,H,Hk", [(1, 1, 1), (3, 8, 4), (2, 16, 2), (20, 2, 1), (64, 12, 2)])
def test_tables_with_room_for_far_more(dtype, T, H, Hk):
    """A table that 2^30 keys of each request would fit, which have none or few: a block is little of a unit of the line they make."""
    x = list(make_tree(T, [0, 1, 40, 0, 300, 2000, 0] * 9 + [0], T, H, Hk, 16384, dtype))
    x[5] = torch.cat([x[5], x[5].new_full((x[5].shape[0], 65536 - x[5].shape[1]), -1)], 1)
    out, lse = torch.full(x[0].shape, math.nan, device="cuda", dtype=TYPES[dtype]), torch.full(x[0].shape[:3], math.nan, device="cuda")
    for lens in (x[6], torch.zeros_like(x[6])):
        x[6] = lens
        got = hk.tree_attention(*x, out=out.fill_(math.nan), lse=lse.fill_(math.nan))
        check(got, trees(*x), dtype)
        again = hk.tree_attention(*x)
        assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])
    assert hk.last_device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T", [1, 6, 30])
def test_rows_that_see_nothing(dtype, T):
    x = list(make_tree(T, [0, 70, 0], T, 4, 2, 16, dtype))
    x[8] = torch.zeros_like(x[8])
    if T > 1:
        x[8][2, 1] = 1 << 0  # sees another, not itself
    if T < 64:
        x[8][0] = -1 << T  # bits of tokens that there are not
    got = hk.tree_attention(*x)
    x[8] = torch.where(x[8] < 0, 0, x[8])
    check(got, trees(*x), dtype)
    assert bool((got[0][0] == 0).all()) and bool((got[1][0] == -math.inf).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,G", [(1, 1), (1, 4), (5, 2), (64, 2)])
def test_large_scores_in_pages(dtype, T, G):
    x = list(make_tree(3, [500, 90, 0, 700], T, 2 * G, 2, 16, dtype))
    x[0].mul_(5.0)
    for scale in (1.0, -0.7, 1e-3):
        x[7] = scale
        check(hk.tree_attention(*x), trees(*x), dtype, scale)
    assert hk.last_device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,G", [(1, 1), (1, 4), (3, 1), (20, 4)])
def test_scores_in_pages_that_are_no_numbers(dtype, T, G):
    x = make_tree(5, [300, 280], T, 2 * G, 2, 16, dtype, tree=None)
    plain = hk.tree_attention(*x)
    check(plain, trees(*x), dtype)
    for at in [0, 1, 2, 7, 8, 15, 16, 63, 64, 100, 127, 128, 200, 279]:
        page = int(x[5][1, at // 16])
        for bad in (math.nan, math.inf):
            keep = x[3][page, 0, at % 16].clone()
            x[3][page, 0, at % 16] = bad
            o, lse = hk.tree_attention(*x)
            x[3][page, 0, at % 16] = keep
            assert bool(o[1, :G].isnan().all()) and bool(lse[1, :G].isnan().all()), (at, bad)
            assert torch.equal(o[0], plain[0][0]) and torch.equal(o[1, G:], plain[0][1, G:]) and torch.equal(lse[1, G:], plain[1][1, G:])
    for j in range(T):  # among the drafts: the rows that see it
        keep = x[1][0, 1, j].clone()
        x[1][0, 1, j] = math.nan
        o, lse = hk.tree_attention(*x)
        x[1][0, 1, j] = keep
        assert bool(o[0, G:, j:].isnan().all()) and torch.equal(o[0, G:, :j], plain[0][0, G:, :j]) and torch.equal(o[0, :G], plain[0][0, :G])
    assert hk.last_device_status() == 0


# ---- calls ----------------------------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype,lens,H,Hk", [("f32", [4000, 100, 900], 4, 4), ("bf16", [6000, 100, 900], 16, 4), ("f16", [500] * 20, 8, 8), ("f32", [30] * 9, 12, 12), ("bf16", [2000] * 3, 8, 1)])
def test_the_same_bits_however_late_the_keys_come(dtype, lens, H, Hk):
    """Every other call finds its keys in the L2, the others in memory: tiles land in other orders and at other times."""
    x = make_prompts(1, lens, H, Hk, dtype)
    y = [make_tree(2, [n // 2 for n in lens] * 4, T, H, Hk, 32, dtype) for T in (1, 5, 40)]
    want = [hk.prompt_attention(*x, SCALE)] + [hk.tree_attention(*t) for t in y]
    check_prompts(want[0], prompts(*x, True), dtype, slice(None))
    for t, w in zip(y, want[1:]):
        check(w, trees(*t), dtype)
    room = torch.empty(1 << 28, device="cuda", dtype=torch.uint8)
    different = torch.zeros((), device="cuda", dtype=torch.int64)
    for i in range(150):
        if i % 2:
            room.fill_(i & 255)
        for (o, lse), w in zip([hk.prompt_attention(*x, SCALE)] + [hk.tree_attention(*t) for t in y], want):
            different += (o != w[0]).any() | (lse != w[1]).any()
    assert int(different) == 0 and hk.last_device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens,H,Hk", [([40, 3], 2, 2), ([2000, 100, 900], 8, 2)])
def test_captured_calls_follow_lengths_and_tables(dtype, lens, H, Hk):
    """Two graphs, each with a workspace of its own, replayed side by side; starts, lengths, tables and trees are read at replay."""
    N, B = sum(lens), len(lens)
    x = make_prompts(1, lens, H, Hk, dtype)
    y = list(make_tree(2, [n // 2 for n in lens], 3, H, Hk, 16, dtype, junk=0.5))
    graphs = []
    hk.prompt_attention(*x, SCALE), hk.tree_attention(*y)
    torch.cuda.synchronize()
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            r = (hk.prompt_attention(*x, SCALE), hk.tree_attention(*y))
        graphs.append((g, r, torch.cuda.Stream()))
    for k in range(4):
        cut = sorted(random.Random(k).randrange(N + 1) for _ in range(B - 1))
        x[3].copy_(ints([0, *cut, N]))
        y[6].copy_(ints([(n // 2 * (k + 1)) // 4 for n in lens]))
        y[5].copy_(y[5].roll(k, 0))
        y[8].copy_(y[8].roll(1, 0))
        y[5].clamp_(0, y[3].shape[0] - 1)
        torch.cuda.synchronize()
        for _ in range(3):
            for g, _, s in graphs:
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        want = (hk.prompt_attention(*x, SCALE), hk.tree_attention(*y))
        for _, r, _ in graphs:
            assert all(torch.equal(a, b) for p, q in zip(r, want) for a, b in zip(p, q))
        check_prompts(want[0], prompts(*x, True), dtype, slice(None))
        check(want[1], trees(*y), dtype)
    assert hk.last_device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,lens,H,Hk,T", [("f32", [3000, 40], 4, 2, 1), ("bf16", [5000, 100], 16, 4, 9), ("f16", [20, 30], 2, 2, 30)])
def test_a_workspace_of_ones_own(dtype, lens, H, Hk, T):
    """Whatever it holds and wherever it starts, the call has the bits of one that allocates it, and stays inside."""
    x, y = make_prompts(1, lens, H, Hk, dtype), make_tree(2, lens, T, H, Hk, 64, dtype)
    for call, need in ((lambda **c: hk.prompt_attention(*x, SCALE, **c), hk.prompt_workspace_bytes(x[0], x[1], x[3])),
                       (lambda **c: hk.tree_attention(*y, **c), hk.tree_workspace_bytes(y[0], y[1], *y[3:6]))):
        want = call()
        room = torch.full((need + 1024,), 0xFF, device="cuda", dtype=torch.uint8)
        for at in (0, 1, 255):
            room.fill_(0xFF)
            got = call(workspace=room[at:at + need])
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
            assert bool((room[:at] == 0xFF).all()) and bool((room[at + need:] == 0xFF).all())
        wide = torch.full((need // 4 + 1,), float("nan"), device="cuda")
        for _ in range(3):  # one after the other in the same memory
            got = call(workspace=wide)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        if need:
            with pytest.raises(AssertionError, match="too small"):
                call(workspace=room[:need - 256 - 1])
            with pytest.raises(AssertionError, match="contiguous"):
                call(workspace=room[:1].expand(need))
    assert hk.last_device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_given_tensors_and_streams(dtype):
    x, y = make_prompts(1, [700, 20, 300], 8, 2, dtype), make_tree(2, [700, 20, 300], 7, 8, 2, 16, dtype)
    want = (hk.prompt_attention(*x, SCALE), hk.tree_attention(*y))
    room = torch.full((3, 9, 9, 64), 7.0, device="cuda", dtype=TYPES[dtype])
    lse_room = torch.full((3, 8, 10), 7.0, device="cuda")
    out = room[:, 1:8, :8].transpose(1, 2)
    got = hk.tree_attention(*y, out=out, lse=lse_room[..., :7])
    assert got[0].data_ptr() == out.data_ptr() and torch.equal(out, want[1][0]) and torch.equal(lse_room[..., :7], want[1][1])
    room[:, 1:8, :8] = 7.0
    assert bool((room == 7.0).all()) and bool((lse_room[..., 7:] == 7.0).all())
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    for stream in (s, s.cuda_stream, 0):
        got = (hk.prompt_attention(*x, SCALE, stream=stream), hk.tree_attention(*y, stream=stream))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for p, q in zip(got, want) for a, b in zip(p, q))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_two_threads_on_streams_of_their_own(dtype):
    from threading import Thread

    lens = [900, 3, 0, 260, 77]
    p = make_prompts(1, lens, 8, 2, dtype)
    t = {T: make_tree(T, [700, 0, 65, 128], T, 8, 2, 16, dtype) for T in (1, 12)}
    call = [lambda: hk.prompt_attention(*p, SCALE)] + [lambda T=T: hk.tree_attention(*t[T]) for T in t]
    want = [f() for f in call]
    torch.cuda.synchronize()
    failed = []

    def run(order):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                got = [(i, call[i]()) for _ in range(20) for i in order]
                torch.cuda.current_stream().synchronize()
            for i, g in got:
                assert all(torch.equal(a, b) for a, b in zip(g, want[i])), i
        except BaseException as e:  # said by the test, not lost with the thread
            failed.append(e)

    threads = [Thread(target=run, args=(o,)) for o in ((0, 1, 2), (2, 0, 1))]
    for x in threads:
        x.start()
    for x in threads:
        x.join()
    assert not failed, failed
    assert hk.last_device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_lengths_and_queries_written_by_the_launch_before(dtype):
    """What a call reads was written a moment ago, over what the call before it read: no older value may come out of a cache."""
    x, y = make_prompts(1, [300, 20, 400], 8, 2, dtype), list(make_tree(2, [700, 20, 300], 3, 8, 2, 16, dtype, junk=0.5, spare=40))
    states = []
    for k in range(2):
        g = torch.Generator(device="cuda").manual_seed(k)
        states.append([torch.randn(x[0].shape, generator=g, device="cuda").to(x[0].dtype), ints([0, 100 + 400 * k, 500 + k, 720]), torch.randn(y[0].shape, generator=g, device="cuda").to(y[0].dtype),
                       ints([700 * k, 20, 300 - 290 * k]), y[5].roll(k, 0).clamp(0, 9), y[8].roll(k, 0)])
    live = [x[0], x[3], y[0], y[6], y[5], y[8]]

    def call():
        return hk.prompt_attention(*x, SCALE) + hk.tree_attention(*y)

    want = []
    for s in states:
        for a, b in zip(live, s):
            a.copy_(b)
        torch.cuda.synchronize()
        want.append(call())
        torch.cuda.synchronize()
    different = torch.zeros((), device="cuda", dtype=torch.int64)
    for i in range(200):
        for a, b in zip(live, states[i % 2]):
            a.copy_(b)
        for a, b in zip(call(), want[i % 2]):
            different += (a != b).any()
    assert int(different) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_offsets_past_32_bits(dtype):
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB")
    P, Hk, page, t = 3, 2, 64, TYPES[dtype]
    e = 4 if dtype == "f32" else 2
    g = torch.Generator(device="cuda").manual_seed(1)
    far = torch.zeros((2, P, (12 << 30) // e // 2), device="cuda", dtype=t)
    kp, vp = (far[i].as_strided((P, Hk, page, 64), (far.stride(1), page * 64, 64, 1), far[i].storage_offset()) for i in range(2))
    kp.copy_(torch.randn(kp.shape, generator=g, device="cuda")), vp.copy_(torch.randn(kp.shape, generator=g, device="cuda"))
    q, k, v = (torch.randn((1, n, 2, 64), generator=g, device="cuda").to(t) for n in (4, 2, 2))
    x = (q, k, v, kp, vp, ints([[2, 0, 1]]), ints([170]), SCALE, None)
    check(hk.tree_attention(*x), trees(*x), dtype)
    del far, kp, vp, x
    # rows of packed tensors a long way apart
    far = torch.zeros((3, 200, (4 << 30) // e // 64), device="cuda", dtype=t)
    q, k, v = (far[i].as_strided((200, 2, 64), (far.stride(1), 64, 1), far[i].storage_offset()) for i in range(3))
    for y in (q, k, v):
        y.copy_(torch.randn(y.shape, generator=g, device="cuda"))
    x = (q, k, v, ints([0, 7, 200]))
    check_prompts(hk.prompt_attention(*x, SCALE), prompts(*x, True), dtype, slice(None))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,N,H,Hk,causal", [("bf16", 1 << 20, 2, 1, False), ("f16", (1 << 20) + 77, 1, 1, True), ("bf16", (1 << 20) - 9, 1, 1, True), ("f16", 1 << 17, 12, 4, True), ("f32", 1 << 18, 2, 2, False)])
def test_very_long_prompts(dtype, N, H, Hk, causal):
    """Values that do not cancel: a sum that is cut off at every step is too low by more with every key.  Some rows are compared."""
    x = q, k, v, starts = make_prompts(1, [3, N - 8, 5], H, Hk, dtype)
    v += 1
    o, lse = hk.prompt_attention(*x, SCALE, causal)
    rows = torch.tensor([3, 4, 130, 131, 16390, N // 3, N // 2 - 1, N // 2, N - 137, N - 7, N - 6], device="cuda")
    check_long((o[rows].transpose(0, 1), lse[:, rows]), attend_rows(q[rows], k[3:N - 5], v[3:N - 5], rows - 3, causal), dtype, N)
    for a, b in ((0, 3), (N - 5, N)):
        check_prompts((o[a:b], lse[:, a:b]), prompts(q[a:b], k[a:b], v[a:b], ints([0, b - a]), causal), dtype, slice(None))
    again = hk.prompt_attention(*x, SCALE, causal)
    assert torch.equal(o, again[0]) and torch.equal(lse, again[1])
    assert hk.last_device_status() == 0


def attend_rows(q, k, v, rows, causal):
    """attend() for some rows [R, H, 64] of a prompt's k, v [n, Hk, 64]: the query heads of a key head as rows of one"""
    (R, H, _), (n, Hk, _) = q.shape, k.shape
    seen = ((torch.arange(n, device="cuda") <= rows[:, None]) | (not causal)).repeat(H // Hk, 1)
    out = attend(q.transpose(0, 1).reshape(Hk, H // Hk * R, 64), k.transpose(0, 1), v.transpose(0, 1), seen, SCALE)
    return tuple(t.reshape(H, R, *t.shape[2:]) for t in out)


@pytest.mark.gpu
@pytest.mark.parametrize("lens,H,Hk", [([(1, 0)], 4, 2), ([(1, 1), (0, 40)], 3, 3), ([(1, 128), (0, 0), (0, 1)], 6, 2), ([(1, 129)], 1, 1), ([(1, 256), (0, 70)], 2, 1), ([(2, 300), (1, 257), (0, 7)], 10, 1),
                                       ([(1, 400)], 130, 1), ([(0, 50), (1, 600), (0, 300), (0, 128)], 24, 24)], ids=lambda x: "-".join(f"{a}p{b}" for a, b in x) if isinstance(x, list) else None)
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("causal", [True, False])
def test_prompts_in_pieces(lens, H, Hk, dtype, causal):
    """Around the length where a block's keys are taken in several pieces, in calls that deal blocks out whole and that cut them; the last rows of each prompt, and some in between."""
    P = PIECE[dtype]
    lens = [a * P + b for a, b in lens]
    x = q, k, v, starts = make_prompts(len(lens), lens, H, Hk, dtype, before=3, after=2)
    v += 1
    out, lse = torch.full(q.shape, 7.0, device="cuda", dtype=TYPES[dtype]), torch.full((H, q.shape[0]), 7.0, device="cuda")
    hk.prompt_attention(*x, SCALE, causal, out=out, lse=lse)
    edges = starts.tolist()
    for a, b in zip(edges, edges[1:]):
        n = b - a
        rows = {0, 1, 128, n // 2, *(P + i for i in (-1, 0, 1, 127, 128, 129, 255, 256)), 2 * P, 2 * P + 255, *(n - i for i in (300, 257, 256, 129, 128, 65, 2, 1))}
        rows = torch.tensor(sorted(i for i in rows if 0 <= i < n), device="cuda", dtype=torch.long)
        if n:
            check_long((out[a + rows].transpose(0, 1), lse[:, a + rows]), attend_rows(q[a + rows], k[a:b], v[a:b], rows, causal), dtype, n, (a, b))
    assert bool((out[:3] == 7.0).all()) and bool((out[-2:] == 7.0).all())
    assert not bool((lse[:, 3:-2] == 7.0).any())
    again = hk.prompt_attention(*x, SCALE, causal)
    assert torch.equal(out[3:-2], again[0][3:-2]) and torch.equal(lse[:, 3:-2], again[1][:, 3:-2])
    assert hk.last_device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,H", [(1, 1), (2, 2), (30, 1), (64, 3)])
def test_very_long_caches(dtype, T, H):
    x = make_tree(T, [1000001, 3, 0, 250000], T, H, 1, 64, dtype)
    x[2].add_(1), x[4].add_(1)
    got, want = hk.tree_attention(*x), trees(*x)
    for b, n in enumerate(x[6].tolist()):
        check_long(tuple(t[b] for t in got), tuple(t[b] for t in want), dtype, n + T, b)
    assert hk.last_device_status() == 0


def shared_pages(seed, lens, T, H, Hk, dtype, layout, tree):
    """Requests over the same pages, each in an order of its own; values that do not cancel"""
    B, page = len(lens), 256
    x = list(make_tree(seed, [cdiv(max(lens), page) * page], T, H, Hk, page, dtype, layout, spare=0))
    pages = x[5][0, :-1]
    g, rng = torch.Generator(device="cuda").manual_seed(seed), random.Random(seed)
    x[0], x[1], x[2] = (torch.randn((B, n, T, 64), generator=g, device="cuda").to(TYPES[dtype]) for n in (H, Hk, Hk))
    x[5] = torch.stack([pages.roll(b) for b in range(B)]).contiguous()
    x[6] = ints(lens)
    x[8] = torch.tensor([[rng.getrandbits(i) | 1 << i if i < 63 else -1 for i in range(T)] for _ in range(B)], device="cuda") if tree else None
    x[2].add_(1), x[4].add_(1)
    return x


def check_shared_pages(x, lens, T, dtype, every):
    got = hk.tree_attention(*x)
    for b in [*range(0, len(lens), every), len(lens) - 2, len(lens) - 1]:
        one = trees(*(t[b:b + 1] if i in (0, 1, 2, 5, 6, 8) and t is not None else t for i, t in enumerate(x)))
        check_long(tuple(t[b:b + 1] for t in got), one, dtype, lens[b] + T, b)
    again = hk.tree_attention(*x)
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])
    assert hk.last_device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("T,H", [(17, 1), (40, 2), (64, 4), (5, 130)])
@pytest.mark.parametrize("tree", ["random", None])
def test_trees_in_pieces(dtype, T, H, tree):
    """So many requests that a block is hardly cut, with caches around the length where a block's keys are taken in several pieces."""
    rng, P = random.Random(T), PIECE[dtype]
    lens = [P + rng.choice([-1, 0, 1, 127, 128, 129, 256, 300, 1000, P + 5]) if b % 5 else rng.choice([0, 1, 300]) for b in range(150)]
    check_shared_pages(shared_pages(T, lens, T, H, 1, dtype, "phd" if T == 40 else "hpd", tree), lens, T, dtype, 11)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("T,H,Hk,B", [(1, 7, 7, 260), (1, 8, 8, 230), (4, 16, 4, 460), (16, 2, 2, 900)])
def test_few_rows_in_pieces(dtype, T, H, Hk, B):
    """The same, for as many requests as there are warps (key heads side by side: CTAs)."""
    rng, P = random.Random(T), PIECE[dtype]
    lens = [P + rng.choice([-16, -1, 0, 1, 15, 16, 17, 32, 1000, P + 5]) if b % 7 else rng.choice([0, 1, 300]) for b in range(B)]
    check_shared_pages(shared_pages(T, lens, T, H, Hk, dtype, "phd" if T == 1 else "hpd", "random" if T == 4 else None), lens, T, dtype, 43)


@pytest.mark.gpu
def test_many_requests_with_a_very_long_cache():
    lens = [1 << 20] * 600 + [5]
    check_shared_pages(shared_pages(3, lens, 1, 4, 4, "f16", "hpd", None), lens, 1, "f16", 150)


# ---- a run of them together --------------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["hpd", "phd"])
def test_serving(dtype, layout):
    """Prompts, their keys into pages, drafts that are verified and accepted, forks, requests that end and start, a pool that is compacted:
    at every step attention is that over the requests' own histories."""
    rng, g = random.Random(1), torch.Generator(device="cuda").manual_seed(1)
    H, Hk, page, width, P, T, t = 8, 2, 16, 24, 120, 6, TYPES[dtype]

    def rand(*shape):
        return torch.randn(shape, generator=g, device="cuda").to(t)

    pools = [rand(P, page, Hk, 64).transpose(1, 2) if layout == "phd" else rand(P, Hk, page, 64) for _ in range(2)]
    users, pages, lens = ints([0] * P), ints([[-1] * width]), ints([0])
    history = [None]  # [Hk, n, 64] of keys and values of each request
    for step in range(8):
        # who goes on, who is forked, who is new
        source = [i for i, h in enumerate(history) if h is not None and rng.random() < 0.8]
        source += [rng.choice(source) for _ in range(2) if source and len(source) < 6]
        news = [rng.randint(1, 90) for _ in range(rng.randint(1, 2))] if len(source) < 6 else []
        rng.shuffle(source)
        room = [T] * len(source) + news
        pages, lens, users, missing = hk.cache_fork(*pools, pages, lens, users, ints(source + [-1] * len(news)), ints(room))
        assert int(missing) == 0
        history = [history[i] for i in source] + [(rand(Hk, 0, 64), rand(Hk, 0, 64)) for _ in news]
        assert lens.tolist() == [h[0].shape[1] for h in history]
        if news:  # prompts of the new ones; the others bring none
            N = sum(news)
            q, k, v = rand(N, H, 64), rand(N, Hk, 64), rand(N, Hk, 64)
            starts = [0] * (len(source) + 1)
            for n in news:
                starts.append(starts[-1] + n)
            starts = ints(starts)
            check_prompts(hk.prompt_attention(q, k, v, starts, SCALE), prompts(q, k, v, starts, True), dtype, slice(None))
            hk.cache_append(k, v, *pools, pages, lens, starts=starts)
            grown = starts[1:] - starts[:-1]
            for i, (a, b) in enumerate(zip(starts.tolist(), starts.tolist()[1:])):
                history[i] = tuple(torch.cat([h, x[a:b].transpose(0, 1)], 1) for h, x in zip(history[i], (k, v)))
            lens = lens + grown
        if step % 3 == 2:
            pages, users, where = hk.cache_compact(*pools, pages, users)
            n = int((users > 0).sum())
            assert int(users[n:].sum()) == 0
            for x in pools:
                x[n:] = math.nan  # nobody's
        B = len(history)
        pages, lens, users, missing = hk.cache_fork(*pools, pages, lens, users, ints(list(range(B))), T)
        assert int(missing) == 0
        for _ in range(2):
            q, k, v = rand(B, H, T, 64), rand(B, Hk, T, 64), rand(B, Hk, T, 64)
            parents = [[rng.randrange(-1, i) if i else -1 for i in range(T)] for _ in range(B)]
            bits = []
            for row in parents:
                r = []
                for i, p in enumerate(row):
                    r.append((r[p] if p >= 0 else 0) | 1 << i)
                bits.append(r)
            tree = torch.tensor(bits, device="cuda")
            got = hk.tree_attention(q, k, v, *pools, pages, lens, SCALE, tree)
            want = []
            for b, h in enumerate(history):
                kk, vv = (torch.cat([x, y[b]], 1).repeat_interleave(H // Hk, 0) for x, y in zip(h, (k, v)))
                sees = (tree[b][:, None] >> torch.arange(T, device="cuda") & 1).bool()
                want.append(attend(q[b], kk, vv, torch.cat([sees.new_ones((T, h[0].shape[1])), sees], 1), SCALE))
            check(got, tuple(torch.stack(x) for x in zip(*want)), dtype, step)
            # a path of the tree is accepted, or none of it
            picks, counts = [], []
            for b in range(B):
                at, path = rng.randrange(-1, T), []
                while at >= 0 and len(path) < 3:
                    path.append(at)
                    at = parents[b][at]
                path = sorted(path)
                if parents[b][path[0]] >= 0 if path else False:
                    path = []
                picks.append(path + [0] * (T - len(path)))
                counts.append(len(path))
            hk.cache_append(k, v, *pools, pages, lens, picks=ints(picks), counts=ints(counts))
            for b in range(B):
                history[b] = tuple(torch.cat([h, x[b][:, picks[b][:counts[b]]]], 1) for h, x in zip(history[b], (k, v)))
            lens = lens + ints(counts)
    assert hk.last_device_status() == 0


# ---- refusals ------------------------------------------------------------------------------------------------------------------------------
i32 = dict(dtype=torch.int32)


def _prompt(**c):
    x = dict(dict(q=torch.zeros(9, 4, 64), k=torch.zeros(9, 2, 64), v=torch.zeros(9, 2, 64), starts=torch.zeros(3, **i32), out=None, lse=None), **c)
    return hk.prompt_attention(x["q"], x["k"], x["v"], x["starts"], SCALE, out=x["out"], lse=x["lse"])


def _tree(**c):
    x = dict(dict(q=torch.zeros(2, 4, 5, 64), k=torch.zeros(2, 2, 5, 64), v=torch.zeros(2, 2, 5, 64), kp=torch.zeros(7, 2, 16, 64), vp=torch.zeros(7, 2, 16, 64), pages=torch.zeros(2, 4, **i32),
                  lens=torch.zeros(2, **i32), tree=None, out=None, lse=None), **c)
    return hk.tree_attention(x["q"], x["k"], x["v"], x["kp"], x["vp"], x["pages"], x["lens"], SCALE, x["tree"], out=x["out"], lse=x["lse"])


@pytest.mark.parametrize("call,name,wrong", [
    (_prompt, "Q", dict(q=torch.zeros(1, 9, 4, 64))), (_prompt, "Q", dict(q=torch.zeros(9, 4, 32))), (_prompt, "Q", dict(q=torch.zeros(9, 4, 64).double())), (_prompt, "K", dict(k=torch.zeros(8, 2, 64))),
    (_prompt, "K", dict(k=torch.zeros(9, 2, 64).half())), (_prompt, "V", dict(v=torch.zeros(9, 1, 64))), (_prompt, "starts", dict(starts=torch.zeros(1, **i32))),
    (_prompt, "starts", dict(starts=torch.zeros(3))), (_prompt, "starts", dict(starts=torch.zeros(6, **i32)[::2])), (_prompt, "out", dict(out=torch.zeros(9, 2, 64))),
    (_prompt, "out", dict(out=torch.zeros(9, 4, 64).half())), (_prompt, "lse", dict(lse=torch.zeros(9, 4))), (_prompt, "lse", dict(lse=torch.zeros(9, 4).T)), (_prompt, "lse", dict(lse=torch.zeros(4, 9).half())),
    (_tree, "Q", dict(q=torch.zeros(2, 4, 64))), (_tree, "K", dict(k=torch.zeros(2, 2, 4, 64))), (_tree, "K", dict(k=torch.zeros(1, 2, 5, 64))), (_tree, "V", dict(v=torch.zeros(2, 4, 5, 64))),
    (_tree, "K_pages", dict(kp=torch.zeros(7, 4, 16, 64))), (_tree, "K_pages", dict(kp=torch.zeros(7, 2, 16, 64).half())), (_tree, "V_pages", dict(vp=torch.zeros(8, 2, 16, 64))),
    (_tree, "K_pages", dict(kp=torch.zeros(1, 7, 2, 16, 64))), (_tree, "pages", dict(pages=torch.zeros(3, 4, **i32))), (_tree, "pages", dict(pages=torch.zeros(2, 4, dtype=torch.int64))),
    (_tree, "lengths", dict(lens=torch.zeros(3, **i32))), (_tree, "lengths", dict(lens=torch.zeros(2))), (_tree, "tree", dict(tree=torch.zeros(2, 5, **i32))), (_tree, "tree", dict(tree=torch.zeros(2, 4, dtype=torch.int64))),
    (_tree, "out", dict(out=torch.zeros(2, 4, 4, 64))), (_tree, "lse", dict(lse=torch.zeros(2, 4, 4)))])
def test_arguments_that_do_not_fit_are_refused(call, name, wrong):
    with pytest.raises(AssertionError, match="^" + name + ":"):
        call(**wrong)


@pytest.mark.parametrize("call,name,wrong", [(_prompt, "starts", dict(starts=[0, 9])), (_prompt, "out", dict(out=3)), (_tree, "tree", dict(tree=[[1]])), (_tree, "lengths", dict(lens=None)),
                                             (_tree, "V_pages", dict(vp=None))])
def test_what_is_no_tensor_is_refused(call, name, wrong):
    with pytest.raises(TypeError, match="^" + name + ":"):
        call(**wrong)


def test_host_tensors_are_refused():
    for call in (_prompt, _tree):
        with pytest.raises(AssertionError, match="CUDA"):
            call()


class View(C.Structure):
    _fields_ = [("ptr", C.c_void_p), ("sB", C.c_int64), ("sM", C.c_int64), ("sH", C.c_int64)]


class Pool(C.Structure):
    _fields_ = [("K", View), ("V", View), ("pages", C.c_void_p), ("stride", C.c_int64), ("width", C.c_int), ("n_pages", C.c_int), ("page", C.c_int)]


class Prompt(C.Structure):
    _fields_ = [("Q", View), ("K", View), ("V", View), ("O", View), ("LSE", C.c_void_p), ("lse_sH", C.c_int64), ("starts", C.c_void_p), ("B", C.c_int), ("nh", C.c_int), ("nh_kv", C.c_int),
                ("dtype", C.c_int), ("N", C.c_int64), ("scale", C.c_float), ("is_causal", C.c_bool), ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t)]


class Tree(C.Structure):
    _fields_ = [("Q", View), ("K", View), ("V", View), ("O", View), ("LSE", C.c_void_p), ("lse_sB", C.c_int64), ("lse_sH", C.c_int64), ("pool", Pool), ("lengths", C.c_void_p), ("tree", C.c_void_p),
                ("tree_stride", C.c_int64), ("B", C.c_int), ("nh", C.c_int), ("nh_kv", C.c_int), ("dtype", C.c_int), ("T", C.c_int64), ("scale", C.c_float), ("workspace", C.c_void_p),
                ("workspace_bytes", C.c_size_t)]


def block(kind):
    """Blocks of a call that fits, on addresses that nothing reads: every check is in front of the first launch"""
    b = kind()
    b.LSE, b.scale, b.nh, b.nh_kv, b.dtype, b.B = 0x1000, 0.125, 4, 2, 0, 2
    if kind is Prompt:
        b.Q = b.O = View(0x1000, 0, 4 * 64, 64)
        b.K = b.V = View(0x1000, 0, 2 * 64, 64)
        b.starts, b.N, b.lse_sH = 0x1000, 9, 9
    else:
        b.Q = b.O = View(0x1000, 4 * 5 * 64, 64, 5 * 64)
        b.K = b.V = View(0x1000, 2 * 5 * 64, 64, 5 * 64)
        b.pool.K = b.pool.V = View(0x1000, 2 * 16 * 64, 64, 16 * 64)
        b.pool.pages, b.pool.stride, b.pool.width, b.pool.n_pages, b.pool.page = 0x1000, 4, 4, 7, 16
        b.lengths, b.T, b.lse_sB, b.lse_sH = 0x1000, 5, 20, 5
    return b


def answer(b):
    f = hk.lib().hk_prompt_attention if type(b) is Prompt else hk.lib().hk_tree_attention
    f.argtypes = [C.c_void_p, C.c_void_p]
    return f(C.byref(b) if b is not None else None, None)


@pytest.mark.parametrize("kind,path,value,status", [
    (Prompt, "Q.ptr", None, -1), (Prompt, "starts", None, -1), (Prompt, "LSE", None, -1), (Prompt, "O.ptr", 0x1004, -3), (Prompt, "K.sM", 130, -3), (Prompt, "K.sH", 0, -6), (Prompt, "V.sM", 0, -6),
    (Prompt, "O.sM", 64, -6), (Prompt, "lse_sH", 8, -6), (Prompt, "N", 0, -2), (Prompt, "B", 0, -2), (Prompt, "nh", 3, -2), (Prompt, "nh_kv", 0, -2), (Prompt, "scale", 0.0, -2),
    (Prompt, "scale", math.inf, -2), (Prompt, "dtype", 3, -6), (Prompt, "starts", 0x1002, -3), (Prompt, "N", 1 << 30, -2),
    (Tree, "K.ptr", None, -1), (Tree, "lengths", None, -1), (Tree, "pool.pages", None, -1), (Tree, "pool.V.ptr", None, -1), (Tree, "pool.K.sB", 0, -6), (Tree, "pool.K.sM", 0, -6), (Tree, "pool.page", 24, -6),
    (Tree, "pool.page", 0, -2), (Tree, "pool.width", 1 << 27, -2), (Tree, "T", 65, -6), (Tree, "T", 0, -2), (Tree, "nh", 5, -2), (Tree, "scale", math.nan, -2), (Tree, "tree", 0x1004, -3), (Tree, "tree_stride", -1, 0),
    (Tree, "lse_sH", 4, -6), (Tree, "Q.sM", 65, -3), (Tree, "dtype", -1, -6), (Tree, "O.sH", 64, -6), (Tree, "pool.K.ptr", 0x1008, -3)])
def test_blocks_that_are_refused(kind, path, value, status):
    b = block(kind)
    at, (*way, last) = b, path.split(".")
    for name in way:
        at = getattr(at, name)
    setattr(at, last, value)
    if path == "tree_stride":
        b.tree, status = 0x1000, -2
    assert answer(b) == status
    for f in (hk.lib().hk_prompt_attention, hk.lib().hk_tree_attention):
        f.argtypes = [C.c_void_p, C.c_void_p]
        assert f(None, None) == -1


# ---- the line of the work --------------------------------------------------------------------------------------------------------------
def line_of(b, lens):
    """All units, units of the narrowest block, tiles lost at blocks' ends, 2^x keys to a unit; lens: [n], so often as there are requests"""
    f = hk.lib().hk_prompt_line if type(b) is Prompt else hk.lib().hk_tree_line
    f.argtypes = [C.c_void_p, C.c_void_p, C.c_void_p]
    all_lens = torch.tensor(lens, dtype=torch.int32).repeat(cdiv(b.B, len(lens)))[:b.B].contiguous()
    out = (C.c_int64 * 4)()
    assert f(C.byref(b), all_lens.data_ptr(), out) == 0
    return list(out)


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("N,B,H,Hk,lens,shift", [
    (9, 2, 4, 2, [9, 0], 0), (1 << 17, 1 << 17, 12, 12, [1], 0), (1 << 20, 1 << 20, 8, 8, [1], 5), (1 << 20, 1000, 64, 8, [5, 2000], None), (1 << 20, 1 << 15, 64, 8, [32], None), (1 << 17, 1 << 17, 64, 64, [1], None),
    (1 << 24, 1 << 20, 64, 1, [16], None), (1 << 24, 3, 1, 1, [100, 0, (1 << 24) - 100], None), (1 << 30, 1 << 20, 1, 1, [1024], None), (1 << 30, 2, 1, 1, [1, (1 << 30) - 1], None), (1 << 21, 7, 300, 1, [300000], None)])
def test_every_block_of_prompts_is_on_the_line(N, B, H, Hk, lens, shift, dtype, causal):
    b = block(Prompt)
    b.N, b.B, b.nh, b.nh_kv, b.dtype, b.is_causal = N, B, H, Hk, dtype, causal
    units, narrowest, lost, unit_shift = line_of(b, lens)
    assert 0 < units < 2 ** 31 and narrowest >= 1 and lost == 0, (units, narrowest, lost, unit_shift)
    assert shift is None or unit_shift == shift or unit_shift == shift + 1


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("B,T,H,Hk,width,page,lens", [
    (2, 1, 4, 4, 64, 16, [9, 0]), (64, 1, 1, 1, 16384, 65536, [0]), (64, 1, 1, 1, 16384, 65536, [0, 1, 70, 5000]), (1 << 16, 1, 32, 8, 16384, 64, [0, 1 << 20, 17]), (1 << 16, 16, 32, 32, 16384, 64, [3, 1 << 20]),
    (1 << 16, 64, 256, 1, 1024, 1024, [1 << 20]), (1 << 24, 64, 1, 1, 64, 16, [0, 1]), (1 << 12, 64, 300, 2, 1 << 18, 4096, [1 << 30, 0]),
    (2900000, 17, 1, 1, 1, 16, [16]), (2900000, 17, 1, 1, 1, 16, [1]), (2900000, 40, 4, 1, 1, 16, [16])])
def test_every_block_of_a_tree_is_on_the_line(B, T, H, Hk, width, page, lens, dtype):
    b = block(Tree)
    b.B, b.T, b.nh, b.nh_kv, b.dtype, b.pool.width, b.pool.page = B, T, H, Hk, dtype, width, page
    units, narrowest, lost, unit_shift = line_of(b, lens)
    assert 0 < units < 2 ** 31 and narrowest >= 1 and lost == 0, (units, narrowest, lost, unit_shift)
