"""The pages of a cache: appending, forking, compacting, against models of them in Python, bit for bit."""
import ctypes as C
import random

import pytest
import torch

import hyperkernels_b200 as hk

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def pool(g, layers, P, Hk, page, dtype, layout):
    """[(layers,) P, Hk, page, 64] with room round it that nothing may touch"""
    lead = () if layers is None else (layers,)
    if layout == "phd":
        x = torch.randn((*lead, P + 2, page, Hk, 64), generator=g, device="cuda").to(TYPES[dtype])
        return x, x.narrow(len(lead), 1, P).transpose(-3, -2)
    if layout == "wide":
        x = torch.randn((*lead, P + 2, Hk, page + 1, 128), generator=g, device="cuda").to(TYPES[dtype])
        return x, x.narrow(len(lead), 1, P)[..., :page, 64:]
    x = torch.randn((*lead, P + 2, Hk, page, 64), generator=g, device="cuda").to(TYPES[dtype])
    return x, x.narrow(len(lead), 1, P)


def ints(x):
    return torch.tensor(x, device="cuda", dtype=torch.int32)


def cdiv(a, b):
    return -(-a // b)


def table(rng, P, counts, width, stray=()):
    """Rows of different pages; -1 and (stray) other entries that are no pages behind them"""
    order = list(range(P))
    rng.shuffle(order)
    rows = []
    for n in counts:
        row = [order.pop() for _ in range(n)]
        rows.append(row + [rng.choice([-1, *stray]) for _ in range(width - n)])
    return rows


# ---- appending ------------------------------------------------------------------------------------------------------------------------
def append_model(k, v, kp, vp, pages, lens, rows):
    """rows[b]: rows of k and v ([Hk, T, 64] each) in their order"""
    P, page = kp.shape[0], kp.shape[2]
    for b, (kb, vb, mine) in enumerate(rows):
        for i, r in enumerate(mine):
            if r is None:
                continue
            at, off = divmod(max(lens[b], 0) + i, page)
            if at < len(pages[b]) and 0 <= pages[b][at] < P:
                kp[pages[b][at], :, off], vp[pages[b][at], :, off] = kb[:, r], vb[:, r]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["hpd", "phd", "wide"])
@pytest.mark.parametrize("Hk,page,lens,news", [
    (1, 16, [0], [1]), (3, 16, [0, 5, 16, 31, 100], [40, 0, 16, 2, 1]), (12, 64, [63, 64, 0, 1], [1, 200, 64, 65]), (8, 48, [0] * 40, list(range(40))),
    (33, 32, [7, -3], [33, 5]), (2, 16, [0] * 300, [1] * 300)])
def test_packed_prompts(dtype, layout, Hk, page, lens, news):
    g, rng, B = torch.Generator(device="cuda").manual_seed(Hk), random.Random(Hk), len(lens)
    width = max(cdiv(max(a, 0) + n, page) for a, n in zip(lens, news)) + 1
    counts = [cdiv(max(a, 0) + n, page) for a, n in zip(lens, news)]
    if B > 2:
        counts[-1] = max(0, counts[-1] - 1)  # a request that lacks a page
    P = sum(counts) + 3
    rows = table(rng, P, counts, width, stray=(P, P + 7, -9))
    before, after = 3, 2  # rows of no sequence
    N = sum(news) + before + after
    starts = [before]
    for n in news:
        starts.append(starts[-1] + n)
    x = torch.randn((N, 2 * Hk + 1, 64), generator=g, device="cuda").to(TYPES[dtype])
    k, v = x[:, :Hk], x[:, Hk:2 * Hk]
    (ka, kp), (va, vp) = pool(g, None, P, Hk, page, dtype, layout), pool(g, None, P, Hk, page, dtype, layout)
    want_k, want_v = ka.clone(), va.clone()
    wk, wv = (torch.as_strided(w, p.shape, p.stride(), p.storage_offset()) for w, p in ((want_k, kp), (want_v, vp)))
    append_model(None, None, wk, wv, rows, lens, [(k.transpose(0, 1), v.transpose(0, 1), range(a, b)) for a, b in zip(starts, starts[1:])])
    wide = ints(rows + [[-1] * width])[:, :width]
    assert hk.cache_append(k, v, kp, vp, wide[:B], ints(lens), starts=ints(starts)) is None
    assert torch.equal(ka, want_k) and torch.equal(va, want_v)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("Hk,page,T", [(1, 16, 1), (3, 16, 7), (12, 64, 64), (2, 32, 100)])
@pytest.mark.parametrize("some", ["picks", "counts", "both", "none"])
def test_accepted_drafts(dtype, Hk, page, T, some):
    g, rng, B = torch.Generator(device="cuda").manual_seed(T), random.Random(T), 9
    lens = [rng.choice([0, 1, page - 1, page, 3 * page + 5]) for _ in range(B)]
    counts = [rng.choice([0, 1, T, T // 2, T + 5, -2]) for _ in range(B)]
    picks = [[rng.randrange(T) for _ in range(T)] for _ in range(B)]  # the same row twice, any order
    picks[1][0], picks[2][-1] = -1, T
    width = cdiv(max(lens) + T, page)
    have = [cdiv(n + T, page) for n in lens]
    P = sum(have) + 2
    rows = table(rng, P, have, width)
    k, v = (torch.randn((B, T, Hk, 64), generator=g, device="cuda").to(TYPES[dtype]).transpose(1, 2) for _ in range(2))
    (ka, kp), (va, vp) = pool(g, None, P, Hk, page, dtype, "phd"), pool(g, None, P, Hk, page, dtype, "hpd")
    want_k, want_v = ka.clone(), va.clone()
    wk, wv = (torch.as_strided(w, p.shape, p.stride(), p.storage_offset()) for w, p in ((want_k, kp), (want_v, vp)))
    mine = []
    for b in range(B):
        n = min(max(counts[b], 0), T) if some in ("counts", "both") else T
        r = picks[b] if some in ("picks", "both") else list(range(T))
        mine.append((k[b], v[b], [i if 0 <= i < T else None for i in r[:n]]))
    append_model(None, None, wk, wv, rows, lens, mine)
    hk.cache_append(k, v, kp, vp, ints(rows), ints(lens), picks=ints(picks) if some in ("picks", "both") else None,
                    counts=ints(counts) if some in ("counts", "both") else None)
    assert torch.equal(ka, want_k) and torch.equal(va, want_v)


@pytest.mark.gpu
def test_starts_that_are_no_starts():
    """Beyond the tensors, descending: rows may go anywhere in the pages of the requests, never elsewhere, and nothing else is read."""
    g = torch.Generator(device="cuda").manual_seed(1)
    k = torch.randn((20, 2, 64), generator=g, device="cuda")
    ka, kp = pool(g, None, 6, 2, 16, "f32", "hpd")
    before = ka.clone()
    for starts in ([-100, 5, 1000], [10, 3, 20], [2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1], [-2 ** 31, -2 ** 31, -2 ** 31], [0, -7, 2 ** 31 - 1]):
        for lens in ([0, 2 ** 31 - 1], [-2 ** 31, 5]):
            hk.cache_append(k, k, kp, kp, ints([[0, 1], [2, 3]]), ints(lens), starts=ints(starts))
    torch.cuda.synchronize()
    assert torch.equal(ka[0], before[0]) and torch.equal(ka[5:], before[5:])


@pytest.mark.gpu
def test_starts_are_taken_into_the_tensor():
    """As the attention takes them: a first prompt that begins in front of the tensor begins with its first row."""
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn((250, 2, 64), generator=g, device="cuda")
    rows, lens = [list(range(6)), list(range(6, 24))], [3, 20]
    want = None
    for starts in ([0, 50, 250], [-7, 50, 100000], [-2 ** 31, 50, 2 ** 31 - 1]):
        _, kp = pool(torch.Generator(device="cuda").manual_seed(3), None, 24, 2, 16, "f32", "hpd")
        _, vp = pool(torch.Generator(device="cuda").manual_seed(4), None, 24, 2, 16, "f32", "phd")
        if want is None:
            want = kp.clone(), vp.clone()
            parts = [(x[a:b].transpose(0, 1), -x[a:b].transpose(0, 1), range(b - a)) for a, b in ((0, 50), (50, 250))]
            append_model(None, None, *want, rows, lens, parts)
        table_ = ints([r + [-1] * (18 - len(r)) for r in rows])
        hk.cache_append(x, -x, kp, vp, table_, ints(lens), starts=ints(starts))
        assert torch.equal(kp, want[0]) and torch.equal(vp, want[1]), starts
    _, kp = pool(torch.Generator(device="cuda").manual_seed(3), None, 24, 2, 16, "f32", "hpd")
    hk.cache_append(x, x, kp, kp.clone(), table_, ints(lens), starts=ints([-9, -4, 250]))  # the first is empty
    first = [(x[:0].transpose(0, 1), None, range(0)), (x.transpose(0, 1), x.transpose(0, 1), range(250))]
    _, wk = pool(torch.Generator(device="cuda").manual_seed(3), None, 24, 2, 16, "f32", "hpd")
    append_model(None, None, wk, wk.clone(), rows, lens, first)
    assert torch.equal(kp, wk)


# ---- forking ------------------------------------------------------------------------------------------------------------------------
def fork_model(kp, vp, pages, lens, users, source, room):
    """Tables, and copies made in kp, vp: [layers, P, Hk, page, 64]"""
    P, page, width = kp.shape[1], kp.shape[3], len(pages[0])
    users = list(users)
    for row in pages:
        for p in row:
            if 0 <= p < P:
                users[p] -= 1
    out, out_lens, missing, begun, copies = [], [], 0, {}, []
    for i, b in enumerate(source):
        alive = 0 <= b < len(pages)
        n = min(max(lens[b], 0), width * page) if alive else 0
        row = [p if 0 <= p < P else -1 for p in pages[b][:cdiv(n, page)]] if alive else []
        if n % page:
            if b in begun:
                copies.append((i, n // page, row.pop(), n % page))
            else:
                begun[b] = i
        for p in row:
            if p >= 0:
                users[p] += 1
        out.append(row)
        out_lens.append(n)
    free = [p for p in range(P) if users[p] == 0]
    for i, row in enumerate(out):
        need = cdiv(out_lens[i] + max(room[i], 0), page)
        missing += max(0, need - width)
        while len(row) < min(need, width):
            row.append(free.pop(0) if free else -1)
            missing += row[-1] < 0
            if row[-1] >= 0:
                users[row[-1]] += 1
        row += [-1] * (width - len(row))
    for i, at, frm, rows in copies:
        if out[i][at] >= 0 and frm >= 0:
            for x in (kp, vp):
                x[:, out[i][at], :, :rows] = x[:, frm, :, :rows]
    return out, out_lens, users, missing


def fork_case(seed):
    """Requests of a random history: some share pages, some pages are somebody else's, entries behind a request's pages may be its too"""
    rng = random.Random(seed)
    B, page, width = rng.choice([1, 2, 5, 16, 40]), rng.choice([16, 32, 48]), rng.choice([1, 3, 8])
    P = rng.choice([B, B * width // 2 + 2, B * width * 2, 1500])
    lens, pages, users, order = [], [], [0] * P, list(range(P))
    rng.shuffle(order)
    for b in range(B):
        n = min(rng.choice([0, 1, page, page + 1, rng.randint(0, width * page), width * page]), width * page)
        if b and rng.random() < 0.3:  # full pages like the one before's
            full = min(n, lens[-1]) // page
            row = pages[-1][:full]
        else:
            row = []
        while len(row) < cdiv(n, page) and order:
            row.append(order.pop())
        n = min(n, len(row) * page)
        if len(row) < width and order and rng.random() < 0.3:
            row.append(order.pop())  # room that it had already
        for p in row:
            users[p] += 1
        lens.append(n)
        pages.append(row + [rng.choice([-1, P, -2 ** 31, 2 ** 31 - 1]) for _ in range(width - len(row))])
    for p in rng.sample(range(P), P // 7):
        users[p] += rng.randint(1, 3)
    B_out = rng.choice([1, B, B + 3, 2 * B, 1100 if seed % 10 == 0 else B])
    source = [rng.choice([rng.randrange(B), rng.randrange(B), -1, B]) for _ in range(B_out)]
    room = [rng.choice([0, 1, 1, page, rng.randint(0, 3 * page), -5]) for _ in range(B_out)]
    return B, page, width, P, lens, pages, users, source, room


@pytest.mark.gpu
@pytest.mark.parametrize("seed", range(60))
def test_the_next_batch(seed):
    B, page, width, P, lens, pages, users, source, room = fork_case(seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    Hk, dtype, layout, layers = [1, 2, 5, 12][seed % 4], list(TYPES)[seed % 3], ["hpd", "phd", "wide"][seed // 3 % 3], [None, 1, 3][seed // 9 % 3]
    (ka, kp), (va, vp) = pool(g, layers, P, Hk, page, dtype, layout), pool(g, layers, P, Hk, page, dtype, layout)
    want_k, want_v = ka.clone(), va.clone()
    wk, wv = (torch.as_strided(w, p.shape, p.stride(), p.storage_offset()) for w, p in ((want_k, kp), (want_v, vp)))
    if layers is None:
        wk, wv = wk[None], wv[None]
    if seed % 5 == 4:
        room = [seed] * len(room)
    want = fork_model(wk, wv, pages, lens, users, source, room)
    args = (ints(pages), ints(lens), ints(users), ints(source), seed if seed % 5 == 4 else ints(room))
    keep = [x.clone() for x in args[:4]]
    for _ in range(2):  # the old batch is still there: the same again
        got = hk.cache_fork(kp, vp, *args)
        assert [x.tolist() for x in got] == [want[0], want[1], want[2], [want[3]]]
        assert torch.equal(ka, want_k) and torch.equal(va, want_v)
    assert all(torch.equal(a, b) for a, b in zip(keep, args))


@pytest.mark.gpu
@pytest.mark.parametrize("B,P", [(2500, 30000), (1300, 20000), (700, 9000)])
def test_large_tables(B, P):
    """More requests and pages than the CTA has threads, and room for"""
    rng, g = random.Random(1), torch.Generator(device="cuda").manual_seed(1)
    page, width = 16, 9
    lens = [rng.randint(0, width * page) for _ in range(B)]
    pages = table(rng, P, [cdiv(n, page) for n in lens], width)
    users = [0] * P
    for p in sum(pages, []):
        if p >= 0:
            users[p] += 1
    source, room = [rng.randrange(-B // 10, B) for _ in range(B + 77)], [rng.randint(0, 20) for _ in range(B + 77)]
    (ka, kp), (va, vp) = pool(g, None, P, 1, page, "bf16", "hpd"), pool(g, None, P, 1, page, "bf16", "hpd")
    wk, wv = ka.clone(), va.clone()
    want = fork_model(wk[None, 1:-1], wv[None, 1:-1], pages, lens, users, source, room)
    got = hk.cache_fork(kp, vp, ints(pages), ints(lens), ints(users), ints(source), ints(room))
    assert [x.tolist() for x in got] == [want[0], want[1], want[2], [want[3]]]
    assert torch.equal(ka, wk) and torch.equal(va, wv)
    rows, users, where = compact_model(wk[None, 1:-1], wv[None, 1:-1], want[0], want[2])
    got = hk.cache_compact(kp, vp, got[0], got[2])
    assert [x.tolist() for x in got] == [rows, users, where]
    assert torch.equal(ka, wk) and torch.equal(va, wv)


@pytest.mark.gpu
def test_more_missing_than_there_are_numbers():
    g = torch.Generator(device="cuda").manual_seed(0)
    (_, kp), (_, vp) = pool(g, None, 4, 1, 16, "f32", "hpd"), pool(g, None, 4, 1, 16, "f32", "hpd")
    for B, room, missing in ((1, 2 ** 31 - 1, 2 ** 27 - 4), (1, 2 ** 30, 2 ** 26 - 4), (3, 2 ** 31 - 1, 3 * 2 ** 27 - 4), (3000, 2 ** 31 - 1, 2 ** 31 - 1), (3000, 0, 0)):
        got = hk.cache_fork(kp, vp, ints([[-1] * 4] * B), ints([0] * B), ints([0] * 4), ints([-1] * B), ints([room] * B))
        assert got[3].tolist() == [missing] and got[0].flatten().tolist() == ([0, 1, 2, 3] if missing else []) + [-1] * (4 * B - 4 * (missing > 0))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["hpd", "phd"])
@pytest.mark.parametrize("beams", [1, 3])
def test_begun_pages_that_are_none(dtype, layout, beams):
    """What an earlier call had no page for counts as rows of zeros: whoever goes on there gets a page that begins with such, as
    soon as there is one.  Full pages that are none are shared as such."""
    g = torch.Generator(device="cuda").manual_seed(beams)
    (ka, kp), (va, vp) = (pool(g, 2, 12, 3, 16, dtype, layout) for _ in range(2))
    ka.fill_(float("nan")), va.fill_(float("nan"))
    rows, lens, users = [[3, -1, 12], [-1, 5, 40], [-7, -1, -1], [9, -1, -1]], [20, 32, 1, 16], [0] * 12
    for p in (3, 5, 9):
        users[p] = 1
    source = [b for b in range(4) for _ in range(beams)]
    want_rows, want_users, free = [], list(users), iter(p for p in range(12) if users[p] == 0)
    begun = []  # new pages that begin with zeros, and how many rows of them
    for b in source:
        new = next(free, -1) if b in (0, 2, 3) else None
        if b in (0, 2) and new >= 0:
            begun.append((new, lens[b] % 16))
        want_rows.append({0: [3, new, -1], 1: [-1, 5, -1], 2: [new, -1, -1], 3: [9, new, -1]}[b])
    for p in range(12):
        want_users[p] = sum(row.count(p) for row in want_rows)
    room = [0 if b != 3 else 1 for b in source]
    got = hk.cache_fork(kp, vp, ints(rows), ints(lens), ints(users), ints(source), ints(room))
    assert [x.tolist() for x in got] == [want_rows, [lens[b] for b in source], want_users, [0]]
    for x in (kp, vp):
        for p in range(12):
            n = dict(begun).get(p, 0)
            assert bool((x[:, p, :, :n] == 0).all()) and bool(x[:, p, :, n:].isnan().all()), p
    # an empty pool: still none, and said so
    full = [max(u, 1) for u in users]
    got = hk.cache_fork(kp, vp, ints(rows), ints(lens), ints(full), ints(source), ints(room))
    assert got[0].tolist() == [[p if p != new else -1 for p, new in zip(r, [{0: r[1], 2: r[0], 3: r[1]}.get(b)] * 3)] for r, b in zip(want_rows, source)]
    assert got[3].tolist() == [3 * beams]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,layout", [("f32", "hpd"), ("bf16", "phd"), ("f16", "wide")])
def test_beams_of_many_layers(dtype, layout):
    """More to copy than the kernel over the tables copies, tables that fit its shared memory: the copies are a kernel of their own."""
    rng, g = random.Random(3), torch.Generator(device="cuda").manual_seed(3)
    B, beams, layers, Hk, page, width = 16, 4, 28, 12, 64, 5
    lens = [rng.randint(0, (width - 1) * page) for _ in range(B)]
    lens[0], lens[1], lens[2] = 0, page, page + 1
    P = sum(cdiv(n, page) for n in lens) + 2 * B * beams - 100  # too few for all
    pages = table(rng, P, [cdiv(n, page) for n in lens], width)
    users = [0] * P
    for p in sum(pages, []):
        if p >= 0:
            users[p] += 1
    source, room = [b for b in range(B) for _ in range(beams)], [1 + 70 * (i % 3) for i in range(B * beams)]
    rng.shuffle(source)
    (ka, kp), (va, vp) = pool(g, layers, P, Hk, page, dtype, layout), pool(g, layers, P, Hk, page, dtype, layout)
    want_k, want_v = ka.clone(), va.clone()
    wk, wv = (torch.as_strided(w, p.shape, p.stride(), p.storage_offset()) for w, p in ((want_k, kp), (want_v, vp)))
    want = fork_model(wk, wv, pages, lens, users, source, room)
    before = hk.launch_count()
    got = hk.cache_fork(kp, vp, ints(pages), ints(lens), ints(users), ints(source), ints(room))
    assert hk.launch_count() - before == 2 and want[3] > 0
    assert [x.tolist() for x in got] == [want[0], want[1], want[2], [want[3]]]
    assert torch.equal(ka, want_k) and torch.equal(va, want_v)
    # and the pages to the front by the same
    rows, users, where = compact_model(wk, wv, [r[:2] for r in want[0]], [u if p % 3 else 0 for p, u in enumerate(want[2])])
    before = hk.launch_count()
    moved = hk.cache_compact(kp, vp, got[0][:, :2], got[2] * ints([1 if p % 3 else 0 for p in range(P)]))
    assert hk.launch_count() - before == 2
    assert [x.tolist() for x in moved] == [rows, users, where]
    assert torch.equal(ka, want_k) and torch.equal(va, want_v)


# ---- compacting ------------------------------------------------------------------------------------------------------------------------
def compact_model(kp, vp, pages, users):
    P = kp.shape[1]
    n = sum(u > 0 for u in users)
    where, out, holes = [-1] * P, [0] * P, [p for p in range(n) if users[p] <= 0]
    for p in range(P):
        if users[p] > 0:
            where[p] = p if p < n else holes.pop(0)
            out[where[p]] = users[p]
            for x in (kp, vp):
                x[:, where[p]] = x[:, p].clone()
    return [[where[p] if 0 <= p < P else -1 for p in row] for row in pages], out, where


@pytest.mark.gpu
@pytest.mark.parametrize("seed", range(40))
def test_pages_to_the_front(seed):
    rng, g = random.Random(seed), torch.Generator(device="cuda").manual_seed(seed)
    P, page, Hk, layers = rng.choice([1, 2, 7, 100, 1024, 3000]), rng.choice([16, 32, 48, 80]), rng.choice([1, 3, 8]), rng.choice([None, 1, 3])
    dtype, layout, share = list(TYPES)[seed % 3], ["hpd", "phd", "wide"][seed // 3 % 3], rng.choice([0.0, 0.1, 0.5, 0.9, 1.0])
    users = [rng.randint(1, 4) if rng.random() < share else rng.choice([0, 0, -1]) for _ in range(P)]
    B, width = rng.choice([1, 7, 40]), rng.choice([1, 5, 33])
    pages = [[rng.randrange(-1, P + 1) for _ in range(width)] for _ in range(B)]
    (ka, kp), (va, vp) = pool(g, layers, P, Hk, page, dtype, layout), pool(g, layers, P, Hk, page, dtype, layout)
    want_k, want_v = ka.clone(), va.clone()
    wk, wv = (torch.as_strided(w, p.shape, p.stride(), p.storage_offset()) for w, p in ((want_k, kp), (want_v, vp)))
    if layers is None:
        wk, wv = wk[None], wv[None]
    want = compact_model(wk, wv, pages, users)
    table_, users_ = ints(pages), ints(users)
    for _ in range(2):
        got = hk.cache_compact(kp, vp, table_, users_)
        assert [x.tolist() for x in got] == list(want)
        assert torch.equal(ka, want_k) and torch.equal(va, want_v)
    again = hk.cache_compact(kp, vp, got[0], got[1])  # nothing to do any more
    assert torch.equal(again[0], got[0]) and torch.equal(again[1], got[1]) and torch.equal(ka, want_k)


# ---- calls ------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
def test_captured_calls_follow_their_tables():
    """Appending, forking and compacting in one graph each, replayed on other tables, two graphs on two streams at once."""
    graphs = []
    for k in range(2):
        g = torch.Generator(device="cuda").manual_seed(k)
        P, Hk, page, B, width = 400, 2, 16, 12, 8
        kp, vp = (torch.randn((P, Hk, page, 64), generator=g, device="cuda") for _ in range(2))
        new = torch.randn((B, Hk, 3, 64), generator=g, device="cuda")
        args = [ints([[0] * width] * B), ints([0] * B), ints([0] * P), ints([0] * B), ints([0] * B)]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            pages, lens, users, missing = hk.cache_fork(kp, vp, *args)
            hk.cache_append(new, new, kp, vp, pages, lens)
            moved = hk.cache_compact(kp, vp, pages, users)
        graphs.append((graph, torch.cuda.Stream(), kp, vp, new, args, (pages, lens, users, missing), moved))
    for seed in range(5):
        wants = []
        for k, (graph, s, kp, vp, new, args, got, moved) in enumerate(graphs):
            rng = random.Random(10 * seed + k)
            lens = [rng.randint(0, 100) for _ in range(12)]
            rows = table(rng, 400, [cdiv(n, 16) for n in lens], 8)
            users = [0] * 400
            for p in sum(rows, []):
                if p >= 0:
                    users[p] += 1
            source = [rng.randrange(-1, 12) for _ in range(12)]
            for x, y in zip(args, (rows, lens, users, source, [3] * 12)):
                x.copy_(torch.tensor(y, dtype=torch.int32))
            wk, wv = kp.clone(), vp.clone()
            w = fork_model(wk[None], wv[None], rows, lens, users, source, [3] * 12)
            append_model(None, None, wk, wv, w[0], w[1], [(new[b], new[b], range(3)) for b in range(12)])
            wants.append((w, compact_model(wk[None], wv[None], w[0], w[2]), wk, wv))
        torch.cuda.synchronize()
        for graph, s, *_ in graphs:
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for (w, c, wk, wv), (_, _, kp, vp, _, _, got, moved) in zip(wants, graphs):
            assert [x.tolist() for x in got] == [w[0], w[1], w[2], [w[3]]]
            assert [x.tolist() for x in moved] == list(c)
            assert torch.equal(kp, wk) and torch.equal(vp, wv)


@pytest.mark.gpu
def test_pages_far_apart():
    """Offsets that pass 32 bits, in bytes and in elements"""
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB")
    P, Hk, page = 3, 2, 16
    far = torch.zeros((2, P, (1 << 32) // 4 + 64), device="cuda", dtype=torch.bfloat16)
    kp, vp = (far[i].as_strided((P, Hk, page, 64), (far.stride(1), page * 64, 64, 1), far[i].storage_offset()) for i in range(2))
    k = torch.arange(1, 33, device="cuda").to(torch.bfloat16)[:, None, None].expand(32, Hk, 64).contiguous()
    hk.cache_append(k, -k, kp, vp, ints([[2, 0]]), ints([0]), starts=ints([0, 32]))
    assert torch.equal(kp[2, :, :, 0].float(), torch.arange(1, 17, device="cuda").float().expand(2, 16)) and torch.equal(vp[0, :, :, 5], -kp[0, :, :, 5])
    got = hk.cache_compact(kp, vp, ints([[2, 0]]), ints([1, 0, 1]))
    assert [x.tolist() for x in got] == [[[1, 0]], [1, 1, 0], [0, -1, 1]] and torch.equal(kp[1], kp[2])
    got = hk.cache_fork(kp, vp, ints([[1, 0]]), ints([21]), ints([1, 1, 0]), ints([0, 0]), 0)
    assert [x.tolist() for x in got] == [[[1, 0], [1, 2]], [21, 21], [1, 2, 1], [0]]
    assert torch.equal(kp[2, :, :5], kp[0, :, :5]) and not torch.equal(kp[2, :, 5:], kp[0, :, 5:])


# ---- refusals ------------------------------------------------------------------------------------------------------------------------------
def _args(**changed):
    x = dict(k=torch.zeros(2, 3, 5, 64), v=torch.zeros(2, 3, 5, 64), kp=torch.zeros(7, 3, 16, 64), vp=torch.zeros(7, 3, 16, 64), pages=torch.zeros(2, 4, dtype=torch.int32),
             lens=torch.zeros(2, dtype=torch.int32), users=torch.zeros(7, dtype=torch.int32), source=torch.zeros(3, dtype=torch.int32), room=1, starts=None, picks=None, counts=None)
    return dict(x, **changed)


def _append(**c):
    x = _args(**c)
    return hk.cache_append(x["k"], x["v"], x["kp"], x["vp"], x["pages"], x["lens"], starts=x["starts"], picks=x["picks"], counts=x["counts"])


def _fork(**c):
    x = _args(**c)
    return hk.cache_fork(x["kp"], x["vp"], x["pages"], x["lens"], x["users"], x["source"], x["room"])


def _compact(**c):
    x = _args(**c)
    return hk.cache_compact(x["kp"], x["vp"], x["pages"], x["users"])


i32 = dict(dtype=torch.int32)


@pytest.mark.parametrize("call,name,wrong", [
    (_append, "K", dict(k=torch.zeros(3, 3, 5, 64))), (_append, "K", dict(k=torch.zeros(2, 3, 5, 32))), (_append, "V", dict(v=torch.zeros(2, 3, 4, 64))),
    (_append, "V", dict(v=torch.zeros(2, 3, 5, 64).half())), (_append, "K", dict(k=torch.zeros(2, 3, 5, 64).double())), (_append, "K_pages", dict(kp=torch.zeros(7, 2, 16, 64))),
    (_append, "V_pages", dict(vp=torch.zeros(6, 3, 16, 64))), (_append, "V_pages", dict(vp=torch.zeros(7, 3, 16, 64).bfloat16())), (_append, "pages", dict(pages=torch.zeros(2, 4))),
    (_append, "pages", dict(pages=torch.zeros(2, 8, **i32)[:, ::2])), (_append, "lengths", dict(lens=torch.zeros(3, **i32))), (_append, "counts", dict(counts=torch.zeros(3, **i32))),
    (_append, "picks", dict(picks=torch.zeros(2, 4, **i32))), (_append, "picks", dict(picks=torch.zeros(2, 5))), (_append, "picks", dict(picks=torch.zeros(5, 2, **i32).T)),
    (_append, "K", dict(starts=torch.zeros(3, **i32))), (_append, "starts", dict(k=torch.zeros(9, 3, 64), v=torch.zeros(9, 3, 64), starts=torch.zeros(2, **i32))),
    (_append, "starts", dict(k=torch.zeros(9, 3, 64), v=torch.zeros(9, 3, 64), starts=torch.zeros(3, **i32), counts=torch.zeros(2, **i32))),
    (_append, "K", dict(k=torch.zeros(9, 3, 64), v=torch.zeros(9, 3, 64))), (_append, "K_pages", dict(kp=torch.zeros(2, 7, 3, 16, 64))),
    (_fork, "K_pages", dict(kp=torch.zeros(3, 16, 64))), (_fork, "V_pages", dict(vp=torch.zeros(2, 7, 3, 16, 64))), (_fork, "lengths", dict(lens=torch.zeros(3, **i32))),
    (_fork, "users", dict(users=torch.zeros(6, **i32))), (_fork, "source", dict(source=torch.zeros(3))), (_fork, "source", dict(source=torch.zeros(3, 1, **i32))),
    (_fork, "room", dict(room=torch.zeros(2, **i32))), (_fork, "pages", dict(pages=torch.zeros(2, 4, dtype=torch.int64))),
    (_compact, "users", dict(users=torch.zeros(7))), (_compact, "V_pages", dict(vp=torch.zeros(7, 3, 32, 64))), (_compact, "pages", dict(pages=torch.zeros(8, **i32)))])
def test_arguments_that_do_not_fit_are_refused(call, name, wrong):
    with pytest.raises(AssertionError, match="^" + name + ":"):
        call(**wrong)


@pytest.mark.parametrize("call,name,wrong", [(_append, "K", dict(k=None)), (_append, "starts", dict(starts=[0, 1, 2])), (_append, "picks", dict(picks=3)), (_fork, "users", dict(users=None)),
                                             (_compact, "V_pages", dict(vp=[]))])
def test_what_is_no_tensor_is_refused(call, name, wrong):
    with pytest.raises(TypeError, match="^" + name + ":"):
        call(**wrong)
    with pytest.raises(TypeError):
        _fork(room="much")


def test_host_tensors_are_refused():
    for call in (_append, _fork, _compact):
        with pytest.raises(AssertionError, match="CUDA"):
            call()


class View(C.Structure):
    _fields_ = [("ptr", C.c_void_p), ("sB", C.c_int64), ("sM", C.c_int64), ("sH", C.c_int64)]


class Pool(C.Structure):
    _fields_ = [("K", View), ("V", View), ("pages", C.c_void_p), ("stride", C.c_int64), ("width", C.c_int), ("n_pages", C.c_int), ("page", C.c_int)]


class Append(C.Structure):
    _fields_ = [("K", View), ("V", View), ("pool", Pool), ("lengths", C.c_void_p), ("starts", C.c_void_p), ("picks", C.c_void_p), ("counts", C.c_void_p), ("B", C.c_int), ("nh_kv", C.c_int),
                ("dtype", C.c_int), ("T", C.c_int64)]


class Fork(C.Structure):
    _fields_ = [("pool", Pool), ("k_sL", C.c_int64), ("v_sL", C.c_int64), ("lengths", C.c_void_p), ("users", C.c_void_p), ("source", C.c_void_p), ("room", C.c_void_p), ("pages_out", C.c_void_p),
                ("lengths_out", C.c_void_p), ("users_out", C.c_void_p), ("missing", C.c_void_p), ("B", C.c_int), ("B_out", C.c_int), ("layers", C.c_int), ("nh_kv", C.c_int), ("dtype", C.c_int),
                ("room_all", C.c_int64), ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t)]


class Compact(C.Structure):
    _fields_ = [("pool", Pool), ("k_sL", C.c_int64), ("v_sL", C.c_int64), ("users", C.c_void_p), ("pages_out", C.c_void_p), ("users_out", C.c_void_p), ("where", C.c_void_p), ("B", C.c_int),
                ("layers", C.c_int), ("nh_kv", C.c_int), ("dtype", C.c_int), ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t)]


def block(kind):
    """Blocks of a call that fits, on addresses that nothing reads: every check is in front of the first launch"""
    b = kind()
    b.pool.K = b.pool.V = View(0x1000, 3 * 16 * 64, 64, 16 * 64)
    b.pool.pages, b.pool.stride, b.pool.width, b.pool.n_pages, b.pool.page = 0x1000, 4, 4, 7, 16
    b.B, b.nh_kv, b.dtype = 2, 3, 0
    for name, _ in kind._fields_:
        if name in ("lengths", "users", "source", "pages_out", "lengths_out", "users_out", "missing", "where"):
            setattr(b, name, 0x1000)
    if kind is Append:
        b.K = b.V = View(0x1000, 3 * 5 * 64, 64, 5 * 64)
        b.T = 5
    else:
        b.layers, b.k_sL, b.v_sL = 2, 7 * 3 * 16 * 64, 7 * 3 * 16 * 64
        if kind is Fork:
            b.B_out = 3
    return b


CALLS = {Append: "hk_cache_append", Fork: "hk_cache_fork", Compact: "hk_cache_compact"}


def answer(b):
    f = getattr(hk.lib(), CALLS[type(b)])
    f.argtypes = [C.c_void_p, C.c_void_p]
    return f(C.byref(b), None)


@pytest.mark.parametrize("kind,path,value,status", [
    (Append, "pool.K.ptr", None, -1), (Append, "pool.pages", None, -1), (Append, "lengths", None, -1), (Append, "V.ptr", None, -1), (Append, "K.ptr", 0x1008, -3), (Append, "K.sM", 66, -3),
    (Append, "pool.V.sB", 3 * 16 * 64 + 2, -3), (Append, "pool.K.sM", 0, -6), (Append, "pool.K.sB", 64, -6), (Append, "pool.page", 8, -6), (Append, "pool.page", 24, -6), (Append, "pool.page", 0, -2),
    (Append, "pool.n_pages", 0, -2), (Append, "pool.width", 0, -2), (Append, "B", 0, -2), (Append, "T", 0, -2), (Append, "nh_kv", 0, -2), (Append, "dtype", 3, -6), (Append, "counts", 0x1001, -3),
    (Append, "pool.width", 1 << 28, -2), (Append, "pool.stride", -1, -2), (Append, "T", 1 << 31, -2),
    (Fork, "users", None, -1), (Fork, "missing", None, -1), (Fork, "source", None, -1), (Fork, "layers", 0, -2), (Fork, "B_out", 0, -2), (Fork, "room_all", -1, -2), (Fork, "k_sL", 64, -6),
    (Fork, "v_sL", 7 * 3 * 16 * 64 + 2, -3), (Fork, "pool.page", 20, -6), (Fork, "room", 0x1002, -3), (Fork, "workspace", None, -5), (Fork, "dtype", -1, -6),
    (Compact, "where", None, -1), (Compact, "users", 0x1001, -3), (Compact, "layers", -1, -2), (Compact, "workspace", None, -5), (Compact, "v_sL", 0, -6), (Compact, "pool.n_pages", -1, -2)])
def test_blocks_that_are_refused(kind, path, value, status):
    b = block(kind)
    if kind is not Append:  # a workspace that is too small, for those that get past all else
        b.workspace, b.workspace_bytes = 0x1000, 16
        assert answer(b) == -5
    at, (*way, last) = b, path.split(".")
    for name in way:
        at = getattr(at, name)
    setattr(at, last, value)
    assert answer(b) == status
    assert answer_of_nothing(kind) == -1


def answer_of_nothing(kind):
    f = getattr(hk.lib(), CALLS[kind])
    f.argtypes = [C.c_void_p, C.c_void_p]
    return f(None, None)


def test_starts_beside_picks_are_refused():
    b = block(Append)
    b.starts, b.picks = 0x1000, 0x1000
    b.K = b.V = View(0x1000, 0, 64, 5 * 64)
    assert answer(b) == -6


def test_workspaces():
    for kind in (Fork, Compact):
        f = getattr(hk.lib(), CALLS[kind] + "_workspace_bytes")
        f.restype, f.argtypes = C.c_size_t, [C.c_void_p]
        b = block(kind)
        need = f(C.byref(b))
        assert need > 0 and need % 256 == 0
        b.workspace, b.workspace_bytes = 0x1000, need - 1
        assert answer(b) == -5
        b.workspace, b.workspace_bytes = 0x1010, need
        assert answer(b) == -5
        b.pool.page = 17
        assert f(C.byref(b)) == 0 and f(None) == 0
