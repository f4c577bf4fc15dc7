"""The operators of serving from a cache of pages, at the sizes their users have: prompts of different lengths behind each other,
drafted tokens (or single ones) against the pages, and what happens to the pages in between.

A case is a dict of plain values; ``op`` picks the entry point.

* ``prompt``   ``prompt_attention``: ``B`` whole prompts, ``N`` tokens in all, packed without gaps.
* ``tree``     ``tree_attention``: ``T`` new tokens of each of ``B`` requests, a tree of drafts (1: plain decoding), against up to
  ``keys`` keys of each in pages of ``page`` tokens.
* ``append``   ``cache_append``: keys and values of new tokens into the pages: of packed prompts, or of those of ``T`` drafts
  that were accepted.
* ``fork``     ``cache_fork``: one step of a batch: requests go on, end, are continued several times (``beams``) or start, with pages for
  the tokens to come (``room``, or a prompt), in the pools of ``L`` layers.
* ``compact``  ``cache_compact``: the pages in use to the front of the pools.

``layout`` is how a page lies in memory: head by head ("hpd") or token by token ("phd").  ``lens`` says how the requests' lengths
spread: "ramp" from (nearly) nothing to the most there is, "halves" each half of the one before, "equal".
"""
import math

import torch

own = False

SCALE = 0.125  # 1 / sqrt(64)
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}


def _named(name, c):
    return dict(c, name=name) if name else c


def _prompt(name, B, N, H, Hk, dtype, lens, causal=True, layout="packed"):
    return _named(name, dict(op="prompt", B=B, N=N, H=H, Hk=Hk, dtype=dtype, lens=lens, causal=causal, layout=layout))


def _tree(name, B, T, H, Hk, keys, page, dtype, lens, layout="hpd"):
    return _named(name, dict(op="tree", B=B, T=T, H=H, Hk=Hk, keys=keys, page=page, dtype=dtype, lens=lens, layout=layout))


def _append(name, B, N, T, Hk, keys, page, dtype, lens, layout="hpd"):
    """T = 0: N tokens of packed prompts; otherwise those of T drafts that were accepted."""
    return _named(name, dict(op="append", B=B, N=N, T=T, Hk=Hk, keys=keys, page=page, dtype=dtype, lens=lens, layout=layout))


def _fork(name, B, beams, L, Hk, keys, page, room, dtype, layout="hpd"):
    return _named(name, dict(op="fork", B=B, beams=beams, L=L, Hk=Hk, keys=keys, page=page, room=room, dtype=dtype, lens="ramp", layout=layout))


def _compact(name, B, L, pool, Hk, page, used, dtype, layout="hpd"):
    return _named(name, dict(op="compact", B=B, L=L, pool=pool, Hk=Hk, page=page, used=used, dtype=dtype, layout=layout))


def listed():
    return [
        # a handful of short questions in one call, fp32, the longest not quite 100 tokens: latency
        _prompt("prompt_b6_n333", 6, 333, 12, 12, "f32", "ramp"),
        # an ordinary batch of prompts, shared key heads, half precision, views of a fused projection
        _prompt("prompt_b16_n8192_bf16", 16, 8192, 32, 8, "bf16", "ramp"),
        # long documents of very different lengths, the largest work
        _prompt("prompt_b4_n16384_bf16", 4, 16384, 32, 8, "bf16", "halves"),
        # one token each for sixteen requests, fp32, small pages
        _tree("tree_b16_t1", 16, 1, 12, 12, 2047, 16, "f32", "ramp"),
        # a full decoding batch, shared key heads, half precision, pages stored token by token
        _tree("tree_b64_t1_bf16", 64, 1, 32, 8, 8192, 64, "bf16", "ramp", "phd"),
        # sixteen drafted tokens of each request are verified at once
        _tree("tree_b16_t16_bf16", 16, 16, 32, 8, 4096, 64, "bf16", "ramp"),
        # the drafts that were accepted go into the cache: a few rows of each request
        _append("append_b16_t16_bf16", 16, 0, 16, 8, 4096, 64, "bf16", "ramp"),
        # the keys and values of packed prompts go into new pages
        _append("append_b16_n8192", 16, 8192, 0, 12, 0, 16, "f32", "ramp"),
        # between two decoding steps: some requests end, all get room for the next token
        _fork("fork_b64_step_bf16", 64, 1, 12, 8, 1000, 16, 1, "bf16"),
        # a step of a beam search, four beams of sixteen requests: full pages are shared, begun ones copied
        _fork("fork_b64_beams4", 64, 4, 12, 12, 512, 64, 1, "f32"),
        # a small pool, one layer
        _compact("compact_p96", 8, 1, 96, 12, 16, 0.5, "f32"),
        # a large one, half of it in use
        _compact("compact_p2048_bf16", 64, 4, 2048, 8, 64, 0.5, "bf16", "phd"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["prompt", "prompt", "tree", "tree", "append", "fork", "compact"])
    dtype, layout, page = rng.choice(["f32", "bf16", "f16"]), rng.choice(["hpd", "phd"]), rng.choice([16, 16, 32, 48, 64, 80, 128, 256])
    Hk, group = rng.choice([1, 2, 3, 4, 8, 12]), rng.choice([1, 1, 2, 3, 4, 7, 8])
    lens = rng.choice(["ramp", "halves", "equal"])
    while True:
        if op == "prompt":
            c = _prompt(None, _log(rng, 1, 64), _log(rng, 1, 16384), Hk * group, Hk, dtype, lens, rng.choice([True, True, False]),
                        rng.choice(["packed", "own"]))
            if work(c)["flops"] <= (3e11 if dtype != "f32" else 5e10):
                return c
        elif op == "tree":
            c = _tree(None, _log(rng, 1, 64), rng.choice([1, 1, _log(rng, 2, 64)]), Hk * group, Hk, _log(rng, 1, 16384), page, dtype, lens, layout)
            if work(c)["bytes"] <= 5e8 and work(c)["flops"] <= (1e11 if dtype != "f32" else 2e10) and c["B"] * c["H"] * c["T"] * c["keys"] <= 4e8:
                return c
        elif op == "append":
            T = rng.choice([0, 1, _log(rng, 2, 64)])
            c = _append(None, _log(rng, 1, 64), 0 if T else _log(rng, 1, 16384), T, Hk, _log(rng, 1, 4096), page, dtype, lens, layout)
            if work(c)["bytes"] <= 1e9:
                return c
        elif op == "fork":
            beams = rng.choice([1, 2, 4, 5])
            c = _fork(None, beams * _log(rng, 1, 32), beams, rng.choice([1, 2, 12]), Hk, _log(rng, 1, 2048), page, rng.choice([1, 1, _log(rng, 1, 100)]), dtype, layout)
            if c["B"] * c["L"] * Hk * (1.1 * c["keys"] + 2 * page + c["room"]) * 256 * BYTES[dtype] <= 6e9:
                return c
        else:
            c = _compact(None, _log(rng, 1, 64), rng.choice([1, 2, 4]), _log(rng, 8, 4000), Hk, page, rng.uniform(0.05, 0.95), dtype, layout)
            if c["L"] * c["pool"] * Hk * page * 128 * BYTES[dtype] <= 2e9:
                return c


def _spread(how, n, total, most):
    """Lengths of n requests: that sum up to `total`, or (None) with `most` as the largest."""
    w = [1.0 if how == "equal" else 0.5 ** i if how == "halves" else i + 0.25 for i in range(n)]
    if total is None:
        return [round(most * x / max(w)) for x in w]
    ends, s = [0], 0.0
    for x in w:
        s += x
        ends.append(round(total * s / sum(w)))
    return [b - a for a, b in zip(ends, ends[1:])]


def _lengths(c):
    if c["op"] == "prompt":
        return _spread(c["lens"], c["B"], c["N"], None)
    if c["op"] == "fork":  # the beams of a request are of one length
        return [n for n in _spread(c["lens"], c["B"] // c["beams"], None, c["keys"]) for _ in range(c["beams"])]
    return _spread(c["lens"], c["B"], None, c["keys"])


def _news(c):
    """New tokens of each request that an append brings into the pages."""
    if c["T"] == 0:
        return _spread(c["lens"], c["B"], c["N"], None)
    return [(5 * b + c["T"] // 2 + 1) % (c["T"] + 1) for b in range(c["B"])]


def _cdiv(a, b):
    return -(-a // b)


def _sources(c):
    """Which request of the old batch each of the new one goes on with (-1: none): without beams one in nine has ended; of a
    group of beams some are continued more than once, others not at all."""
    B, W = c["B"], c["beams"]
    if W == 1:
        return [-1 if b % 9 == 4 else b for b in range(B)]
    return [b - b % W + (b * b // W + b % W * (b // W % 2)) % W for b in range(B)]


def _rooms(c):
    """Tokens that each request of the new batch needs pages for: those that go on some, of the places of those that have ended
    every other one is a new prompt's."""
    return [c["room"] if s >= 0 else c["keys"] // 2 * (b % 2) for b, s in enumerate(_sources(c))]


def work(c):
    e = 64 * BYTES[c["dtype"]]  # bytes of a row
    if c["op"] == "prompt":
        lens = _lengths(c)
        seen = sum(n * (n + 1) // 2 if c["causal"] else n * n for n in lens)
        return {"bytes": 2 * c["N"] * (c["H"] + c["Hk"]) * e + 4 * c["N"] * c["H"] + 4 * (c["B"] + 1), "flops": 256 * c["H"] * seen}
    if c["op"] == "tree":
        lens, T = _lengths(c), c["T"]
        seen = sum(lens) * T + c["B"] * sum(_depth(i) + 1 for i in range(T))
        held = sum(lens) + c["B"] * T
        table = 4 * sum(_cdiv(n, c["page"]) for n in lens) + 4 * c["B"] + 8 * c["B"] * T
        return {"bytes": 2 * held * c["Hk"] * e + c["B"] * c["H"] * T * (2 * e + 4) + table, "flops": 256 * c["H"] * seen}
    if c["op"] == "append":
        return {"bytes": 4 * sum(_news(c)) * c["Hk"] * e + 4 * sum(_cdiv(n, c["page"]) + 2 for n in _news(c)), "flops": 0}
    if c["op"] == "fork":
        lens, seen, rows = _lengths(c), set(), 0
        for s in _sources(c):
            if s >= 0:
                rows += lens[s] % c["page"] if s in seen else 0
                seen.add(s)
        return {"bytes": 4 * rows * c["L"] * c["Hk"] * e + 8 * c["B"] * (_width(c) + 2) + 8 * _pool(c), "flops": 0}
    P, used = c["pool"], max(1, round(c["used"] * c["pool"]))
    moved = used * (P - used) // P  # of pages in use that lie anywhere
    return {"bytes": 4 * moved * c["L"] * c["Hk"] * c["page"] * e + 12 * P + 8 * used, "flops": 0}


def _depth(i):
    """The tree of drafts that the cases have: the first two in a row, then branches of two."""
    d = 0
    while i > 0:
        i = 0 if i < 2 else (i - 1) // 2
        d += 1
    return d


def _width(c):
    """Pages that a row of the table has room for."""
    if c["op"] == "append":
        return max(_cdiv(n + m + c["T"], c["page"]) for n, m in zip(_olds(c), _news(c))) + 1
    return _cdiv(c["keys"] + (c["room"] if c["op"] == "fork" else 0), c["page"]) + 1


def _olds(c):
    return [0] * c["B"] if c["T"] == 0 else _lengths(c)


def _pool(c):
    """Pages of a pool: what the requests need and some that are free."""
    if c["op"] == "append":
        need = sum(_cdiv(n + max(m, c["T"]), c["page"]) for n, m in zip(_olds(c), _news(c)))
    else:
        need = sum(_cdiv(n, c["page"]) for n in _lengths(c))
    if c["op"] == "fork":
        need += sum(_cdiv(r, c["page"]) + 2 for r in _rooms(c))
    return need + need // 8 + 3


def _tensor(g, shape, dtype, sigma=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * sigma).to(TYPES[dtype])


def _pages(c, g, P, L=None):
    """A pool and one page more behind it, which the plain forms write to in place of nowhere: [(L,) P + 1, Hk, page, 64]."""
    lead = () if L is None else (L,)
    if c["layout"] == "phd":
        return _tensor(g, (*lead, P + 1, c["page"], c["Hk"], 64), c["dtype"]).transpose(-3, -2)
    return _tensor(g, (*lead, P + 1, c["Hk"], c["page"], 64), c["dtype"])


def _table(c, g, counts, P, width):
    """Pages of each request, anywhere in the pool, -1 behind them."""
    order = torch.randperm(P, generator=g, device="cuda").to(torch.int32)
    have = torch.tensor(counts, device="cuda")
    j = torch.arange(width, device="cuda")
    at = (have.cumsum(0) - have)[:, None] + j
    return torch.where(j < have[:, None], order[at.clamp(max=P - 1)], -1).contiguous()


def _shuffled(g, values):
    return [values[i] for i in torch.randperm(len(values), generator=g, device="cuda").tolist()]


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(c)
    if c["op"] == "prompt":
        N, H, Hk = c["N"], c["H"], c["Hk"]
        lens = _shuffled(g, _lengths(c))
        starts = torch.zeros(c["B"] + 1, device="cuda", dtype=torch.int32)
        starts[1:] = torch.tensor(lens, device="cuda").cumsum(0)
        if c["layout"] == "packed":
            x = _tensor(g, (N, H + 2 * Hk, 64), c["dtype"])
            q, k, v = x[:, :H], x[:, H:H + Hk], x[:, H + Hk:]
            q.mul_(1.5)
        else:
            q, k, v = _tensor(g, (N, H, 64), c["dtype"], 1.5), _tensor(g, (N, Hk, 64), c["dtype"]), _tensor(g, (N, Hk, 64), c["dtype"])
        return dict(s, q=q, k=k, v=v, starts=starts, host_lens=lens)
    if c["op"] == "compact":
        P = c["pool"]
        used = max(1, round(c["used"] * P))
        # a random half is in use, some of it by two requests
        order = torch.randperm(P, generator=g, device="cuda")
        shared = used // 4
        users = torch.zeros(P, device="cuda", dtype=torch.int32)
        users[order[:used]] = 1
        users[order[:shared]] += 1
        entries = torch.cat([order[:used], order[:shared]]).to(torch.int32)
        width = _cdiv(len(entries), c["B"])
        pages = torch.full((c["B"] * width,), -1, device="cuda", dtype=torch.int32)
        pages[:len(entries)] = entries
        k, v = _pages(c, g, P, c["L"]), _pages(c, g, P, c["L"])
        return dict(s, P=P, k_all=k, v_all=v, users=users, pages=pages.view(c["B"], width))
    P, width = _pool(c), _width(c)
    if c["op"] == "append":
        pairs = _shuffled(g, list(zip(_olds(c), _news(c))))
        lens = torch.tensor([n for n, _ in pairs], device="cuda", dtype=torch.int32)
        news = torch.tensor([m for _, m in pairs], device="cuda", dtype=torch.int32)
        pages = _table(c, g, [_cdiv(n + max(m, c["T"]), c["page"]) for n, m in pairs], P, width)
        s.update(P=P, lens=lens, pages=pages, k_all=_pages(c, g, P), v_all=_pages(c, g, P))
        if c["T"] == 0:
            starts = torch.zeros(c["B"] + 1, device="cuda", dtype=torch.int32)
            starts[1:] = news.cumsum(0)
            x = _tensor(g, (c["N"], 2 * c["Hk"], 64), c["dtype"])
            return dict(s, starts=starts, k=x[:, :c["Hk"]], v=x[:, c["Hk"]:])
        # the accepted drafts come in their order, but not all of them
        picks = torch.rand((c["B"], c["T"]), generator=g, device="cuda").argsort(1)
        j = torch.arange(c["T"], device="cuda")
        picks = torch.where(j < news[:, None], picks, c["T"]).sort(1).values.clamp(max=c["T"] - 1).to(torch.int32)
        k, v = (_tensor(g, (c["B"], c["T"], c["Hk"], 64), c["dtype"]).transpose(1, 2) for _ in range(2))
        return dict(s, picks=picks, counts=news, k=k, v=v)
    lens = _lengths(c)
    if c["op"] == "tree":
        lens = _shuffled(g, lens)
    on_device = torch.tensor(lens, device="cuda", dtype=torch.int32)
    pages = _table(c, g, [_cdiv(n, c["page"]) for n in lens], P, width)
    if c["op"] == "tree":
        B, T, H, Hk = c["B"], c["T"], c["H"], c["Hk"]
        q = _tensor(g, (B, T, H, 64), c["dtype"], 1.5).transpose(1, 2)
        k, v = (_tensor(g, (B, T, Hk, 64), c["dtype"]).transpose(1, 2) for _ in range(2))
        rows = []
        for i in range(T):
            rows.append((rows[0 if i < 2 else (i - 1) // 2] if i else 0) | 1 << i)
        tree = torch.tensor([r - (1 << 64) if r >> 63 else r for r in rows], device="cuda").expand(B, T).contiguous()
        return dict(s, P=P, q=q, k=k, v=v, k_all=_pages(c, g, P), v_all=_pages(c, g, P), pages=pages, lens=on_device, tree=tree)
    users = torch.zeros(P + 1, device="cuda", dtype=torch.int32)
    users.scatter_add_(0, torch.where(pages >= 0, pages, P).flatten().long(), torch.ones(pages.numel(), device="cuda", dtype=torch.int32))
    group = torch.arange(c["B"], device="cuda") // c["beams"]
    shift = torch.randint(0, c["beams"], (c["B"] // c["beams"],), generator=g, device="cuda")[group]
    source = torch.tensor(_sources(c), device="cuda")
    if c["beams"] > 1:
        source = group * c["beams"] + (source + shift) % c["beams"]
    return dict(s, P=P, k_all=_pages(c, g, P, c["L"]), v_all=_pages(c, g, P, c["L"]), pages=pages, lens=on_device, users=users[:P].clone(),
                source=source.to(torch.int32), rooms=torch.tensor(_rooms(c), device="cuda", dtype=torch.int32))


# ---- the operators' plain forms ------------------------------------------------------------------------------------------
def _plain_prompt(s):
    H, Hk, N = s["H"], s["Hk"], s["N"]
    G = H // Hk
    o = torch.empty((N, H, 64), device="cuda", dtype=TYPES[s["dtype"]])
    lse = torch.empty((H, N), device="cuda")
    at = 0
    for n in s["host_lens"]:
        r, at = slice(at, at + n), at + n
        if n == 0:
            continue
        i = torch.arange(n, device="cuda")
        for h in range(Hk):
            heads = slice(h * G, h * G + G)
            x = (s["q"][r, heads].float().transpose(0, 1) * SCALE) @ s["k"][r, h].float().T  # [G, n, n]
            if s["causal"]:
                x = x.masked_fill(i > i[:, None], -math.inf)
            m = x.amax(-1, keepdim=True)
            x = (x - m).exp()
            total = x.sum(-1, keepdim=True)
            o[r, heads] = (x @ s["v"][r, h].float() / total).transpose(0, 1).to(o.dtype)
            lse[heads, r] = (m + total.log())[..., 0]
    return {"o": o, "lse": lse}


def _plain_tree(s):
    B, T, H, Hk, page = s["B"], s["T"], s["H"], s["Hk"], s["page"]
    G, M = H // Hk, s["pages"].shape[1]
    at = s["pages"].clamp(min=0).long()
    k, v = (x[at].transpose(1, 2).reshape(B, Hk, M * page, 64).float() for x in (s["k_all"], s["v_all"]))
    q = s["q"].float().reshape(B, Hk, G * T, 64) * SCALE
    old = q @ k.transpose(2, 3)
    old = old.masked_fill(torch.arange(M * page, device="cuda") >= s["lens"][:, None, None, None], -math.inf)
    new = (q @ s["k"].float().transpose(2, 3)).view(B, Hk, G, T, T)
    sees = (s["tree"][:, :, None] >> torch.arange(T, device="cuda") & 1).bool()
    new = new.masked_fill(~sees[:, None, None], -math.inf).view(B, Hk, G * T, T)
    m = torch.maximum(old.amax(-1, keepdim=True), new.amax(-1, keepdim=True))
    old, new = (old - m).exp(), (new - m).exp()
    total = old.sum(-1, keepdim=True) + new.sum(-1, keepdim=True)
    o = (old @ v + new @ s["v"].float()) / total
    return {"o": o.reshape(B, H, T, 64).to(TYPES[s["dtype"]]), "lse": (m + total.log()).reshape(B, H, T)}


def _plain_append(s):
    page = s["page"]
    if s["T"] == 0:
        n = torch.arange(s["N"], device="cuda", dtype=torch.int32)
        b = torch.bucketize(n, s["starts"][1:], right=True)
        pos = s["lens"][b] + n - s["starts"][b]
        to = s["pages"][b, pos // page].long()
        s["k_all"][to, :, pos % page] = s["k"]
        s["v_all"][to, :, pos % page] = s["v"]
    else:
        j = torch.arange(s["T"], device="cuda")
        pos = s["lens"][:, None] + j
        to = torch.where(j < s["counts"][:, None], s["pages"].gather(1, (pos // page).long()), s["P"]).long()
        b = torch.arange(s["B"], device="cuda")[:, None]
        s["k_all"][to, :, pos % page] = s["k"][b, :, s["picks"].long()]
        s["v_all"][to, :, pos % page] = s["v"][b, :, s["picks"].long()]
    return {"k": s["k_all"][:s["P"]], "v": s["v_all"][:s["P"]]}


def _count(pages, P, sign, into):
    """Adds `sign` for every entry of a table to its page."""
    into = torch.cat([into, into.new_zeros(1)])
    into.scatter_add_(0, torch.where(pages >= 0, pages, P).flatten().long(), torch.full((pages.numel(),), sign, device="cuda", dtype=torch.int32))
    return into[:P]


def _plain_fork(s):
    B, P, page, M = s["B"], s["P"], s["page"], s["pages"].shape[1]
    src, live = s["source"].clamp(min=0).long(), s["source"] >= 0
    lens = torch.where(live, s["lens"][src], 0)
    i, j = torch.arange(B, device="cuda", dtype=torch.int32), torch.arange(M, device="cuda")
    first = torch.full((B,), B, device="cuda", dtype=torch.int32).scatter_reduce_(0, src, torch.where(live, i, B), "amin")
    full, begun = lens // page, lens % page
    shared = (j < full[:, None]) | ((j == full[:, None]) & (begun > 0)[:, None] & (first[src] == i)[:, None])
    needed = j < ((lens + s["rooms"] + page - 1) // page)[:, None]
    kept = torch.where(shared, s["pages"][src], -1)
    users = _count(kept, P, 1, _count(s["pages"], P, -1, s["users"]))
    order = (users != 0).to(torch.int8).argsort(stable=True)
    free = (users == 0).sum()
    fresh = needed & ~shared
    rank = fresh.flatten().cumsum(0).view(B, M) - 1
    given = torch.where(fresh & (rank < free), order[rank.clamp(0, P - 1)].to(torch.int32), -1)
    pages = torch.where(shared, kept, given)
    users = _count(given, P, 1, users)
    at = full.clamp(max=M - 1).long()[:, None]
    copied = ((begun > 0) & (first[src] != i))[:, None] & (given.gather(1, at) >= 0)
    frm = torch.where(copied, s["pages"][src].gather(1, at), P)[:, 0].long()
    to = torch.where(copied, given.gather(1, at), P)[:, 0].long()
    rows = (torch.arange(page, device="cuda") < begun[:, None])[:, None, :, None]
    for x in (s["k_all"], s["v_all"]):
        for layer in x:
            layer[to] = torch.where(rows, layer[frm], layer[to])
    return {"pages": pages, "lens": lens, "users": users, "missing": (fresh.sum() - free).clamp(min=0).to(torch.int32).view(1),
            "k": s["k_all"][:, :P], "v": s["v_all"][:, :P]}


def _plain_compact(s):
    P = s["P"]
    p = torch.arange(P, device="cuda", dtype=torch.int32)
    used = s["users"] > 0
    n = used.sum()
    hole, moves = ~used & (p < n), used & (p >= n)
    few = max(1, P // 2)  # more cannot move
    k = torch.arange(few, device="cuda") < moves.sum()
    frm = torch.where(k, (~moves).to(torch.int8).argsort(stable=True)[:few], P)
    to = torch.where(k, (~hole).to(torch.int8).argsort(stable=True)[:few], P)
    where = torch.cat([torch.where(used, p, -1), p[:1]])
    where[frm] = to.to(torch.int32)
    where = where[:P]
    users = torch.zeros(P + 1, device="cuda", dtype=torch.int32)
    users[torch.where(used, where, P).long()] = s["users"]
    for x in (s["k_all"], s["v_all"]):
        for layer in x:
            layer[to] = layer[frm]
    pages = torch.where(s["pages"] >= 0, where[s["pages"].clamp(min=0).long()], -1)
    return {"pages": pages, "users": users[:P], "where": where, "k": s["k_all"][:, :P], "v": s["v_all"][:, :P]}


def run(s):
    if own:
        import hyperkernels_b200 as hk

        if s["op"] == "prompt":
            o, lse = hk.prompt_attention(s["q"], s["k"], s["v"], s["starts"], SCALE, s["causal"])
            return {"o": o, "lse": lse}
        P = s["P"]
        if s["op"] == "tree":
            o, lse = hk.tree_attention(s["q"], s["k"], s["v"], s["k_all"][:P], s["v_all"][:P], s["pages"], s["lens"], SCALE, s["tree"])
            return {"o": o, "lse": lse}
        if s["op"] == "append":
            k_pages, v_pages = s["k_all"][:P], s["v_all"][:P]
            if s["T"] == 0:
                hk.cache_append(s["k"], s["v"], k_pages, v_pages, s["pages"], s["lens"], starts=s["starts"])
            else:
                hk.cache_append(s["k"], s["v"], k_pages, v_pages, s["pages"], s["lens"], picks=s["picks"], counts=s["counts"])
            return {"k": k_pages, "v": v_pages}
        k_pages, v_pages = s["k_all"][:, :P], s["v_all"][:, :P]
        if s["op"] == "fork":
            pages, lens, users, missing = hk.cache_fork(k_pages, v_pages, s["pages"], s["lens"], s["users"], s["source"], s["rooms"])
            return {"pages": pages, "lens": lens, "users": users, "missing": missing, "k": k_pages, "v": v_pages}
        pages, users, where = hk.cache_compact(k_pages, v_pages, s["pages"], s["users"])
        return {"pages": pages, "users": users, "where": where, "k": k_pages, "v": v_pages}
    return {"prompt": _plain_prompt, "tree": _plain_tree, "append": _plain_append, "fork": _plain_fork, "compact": _plain_compact}[s["op"]](s)


# ---- the definitions in 64 bits: request by request and head by head, pages one at a time ----------------------------------
def _exact_rows(q, k, v, hidden):
    x = q.double() @ k.double().T * SCALE
    x[hidden] = -math.inf
    return torch.softmax(x, -1) @ v.double(), torch.logsumexp(x, -1)


def _exact_prompt(s):
    G, N = s["H"] // s["Hk"], s["N"]
    o = torch.zeros((N, s["H"], 64), device="cuda", dtype=torch.float64)
    lse = torch.zeros((s["H"], N), device="cuda", dtype=torch.float64)
    edges = s["starts"].tolist()
    for a, b in zip(edges, edges[1:]):
        for t in range(a, b, 2048):  # rows of queries
            e = min(b, t + 2048)
            last = e if s["causal"] else b
            hidden = (torch.arange(a, last, device="cuda") > torch.arange(t, e, device="cuda")[:, None]) & s["causal"]
            for h in range(s["H"]):
                o[t:e, h], lse[h, t:e] = _exact_rows(s["q"][t:e, h], s["k"][a:last, h // G], s["v"][a:last, h // G], hidden)
    return {"o": o, "lse": lse}


def _exact_tree(s):
    B, H, T, G = s["B"], s["H"], s["T"], s["H"] // s["Hk"]
    o = torch.zeros((B, H, T, 64), device="cuda", dtype=torch.float64)
    lse = torch.zeros((B, H, T), device="cuda", dtype=torch.float64)
    lens, table, tree = s["lens"].tolist(), s["pages"].tolist(), s["tree"].tolist()
    for b in range(B):
        ids = torch.tensor(table[b][:_cdiv(lens[b], s["page"])], device="cuda", dtype=torch.long)
        old_k, old_v = s["k_all"][ids], s["v_all"][ids]  # [pages, Hk, page, 64]
        hidden = torch.tensor([[False] * lens[b] + [tree[b][i] >> j & 1 == 0 for j in range(T)] for i in range(T)], device="cuda")
        for h in range(H):
            k = torch.cat([old_k[:, h // G].flatten(0, 1)[:lens[b]], s["k"][b, h // G]])
            v = torch.cat([old_v[:, h // G].flatten(0, 1)[:lens[b]], s["v"][b, h // G]])
            o[b, h], lse[b, h] = _exact_rows(s["q"][b, h], k, v, hidden)
    return {"o": o, "lse": lse}


def _exact_append(s):
    lens, table, page = s["lens"].tolist(), s["pages"].tolist(), s["page"]
    for b in range(s["B"]):
        if s["T"] == 0:
            a, e = s["starts"][b:b + 2].tolist()
            k, v = s["k"][a:e].transpose(0, 1), s["v"][a:e].transpose(0, 1)  # [Hk, tokens, 64]
        else:
            rows = s["picks"][b, :int(s["counts"][b])].long()
            k, v = s["k"][b][:, rows], s["v"][b][:, rows]
        i = 0
        while i < k.shape[1]:
            at, off = divmod(lens[b] + i, page)
            m = min(page - off, k.shape[1] - i)
            s["k_all"][table[b][at], :, off:off + m] = k[:, i:i + m]
            s["v_all"][table[b][at], :, off:off + m] = v[:, i:i + m]
            i += m
    return {"k": s["k_all"][:s["P"]], "v": s["v_all"][:s["P"]]}


def _exact_fork(s):
    P, page, width = s["P"], s["page"], s["pages"].shape[1]
    users, old, lens = s["users"].tolist(), s["pages"].tolist(), s["lens"].tolist()
    for row in old:
        for p in row:
            if p >= 0:
                users[p] -= 1
    new, new_lens, missing, begun_by, copies = [], [], 0, {}, []
    for i, b in enumerate(s["source"].tolist()):
        n = lens[b] if b >= 0 else 0
        row = old[b][:_cdiv(n, page)] if b >= 0 else []
        if n % page:
            if b in begun_by:
                copies.append((i, n // page, row[-1], n % page))
                row = row[:-1]
            else:
                begun_by[b] = i
        for p in row:
            users[p] += 1
        new.append(row)
        new_lens.append(n)
    free = [p for p in range(P) if users[p] == 0]
    for i, room in enumerate(s["rooms"].tolist()):
        while len(new[i]) < _cdiv(new_lens[i] + room, page):
            p = free.pop(0) if free else -1
            missing += p < 0
            if p >= 0:
                users[p] += 1
            new[i].append(p)
        new[i] += [-1] * (width - len(new[i]))
    for i, at, frm, rows in copies:
        for x in (s["k_all"], s["v_all"]):
            if new[i][at] >= 0:
                x[:, new[i][at], :, :rows] = x[:, frm, :, :rows]
    ints = dict(device="cuda", dtype=torch.int32)
    return {"pages": torch.tensor(new, **ints), "lens": torch.tensor(new_lens, **ints), "users": torch.tensor(users, **ints),
            "missing": torch.tensor([missing], **ints), "k": s["k_all"][:, :P], "v": s["v_all"][:, :P]}


def _exact_compact(s):
    P, users = s["P"], s["users"].tolist()
    n = sum(u > 0 for u in users)
    where, counts, holes = [-1] * P, [0] * P, [p for p in range(n) if users[p] == 0]
    for p in range(P):
        if users[p] > 0:
            where[p] = p if p < n else holes.pop(0)
            counts[where[p]] = users[p]
            if where[p] != p:
                for x in (s["k_all"], s["v_all"]):
                    x[:, where[p]] = x[:, p]
    pages = [[where[p] if p >= 0 else -1 for p in row] for row in s["pages"].tolist()]
    ints = dict(device="cuda", dtype=torch.int32)
    return {"pages": torch.tensor(pages, **ints), "users": torch.tensor(counts, **ints), "where": torch.tensor(where, **ints),
            "k": s["k_all"][:, :P], "v": s["v_all"][:, :P]}


def exact(case, seed):
    s = prepare(case, seed)
    return {"prompt": _exact_prompt, "tree": _exact_tree, "append": _exact_append, "fork": _exact_fork, "compact": _exact_compact}[s["op"]](s)
