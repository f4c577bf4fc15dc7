"""The operators round the attention calls, at the sizes their users have: rotary positions with several axes, norms of
queries and keys with the rotation in the same pass, and the attention of a batch that shares a prefix.

A case is a dict of plain values; ``op`` picks the entry point, ``back`` its backward pass.

* ``rotary``  ``rotary_forward`` / ``rotary_backward``: queries and keys as a fused QKV projection leaves them ([B, T, heads,
  64], or head by head with ``layout`` "bhtd"), tokens of text and of images with a position on every axis.
* ``norm``    ``qk_norm_rotary_forward`` / ``qk_norm_rotary_backward``: the same behind an RMS norm of each head's row.
* ``prefix``  ``shared_prefix_attention``: ``T`` new tokens of each of ``B`` requests (1: decoding) against a prompt of
  ``prefix`` keys that all share and up to ``own`` keys of each request, in a cache of ``own`` rows a request.

``dtype`` is the type of what the projection or the cache holds, ``out`` that of what goes on to (forward) or comes back
from (backward) the attention.
"""
import math

import torch

own = False

SCALE = 0.125  # 1 / sqrt(64)
EPS = 1e-6
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}


def _rows(name, op, back, B, H, Hk, T, dtype, out, sections, interleaved=False, layout="packed", far=0):
    c = dict(op=op, back=back, B=B, H=H, Hk=Hk, T=T, dtype=dtype, out=out, sections=sections, interleaved=interleaved,
             layout=layout, far=far)
    return dict(c, name=name) if name else c


def _prefix(name, B, H, Hk, T, prefix, own_keys, dtype, layout="bhtd"):
    c = dict(op="prefix", B=B, H=H, Hk=Hk, T=T, prefix=prefix, own=own_keys, dtype=dtype, layout=layout)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one decoding step of 16 sequences with image tokens behind them: latency is all there is
        _rows("rotary_decode_b16", "rotary", False, 16, 12, 12, 1, "f32", "f32", "8,12,12", far=4000),
        # a batch of text and images on its way into the attention
        _rows("rotary_b8_t1024", "rotary", False, 8, 12, 12, 1024, "f32", "f32", "8,12,12"),
        # the gradients of one long sequence of patches (height, width; neighbours paired), back to half precision, an odd length
        _rows("rotary_back_t32767_bf16", "rotary", True, 1, 32, 8, 32767, "bf16", "f32", "16,16", interleaved=True, far=100000),
        # one decoding step of 64 sequences, shared key heads, half precision throughout
        _rows("norm_decode_b64_bf16", "norm", False, 64, 32, 8, 1, "bf16", "bf16", "32", far=8000),
        # the training batch in fp32, both directions
        _rows("norm_b8_t1024", "norm", False, 8, 12, 12, 1024, "f32", "f32", "32"),
        _rows("norm_back_b8_t1024", "norm", True, 8, 12, 12, 1024, "f32", "f32", "32", layout="bhtd"),
        # one long sequence: half-precision projections, fp32 gradients from the attention, three axes
        _rows("norm_back_t32768_bf16", "norm", True, 1, 32, 32, 32768, "bf16", "f32", "8,12,12"),
        # the smallest serving batch: four requests behind a short prompt
        _prefix("prefix_decode_b4", 4, 12, 12, 1, 333, 64, "f32"),
        # sixteen requests behind a prompt of an odd length, fp32 cache
        _prefix("prefix_decode_b16", 16, 12, 12, 1, 2047, 512, "f32"),
        # a full serving batch, shared key heads, half-precision cache stored token by token
        _prefix("prefix_decode_b64_bf16", 64, 32, 8, 1, 8192, 1000, "bf16", layout="bthd"),
        # chunks of eight requests, fp32
        _prefix("prefix_chunk_b8_t77", 8, 12, 12, 77, 4096, 333, "f32"),
        # prompts' own parts behind a long common part, the largest work
        _prefix("prefix_prefill_b8_t512_bf16", 8, 32, 8, 512, 8192, 1024, "bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["rotary", "norm", "prefix"])
    if op == "prefix":
        while True:
            Hk, group = rng.choice([1, 2, 3, 4, 8, 12, 16]), rng.choice([1, 1, 2, 3, 4, 8])
            T = rng.choice([1, 1, 1, 2, _log(rng, 3, 600)])
            c = _prefix(None, _log(rng, 1, 64), Hk * group, Hk, T, _log(rng, 1, 16384), _log(rng, T, 2048), rng.choice(["f32", "bf16", "f16"]),
                        layout=rng.choice(["bhtd", "bthd"]))
            w = work(c)
            if w["bytes"] <= 4e8 and w["flops"] <= (2e11 if c["dtype"] != "f32" else 4e10) and c["B"] * c["H"] * T * (c["prefix"] + c["own"]) <= 1.0e9:
                return c
    while True:
        B, Hk, group = _log(rng, 1, 64), rng.choice([1, 2, 4, 8, 12, 25]), rng.choice([1, 1, 2, 3, 4])
        T = rng.choice([1, _log(rng, 1, 33000), _log(rng, 1, 33000)])
        dtype = rng.choice(["f32", "bf16", "f16"])
        axes = rng.choice(["32", "16,16", "8,12,12", "10,11", "5,9,9,9"])  # the fourth leaves elements as they are
        c = _rows(None, op, rng.choice([False, True]), B, Hk * group, Hk, T, dtype, rng.choice(["f32", dtype]), axes,
                  interleaved=rng.choice([False, True]), layout=rng.choice(["packed", "bhtd"]), far=_log(rng, 1, 500000))
        if work(c)["bytes"] <= 1.0e9:
            return c


def _sections(case):
    return tuple(int(x) for x in case["sections"].split(","))


def _lengths(case):
    """Keys each request has of its own: spread over what the cache holds (an idle place among them when decoding)."""
    lo = 0 if case["T"] == 1 else case["T"]
    if case["B"] == 1:
        return [case["own"]]
    return [lo + round((case["own"] - lo) * i / (case["B"] - 1)) for i in range(case["B"])]


def work(case):
    if case["op"] == "prefix":
        B, H, Hk, T, b = case["B"], case["H"], case["Hk"], case["T"], BYTES[case["dtype"]]
        lens = _lengths(case)
        seen = sum(sum(max(0, n - T + i + 1) for i in range(T)) for n in lens) + B * T * case["prefix"]
        kept = case["prefix"] + sum(lens)
        return {"bytes": 2 * Hk * kept * 64 * b + B * H * T * (64 * 2 * b + 4) + 4 * B, "flops": 256 * H * seen}
    n = case["B"] * (case["H"] + case["Hk"]) * case["T"] * 64
    x, y = BYTES[case["dtype"]], BYTES[case["out"]]
    pos = 4 * len(_sections(case)) * case["B"] * case["T"]
    if case["op"] == "rotary":
        return {"bytes": n * (x + y) + pos, "flops": 3 * n}
    if not case["back"]:
        return {"bytes": n * (x + y) + pos + 512, "flops": 7 * n}
    return {"bytes": n * (2 * x + y) + pos + 1024, "flops": 14 * n}


def _positions(case, g):
    """Text counts up on every axis; every other run of 64 tokens is a picture of 8 x 8 patches at one time.  The rows start
    at different places up to ``far``."""
    A, B, T = len(_sections(case)), case["B"], case["T"]
    t = torch.arange(T, device="cuda")
    start = torch.randint(0, case["far"] + 1, (B, 1), generator=g, device="cuda")
    picture = (t // 64) % 2 == 1
    here = t - t % 64
    axes = [torch.where(picture, here, t), torch.where(picture, here + (t % 64) // 8, t), torch.where(picture, here + t % 8, t),
            t // 64]
    if A == 2:
        axes = axes[1:]
    return torch.stack([a + start for a in axes[:A]]).to(torch.int32)


def _tensor(g, shape, dtype, sigma=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * sigma).to(TYPES[dtype])


def _qk(case, g, dtype, sigma=1.0):
    """Queries and keys [B, heads, T, 64]: views of a fused projection's output (values behind them), or tensors of their own."""
    B, H, Hk, T = case["B"], case["H"], case["Hk"], case["T"]
    if case["layout"] == "packed":
        x = _tensor(g, (B, T, H + 2 * Hk, 64), dtype, sigma)
        return x[:, :, :H].transpose(1, 2), x[:, :, H:H + Hk].transpose(1, 2)
    return _tensor(g, (B, H, T, 64), dtype, sigma), _tensor(g, (B, Hk, T, 64), dtype, sigma)


def _cache(case, g):
    """Keys or values of each request, [B, Hk, own, 64], stored head by head or token by token."""
    B, Hk, S = case["B"], case["Hk"], case["own"]
    if case["layout"] == "bthd":
        return _tensor(g, (B, S, Hk, 64), case["dtype"]).transpose(1, 2)
    return _tensor(g, (B, Hk, S, 64), case["dtype"])


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    if case["op"] == "prefix":
        B, H, Hk, T, P = case["B"], case["H"], case["Hk"], case["T"], case["prefix"]
        q = _tensor(g, (B, T, H, 64), case["dtype"], 1.5).transpose(1, 2)
        if case["layout"] == "bthd":
            kp, vp = (_tensor(g, (P, Hk, 64), case["dtype"]).transpose(0, 1) for _ in range(2))
        else:
            kp, vp = (_tensor(g, (Hk, P, 64), case["dtype"]) for _ in range(2))
        k, v = _cache(case, g), _cache(case, g)
        order = torch.randperm(B, generator=g, device="cuda")
        lens = torch.tensor(_lengths(case), device="cuda", dtype=torch.int32)[order].contiguous()
        return dict(s, q=q, kp=kp, vp=vp, k=k, v=v, lens=lens)
    s["sections"] = _sections(case)
    s["positions"] = _positions(case, g)
    n = sum(s["sections"])
    s["axis"] = torch.tensor([a for a, m in enumerate(s["sections"]) for _ in range(m)], device="cuda")  # of every pair
    s["frequency"] = 10000.0 ** (-torch.arange(n, device="cuda", dtype=torch.float64) / 32)
    if case["op"] == "norm":
        s["q"], s["k"] = _qk(case, g, case["dtype"], 1.7)
        s["wq"], s["wk"] = (1 + 0.2 * torch.randn(64, generator=g, device="cuda") for _ in range(2))
    elif not case["back"]:
        s["q"], s["k"] = _qk(case, g, case["dtype"])
    if case["back"]:  # gradients as the attention's backward leaves them: tensors of their own
        s["dq"], s["dk"] = _qk(dict(case, layout="bhtd"), g, case["out"], 0.3)
    return s


# ---- the operators' plain forms ------------------------------------------------------------------------------------------
def _angles(s):
    """cos and sin of every pair, [B, 1, T, 32], from angles in 64 bits: at position 100 000 an angle in 32 bits is off by 0.004."""
    a = torch.zeros((*s["positions"].shape[1:], 32), device="cuda", dtype=torch.float64)
    a[..., :len(s["axis"])] = s["positions"][s["axis"]].permute(1, 2, 0) * s["frequency"]
    return a.cos().float()[:, None], a.sin().float()[:, None]


def _turn(x, cos, sin, interleaved):
    if interleaved:
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2)
    a, b = x[..., :32], x[..., 32:]
    return torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1)


def _plain_rotary(s):
    cos, sin = _angles(s)
    if s["back"]:
        return {n: _turn(s[n].float(), cos, -sin, s["interleaved"]).to(TYPES[s["dtype"]]) for n in ("dq", "dk")}
    return {n: _turn(s[n].float(), cos, sin, s["interleaved"]).to(TYPES[s["out"]]) for n in ("q", "k")}


def _plain_norm(s, x, w, dy, cos, sin):
    x = x.float()
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
    if dy is None:
        return _turn(x * r * w, cos, sin, s["interleaved"]).to(TYPES[s["out"]])
    z = _turn(dy.float(), cos, -sin, s["interleaved"])
    n = x * r
    wz = w * z
    return (r * (wz - n * (wz * n).mean(-1, keepdim=True))).to(TYPES[s["dtype"]]), (z * n).sum((0, 1, 2))


def _plain_prefix(s):
    B, H, Hk, T, P = s["B"], s["H"], s["Hk"], s["T"], s["prefix"]
    G = H // Hk
    q = s["q"].float().reshape(B, Hk, G, T, 64) * SCALE
    sp = (q.transpose(0, 1).reshape(Hk, B * G * T, 64) @ s["kp"].float().transpose(1, 2)).view(Hk, B, G * T, P).transpose(0, 1)
    so = q.reshape(B, Hk, G * T, 64) @ s["k"].float().transpose(2, 3)
    j = torch.arange(s["own"], device="cuda")
    last = s["lens"][:, None] - T + torch.arange(T, device="cuda")
    seen = (j < s["lens"][:, None, None]) & (j <= last[:, :, None])  # [B, T, own]
    so = so.view(B, Hk, G, T, -1).masked_fill(~seen[:, None, None], -math.inf).view(B, Hk, G * T, -1)
    m = torch.maximum(sp.amax(-1, keepdim=True), so.amax(-1, keepdim=True))
    sp, so = (sp - m).exp(), (so - m).exp()
    total = sp.sum(-1, keepdim=True) + so.sum(-1, keepdim=True)
    o = (sp.transpose(0, 1).reshape(Hk, B * G * T, P) @ s["vp"].float()).view(Hk, B, G * T, 64).transpose(0, 1) + so @ s["v"].float()
    return {"o": (o / total).reshape(B, H, T, 64).to(TYPES[s["dtype"]]), "lse": (m + total.log()).reshape(B, H, T)}


def run(s):
    if own:
        import hyperkernels_b200 as hk

        if s["op"] == "prefix":
            o, lse = hk.shared_prefix_attention(s["q"], s["kp"], s["vp"], s["k"], s["v"], s["lens"], SCALE, True)
            return {"o": o, "lse": lse}
        if s["op"] == "rotary":
            if s["back"]:
                dq, dk = hk.rotary_backward(s["dq"], s["dk"], s["positions"], s["sections"], interleaved=s["interleaved"], out_dtype=TYPES[s["dtype"]])
                return {"dq": dq, "dk": dk}
            q, k = hk.rotary_forward(s["q"], s["k"], s["positions"], s["sections"], interleaved=s["interleaved"], out_dtype=TYPES[s["out"]])
            return {"q": q, "k": k}
        if s["back"]:
            dq, dk, dwq, dwk = hk.qk_norm_rotary_backward(s["q"], s["k"], s["dq"], s["dk"], s["wq"], s["wk"], s["positions"], s["sections"],
                                                          eps=EPS, interleaved=s["interleaved"])
            return {"dq": dq, "dk": dk, "dwq": dwq, "dwk": dwk}
        q, k = hk.qk_norm_rotary_forward(s["q"], s["k"], s["wq"], s["wk"], s["positions"], s["sections"], eps=EPS, interleaved=s["interleaved"],
                                         out_dtype=TYPES[s["out"]])
        return {"q": q, "k": k}
    if s["op"] == "prefix":
        return _plain_prefix(s)
    if s["op"] == "rotary":
        return _plain_rotary(s)
    cos, sin = _angles(s)
    if s["back"]:
        dq, dwq = _plain_norm(s, s["q"], s["wq"], s["dq"], cos, sin)
        dk, dwk = _plain_norm(s, s["k"], s["wk"], s["dk"], cos, sin)
        return {"dq": dq, "dk": dk, "dwq": dwq, "dwk": dwk}
    return {"q": _plain_norm(s, s["q"], s["wq"], None, cos, sin), "k": _plain_norm(s, s["k"], s["wk"], None, cos, sin)}


# ---- the definitions in 64 bits: rotations as products of complex numbers, request by request and head by head ---------------
def _exact_prefix(s):
    B, H, Hk, T, G = s["B"], s["H"], s["Hk"], s["T"], s["H"] // s["Hk"]
    o = torch.zeros((B, H, T, 64), device="cuda", dtype=torch.float64)
    lse = torch.zeros((B, H, T), device="cuda", dtype=torch.float64)
    lens = s["lens"].tolist()
    for h in range(H):
        kp, vp = s["kp"][h // G].double(), s["vp"][h // G].double()
        for b in range(B):
            n = lens[b]
            k, v = torch.cat([kp, s["k"][b, h // G, :n].double()]), torch.cat([vp, s["v"][b, h // G, :n].double()])
            x = s["q"][b, h].double() @ k.T * SCALE
            ahead = torch.arange(len(k), device="cuda") - (len(k) - T) > torch.arange(T, device="cuda")[:, None]
            x[ahead & (torch.arange(len(k), device="cuda") >= s["prefix"])] = -math.inf
            lse[b, h] = torch.logsumexp(x, -1)
            o[b, h] = torch.softmax(x, -1) @ v
    return {"o": o, "lse": lse}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "prefix":
        return _exact_prefix(s)
    turn = torch.zeros((case["B"], case["T"], 32), device="cuda", dtype=torch.float64)
    p = 0
    for a, n in enumerate(s["sections"]):
        for _ in range(n):
            turn[..., p] = s["positions"][a].double() * math.exp(-math.log(10000.0) * p / 32)
            p += 1
    unit = torch.polar(torch.ones_like(turn), turn)[:, None]

    def pairs(x):
        x = x.double()
        return torch.complex(x[..., 0::2], x[..., 1::2]) if case["interleaved"] else torch.complex(x[..., :32], x[..., 32:])

    def elements(c):
        return torch.view_as_real(c).flatten(-2) if case["interleaved"] else torch.cat([c.real, c.imag], -1)

    if case["op"] == "rotary":
        return {n: elements(pairs(s[n]) * (unit.conj() if case["back"] else unit)) for n in (("dq", "dk") if case["back"] else ("q", "k"))}
    got = {}
    for n in ("q", "k"):
        x, w = s[n].double(), s["w" + n].double()
        rms = (x.square().sum(-1, keepdim=True) / 64 + EPS).sqrt()
        if not case["back"]:
            got[n] = elements(pairs(x * w / rms) * unit)
            continue
        z = elements(pairs(s["d" + n]) * unit.conj())
        got["dw" + n] = (z * x / rms).sum((0, 1, 2))
        got["d" + n] = w * z / rms - x * (w * z * x).sum(-1, keepdim=True) / (64 * rms ** 3)
    return got
