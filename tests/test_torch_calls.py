"""CPU tests of the calls on torch tensors (csrc/hk_torch.cpp): what they refuse, and that nothing they meet ends the
process.  No call here gets as far as a launch."""
import os
import subprocess
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# (what throws, the call): each in a process of its own, which an exception that escapes the native code would end
THROWS = {
    "forward: the current stream of a machine without a device": "hk.attention_forward(x, x, x, 0.125, True)",
    "backward: the same": "hk.attention_backward(x, x, x, x, x, l, 0.125, True)",
    "zero_dq: the same": "att.zero_dq(x)",
    "forward: a tensor without data": "vmap(lambda y: hk.attention_forward(x, y, x, 0.125, True, stream=0))(x[None])",
    "backward: the same ": "vmap(lambda y: hk.attention_backward(x, x, x, x, y, l, 0.125, True, stream=0))(x[None])",
    "zero_dq: the same ": "vmap(lambda y: att.zero_dq(y, 0))(x[None])",
    "forward: no memory for the result": "hk.attention_forward(x.expand(1 << 24, 1 << 24, 64, 64), x, x, 0.125, True, stream=0)",
    "backward: the same  ": "hk.attention_backward(x.expand(1 << 24, 1 << 24, 64, 64), x, x, x, x, l, 0.125, True, stream=0)",
    "forward: a result without the dimensions": "hk.attention_forward(x, x, x, 0.125, True, lse=l[0, 0], stream=0)",
}


@pytest.mark.skipif(torch.cuda.is_available(), reason="host tensors: a kernel must not get them")
@pytest.mark.parametrize("what", THROWS)
def test_exceptions_of_the_native_calls_reach_the_caller(what):
    code = f"""
import torch, hyperkernels_b200 as hk, hyperkernels_b200.attention as att
from torch.func import vmap
x, l = torch.zeros(1, 1, 64, 64), torch.zeros(1, 1, 64)
try:
    {THROWS[what]}
except (RuntimeError, IndexError) as e:
    print("caught", not isinstance(e, hk.HKError))
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "caught True", (r.returncode, r.stdout, r.stderr[-400:])


FORWARD_TENSORS = ["Q", "K", "V", "dropout_mask", "workspace", "out", "lse"]
BACKWARD_TENSORS = ["Q", "K", "V", "O", "dO", "LSE", "dropout_mask", "workspace", "D", "dQ", "dK", "dV"]


@pytest.mark.parametrize("call,name", [("forward", n) for n in FORWARD_TENSORS] + [("backward", n) for n in BACKWARD_TENSORS])
@pytest.mark.parametrize("kind", ["numpy array", "list", "address", "False"])
def test_what_is_no_tensor_is_refused(call, name, kind):
    """A mask that is no tensor must not run without dropout, a buffer that is none must not be left unwritten."""
    import numpy as np

    import hyperkernels_b200 as hk

    x, l = torch.zeros(1, 1, 64, 64), torch.zeros(1, 1, 64)
    wrong = {"numpy array": np.ones((1, 64, 64), np.float32), "list": [1.0], "address": 4096, "False": False}[kind]
    args = dict(Q=x, K=x, V=x) if call == "forward" else dict(Q=x, K=x, V=x, O=x, dO=x, LSE=l)
    args.update(scale=0.125, causal=True, dropout_p=0.1)
    args[name] = wrong
    with pytest.raises(TypeError, match=f"^{name}: expected a tensor"):
        (hk.attention_forward if call == "forward" else hk.attention_backward)(**args)


@pytest.mark.parametrize("name", ["Q", "K", "V", "dO", "LSE"])
def test_none_is_refused_where_a_tensor_is_needed(name):
    import hyperkernels_b200 as hk
    import hyperkernels_b200.attention as att

    x, l = torch.zeros(1, 1, 64, 64), torch.zeros(1, 1, 64)
    args = dict(Q=x, K=x, V=x, O=x, dO=x, LSE=l, scale=0.125, causal=True)
    args[name] = None
    with pytest.raises(TypeError, match=f"^{name}: expected a tensor"):
        hk.attention_backward(**args)
    with pytest.raises(TypeError, match="^dQ: expected a tensor"):
        att.zero_dq(None)


def test_an_offset_without_a_seed_is_not_read():
    """philox_offset=None beside philox_seed=None, as a caller that forwards its own defaults passes them."""
    import hyperkernels_b200 as hk

    x, l = torch.zeros(1, 1, 64, 64), torch.zeros(1, 1, 64)
    # dropout_p = 1 is refused by the library, behind all reading of arguments and in front of any launch
    for call in (lambda **kw: hk.attention_forward(x, x, x, 0.125, True, dropout_p=1.0, stream=0, **kw),
                 lambda **kw: hk.attention_backward(x, x, x, x, x, l, 0.125, True, dropout_p=1.0, stream=0, **kw)):
        with pytest.raises(hk.HKError, match="dropout"):
            call(philox_offset=None)
        with pytest.raises(TypeError):
            call(philox_seed=1, philox_offset=None)


@pytest.mark.parametrize("status,address,dims,strides", [
    (-1, 0, (1, 1, 64), (4096, 4096, 64)), (-2, 4096, (1, 1, 0), (4096, 4096, 64)), (-2, 4096, (0, 1, 64), (4096, 4096, 64)),
    (-2, 4096, (1, 0, 64), (4096, 4096, 64)), (-3, 4100, (1, 1, 64), (4096, 4096, 64)), (-3, 4096, (1, 1, 64), (4096, 4096, 66)),
    (-3, 4096, (2, 1, 64), (4097, 4096, 64)), (-3, 4096, (1, 2, 64), (4096, 4098, 64))])
def test_zero_dq_refuses_what_its_kernel_cannot_write(status, address, dims, strides):
    """No rows (a division by zero on the host), no memory, or rows that are not on 16 bytes (a fault on the device).
    In a process of its own: the unchecked call ended it."""
    code = f"""
import ctypes as C, hyperkernels_b200 as hk
p = hk.MemEfficientBwdParams()
p.dQ = {address} or None
p.B, p.nh, p.T = {dims}
p.dq_strideB, p.dq_strideH, p.dq_strideM = {strides}
print(hk.lib().hk_attn_zero_dq(C.byref(p), None))
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == str(status), (r.returncode, r.stdout, r.stderr[-400:])


@pytest.mark.gpu
def test_no_memory_for_the_result_is_torchs_own_error():
    """torch.OutOfMemoryError, which programs catch to free memory and try again, not a bare RuntimeError."""
    import hyperkernels_b200 as hk

    x = torch.zeros(1, 1, 64, 64, device="cuda")
    with pytest.raises(torch.OutOfMemoryError):
        hk.attention_forward(x.expand(1 << 20, 1 << 10, 64, 64), x, x, 0.125, True)


@pytest.mark.gpu
def test_slabs_of_a_backward_on_another_stream_are_not_handed_on():
    """The slabs of the deterministic dQ are given back when the call returns.  Called with a stream that is not the
    current one and still busy, the kernels write them later: a tensor made meanwhile must not get that memory."""
    import hyperkernels_b200 as hk

    B, H, T = 1, 8, 1000
    g = torch.Generator(device="cuda").manual_seed(5)
    Q, K, V, dO = (torch.randn((B, H, T, 64), generator=g, device="cuda") for _ in range(4))
    O, LSE = hk.attention_forward(Q, K, V, 0.125, True)
    want = hk.attention_backward(Q, K, V, O, dO, LSE, 0.125, True, deterministic_dq=True)
    dQ, dK, dV = (torch.empty_like(Q) for _ in range(3))
    D = torch.empty_like(LSE)
    slab_floats = (T + 127) // 128 * B * H * T * 64 + 64
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)  # about 0.1 s
    hk.attention_backward(Q, K, V, O, dO, LSE, 0.125, True, deterministic_dq=True, dQ=dQ, dK=dK, dV=dV, D=D, stream=side)
    others = [torch.full((slab_floats,), 7.0, device="cuda") for _ in range(4)]
    torch.cuda.synchronize()
    assert hk.last_device_status() == 0
    assert all(bool((t == 7.0).all()) for t in others)
    assert torch.equal(dQ, want[0]) and torch.equal(dK, want[1]) and torch.equal(dV, want[2])


@pytest.mark.gpu
@pytest.mark.parametrize("handle", [0, 1, 2])
def test_slabs_under_the_streams_that_have_no_object(handle):
    """0, cudaStreamLegacy and cudaStreamPerThread, as numbers."""
    import hyperkernels_b200 as hk

    g = torch.Generator(device="cuda").manual_seed(6)
    Q, K, V, dO = (torch.randn((1, 2, 300, 64), generator=g, device="cuda") for _ in range(4))
    O, LSE = hk.attention_forward(Q, K, V, 0.125, True)
    want = hk.attention_backward(Q, K, V, O, dO, LSE, 0.125, True, deterministic_dq=True)
    torch.cuda.synchronize()
    got = hk.attention_backward(Q, K, V, O, dO, LSE, 0.125, True, deterministic_dq=True, stream=handle)
    torch.cuda.synchronize()
    assert hk.last_device_status() == 0
    assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---- what the kernels would read or write past its end -------------------------------------------------------------------
def _attention_arguments(call):
    x, kv, l = torch.zeros(2, 3, 5, 64), torch.zeros(2, 3, 9, 64), torch.zeros(2, 3, 5)
    args = dict(Q=x, K=kv, V=kv, scale=0.125, causal=True, dropout_p=0.1, dropout_mask=torch.ones(6, 5, 9), stream=0)
    return dict(args, out=x, lse=l) if call == "attention_forward" else dict(args, O=x, dO=x, LSE=l, D=l, dQ=x, dK=kv, dV=kv)


_LIKE_Q, _LIKE_K, _LIKE_L = ("Q", "out", "O", "dO", "dQ"), ("K", "V", "dK", "dV"), ("lse", "LSE", "D")
_WRONG = [(n, torch.zeros(2, 3, t, 64, dtype=d)) for names, t in ((_LIKE_Q, 5), (_LIKE_K, 9)) for n in names for d in (torch.bfloat16, torch.float16, torch.float64)]
_WRONG += [(n, torch.zeros(*s, 64)) for n in _LIKE_Q[1:] for s in ((1, 3, 5), (2, 1, 5), (2, 2, 5), (2, 3, 4))]
_WRONG += [(n, torch.zeros(*s, 64)) for n in _LIKE_K for s in ((1, 3, 9), (2, 1, 9), (2, 2, 9))]  # a group's shared heads among them
_WRONG += [(n, torch.zeros(2, 3, 8, 64)) for n in _LIKE_K[1:]]
_WRONG += [(n, x) for n in _LIKE_L for x in (torch.zeros(2, 3, 5, dtype=torch.bfloat16), torch.zeros(1, 3, 5), torch.zeros(2, 2, 5), torch.zeros(2, 3, 4), torch.zeros(6, 5),
                                             torch.zeros(2, 3, 10)[..., ::2])]
_WRONG += [("dropout_mask", x) for x in (torch.ones(6, 5, 9, dtype=torch.bool), torch.ones(6, 5, 8), torch.ones(6, 9, 5).transpose(1, 2), torch.ones(1, 5, 9).expand(6, 5, 9))]


@pytest.mark.parametrize("call,name,wrong", [(c, n, x) for c in ("attention_forward", "attention_backward") for n, x in _WRONG if n in _attention_arguments(c)])
def test_tensors_that_the_kernels_would_leave_are_refused(call, name, wrong):
    """Half-precision rows or shared key heads, as the operators round the attention give them, read as fp32 of Q's heads."""
    import hyperkernels_b200 as hk

    with pytest.raises(AssertionError, match=f"^{name}: "):
        getattr(hk, call)(**{**_attention_arguments(call), name: wrong})


def test_zero_dq_refuses_what_is_not_fp32():
    import hyperkernels_b200.attention as att

    with pytest.raises(AssertionError, match="^dQ: expected float32"):
        att.zero_dq(torch.zeros(1, 2, 5, 64, dtype=torch.bfloat16), 0)


def test_larger_tensors_and_masks_without_use_are_taken():
    """Room behind the rows, as before; a mask is looked at where the call drops anything by it.  (dropout_p = 1 and a mask beside a seed are
    refused by the library, behind these checks and in front of any launch.)"""
    import hyperkernels_b200 as hk

    room, rows = torch.zeros(3, 4, 9, 64), torch.zeros(3, 4, 9, 1)
    for call, more in (("attention_forward", dict(out=room, lse=rows[..., 0])), ("attention_backward", dict(O=room, dO=room, LSE=rows, D=rows, dQ=room, dK=room, dV=room))):
        args = {**_attention_arguments(call), **more, "V": torch.zeros(3, 3, 12, 64), "dropout_p": 1.0}
        with pytest.raises(hk.HKError, match="dropout"):
            getattr(hk, call)(**args)
        with pytest.raises(hk.HKError, match="dropout"):
            getattr(hk, call)(**{**args, "dropout_p": 0.5, "philox_seed": 3, "dropout_mask": torch.ones(1)})
        if call == "attention_backward":  # with D there, O is not read
            with pytest.raises(hk.HKError, match="dropout"):
                getattr(hk, call)(**{**args, "d_precomputed": True, "O": torch.zeros(1, 1, 1, 64, dtype=torch.bfloat16)})


@pytest.mark.parametrize("call", ["attention_forward", "attention_backward"])
def test_a_workspace_is_as_large_as_its_memory(call):
    """An expanded tensor has less memory than elements, one of a wider type more bytes than elements.  Those that are large enough get as
    far as the library, which refuses dropout_p = 1 in front of any launch."""
    import hyperkernels_b200 as hk

    x, l = torch.zeros(1, 2, 64, 64), torch.zeros(1, 2, 64)
    args = dict(Q=x, K=x, V=x, scale=0.125, causal=True, round_in_hbm=True, dropout_p=1.0, stream=0)
    args.update({} if call == "attention_forward" else dict(O=x, dO=x, LSE=l))
    need = 6 * 64 * 256 if call == "attention_forward" else 8 * 64 * 256
    for wrong, why in ((torch.zeros(1, dtype=torch.uint8).expand(1 << 20), "contiguous"), (torch.zeros(1 << 20, 2, dtype=torch.uint8)[:, 0], "contiguous"),
                       (torch.zeros(need - 1, dtype=torch.uint8), "too small"), (torch.zeros(need // 4 - 1), "too small"), (torch.zeros(0), "too small")):
        with pytest.raises(AssertionError, match=why):
            getattr(hk, call)(**args, workspace=wrong)
    for enough in (torch.zeros(need + 256, dtype=torch.uint8), torch.zeros(need // 4 + 64), torch.zeros(need // 512 + 1, 64, dtype=torch.float64)):
        with pytest.raises(hk.HKError, match="dropout"):
            getattr(hk, call)(**args, workspace=enough)
