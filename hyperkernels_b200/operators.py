"""Operators round the attention calls, over torch tensors: rotary positions with several axes, norms of queries and keys with
the rotation in the same pass, both with their backward passes, and the attention of a batch that shares a prefix.

They have no counterpart in the reference.  Tensors are ``[B, heads, T, 64]`` views with any strides whose last is 1 (rows on
16 bytes), of float32, bfloat16 or float16; arithmetic is fp32 (shared prefixes of 16-bit types: but for the
weights that multiply values, see there).  A call runs on the tensors' device, on that device's current
stream or the one given; results and workspaces that were not given are allocated for that stream.
"""
from __future__ import annotations

import ctypes as C
import functools
from typing import Optional, Sequence

from . import attention as _att
from .attention import HKError, _stream_handle


class RotaryPlan(C.Structure):
    """hk_rotary_plan: what each of a row's 32 pairs turns by, per position and on which axis."""

    _fields_ = [("turn", C.c_uint64 * 32), ("axis", C.c_uint8 * 32), ("n_axes", C.c_int32), ("interleaved", C.c_int32)]


@functools.lru_cache(maxsize=64)
def _plan(sections, base, frequencies, interleaved) -> bytes:
    n = sum(sections)
    if frequencies is not None and len(frequencies) != n:
        raise ValueError(f"frequencies: expected {n}, one for each pair of the sections")
    plan = RotaryPlan()
    status = _att.lib().hk_rotary_plan_fill(C.byref(plan), len(sections), (C.c_int * len(sections))(*sections), float(base),
                                            None if frequencies is None else (C.c_double * n)(*frequencies), int(bool(interleaved)))
    if status != 0:
        raise HKError(status, "hk_rotary_plan_fill")
    return bytes(plan)


def rotary_plan(sections: Sequence[int], base: float = 10000.0, frequencies: Optional[Sequence[float]] = None,
                interleaved: bool = False) -> RotaryPlan:
    """The plan that the calls below make of these arguments, for callers of the C ABI."""
    return RotaryPlan.from_buffer_copy(_plan(tuple(sections), base, None if frequencies is None else tuple(frequencies), interleaved))


_dtype_codes = {}


def _code(dtype) -> int:
    if dtype is None:
        return -1
    if not _dtype_codes:
        import torch

        _dtype_codes.update({torch.float32: 0, torch.bfloat16: 1, torch.float16: 2})
    if dtype not in _dtype_codes:
        raise TypeError(f"out_dtype: expected float32, bfloat16 or float16, not {dtype}")
    return _dtype_codes[dtype]


def _qk(which, where, Q, K, dQ, dK, w_q, w_k, positions, sections, base, frequencies, interleaved, eps, out_dtype, out_q, out_k, stream):
    plan = _plan(tuple(sections), base, None if frequencies is None else tuple(frequencies), interleaved)
    r = (_att._native or _att._torch_calls()).qk(which, Q, K, dQ, dK, w_q, w_k, positions, plan, eps, _code(out_dtype), out_q, out_k,
                                                 stream if stream is None else _stream_handle(stream))
    if type(r) is int:
        raise HKError(r, where)
    return r


def rotary_forward(Q, K, positions, sections, *, base: float = 10000.0, frequencies=None, interleaved: bool = False,
                   out_dtype=None, out_q=None, out_k=None, stream=None):
    """Q, K turned by their positions: rotary embedding with one or several axes (text: one; images, video: time, height, width).

    ``positions``: [axes, B, T] of int32 or int64, any strides (expanded ones too).  ``sections``: how many of a row's 32 pairs
    turn with each axis, in order; pairs behind the last section are left as they are.  Pair p of all is elements (p, p + 32), or
    (2 p, 2 p + 1) with ``interleaved``, and turns by ``base ** (-p / 32)`` radians per position, or by ``frequencies[p]``.  The
    turns per position are rounded once, to 2^-64 of a turn; their product with an integer position is exact, modulo a turn.
    ``K`` may be None.  Results are new tensors of ``out_dtype`` (default: Q's type), or ``out_q`` / ``out_k``, which may be Q
    and K themselves and must not lie on top of each other.  A 16-bit type becomes float32 (what ``attention_forward`` reads) or
    stays; float32 becomes any."""
    return _qk(0, "hk_rotary_forward", Q, K, None, None, None, None, positions, sections, base, frequencies, interleaved, 0.0,
               out_dtype, out_q, out_k, stream)


def rotary_backward(dQ, dK, positions, sections, *, base: float = 10000.0, frequencies=None, interleaved: bool = False,
                    out_dtype=None, out_q=None, out_k=None, stream=None):
    """Gradients of ``rotary_forward``'s Q and K from those of its results; ``out_dtype`` is the type Q and K had."""
    return _qk(1, "hk_rotary_backward", None, None, dQ, dK, None, None, positions, sections, base, frequencies, interleaved, 0.0,
               out_dtype, out_q, out_k, stream)


def qk_norm_rotary_forward(Q, K, w_q, w_k, positions, sections, *, eps: float = 1e-6, base: float = 10000.0, frequencies=None,
                           interleaved: bool = False, out_dtype=None, out_q=None, out_k=None, stream=None):
    """``rotary_forward`` of ``x / sqrt(mean(x^2) + eps) * w`` for every row x of 64 of Q (``w_q``) and K (``w_k``), in one pass.

    The weights are [64] of float32 or Q's type, or None for ones.  ``out_dtype``: Q's type or float32."""
    return _qk(2, "hk_qk_norm_rotary_forward", Q, K, None, None, w_q, w_k, positions, sections, base, frequencies, interleaved, eps,
               out_dtype, out_q, out_k, stream)


def qk_norm_rotary_backward(Q, K, dQ, dK, w_q, w_k, positions, sections, *, eps: float = 1e-6, base: float = 10000.0,
                            frequencies=None, interleaved: bool = False, out_q=None, out_k=None, stream=None):
    """Gradients (of Q, of K, of w_q, of w_k) of ``qk_norm_rotary_forward`` from its arguments and the gradients dQ, dK of its
    results (Q's type or float32).  Those of Q and K are of Q's type, those of the weights float32 (None without a weight).
    The same call gives the same bits."""
    return _qk(3, "hk_qk_norm_rotary_backward", Q, K, dQ, dK, w_q, w_k, positions, sections, base, frequencies, interleaved, eps,
               None, out_q, out_k, stream)


def shared_prefix_workspace_bytes(Q, K_prefix, K) -> int:
    """Bytes that a ``workspace`` of ``shared_prefix_attention`` needs for these tensors' sizes and type, on Q's device; 0: none.

    It goes by how the work is cut: other sizes, even smaller ones, may need more."""
    return (_att._native or _att._torch_calls()).prefix_workspace(Q, K_prefix, K)


def shared_prefix_attention(Q, K_prefix, V_prefix, K, V, lengths, scale: float, causal: bool = True, *, workspace=None, out=None,
                            lse=None, stream=None):
    """O, LSE of the new tokens Q [B, H, T, 64] of B requests that share a prefix: forward only, for serving (T = 1: decoding).

    ``K_prefix``, ``V_prefix``: [Hkv, P, 64], the prefix's keys and values, read once for the whole batch.  ``K``, ``V``:
    [B, Hkv, S, 64], each request's own, of which the first ``lengths[b]`` rows (int32 on the device; None: S) are its keys,
    those of the new tokens among them.  Rows behind them may hold anything.  H is a multiple of Hkv; query head h reads head
    ``h // (H // Hkv)``.  Every new token sees the whole prefix and its request's own keys, with ``causal`` those up to its
    own: token i of T sees j <= lengths[b] - T + i.  A row that sees no key gives O = 0, LSE = -inf.  P and S may be 0.
    A key that only ``causal`` hides from a row takes part in it with weight 0, so its values have to be finite.  Keys and values
    may not be expanded (a stride of 0).  The same call gives the same bits.
    ``workspace``: contiguous memory of ``shared_prefix_workspace_bytes`` on the device, of any type, for this call alone until it
    is done (None: allocated).  It needs no contents and keeps none; each captured call needs its own.
    All of one type, which O has too; LSE is float32.  Scores, exponentials and sums are fp32; with 16-bit types the weights that
    multiply the values are rounded to that type, half a step each, as O is."""
    r = (_att._native or _att._torch_calls()).prefix(Q, K_prefix, V_prefix, K, V, lengths, scale, causal, workspace, out, lse,
                                                     stream if stream is None else _stream_handle(stream))
    if type(r) is int:
        raise HKError(r, "hk_shared_prefix_attention")
    return r
