"""Serving from a cache of pages, over torch tensors: attention within packed prompts and of new tokens (one, or a tree of drafts)
against the pages, and what happens to the pages in between.

They have no counterpart in the reference.  A pool of pages is a view ``[pages, heads, page, 64]`` with any strides whose last is 1 (rows
on 16 bytes), ``page`` a multiple of 16; pages stored token by token are one with the middle dimensions transposed.  Keys and values have a
pool each.  ``pages`` is the table, ``[B, width]`` of int32: token i of request b lies in row ``i % page`` of page ``pages[b, i // page]``.  An
entry outside the pool stands for no page: nothing is written there, and attention takes its keys and values for zeros.  Types are float32,
bfloat16 or float16, one for all of a call; arithmetic is fp32 (16-bit types: but for the weights that multiply values, which are rounded to
the type).  Tables, lengths and starts are read by the kernels, so a captured call follows them.  A call runs on the tensors' device, on
that device's current stream or the one given; results and workspaces that were not given are allocated for that stream.  All are for
serving: there is no backward pass, and tensors that require a gradient are taken as they are: the results are part of no graph.
"""
from __future__ import annotations

from . import attention as _att
from .attention import HKError, _stream_handle


def _native():
    return _att._native or _att._torch_calls()


def _result(r, where):
    if type(r) is int:
        raise HKError(r, where)
    return r


def _handle(stream):
    return stream if stream is None else _stream_handle(stream)


def prompt_workspace_bytes(Q, K, starts) -> int:
    """Bytes that a ``workspace`` of ``prompt_attention`` needs for these tensors' sizes and type, on Q's device; 0: none."""
    return _native().prompt_workspace(Q, K, starts)


def prompt_attention(Q, K, V, starts, scale: float, causal: bool = True, *, workspace=None, out=None, lse=None, stream=None):
    """O [N, H, 64], LSE [H, N] of whole prompts of different lengths, packed behind each other.

    ``Q``: [N, H, 64], ``K``, ``V``: [N, Hkv, 64], all prompts' tokens; H is a multiple of Hkv, and query head h reads head
    ``h // (H // Hkv)``.  ``starts``: [B + 1] of int32 on the device, ascending, taken into [0, N]: prompt b is the tokens
    ``starts[b] <= i < starts[b + 1]``, which may be none.  A token sees the keys of its prompt, with ``causal`` those up to its own.  Tokens
    before the first prompt and behind the last are left as they are in ``out`` and ``lse``.  A key that only ``causal`` hides from a token
    takes part with weight 0, so its values have to be finite; what other prompts hold does not matter.  The same call gives the same bits.
    ``workspace``: contiguous memory of ``prompt_workspace_bytes`` on the device, of any type, for this call alone until it is done (None:
    allocated).  It needs no contents and keeps none; each captured call needs its own."""
    return _result(_native().prompt(Q, K, V, starts, scale, causal, workspace, out, lse, _handle(stream)), "hk_prompt_attention")


def tree_workspace_bytes(Q, K, K_pages, V_pages, pages) -> int:
    """Bytes that a ``workspace`` of ``tree_attention`` needs for these tensors' sizes and type, on Q's device; 0: none."""
    return _native().tree_workspace(Q, K, K_pages, V_pages, pages)


def tree_attention(Q, K, V, K_pages, V_pages, pages, lengths, scale: float, tree=None, *, workspace=None, out=None, lse=None, stream=None):
    """O [B, H, T, 64], LSE [B, H, T] of T <= 64 new tokens of each of B requests: decoding (T = 1), or a tree of drafts to verify.

    ``Q``: [B, H, T, 64], ``K``, ``V``: [B, Hkv, T, 64], the new tokens'; they need not be in the cache yet (``cache_append`` brings those
    there that were accepted).  ``lengths``: [B] of int32 on the device, the keys each request has in its pages (taken into what the table
    has room for); rows behind them may hold anything.  ``tree``: [B, T] of int64: bit j of ``tree[b, i]`` says that token i sees new token j,
    itself and its ancestors; None: all up to itself, a chain.  Every token sees its request's keys in the pages.  A token that sees nothing
    gives O = 0, LSE = -inf.  A new token that the tree hides takes part with weight 0, so its values have to be finite.  The same call
    gives the same bits.  ``workspace``: as of ``prompt_attention``, with ``tree_workspace_bytes``."""
    return _result(_native().tree(Q, K, V, K_pages, V_pages, pages, lengths, scale, tree, workspace, out, lse, _handle(stream)), "hk_tree_attention")


def cache_append(K, V, K_pages, V_pages, pages, lengths, *, starts=None, picks=None, counts=None, stream=None) -> None:
    """Keys and values of new tokens into the pages, behind the ``lengths[b]`` tokens that are there; ``lengths`` itself stays.

    With ``starts``, as of ``prompt_attention``: ``K``, ``V`` are [N, Hkv, 64], the tokens of packed prompts.  Otherwise they are [B, Hkv, T,
    64], and request b gets the rows ``picks[b, k]`` for ``k < counts[b]``: the drafts that were accepted, in their order (``picks``: [B, T]
    of int32, None: 0, 1, ..; ``counts``: [B] of int32, None: T).  ``starts`` are taken into the tensor, as there.  A pick outside [0, T) is left out, and so is a token that has no page.
    Requests may not share the pages that are written."""
    r = _native().append(K, V, K_pages, V_pages, pages, lengths, starts, picks, counts, _handle(stream))
    if r != 0:
        raise HKError(r, "hk_cache_append")


def cache_fork(K_pages, V_pages, pages, lengths, users, source, room=1, *, stream=None):
    """The next batch out of this one: requests go on, end, are forked (beams) or start, and get pages for the tokens to come.

    Pools are [pages, Hkv, page, 64], or [layers, pages, Hkv, page, 64].  ``source``: [B'] of int32 on the device: request i of the next batch
    goes on where request ``source[i]`` of this one is; with any entry outside [0, B) it starts anew, with a length of 0.  ``room``: how many
    more tokens each of them gets pages for, [B'] of int32 on the device, or one number for all.  ``users``:
    [pages] of int32, how many hold each page: the entries of the table, and whoever else (a kept prefix, say) counts on.  Full pages are
    shared by all that go on with them.  One that is begun stays with the first of these; the others get one of their own and its rows
    copied.  Where a request's begun page is none (an earlier call had none to give), all that go on with it get one whose rows are zeros, which is what
    they counted for.  Who keeps a begun page beside the table keeps the rows that there are; behind them a request goes on, so let one row of the
    table at a time hold it.  Pages nobody holds any longer are given out at once, lowest first.
    Returns the next batch's ``pages`` [B', width], ``lengths`` [B'], ``users`` [pages], and ``missing`` [1]: how many pages could not be
    given because the pool is empty or the table is full (their entries are -1, rows that were to be copied there are lost)."""
    return _result(_native().fork(K_pages, V_pages, pages, lengths, users, source, room, _handle(stream)), "hk_cache_fork")


def cache_compact(K_pages, V_pages, pages, users, *, stream=None):
    """Brings the pages that somebody holds (``users`` > 0) to the front of the pools, so that what is behind them can be given back.

    Pools, ``pages`` and ``users`` as of ``cache_fork``.  Of n such pages those at n and behind it are copied, in their order, to the free ones
    in front of it, in theirs.  Returns ``pages`` and ``users`` as they are then, and ``where`` [pages]: each page's new place, -1 if it was free
    (for whoever else holds pages)."""
    return _result(_native().compact(K_pages, V_pages, pages, users, _handle(stream)), "hk_cache_compact")
