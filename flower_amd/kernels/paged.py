"""The paged key-value cache's operators on the HIP library (gfx950): new tokens written to their pages, attention of the
newest tokens over them, and the pages' bookkeeping. The reference has no incremental decoding: it computes every key anew
(flower/models/base.py:553-665).

A layer's pool: ``k_pages`` (pages, kv heads, page size, D) and ``v_pages`` (pages, kv heads, D, page size), bfloat16 or
float8_e4m3fn with one float32 scale a kv head (``k_scale``, ``v_scale``). ``tables`` (S, entries) int32: the page of each
run of ``page size`` positions of a sequence, -1 where it holds none; ``lens`` (S,) int32: its positions; ``refs`` (pages,)
int32: how many table entries hold a page. Nothing of this comes back to the host: every call is asynchronous on the
current stream and can be captured in a graph. ``flower_amd.kv_cache.PagedKVCache`` keeps the state for a model.

``paged_append``     QK-norm and rotary positions of the new tokens' q and k, k and v written to their pages
``paged_attention``  the new tokens' attention over their sequences' pages, causal, optionally windowed
``reserve_pages``    room for the next tokens; pages behind the window given back
``reorder_pages``    sequences forked, dropped, or put in another order (a beam search's step)
``compact_pages``    the pages in use moved to the front of the pool
"""

from __future__ import annotations

import torch

from .. import _lib
from .rotary import ROTARY_LAYOUTS

_FULL = 0x7FFFFFFF                # a window longer than any table


def paged_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                 tables: torch.Tensor, lens: torch.Tensor, counts: torch.Tensor | None = None, *,
                 cos: torch.Tensor | None = None, sin: torch.Tensor | None = None, layout: str = "interleaved",
                 norm_eps: float | None = None, k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None,
                 return_k: bool = False):
    """The new tokens' heads into the cache, in one launch: q' (B, H, T, D), contiguous (and, with ``return_k``, k' as it
    was written, before an e4m3 cache's cast).

    q (B, H, T, D), k and v (B, KV, T, D) bf16, any strides with contiguous 16-byte rows (views of a projection's output).
    Token t of sequence b stands at position lens[b] - counts[b] + t (``lens`` counts the new tokens in; ``counts`` None: T
    each); tokens t >= counts[b] are padding: nothing is written for them and their q' (and k') is zero. norm_eps: q and k are normed
    over the head first (x / sqrt(mean(x^2) + eps), HeadRMSNorm). cos, sin, layout: rotary positions as in ``apply_rotary``.
    fp32 arithmetic, rounded once. A position without a page is not written. Forward-only.
    """
    if layout not in ROTARY_LAYOUTS:
        raise ValueError(f"layout must be one of {ROTARY_LAYOUTS}, got {layout!r}")
    qo, ko = _lib.native().paged_append(q, k, v, k_pages, v_pages, tables, lens, counts, cos, sin, layout == "half", norm_eps,
                                        k_scale, v_scale, return_k, _lib.stream_or_none(q))
    return (qo, ko) if return_k else qo


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, tables: torch.Tensor, lens: torch.Tensor,
                    counts: torch.Tensor | None = None, *, window: int | None = None, scale: float | None = None,
                    k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None, return_lse: bool = False):
    """Attention of the newest tokens over their sequences' pages: (B, H, T, D) bf16, a view of (B, T, H, D) storage (so
    ``out.transpose(1, 2).reshape(B, T, H * D)`` is a view), with the log-sum-exp (B, H, T) fp32 when ``return_lse``.

    q (B, H, T, D) bf16 as ``paged_append`` gives it; ``lens`` and ``counts`` as there: the query of token t stands at
    i = lens[b] - counts[b] + t and sees the keys j <= i, with i - j < window when a window is given (window <= 0: none, the
    result is zero). H is a multiple of the pool's kv heads: query head h reads kv head h // (H / KV). scale: of the scores,
    1 / sqrt(D) by default. A query without keys, and a padding token, gives zeros (lse -inf). Softmax and sums in fp32; an
    e4m3 cache's codes are multiplied as they are. Keys and values that are not finite reach only the rows that see them (where an
    infinite value may come out as NaN). The work is cut by the width of ``tables``, which must be contiguous: narrower
    ones serve short sequences faster. Made for few tokens a sequence: up to 64 rows (T H / KV) of a kv head read
    the cache once, each further 64 read it again. Forward-only.
    """
    out, lse = _lib.native().paged_attention(q, k_pages, v_pages, tables, lens, counts, _FULL if window is None else window,
                                             scale, k_scale, v_scale, return_lse, _lib.stream_or_none(q))
    return (out, lse) if return_lse else out


def reserve_pages(tables: torch.Tensor, lens: torch.Tensor, refs: torch.Tensor, counts: torch.Tensor, page_size: int, *,
                  window: int | None = None, out=None):
    """(tables, lens, refs, granted): room for counts[s] more tokens of each sequence.

    With a window, entries wholly behind what a sequence's next token sees are given back first. Then the new positions'
    empty entries are filled with free pages, the lowest numbers first, in the order of the sequences, and lens grows by
    counts. A sequence whose pages cannot be had (the wants up to it exceed the free pages, or its table is too short) is
    left as it was, with granted[s] = 0, as one with counts[s] <= 0 is; else granted[s] = counts[s]: pass ``lens`` and
    ``granted`` on to ``paged_append`` and ``paged_attention``. out: (tables, lens, refs) to write, which may be the inputs.
    """
    return _lib.native().reserve_pages(tables, lens, refs, counts, page_size, window, out, _lib.stream_or_none(tables))


def reorder_pages(k_pages: torch.Tensor, v_pages: torch.Tensor, tables: torch.Tensor, lens: torch.Tensor, refs: torch.Tensor,
                  parents: torch.Tensor, *, out=None, return_kept: bool = False):
    """(tables, lens, refs), with place s holding a copy of the sequence that stood at parents[s] (int32): itself stays, any
    other forks it, a number that is no place (-1) leaves s empty and its pages to whoever else holds them.

    Full pages are shared. A last page that is not full stays with one child (the one in its parent's place, or else the
    first), each other child gets a free page (the lowest numbers first, in the order of s) and a copy of its positions, in
    the pools of all layers: k_pages (layers, pages, ..), v_pages, or one layer's. A place whose page cannot be had is
    emptied: its lens is 0. Pages that nobody holds any more can be taken in the same call. out: as in ``reserve_pages``.
    ``return_kept`` adds kept (S,) int32: 1 where place s holds positions of its parent, 0 where it is empty: for want of a page,
    because it was to be emptied, or as its parent was.
    """
    *state, kept = _lib.native().reorder_pages(k_pages, v_pages, tables, lens, refs, parents, out, return_kept,
                                               _lib.stream_or_none(tables))
    return (*state, kept) if return_kept else tuple(state)


def compact_pages(k_pages: torch.Tensor, v_pages: torch.Tensor, tables: torch.Tensor, refs: torch.Tensor, *, out=None):
    """(tables, refs, live): the pages in use moved to the numbers 0 .. live[0] - 1, in the pools of all layers. The pages
    of higher numbers, in ascending order, take the free numbers below, in ascending order. out: (tables, refs) to write,
    which may be the inputs."""
    return _lib.native().compact_pages(k_pages, v_pages, tables, refs, out, _lib.stream_or_none(tables))


__all__ = ["paged_append", "paged_attention", "reserve_pages", "reorder_pages", "compact_pages"]
