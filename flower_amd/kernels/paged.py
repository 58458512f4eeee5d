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

import math

import torch

from .. import _lib
from .rotary import check_tables

_FULL = 0x7FFFFFFF                # a window longer than any table


def _check_pool(k_pages: torch.Tensor, v_pages: torch.Tensor, dims: int) -> None:
    """Pools of one layer (dims 4) or of all layers (dims 5)."""
    if k_pages.dim() != dims or v_pages.dim() != dims:
        raise ValueError(f"k_pages and v_pages must have {dims} dimensions, got {tuple(k_pages.shape)}, {tuple(v_pages.shape)}")
    shape = k_pages.shape
    if v_pages.shape != (*shape[:-2], shape[-1], shape[-2]):
        raise ValueError("k_pages (.., pages, kv heads, page size, D) and v_pages (.., pages, kv heads, D, page size) do not "
                         f"match: {tuple(shape)}, {tuple(v_pages.shape)}")
    if k_pages.dtype != v_pages.dtype or k_pages.dtype not in (torch.bfloat16, torch.float8_e4m3fn):
        raise TypeError(f"the cache holds bfloat16 or float8_e4m3fn, got {k_pages.dtype} and {v_pages.dtype}")
    if not (k_pages.is_contiguous() and v_pages.is_contiguous()):
        raise ValueError("k_pages and v_pages must be contiguous")
    if k_pages.device != v_pages.device:
        raise ValueError("k_pages and v_pages must be on one device")


def _check_ints(device, **tensors) -> None:
    for name, (t, shape) in tensors.items():
        if t.dtype != torch.int32 or tuple(t.shape) != shape or not t.is_contiguous() or t.device != device:
            raise ValueError(f"{name} must be a contiguous int32 tensor {shape} on {device}, got {tuple(t.shape)} {t.dtype} "
                             f"on {t.device}")


def _check_scales(k_pages, k_scale, v_scale) -> None:
    if k_pages.dtype == torch.bfloat16:
        if k_scale is not None or v_scale is not None:
            raise ValueError("a bfloat16 cache takes no scales")
        return
    for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
        if t is None or t.dtype != torch.float32 or tuple(t.shape) != (k_pages.shape[1],) or not t.is_contiguous() \
                or t.device != k_pages.device:
            raise ValueError(f"an e4m3 cache needs {name}, contiguous float32 ({k_pages.shape[1]},) on {k_pages.device}")


def _check_heads(q: torch.Tensor, k_pages: torch.Tensor, tables: torch.Tensor) -> None:
    if q.dim() != 4:
        raise ValueError(f"expected (B, H, T, D), got {tuple(q.shape)}")
    if q.dtype != torch.bfloat16:
        raise TypeError(f"the paged cache's operators take bfloat16 heads; got {q.dtype}")
    if q.shape[3] not in (32, 64, 128):
        raise ValueError(f"head_dim must be 32/64/128, got {q.shape[3]}")
    if q.shape[3] != k_pages.shape[3] or q.shape[1] % k_pages.shape[1]:
        raise ValueError(f"q {tuple(q.shape)} does not match the pool's {k_pages.shape[1]} kv heads of {k_pages.shape[3]} values")
    if q.numel() == 0:
        raise ValueError("q must not be empty")
    if tables.dim() != 2 or tables.shape[0] != q.shape[0]:
        raise ValueError(f"tables must be ({q.shape[0]}, entries), got {tuple(tables.shape)}")
    if q.device != k_pages.device:
        raise ValueError(f"q is on {q.device}, the pages on {k_pages.device}")
    _lib.require_gpu(q)


def _refuse_grad(what: str, *tensors) -> None:
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise RuntimeError(f"{what} is forward-only: call it under torch.no_grad() or on detached tensors")


def paged_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                 tables: torch.Tensor, lens: torch.Tensor, counts: torch.Tensor | None = None, *,
                 cos: torch.Tensor | None = None, sin: torch.Tensor | None = None, layout: str = "interleaved",
                 norm_eps: float | None = None, k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None,
                 return_k: bool = False):
    """The new tokens' heads into the cache, in one launch: q' (B, H, T, D), contiguous (and, with ``return_k``, k' as it
    was written, before an e4m3 cache's cast).

    q (B, H, T, D), k and v (B, KV, T, D) bf16, any strides with contiguous 16-byte rows (views of a projection's output).
    Token t of sequence b stands at position lens[b] - counts[b] + t (``lens`` counts the new tokens in; ``counts`` None: T
    each); tokens t >= counts[b] are padding: nothing is written for them and their q' is zero. norm_eps: q and k are normed
    over the head first (x / sqrt(mean(x^2) + eps), HeadRMSNorm). cos, sin, layout: rotary positions as in ``apply_rotary``.
    fp32 arithmetic, rounded once. A position without a page is not written. Forward-only.
    """
    _check_pool(k_pages, v_pages, 4)
    _check_heads(q, k_pages, tables)
    B, _, T, D = q.shape
    if k.shape != (B, k_pages.shape[1], T, D) or v.shape != k.shape or k.dtype != q.dtype or v.dtype != q.dtype \
            or k.device != q.device or v.device != q.device:
        raise ValueError(f"k and v must be {(B, k_pages.shape[1], T, D)} {q.dtype}, got {tuple(k.shape)} {k.dtype}, "
                         f"{tuple(v.shape)} {v.dtype}")
    _refuse_grad("paged_append", q, k, v)
    _check_ints(q.device, tables=(tables, tuple(tables.shape)), lens=(lens, (B,)))
    if counts is not None:
        _check_ints(q.device, counts=(counts, (B,)))
    _check_scales(k_pages, k_scale, v_scale)
    if (cos is None) != (sin is None):
        raise ValueError("give both cos and sin, or neither")
    if cos is not None:
        check_tables(cos, sin, D, layout, q.device)
    qo, ko = _lib.native().paged_append(q, k, v, k_pages, v_pages, tables, lens, counts, norm_eps, cos, sin,
                                        layout == "half", k_scale, v_scale, return_k, _lib.stream_of(q))
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
    e4m3 cache's codes are multiplied as they are. Made for few tokens a sequence (T H / KV up to 16 read the cache once;
    each further 16 read it again). Forward-only.
    """
    _check_pool(k_pages, v_pages, 4)
    _check_heads(q, k_pages, tables)
    _refuse_grad("paged_attention", q)
    B = q.shape[0]
    _check_ints(q.device, tables=(tables, tuple(tables.shape)), lens=(lens, (B,)))
    if counts is not None:
        _check_ints(q.device, counts=(counts, (B,)))
    _check_scales(k_pages, k_scale, v_scale)
    scale = 1.0 / math.sqrt(q.shape[3]) if scale is None else float(scale)
    out, lse = _lib.native().paged_attention(q, k_pages, v_pages, tables, lens, counts, _FULL if window is None else int(window),
                                             scale, k_scale, v_scale, return_lse, _lib.stream_of(q))
    return (out, lse) if return_lse else out


def _check_state(tables, refs, lens=None) -> None:
    if tables.dim() != 2 or refs.dim() != 1:
        raise ValueError(f"tables must be (S, entries) and refs (pages,), got {tuple(tables.shape)}, {tuple(refs.shape)}")
    _lib.require_gpu(tables)
    _check_ints(tables.device, tables=(tables, tuple(tables.shape)), refs=(refs, tuple(refs.shape)))
    if lens is not None:
        _check_ints(tables.device, lens=(lens, (tables.shape[0],)))


def _outputs(out, *like):
    """The tensors to write: ``out``, one for each of ``like`` (each may be that one itself), or new ones."""
    if out is None:
        return tuple(torch.empty_like(t) for t in like)
    if len(out) != len(like):
        raise ValueError(f"out takes {len(like)} tensors, got {len(out)}")
    for o, t in zip(out, like):
        _check_ints(t.device, out=(o, tuple(t.shape)))
        for x in like:
            if o.data_ptr() != x.data_ptr() and o.untyped_storage().data_ptr() == x.untyped_storage().data_ptr() \
                    and o.data_ptr() < x.data_ptr() + 4 * x.numel() and x.data_ptr() < o.data_ptr() + 4 * o.numel():
                raise ValueError("an output may be an input, but not overlap one")
        if any(o.data_ptr() == x.data_ptr() for x in like if x is not t):
            raise ValueError("an output may only be its own input")
    return tuple(out)


def reserve_pages(tables: torch.Tensor, lens: torch.Tensor, refs: torch.Tensor, counts: torch.Tensor, page_size: int, *,
                  window: int | None = None, out=None):
    """(tables, lens, refs, granted): room for counts[s] more tokens of each sequence.

    With a window, entries wholly behind what a sequence's next token sees are given back first. Then the new positions'
    empty entries are filled with free pages, the lowest numbers first, in the order of the sequences, and lens grows by
    counts. A sequence whose pages cannot be had (the wants up to it exceed the free pages, or its table is too short) is
    left as it was, with granted[s] = 0, as one with counts[s] <= 0 is; else granted[s] = counts[s]: pass ``lens`` and
    ``granted`` on to ``paged_append`` and ``paged_attention``. out: (tables, lens, refs) to write, which may be the inputs.
    """
    _check_state(tables, refs, lens)
    _check_ints(tables.device, counts=(counts, (tables.shape[0],)))
    if window is not None and window <= 0:
        raise ValueError("window must be positive")
    to = _outputs(out, tables, lens, refs)
    granted = _lib.native().reserve_pages(tables, lens, refs, counts, int(page_size), int(window or 0), *to,
                                          _lib.stream_of(tables))
    return (*to, granted)


def _all_layers(k_pages, v_pages, refs):
    if k_pages.dim() == 4:
        k_pages, v_pages = k_pages[None], v_pages[None]
    _check_pool(k_pages, v_pages, 5)
    if k_pages.shape[1] != refs.shape[0] or k_pages.device != refs.device:
        raise ValueError(f"the pool {tuple(k_pages.shape)} on {k_pages.device} is not of refs' {refs.shape[0]} pages")
    if k_pages.numel() == 0:
        raise ValueError("the pool must not be empty")
    return k_pages, v_pages


def reorder_pages(k_pages: torch.Tensor, v_pages: torch.Tensor, tables: torch.Tensor, lens: torch.Tensor, refs: torch.Tensor,
                  parents: torch.Tensor, *, out=None):
    """(tables, lens, refs) with place s holding a copy of the sequence that stood at parents[s] (int32): itself stays, any
    other forks it, a number that is no place (-1) leaves s empty and its pages to whoever else holds them.

    Full pages are shared. A last page that is not full stays with one child (the one in its parent's place, or else the
    first), each other child gets a free page (the lowest numbers first, in the order of s) and a copy of its positions, in
    the pools of all layers: k_pages (layers, pages, ..), v_pages, or one layer's. A place whose page cannot be had is
    emptied: its lens is 0. Pages that nobody holds any more can be taken in the same call. out: as in ``reserve_pages``.
    """
    _check_state(tables, refs, lens)
    _check_ints(tables.device, parents=(parents, (tables.shape[0],)))
    k_pages, v_pages = _all_layers(k_pages, v_pages, refs)
    to = _outputs(out, tables, lens, refs)
    _lib.native().reorder_pages(k_pages, v_pages, tables, lens, refs, parents, *to, _lib.stream_of(tables))
    return to


def compact_pages(k_pages: torch.Tensor, v_pages: torch.Tensor, tables: torch.Tensor, refs: torch.Tensor, *, out=None):
    """(tables, refs, live): the pages in use moved to the numbers 0 .. live[0] - 1, in the pools of all layers. The pages
    of higher numbers, in ascending order, take the free numbers below, in ascending order. out: (tables, refs) to write,
    which may be the inputs."""
    _check_state(tables, refs)
    k_pages, v_pages = _all_layers(k_pages, v_pages, refs)
    to = _outputs(out, tables, refs)
    live = _lib.native().compact_pages(k_pages, v_pages, tables, refs, *to, _lib.stream_of(tables))
    return (*to, live)


__all__ = ["paged_append", "paged_attention", "reserve_pages", "reorder_pages", "compact_pages"]
