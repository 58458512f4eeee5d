"""A model's paged key-value cache: the pools of all layers, and each sequence's table of pages.

The reference computes every key anew (flower/models/base.py:553-665); with this cache a model decodes: ``reserve`` makes
room for the next tokens, each layer then writes and reads its own pool (``append``, ``attend``, or
``CausalSelfAttention.forward_cached``), ``reorder`` forks and drops sequences. All state stays on the GPU, is updated in
place and never read by the host, so that a step can be captured in a graph and replayed.
"""

from __future__ import annotations

import torch

from .kernels.paged import compact_pages, paged_append, paged_attention, reorder_pages, reserve_pages


class PagedKVCache:
    """``num_pages`` pages of ``page_size`` positions for ``sequences`` places of at most ``max_len`` positions, for
    ``layers`` layers of ``kv_heads`` heads of ``head_dim`` values.

    dtype: bfloat16, or float8_e4m3fn with float32 scales ``k_scale``, ``v_scale`` (layers, kv_heads), ones by default.
    window: positions that a query sees; pages behind it are given back by ``reserve`` (give the longest of the layers'
    windows, None if a layer sees everything). A sequence holds max_len / page_size pages at most, or with a window
    window / page_size and two more beside those of the tokens of one ``reserve``.

    ``tables`` (sequences, entries), ``lens`` (sequences,), ``refs`` (num_pages,) and ``counts`` (sequences,) int32 are the
    state: counts are the tokens that the last ``reserve`` granted (less those taken back), which ``append`` and ``attend``
    work on.
    """

    def __init__(self, layers: int, num_pages: int, kv_heads: int, head_dim: int, *, sequences: int, max_len: int,
                 page_size: int = 64, dtype: torch.dtype = torch.bfloat16, window: int | None = None,
                 k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None, device="cuda") -> None:
        if min(layers, num_pages, kv_heads, sequences, max_len) <= 0:
            raise ValueError("layers, num_pages, kv_heads, sequences and max_len must be positive")
        if head_dim not in (32, 64, 128):
            raise ValueError(f"head_dim must be 32/64/128, got {head_dim}")
        if page_size not in (16, 32, 64, 128, 256, 512, 1024):
            raise ValueError(f"page size must be a power of two from 16 to 1024, got {page_size}")
        if dtype not in (torch.bfloat16, torch.float8_e4m3fn):
            raise TypeError(f"the cache holds bfloat16 or float8_e4m3fn, got {dtype}")
        if window is not None and window <= 0:
            raise ValueError("window must be positive")
        self.page_size, self.window, self.dtype, self.layers = page_size, window, dtype, layers
        self.k_scale, self.v_scale = None, None
        if dtype == torch.float8_e4m3fn:
            scales = []
            for name, s in (("k_scale", k_scale), ("v_scale", v_scale)):
                if s is None:
                    s = torch.ones((layers, kv_heads))
                if tuple(s.shape) != (layers, kv_heads):
                    raise ValueError(f"{name} must be (layers, kv_heads) = {(layers, kv_heads)}, got {tuple(s.shape)}")
                scales.append(s.detach().to(device=device, dtype=torch.float32, copy=True).contiguous())
            self.k_scale, self.v_scale = scales
        elif k_scale is not None or v_scale is not None:
            raise ValueError("scales are for a float8_e4m3fn cache")
        pool = dict(dtype=dtype, device=device)
        self.k_pages = torch.empty((layers, num_pages, kv_heads, page_size, head_dim), **pool)
        self.v_pages = torch.empty((layers, num_pages, kv_heads, head_dim, page_size), **pool)
        entries = -(-max_len // page_size)
        self.tables = torch.full((sequences, entries), -1, dtype=torch.int32, device=device)
        self.lens, self.counts = (torch.zeros(sequences, dtype=torch.int32, device=device) for _ in range(2))
        self.refs = torch.zeros(num_pages, dtype=torch.int32, device=device)

    @property
    def sequences(self) -> int:
        return self.tables.shape[0]

    @property
    def max_len(self) -> int:
        return self.tables.shape[1] * self.page_size

    def _scales(self, layer: int):
        return {} if self.k_scale is None else dict(k_scale=self.k_scale[layer], v_scale=self.v_scale[layer])

    def _ints(self, values) -> torch.Tensor:
        if isinstance(values, int):
            return torch.full((self.sequences,), values, dtype=torch.int32, device=self.lens.device)
        values = torch.as_tensor(values)
        if values.is_floating_point() or values.is_complex():
            raise TypeError(f"counts and places are whole numbers, got {values.dtype}")
        if values.dtype == torch.int64:                  # beyond 32 bits: as far as those go, not what is left of it
            values = values.clamp(-2 ** 31, 2 ** 31 - 1)
        return values.to(device=self.lens.device, dtype=torch.int32).contiguous()

    def reserve(self, counts) -> torch.Tensor:
        """Room for counts[s] (a tensor, a list, or one number for all) more tokens of each sequence, as ``reserve_pages``
        grants it; returns ``counts`` as granted, 0 for a sequence that found no room and for one that wanted none. The
        tokens are then given to every layer together: no more than the T that its heads have room for."""
        *_, granted = reserve_pages(self.tables, self.lens, self.refs, self._ints(counts), self.page_size, window=self.window,
                                    out=(self.tables, self.lens, self.refs))
        return self.counts.copy_(granted)

    def take_back(self, counts) -> None:
        """The last counts[s] (as ``reserve`` takes them) of the tokens that the last ``reserve`` granted are no more: drafted
        tokens that were not accepted. No more than were granted, so that a sequence never becomes shorter than a fork of it
        was, whose full pages it shares, nor than its window needs: lower ``lens`` by this alone. The pages stay with the
        sequence for its next tokens."""
        counts = self._ints(counts)
        if counts.shape != self.counts.shape:
            raise ValueError(f"counts must be ({self.sequences},), got {tuple(counts.shape)}")
        counts = torch.minimum(counts.clamp(min=0), self.counts)
        self.lens.sub_(counts)
        self.counts.sub_(counts)

    def append(self, layer: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, **how):
        """``paged_append`` of the reserved tokens' heads to a layer's pool (``how``: its rotary and norm arguments)."""
        return paged_append(q, k, v, self.k_pages[layer], self.v_pages[layer], self.tables, self.lens, self.counts,
                            **self._scales(layer), **how)

    def attend(self, layer: int, q: torch.Tensor, *, window: int | None = None, **how):
        """``paged_attention`` of the reserved tokens over a layer's pool, within ``window`` (the cache's own by default)."""
        window = self.window if window is None else window
        if self.window is not None and window > self.window:
            raise ValueError(f"the cache keeps a window of {self.window} positions, not {window}")
        return paged_attention(q, self.k_pages[layer], self.v_pages[layer], self.tables, self.lens, self.counts, window=window,
                               **self._scales(layer), **how)

    def reorder(self, parents) -> torch.Tensor:
        """Place s becomes a copy of the sequence at parents[s], or empty (-1), as ``reorder_pages`` does; returns its kept (S,)
        int32, on the GPU: 0 for an empty place, as one is whose copy found no page. Such a place must not go on as its parent:
        ``reserve(kept)`` gives one more token to the others only, on this step and on the next ones. ``counts`` is then of no
        sequence: ``reserve`` comes next."""
        *_, kept = reorder_pages(self.k_pages, self.v_pages, self.tables, self.lens, self.refs, self._ints(parents),
                                 out=(self.tables, self.lens, self.refs), return_kept=True)
        self.counts.zero_()
        return kept

    def free(self, places) -> None:
        """Empties the given places (numbers); their pages can be taken again where no fork holds them."""
        parents = list(range(self.sequences))
        for s in places:
            if not 0 <= s < self.sequences:
                raise ValueError(f"no place {s} of {self.sequences}")
            parents[s] = -1
        self.reorder(parents)

    def compact(self) -> torch.Tensor:
        """Moves the pages in use to the pool's front; returns their number (1,) int32, on the GPU."""
        *_, live = compact_pages(self.k_pages, self.v_pages, self.tables, self.refs, out=(self.tables, self.refs))
        return live


__all__ = ["PagedKVCache"]
