"""A paged KV cache: sequences of different lengths in pages of one pool, in fp16 or quantised to int8 as they are written.

Stands beside the contiguous cache of `llama.Attention` (jsgrad/models/llama.ts:78-87), which holds equally long sequences at one
position and reserves max_context positions for each.  `PageTable` is the bookkeeping, on the host alone; `PagedCache` has the pools of every
layer and the calls on them; `PagedBatch` is one ragged batch: which sequences, how many new rows of each.  `Transformer.forward_paged`
runs a model on it.
"""
from __future__ import annotations

from math import prod

import numpy as np

from . import ffi
from .ffi import check
from .tensor import Tensor


class PageTable:
    """Which pages of a pool belong to which sequence."""

    def __init__(self, n_pages: int, page_size: int):
        if n_pages < 1 or page_size < 16 or page_size > 256 or page_size & (page_size - 1):
            raise ValueError(f"{n_pages} pages of {page_size} positions: page_size is a power of two from 16 to 256")
        self.n_pages, self.page_size = n_pages, page_size
        self.free = list(range(n_pages - 1, -1, -1))
        self.pages: dict[int, list[int]] = {}                 # per sequence; -1: given away behind the window
        self.lengths: dict[int, int] = {}
        self._next = 0

    @staticmethod
    def pages_for(prompts, n_new: int, page_size: int, window: int = 0, sinks: int = 0) -> int:
        """The most pages that sequences hold at a time which begin with these numbers of positions and grow by one n_new - 1 times, all at once; with a window,
        `slide` comes behind every step."""
        steps = np.asarray(prompts, np.int64)[:, None] + np.arange(n_new)
        held = -(-steps // page_size)
        if window:
            given = np.maximum(steps[:, :-1] - window + 1, 0) // page_size - -(-sinks // page_size)
            held[:, 1:] -= np.maximum(given, 0)
        return int(held.sum(0).max())

    def add(self) -> int:
        """A new, empty sequence."""
        seq, self._next = self._next, self._next + 1
        self.pages[seq], self.lengths[seq] = [], 0
        return seq

    def drop(self, seq: int) -> None:
        """The sequence is over; its pages are free."""
        self.free += [p for p in reversed(self.pages.pop(seq)) if p >= 0]
        del self.lengths[seq]

    def grow(self, seqs, counts) -> None:
        """Room for counts[i] more positions of seqs[i].  Nothing changes where the pool has too few pages left."""
        seqs, counts = list(seqs), [int(c) for c in counts]
        if len(seqs) != len(counts) or len(set(seqs)) != len(seqs) or any(c < 0 for c in counts):
            raise ValueError(f"sequences {seqs} with {counts} new positions: one count of 0 and more for each, no sequence twice")
        need = [-(-(self.lengths[s] + c) // self.page_size) - len(self.pages[s]) for s, c in zip(seqs, counts)]
        if sum(need) > len(self.free):
            raise MemoryError(f"{sum(need)} pages are needed and {len(self.free)} of {self.n_pages} are free")
        for s, c, n in zip(seqs, counts, need):
            self.pages[s] += [self.free.pop() for _ in range(n)]
            self.lengths[s] += c

    def _held(self, seqs) -> list[tuple[int, int, int]]:
        return [(s, len(self.pages[s]), self.lengths[s]) for s in seqs]

    def _put_back(self, held) -> None:
        """Takes a grow back: held is what the sequences had before it."""
        for s, n, length in reversed(held):
            if s in self.pages:
                self.free += [p for p in reversed(self.pages[s][n:]) if p >= 0]
                del self.pages[s][n:]
                self.lengths[s] = length

    def slide(self, seq: int, window: int, sinks: int = 0) -> int:
        """Gives away the pages that no later row of the sequence sees through this window; how many those were."""
        if window < 1 or sinks < 0:
            raise ValueError(f"window {window}, sinks {sinks}")
        pages, n = self.pages[seq], 0
        # the next row is at position lengths[seq] and sees positions > lengths[seq] - window
        for i in range(-(-sinks // self.page_size), max(0, self.lengths[seq] - window + 1) // self.page_size):
            if pages[i] >= 0:
                self.free.append(pages[i])
                pages[i], n = -1, n + 1
        return n


class PagedCache(PageTable):
    """Pools of n_layers layers under one page table.  dtype: "float16", or "int8" with a float scale per position and head."""

    def __init__(self, n_layers: int, n_kv_heads: int, head_dim: int, n_pages: int, page_size: int = 64, dtype: str = "float16", device: str = "HIP"):
        super().__init__(n_pages, page_size)
        if dtype not in ("float16", "int8"):
            raise ValueError(f"pages are float16 or int8, not {dtype}")
        if n_layers < 1 or not 0 < n_kv_heads <= 1024 or head_dim not in (64, 128):
            raise ValueError(f"{n_layers} layers of {n_kv_heads} heads of {head_dim}: one layer and more, 1 to 1024 heads of 64 or 128")
        self.n_layers, self.n_kv_heads, self.head_dim, self.dtype, self.device = n_layers, n_kv_heads, head_dim, dtype, device
        rows = (2, n_pages, n_kv_heads, page_size)
        self.pools = [Tensor.zeros((*rows, head_dim), dtype, device) for _ in range(n_layers)]       # k, then v
        self.scales = [Tensor.ones(rows, "float32", device) if dtype == "int8" else None for _ in range(n_layers)]
        self._plan: Tensor | None = None                      # row_starts, lengths and page table of the batch last begun
        self._batches = 0
        self._ws: dict[int, Tensor] = {}

    def begin(self, seqs, counts) -> "PagedBatch":
        """A batch of counts[i] new rows of seqs[i], with pages for them.  The batch before it is over: they share the arrays that the device
        reads, which move when a batch needs more room than any before it (a captured graph is of no more use then).  Where this raises, no sequence has
        changed."""
        seqs, counts = list(seqs), [int(c) for c in counts]
        if not 0 < len(seqs) <= 65535 or not 0 < sum(counts) < 1 << 24:
            raise ValueError(f"a batch has 1 to 65535 sequences and fewer than 2^24 rows, one at least: {len(seqs)} with {sum(counts)}")
        held = self._held(seqs)
        self.grow(seqs, counts)
        try:
            return self._plan_batch(seqs, counts, held)
        except BaseException:
            self._put_back(held)
            raise

    def _plan_batch(self, seqs, counts, held) -> "PagedBatch":
        width = max(1, max(len(self.pages[s]) for s in seqs))
        n = len(seqs)
        plan = np.full(2 * n + 1 + n * width, -1, np.int32)
        plan[0] = 0
        plan[1:n + 1] = np.cumsum(counts)
        plan[n + 1:2 * n + 1] = [self.lengths[s] for s in seqs]
        table = plan[2 * n + 1:].reshape(n, width)
        for i, s in enumerate(seqs):
            table[i, :len(self.pages[s])] = self.pages[s]
        self._batches += 1                                    # in front of what ends the batch before it
        if self._plan is None or self._plan.numel < plan.size:
            self._plan = Tensor.empty((2 * plan.size,), "int32", self.device)
        self._plan.lazydata.view(plan.size, "int32", 0).ensure_allocated().copyin(plan)
        return PagedBatch(self, n, int(plan[n]), width, held)

    def workspace(self, n_heads: int) -> Tensor:
        if n_heads not in self._ws:
            self._ws[n_heads] = Tensor.zeros((ffi.load().jsgrad_hip_attn_paged_workspace_bytes(n_heads, self.n_kv_heads, self.head_dim),), "uint8", self.device)
        return self._ws[n_heads]


class PagedBatch:
    """The rows of one ragged batch, in the order of its sequences: row i of a sequence is its position length - count + i."""

    def __init__(self, cache: PagedCache, n_seqs: int, rows: int, width: int, held: list[tuple[int, int, int]]):
        self.cache, self.n_seqs, self.rows, self.width, self._held = cache, n_seqs, rows, width, held
        self._number = cache._batches
        self._layers: dict[int, tuple] = {}                   # what the calls on a layer take

    def _cancel(self) -> None:
        """An error ended the batch between its layers: its sequences have the lengths and pages again that they had in front of it."""
        if self._number == self.cache._batches:
            self.cache._batches += 1
            self.cache._put_back(self._held)

    def _args(self, layer: int) -> tuple:
        if self._number != self.cache._batches:
            raise RuntimeError("another batch has begun on this cache")
        if layer in self._layers:
            return self._layers[layer]
        c, plan = self.cache, self.cache._plan.ptr
        pool, scales = c.pools[layer], c.scales[layer]
        half = pool.nbytes // 2
        sp = (scales.ptr, scales.ptr + scales.nbytes // 2) if scales is not None else (None, None)
        desc = ffi.PagesDesc(ffi.W_I8 if c.dtype == "int8" else ffi.W_F16, c.n_pages, c.page_size, c.n_kv_heads, c.head_dim, self.width,
                             pool.ptr, pool.ptr + half, *sp, plan + 4 * (2 * self.n_seqs + 1))
        self._layers[layer] = desc, plan, plan + 4 * (self.n_seqs + 1), self.n_seqs, self.rows
        return self._layers[layer]

    def _check(self, what: str, t: Tensor, heads: int) -> None:
        if t.dtype != "float16" or prod(t.shape) < self.rows * heads * self.cache.head_dim:
            raise ValueError(f"{what}: {self.rows} float16 rows of {heads} heads of {self.cache.head_dim} are wanted, got {t.dtype} {t.shape}")

    def write(self, layer: int, k: Tensor, v: Tensor, q: Tensor | None = None, freqs_cis: Tensor | None = None, n_heads: int = 0, q_out: Tensor | None = None) -> Tensor | None:
        """Rotates k (and q, into q_out or in place) by freqs_cis, as precompute_freqs_cis makes it, and writes k and v into the pages."""
        for what, t in (("k", k), ("v", v)):
            self._check(what, t, self.cache.n_kv_heads)
        if q is not None:
            q_out = q if q_out is None else q_out
            self._check("q", q, n_heads)
            self._check("q_out", q_out, n_heads)
        positions, odd = divmod(prod(freqs_cis.shape), self.cache.head_dim) if freqs_cis is not None else (0, 0)
        if freqs_cis is not None and (freqs_cis.dtype != "float16" or odd):
            raise ValueError(f"freqs_cis: float16 rows of {self.cache.head_dim} are wanted, got {freqs_cis.dtype} {freqs_cis.shape}")
        p = lambda t: t.ptr if t is not None else None
        check(ffi.load().jsgrad_hip_paged_write(*self._args(layer), p(q), k.ptr, v.ptr, p(freqs_cis), positions,
                                                p(q_out) if q is not None else None, n_heads))
        return q_out if q is not None else None

    def read(self, layer: int) -> tuple[Tensor, Tensor]:
        """The rows of the batch out of the pages, as float16 [rows, n_kv_heads, head_dim]."""
        shape = (self.rows, self.cache.n_kv_heads, self.cache.head_dim)
        k, v = Tensor.empty(shape, "float16", self.cache.device), Tensor.empty(shape, "float16", self.cache.device)
        check(ffi.load().jsgrad_hip_paged_read(*self._args(layer), k.ptr, v.ptr))
        return k, v

    def attend(self, layer: int, q: Tensor, n_heads: int, out: Tensor | None = None, window: int = 0, sinks: int = 0) -> Tensor:
        """Attention of q [rows, n_heads, head_dim] over the pages: everything up to a row's own position or, with window > 0, the last
        `window` positions of that and the first `sinks`."""
        self._check("q", q, n_heads)
        out = out if out is not None else Tensor.empty((self.rows, n_heads, self.cache.head_dim), "float16", self.cache.device)
        self._check("out", out, n_heads)
        check(ffi.load().jsgrad_hip_attn_paged(*self._args(layer), q.ptr, out.ptr, n_heads, window, sinks, self.cache.workspace(n_heads).ptr))
        return out
