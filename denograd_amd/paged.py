"""A paged KV cache: sequences of different lengths in pages of one pool, in fp16 or quantised to int8 as they are written.
Sequences that begin alike may share pages (`fork`): whoever writes into a shared page gets a copy of it first.

Stands beside the contiguous cache of `llama.Attention` (jsgrad/models/llama.ts:78-87), which holds equally long sequences at one
position and reserves max_context positions for each.  `PageTable` is the bookkeeping, on the host alone; `PagedCache` has the pools of every
layer and the calls on them; `PagedBatch` is one ragged batch: which sequences, how many new rows of each.  `Transformer.forward_paged`
runs a model on it.
"""
from __future__ import annotations

from math import prod
from typing import TYPE_CHECKING

import numpy as np

from . import ffi
from .ffi import check
from .tensor import Tensor

if TYPE_CHECKING:
    from .nn import RMSNorm


class PageTable:
    """Which pages of a pool belong to which sequence."""

    def __init__(self, n_pages: int, page_size: int):
        if n_pages < 1 or page_size < 16 or page_size > 256 or page_size & (page_size - 1):
            raise ValueError(f"{n_pages} pages of {page_size} positions: page_size is a power of two from 16 to 256")
        self.n_pages, self.page_size = n_pages, page_size
        self.free = list(range(n_pages - 1, -1, -1))
        self.pages: dict[int, list[int]] = {}                 # per sequence; -1: given away behind the window
        self.lengths: dict[int, int] = {}
        self.shared: dict[int, int] = {}                      # pages with more than one holder: how many
        self.gaps: set[int] = set()                           # sequences with pages that were given away
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

    def _let_go(self, pages) -> None:
        """One holder less of each of these; those that had no other are free."""
        for p in pages:
            if p < 0:
                continue
            if p in self.shared:
                self.shared[p] -= 1
                if self.shared[p] == 1:
                    del self.shared[p]
            else:
                self.free.append(p)

    def drop(self, seq: int) -> None:
        """The sequence is over; pages that no other one holds are free."""
        self._let_go(reversed(self.pages.pop(seq)))
        del self.lengths[seq]
        self.gaps.discard(seq)

    def fork(self, seq: int, at: int | None = None) -> int:
        """A new sequence that begins with the first `at` positions of this one (default: all), in the same pages; those that were given away behind a window it does not have either."""
        at = self.lengths[seq] if at is None else int(at)
        if not 0 <= at <= self.lengths[seq]:
            raise ValueError(f"a fork at position {at} of a sequence of {self.lengths[seq]}")
        pages = self.pages[seq][:-(-at // self.page_size)]
        if at % self.page_size and pages[-1] < 0:
            raise ValueError(f"a fork at position {at}, in a page that was given away")
        new = self.add()
        self.pages[new], self.lengths[new] = list(pages), at
        if seq in self.gaps:
            self.gaps.add(new)
        for p in pages:
            if p >= 0:
                self.shared[p] = self.shared.get(p, 1) + 1
        return new

    def grow(self, seqs, counts) -> list[tuple[int, int, int]]:
        """Room for counts[i] more positions of seqs[i].  A begun last page that others hold as well is replaced by one of the sequence's own; returns what is to be copied
        before anything is written, as (from, to, positions).  Nothing changes where the pool has too few pages left."""
        seqs, counts = list(seqs), [int(c) for c in counts]
        if len(seqs) != len(counts) or len(set(seqs)) != len(seqs) or any(c < 0 for c in counts):
            raise ValueError(f"sequences {seqs} with {counts} new positions: one count of 0 and more for each, no sequence twice")
        need = [-(-(self.lengths[s] + c) // self.page_size) - len(self.pages[s]) for s, c in zip(seqs, counts)]
        # Holders of one page who all write: the longest of them into the page itself, behind what the others have there, so that a batch which is taken back leaves every one's rows.
        writers: dict[int, list[int]] = {}
        for i, (s, c) in enumerate(zip(seqs, counts)):
            if c and self.lengths[s] % self.page_size:
                writers.setdefault(self.pages[s][self.lengths[s] // self.page_size], []).append(i)
        own = [-1] * len(seqs)
        for page, held_by in writers.items():
            stays = max(held_by, key=lambda i: (self.lengths[seqs[i]], i)) if len(held_by) == self.shared.get(page, 1) else -1
            for i in held_by:
                own[i] = page if i != stays else -1
        wanted = sum(need) + sum(p >= 0 for p in own)
        if wanted > len(self.free):
            raise MemoryError(f"{wanted} pages are needed and {len(self.free)} of {self.n_pages} are free")
        moves = []
        for s, c, n, old in zip(seqs, counts, need, own):
            if old >= 0:
                at = self.lengths[s] // self.page_size
                self.pages[s][at] = self.free.pop()
                self._let_go([old])
                moves.append((old, self.pages[s][at], self.lengths[s] % self.page_size))
            self.pages[s] += [self.free.pop() for _ in range(n)]
            self.lengths[s] += c
        return moves

    def _held(self, seqs) -> list[tuple[int, list[int], int]]:
        return [(s, list(self.pages[s]), self.lengths[s]) for s in seqs]

    def _put_back(self, held) -> None:
        """Takes a grow back: held is what the sequences had before it."""
        for s, pages, length in reversed(held):
            if s not in self.pages:
                continue
            n = len(pages)
            self._let_go(reversed(self.pages[s][n:]))
            for at, (mine, old) in enumerate(zip(self.pages[s], pages)):
                if mine == old or mine < 0:                   # a page that was given away in the meantime stays so
                    pages[at] = mine
                    continue
                self._let_go([mine])
                if old in self.free:                          # its other holders are gone
                    self.free.remove(old)
                else:
                    self.shared[old] = self.shared.get(old, 1) + 1
            self.pages[s], self.lengths[s] = pages, length

    def slide(self, seq: int, window: int, sinks: int = 0) -> int:
        """Gives away the pages that no later row of the sequence sees through this window; how many those were."""
        if window < 1 or sinks < 0:
            raise ValueError(f"window {window}, sinks {sinks}")
        pages, n = self.pages[seq], 0
        # the next row is at position lengths[seq] and sees positions > lengths[seq] - window
        for i in range(-(-sinks // self.page_size), max(0, self.lengths[seq] - window + 1) // self.page_size):
            if pages[i] >= 0:
                self._let_go([pages[i]])
                pages[i], n = -1, n + 1
        if n:
            self.gaps.add(seq)
        return n

    def _pack(self) -> list[tuple[int, int, int]]:
        """Renumbers the pages so that those in use are the first ones; what has to be copied for that, from the upper ones to free lower ones."""
        used = {p for pages in self.pages.values() for p in pages if p >= 0}
        holes = [p for p in range(len(used)) if p not in used]
        to = dict(zip(sorted(p for p in used if p >= len(used)), holes))
        for pages in self.pages.values():
            pages[:] = [to.get(p, p) for p in pages]
        self.shared = {to.get(p, p): n for p, n in self.shared.items()}
        self.free = list(range(self.n_pages - 1, len(used) - 1, -1))
        return [(a, b, self.page_size) for a, b in to.items()]


class PagedCache(PageTable):
    """Pools of n_layers layers under one page table.  dtype: "float16", or "int8" with a float scale per position and head.  bounds: what PagedBatch.attend_chosen goes by is kept with
    every write."""

    def __init__(self, n_layers: int, n_kv_heads: int, head_dim: int, n_pages: int, page_size: int = 64, dtype: str = "float16", device: str = "HIP", bounds: bool = False):
        super().__init__(n_pages, page_size)
        if dtype not in ("float16", "int8"):
            raise ValueError(f"pages are float16 or int8, not {dtype}")
        if n_layers < 1 or not 0 < n_kv_heads <= 1024 or head_dim not in (64, 128):
            raise ValueError(f"{n_layers} layers of {n_kv_heads} heads of {head_dim}: one layer and more, 1 to 1024 heads of 64 or 128")
        self.n_layers, self.n_kv_heads, self.head_dim, self.dtype, self.device = n_layers, n_kv_heads, head_dim, dtype, device
        rows = (2, n_pages, n_kv_heads, page_size)
        self.pools = [Tensor.zeros((*rows, head_dim), dtype, device) for _ in range(n_layers)]       # k, then v
        self.scales = [Tensor.ones(rows, "float32", device) if dtype == "int8" else None for _ in range(n_layers)]
        # per layer: the least and largest of each feature of a page's keys, as whole numbers, and their unit
        self.bounds = [(Tensor.zeros((n_pages, n_kv_heads, 2, head_dim), "int8", device), Tensor.ones((n_pages, n_kv_heads), "float32", device)) for _ in range(n_layers)] if bounds else []
        self._chosen: Tensor | None = None
        self._moves: Tensor | None = None                     # what is copied next
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
        moves = self.grow(seqs, counts)
        try:
            if moves:
                self._copy(moves)
            return self._plan_batch(seqs, counts, held)
        except BaseException:
            self._put_back(held)
            raise

    def _page_pools(self) -> list[ffi.Pool]:
        """Every pool of every layer."""
        pools, row = [], self.head_dim * (2 if self.dtype == "float16" else 1)
        for pool, scales in zip(self.pools, self.scales):
            for i in (0, 1):
                pools.append(ffi.Pool(pool.ptr + i * (pool.nbytes // 2), self.n_kv_heads, self.page_size, row))
                if scales is not None:
                    pools.append(ffi.Pool(scales.ptr + i * (scales.nbytes // 2), self.n_kv_heads, self.page_size, 4))
        for codes, scales in self.bounds:
            pools += [ffi.Pool(codes.ptr, 1, 1, codes.nbytes // self.n_pages), ffi.Pool(scales.ptr, 1, 1, scales.nbytes // self.n_pages)]
        return pools

    def _copy(self, moves) -> None:
        moves = np.array(moves, np.int32).reshape(-1, 3)
        if self._moves is None or self._moves.numel < moves.size:
            self._moves = Tensor.empty((2 * moves.size,), "int32", self.device)
        self._moves.lazydata.view(moves.size, "int32", 0).ensure_allocated().copyin(moves.reshape(-1))
        pools = self._page_pools()
        check(ffi.load().jsgrad_hip_paged_copy((ffi.Pool * len(pools))(*pools), len(pools), self.n_pages, self._moves.ptr, len(moves)))

    def compact(self) -> int:
        """Packs the pages in use into the first ones of the pools, in all layers; how many those are.  A batch that had begun is over."""
        kept = {s: list(p) for s, p in self.pages.items()}, dict(self.shared), list(self.free)
        moves = self._pack()
        self._batches += 1
        try:
            if moves:
                self._copy(moves)
        except BaseException:
            self.pages, self.shared, self.free = kept
            raise
        return self.n_pages - len(self.free)

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
        return PagedBatch(self, n, int(plan[n]), width, held, counts)

    def workspace(self, n_heads: int, chosen: bool = False) -> Tensor:
        key = -n_heads if chosen else n_heads
        if key not in self._ws:
            call = ffi.load().jsgrad_hip_attn_selected_workspace_bytes if chosen else ffi.load().jsgrad_hip_attn_paged_workspace_bytes
            self._ws[key] = Tensor.zeros((call(n_heads, self.n_kv_heads, self.head_dim),), "uint8", self.device)
        return self._ws[key]


class PagedBatch:
    """The rows of one ragged batch, in the order of its sequences: row i of a sequence is its position length - count + i."""

    def __init__(self, cache: PagedCache, n_seqs: int, rows: int, width: int, held: list[tuple[int, list[int], int]], counts: list[int]):
        self.cache, self.n_seqs, self.rows, self.width, self._held = cache, n_seqs, rows, width, held
        self._gaps = [h for h, n in zip(held, counts) if n and h[0] in cache.gaps]     # what _check_seen looks at
        self._seen: set[tuple[int, int]] = set()              # windows and sinks that it has looked at
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

    def _check_seen(self, window: int, sinks: int) -> None:
        """Raises where a row's window reaches positions that were given away, as those of a fork behind the window of the sequence it comes from: they would be left out in silence."""
        if (window, sinks) in self._seen:
            return
        size = self.cache.page_size
        for s, pages, length in self._gaps:
            seen = pages[max(0, length - window + 1) // size if window else 0:] + (pages[:-(-min(sinks, length) // size)] if window else [])
            if -1 in seen:
                raise ValueError(f"sequence {s} has given away pages that its row at position {length} sees with window {window} and sinks {sinks}")
        self._seen.add((window, sinks))

    def write(self, layer: int, k: Tensor, v: Tensor, q: Tensor | None = None, freqs_cis: Tensor | None = None, n_heads: int = 0, q_out: Tensor | None = None,
              q_norm: "RMSNorm | None" = None, k_norm: "RMSNorm | None" = None) -> Tensor | None:
        """Rotates k (and q, into q_out or in place) by freqs_cis, as precompute_freqs_cis makes it, and writes k and v into the pages.  With k_norm and q_norm, the
        RMSNorms of a model that norms keys and queries per head, these come in front of the rotation."""
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
        norms = []
        if k_norm is not None or q_norm is not None:
            if k_norm is None or (q is None) != (q_norm is None) or (q is not None and q_norm.eps != k_norm.eps):
                raise ValueError("the norms of q and k go together, with one eps")
            for norm in (q_norm, k_norm):
                if norm is not None and (norm.weight.dtype != "float16" or norm.weight.numel != self.cache.head_dim):
                    raise ValueError(f"norms of q and k: {self.cache.head_dim} float16 weights are wanted, got {norm.weight.dtype} {norm.weight.shape}")
            norms = [q_norm.weight.ptr if q_norm is not None else None, k_norm.weight.ptr, k_norm.eps]
        call = ffi.load().jsgrad_hip_paged_write_norm if norms else ffi.load().jsgrad_hip_paged_write
        check(call(*self._args(layer), p(q), k.ptr, v.ptr, *norms, p(freqs_cis), positions, p(q_out) if q is not None else None, n_heads))
        if self.cache.bounds:
            codes, scales = self.cache.bounds[layer]
            check(ffi.load().jsgrad_hip_paged_bounds(*self._args(layer), codes.ptr, scales.ptr))
        return q_out if q is not None else None

    def read(self, layer: int) -> tuple[Tensor, Tensor]:
        """The rows of the batch out of the pages, as float16 [rows, n_kv_heads, head_dim]."""
        shape = (self.rows, self.cache.n_kv_heads, self.cache.head_dim)
        k, v = Tensor.empty(shape, "float16", self.cache.device), Tensor.empty(shape, "float16", self.cache.device)
        check(ffi.load().jsgrad_hip_paged_read(*self._args(layer), k.ptr, v.ptr))
        return k, v

    def attend(self, layer: int, q: Tensor, n_heads: int, out: Tensor | None = None, window: int = 0, sinks: int = 0) -> Tensor:
        """Attention of q [rows, n_heads, head_dim] over the pages: everything up to a row's own position or, with window > 0, the last
        `window` positions of that and the first `sinks`; these have to be there still (PageTable.slide)."""
        self._check("q", q, n_heads)
        self._check_seen(window, sinks)
        out = out if out is not None else Tensor.empty((self.rows, n_heads, self.cache.head_dim), "float16", self.cache.device)
        self._check("out", out, n_heads)
        check(ffi.load().jsgrad_hip_attn_paged(*self._args(layer), q.ptr, out.ptr, n_heads, window, sinks, self.cache.workspace(n_heads).ptr))
        return out

    def choose(self, layer: int, q: Tensor, n_heads: int, first: int, recent: int, top: int, out: Tensor | None = None) -> Tensor:
        """The pages of each row of q [rows, n_heads, head_dim] per kv head, by the bounds of their keys: int32 [rows, n_kv_heads, top], rising, -1 behind the last.  The first `first` and the last `recent` ones,
        the row's own among them, and of the others those on which its queries may score most."""
        self._check("q", q, n_heads)
        c = self.cache
        if not c.bounds:
            raise ValueError("pages are chosen by their bounds: a cache with bounds=True is wanted")
        shape = (self.rows, c.n_kv_heads, top)
        out = out if out is not None else Tensor.empty((self.rows, c.n_kv_heads, max(top, 1)), "int32", c.device)
        if out.dtype != "int32" or out.numel < prod(shape):
            raise ValueError(f"out: int32 {shape} are wanted, got {out.dtype} {out.shape}")
        codes, scales = c.bounds[layer]
        check(ffi.load().jsgrad_hip_paged_select(*self._args(layer), q.ptr, n_heads, codes.ptr, scales.ptr, first, recent, top, out.ptr))
        return out if out.shape == shape else Tensor(buffer=out.lazydata.view(prod(shape), "int32", 0), shape=shape, dtype="int32", device=c.device)

    def attend_pages(self, layer: int, q: Tensor, n_heads: int, chosen: Tensor, out: Tensor | None = None) -> Tensor:
        """Attention of q [rows, n_heads, head_dim] over the positions up to a row's own on the pages in chosen [rows, n_kv_heads, any number]."""
        self._check("q", q, n_heads)
        c = self.cache
        if chosen.dtype != "int32" or len(chosen.shape) != 3 or chosen.shape[0] < self.rows or chosen.shape[1] != c.n_kv_heads:
            raise ValueError(f"chosen: int32 [{self.rows}, {c.n_kv_heads}, pages] are wanted, got {chosen.dtype} {chosen.shape}")
        out = out if out is not None else Tensor.empty((self.rows, n_heads, c.head_dim), "float16", c.device)
        self._check("out", out, n_heads)
        check(ffi.load().jsgrad_hip_attn_selected(*self._args(layer), q.ptr, out.ptr, n_heads, chosen.ptr, chosen.shape[2], c.workspace(n_heads, True).ptr))
        return out

    def attend_chosen(self, layer: int, q: Tensor, n_heads: int, first: int, recent: int, top: int, out: Tensor | None = None) -> Tensor:
        """Attention over the pages that `choose` names, in a list that the cache keeps for every layer and batch."""
        c, n = self.cache, self.rows * self.cache.n_kv_heads * max(top, 1)
        if c._chosen is None or c._chosen.numel < n:
            c._chosen = Tensor.empty((n,), "int32", c.device)
        return self.attend_pages(layer, q, n_heads, self.choose(layer, q, n_heads, first, recent, top, c._chosen), out)
