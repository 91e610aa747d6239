"""Tokens for the rows of a batch, each by its own settings, from random numbers that the host draws.

Stands beside the sampler of one sequence (`Transformer.forward` at a temperature, jsgrad/models/llama.ts:131-185), which has a random stream of its own on the
device; `Transformer.forward_paged` takes a RowSampler for its batch.
"""
from __future__ import annotations

import numpy as np

from . import ffi
from .ffi import check
from .llama import act_code
from .tensor import Tensor


class RowSampler:
    """Settings of the rows of a batch: a number for all of them, or one for each.  min_p comes first, then top_k (0: all), then top_p; or,
    min_p_last, on what these two leave, whose mass then counts for top_p; a temperature of 0 is the greedy token."""

    def __init__(self, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, seed: int = 0, device: str = "HIP", min_p_last: bool = False):
        self.order = ffi.MIN_P_LAST if min_p_last else ffi.MIN_P_FIRST
        self.device, self.rng = device, np.random.default_rng(seed)
        self.settings = [np.atleast_1d(np.asarray(x, t)) for x, t in ((temperature, np.float32), (top_k, np.int32), (top_p, np.float32), (min_p, np.float32))]
        temperature, top_k, top_p, min_p = self.settings
        if any(x.ndim != 1 for x in self.settings) or len({x.size for x in self.settings if x.size != 1}) > 1 or any(x.size == 0 for x in self.settings):
            raise ValueError("settings of rows: one number, or as many as there are rows")
        if not (np.all(temperature >= 0) and np.all(np.isfinite(temperature)) and np.all(top_k >= 0) and np.all((top_p >= 0) & (top_p <= 1)) and np.all((min_p >= 0) & (min_p <= 1))):
            raise ValueError("a temperature and a top_k of 0 and more, top_p and min_p between 0 and 1")
        self.probs: Tensor | None = None                      # of the tokens last picked
        self._held: Tensor | None = None                      # temperature, top_k, top_p, min_p and uniforms of up to this many rows
        self._ws: Tensor | None = None
        self._rows = 0

    def check(self, rows: int) -> None:
        """Raises where the settings are not those of so many rows."""
        if rows < 1 or any(x.size not in (1, rows) for x in self.settings):
            raise ValueError(f"{rows} rows, settings of {max(x.size for x in self.settings)}")

    def pick(self, logits: Tensor, tokens_out: Tensor | None = None, rows: int | None = None) -> Tensor:
        """The next token of every row of logits [rows, n], float16 or float32, int32 [rows]; -1 where a row has nothing above minus infinity.  probs: the share that each had."""
        lib = ffi.load()
        if len(logits.shape) != 2 or logits.dtype not in ("float16", "float32"):
            raise ValueError(f"logits: float16 or float32 [rows, n] are wanted, got {logits.dtype} {logits.shape}")
        rows, n = logits.shape[0] if rows is None else rows, logits.shape[1]
        if rows > logits.shape[0]:
            raise ValueError(f"{rows} rows of {logits.shape[0]}")
        self.check(rows)
        tokens_out = Tensor.empty((rows,), "int32", self.device) if tokens_out is None else tokens_out
        if tokens_out.dtype != "int32" or tokens_out.numel < rows:
            raise ValueError(f"tokens_out: {rows} int32 are wanted, got {tokens_out.dtype} {tokens_out.shape}")
        if self._held is None or self._rows < rows:
            self._held, self._rows = Tensor.empty((6, rows), "int32", self.device), 0
        if self._rows != rows:                                # the settings stay, the numbers are new in every call
            self._rows = rows
            self._held.lazydata.view(4 * rows, "int32", 0).ensure_allocated().copyin(np.concatenate([np.broadcast_to(x, (rows,)).view(np.int32) for x in self.settings]))
        at = [self._held.ptr + 4 * rows * i for i in range(6)]
        self._held.lazydata.view(rows, "float32", 16 * rows).ensure_allocated().copyin(self.rng.random(rows, np.float32))
        need = lib.jsgrad_hip_sample_rows_workspace_bytes(rows, n)
        if self._ws is None or self._ws.nbytes < need:
            self._ws = Tensor.empty((need,), "uint8", self.device)
        check(lib.jsgrad_hip_sample_rows_ordered(logits.ptr, rows, n, n, act_code(logits.dtype), at[0], at[1], at[2], at[3], self.order, at[4], tokens_out.ptr, at[5], self._ws.ptr))
        self.probs = Tensor(buffer=self._held.lazydata.view(rows, "float32", 20 * rows), shape=(rows,), dtype="float32", device=self.device)
        return Tensor(buffer=tokens_out.lazydata if tokens_out.shape == (rows,) else tokens_out.lazydata.view(rows, "int32", 0), shape=(rows,), dtype="int32", device=self.device)
