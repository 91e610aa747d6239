"""The operators of the paged cache in float64 numpy, written from their definition, and batches for them."""
import numpy as np

from denograd_amd import ffi
from denograd_amd.tensor import Tensor

U16 = 2.0 ** -11      # half a step of fp16, relative
U32 = 2.0 ** -24


def quantise(x):
    """(codes, scales) of rows [..., HD] as the header defines them, in float32."""
    x = np.asarray(x, np.float32)
    with np.errstate(invalid="ignore"):
        top = np.abs(x).max(-1)
        scale = np.where(top == 0, np.float32(1), top / np.float32(127)).astype(np.float32)
        bad = ~np.isfinite(x).all(-1)
        codes = np.where(bad[..., None], 0, np.rint(x / scale[..., None])).astype(np.int8)
    return codes, np.where(bad, np.float32(np.nan), scale)


class Case:
    """Pools with random rows, a page table in random order, and a batch: news[i] new rows of a sequence of lens[i] positions."""

    def __init__(self, rng, kind, hd, KV, page, news, lens, spare=2, k=None, v=None, extra_rows=0):
        self.kind, self.hd, self.KV, self.page, self.news, self.lens = kind, hd, KV, page, list(news), list(lens)
        held = [-(-max(0, l) // page) for l in lens]
        self.n_pages, self.width = sum(held) + spare, max(1, max(held))
        order = rng.permutation(self.n_pages).astype(np.int32)
        self.table, at = np.full((len(lens), self.width), -1, np.int32), 0
        for b, n in enumerate(held):
            self.table[b, :n] = order[at:at + n]
            at += n
        shape = (self.n_pages, KV, page, hd)
        self.k = rng.standard_normal(shape).astype(np.float16) if k is None else k
        self.v = rng.standard_normal(shape).astype(np.float16) if v is None else v
        self.starts = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
        self.rows = int(self.starts[-1]) + extra_rows
        if kind == "int8":
            (self.ck, self.sk), (self.cv, self.sv) = quantise(self.k), quantise(self.v)

    def device(self):
        """Uploads; self.desc is what the calls take."""
        i8 = self.kind == "int8"
        self.t = {"k": Tensor(self.ck if i8 else self.k), "v": Tensor(self.cv if i8 else self.v), "table": Tensor(self.table), "starts": Tensor(self.starts),
                  "lens": Tensor(np.array(self.lens, np.int32))}
        if i8:
            self.t["sk"], self.t["sv"] = Tensor(self.sk), Tensor(self.sv)
        p = lambda n: self.t[n].ptr if n in self.t else None
        self.desc = ffi.PagesDesc(ffi.W_I8 if i8 else ffi.W_F16, self.n_pages, self.page, self.KV, self.hd, self.table.shape[1], p("k"), p("v"), p("sk"), p("sv"), p("table"))
        return self

    @property
    def batch(self):
        return self.desc, self.t["starts"].ptr, self.t["lens"].ptr, len(self.lens), self.rows

    def values(self, name):
        """The pool in float64, as the attention counts it."""
        if self.kind == "int8":
            c, s = (self.ck, self.sk) if name == "k" else (self.cv, self.sv)
            return c.astype(np.float64) * s.astype(np.float64)[..., None]
        return getattr(self, name).astype(np.float64)

    def places(self, b, lo, hi):
        """Pages and slots of positions [lo, hi); page -1 where there is none."""
        pos = np.arange(lo, hi)
        col = pos // self.page
        ok = (pos >= 0) & (col < self.table.shape[1])
        ids = np.where(ok, self.table[b, np.clip(col, 0, self.table.shape[1] - 1)], -1)
        return np.where((ids >= 0) & (ids < self.n_pages), ids, -1), pos % self.page


def attention(case: Case, q, H, window=0, sinks=0):
    """(result, bound) of attn_paged on q [rows, H, hd], float64, rows in the order of the batch.

    Bound of one element: the result's rounding U16 |out|; the rounding of the weights to fp16 for the matrix unit, each off by U16 of itself, so U16 A with A = sum
    w |V|, and by 2^-25 of the largest where it is below the normal numbers, so 2^-25 n max |V|; scores as float sums of hd products, times
    scales, into an exponential: each weight is off by 2 E relative, with E = U32 (hd S + 8 max |s| + 16) and S = max sum |q k| / sqrt(hd), so 2 E A for the
    weights and as much for their sum; float sums over n keys: U32 n A."""
    k, v = case.values("k"), case.values("v")
    out, tol = np.zeros((case.rows, H, case.hd)), np.zeros((case.rows, H, case.hd))
    rep = H // case.KV
    for b, (n, l) in enumerate(zip(case.news, case.lens)):
        ids, slots = case.places(b, 0, max(l, 0))
        for i in range(n):
            p = l - n + i
            j = np.arange(max(0, min(p + 1, l)))
            seen = ids[j] >= 0
            if window:
                seen &= (j > p - window) | (j < sinks)
            j = j[seen]
            if not j.size:
                continue
            r = case.starts[b] + i
            kk, vv = k[ids[j], :, slots[j]], v[ids[j], :, slots[j]]               # [keys, KV, hd]
            for h in range(H):
                g = h // rep
                x = q[r, h].astype(np.float64)
                with np.errstate(invalid="ignore", over="ignore"):
                    s = kk[:, g] @ x / np.sqrt(case.hd)
                    w = np.exp(s - s.max())
                    w /= w.sum()
                    out[r, h] = w @ vv[:, g]
                    A = w @ np.abs(vv[:, g])
                    E = U32 * (case.hd * (np.abs(kk[:, g]) @ np.abs(x)).max() / np.sqrt(case.hd) + 8 * np.abs(s).max() + 16)
                    tol[r, h] = U16 * np.abs(out[r, h]) + (U16 + 4 * E + U32 * j.size) * A + 2.0 ** -25 * (j.size * np.abs(vv[:, g]).max(0) + 1)
    return out, tol
