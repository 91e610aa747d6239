"""Bounds of pages, the pages that rows choose by them, and attention over these, in numpy from their definitions."""
import numpy as np

from tests.paged_ref import U16, U32


def step(most):
    """The smallest power of two, 2^-126 and more, that 127 times is `most` and more; 1 for 0."""
    most = np.asarray(most, np.float64)
    e = np.ceil(np.log2(np.where(most > 0, most, 1) / 127))
    e = np.where(127 * 2.0 ** (e - 1) >= most, e - 1, e)
    e = np.where(127 * 2.0 ** e < most, e + 1, e)
    return np.where(most == 0, 1.0, 2.0 ** np.maximum(e, -126))


def pool_keys(case):
    """The K pool as the bounds count it: int8 ones as float products."""
    if case.kind == "int8":
        with np.errstate(invalid="ignore", over="ignore"):
            return (case.ck.astype(np.float32) * case.sk[..., None]).astype(np.float64)
    return case.k.astype(np.float64)


def bounds(case, codes, scales):
    """The arrays [n_pages, KV, 2, hd] and [n_pages, KV] behind the call."""
    codes, scales, k = codes.copy(), scales.copy(), pool_keys(case)
    for b, (n, l) in enumerate(zip(case.news, case.lens)):
        for i in sorted({p // case.page for p in range(max(0, l - n), l)}):
            (at,), _ = case.places(b, i * case.page, i * case.page + 1)
            if at < 0:
                continue
            rows = k[at, :, :min(case.page, l - i * case.page)]
            for g in range(case.KV):
                if not np.isfinite(rows[g]).all():
                    codes[at, g], scales[at, g] = 0, np.inf
                    continue
                lo, hi = rows[g].min(0), rows[g].max(0)
                s = step(np.maximum(np.abs(lo), np.abs(hi)).max())
                codes[at, g, 0], codes[at, g, 1], scales[at, g] = np.floor(lo / s), np.ceil(hi / s), s
    return codes, scales


def choose(case, q, H, codes, scales, first, recent, top, before):
    """selected [rows, KV, top]; rows that belong to no sequence as in `before`."""
    out, rep = before.copy(), H // case.KV
    for b, (n, l) in enumerate(zip(case.news, case.lens)):
        for i in range(n):
            p, r = l - n + i, case.starts[b] + i
            last = p // case.page
            pages = np.arange(min(last + 1, case.table.shape[1])) if p >= 0 else np.arange(0)
            ids, _ = case.places(b, 0, pages.size * case.page) if pages.size else (np.zeros(0, int), None)
            ids = ids[::case.page]
            for g in range(case.KV):
                x = q[r, g * rep:(g + 1) * rep].astype(np.float64)
                c = np.rint(x / step(np.abs(x).max())) if np.isfinite(x).all() else np.zeros_like(x)
                score = []
                for at, col in zip(ids, pages):
                    if at < 0:
                        score.append(None)
                    elif col < first or col > last - recent or scales[at, g] == np.inf:
                        score.append((0 if col < first or col > last - recent else 1, 0.0))
                    else:
                        box = codes[at, g].astype(np.float64)
                        score.append((2, -(np.where(c > 0, c * box[1], c * box[0]).sum(-1).max() * float(scales[at, g]))))
                order = sorted((s, int(col)) for s, col in zip(score, pages) if s is not None)[:top]
                mine = sorted(col for _, col in order)
                out[r, g] = mine + [-1] * (top - len(mine))
    return out


def choose_many(case, q, H, codes, scales, first, recent, top, before):
    """choose() for many rows at once, each sequence's as one array."""
    out, rep = before.copy(), H // case.KV
    for b, (n, l) in enumerate(zip(case.news, case.lens)):
        if not n:
            continue
        rows, cols = slice(case.starts[b], case.starts[b] + n), np.arange(case.table.shape[1])
        last = np.arange(l - n, l) // case.page
        ids, _ = case.places(b, 0, cols.size * case.page)
        ids = ids[::case.page]
        for g in range(case.KV):
            x = q[rows, g * rep:(g + 1) * rep].astype(np.float64)
            top_of = np.abs(x).max((1, 2))
            fine = np.isfinite(top_of)
            c = np.where(fine[:, None, None], np.rint(x / step(np.where(fine, top_of, 0))[:, None, None]), 0.0)
            lo, hi = (codes[np.maximum(ids, 0), g, i].astype(np.float64) for i in range(2))
            scale = scales[np.maximum(ids, 0), g].astype(np.float64)
            always = (cols < first) | (cols > last[:, None] - recent)
            with np.errstate(invalid="ignore"):
                score = (np.maximum(c, 0) @ hi.T + np.minimum(c, 0) @ lo.T).max(1) * scale
            rank = np.where(always, 0, np.where(np.isinf(scale), 1, 2))
            score = np.where(rank == 2, score, 0.0)
            rank = np.where((ids < 0) | (cols > last[:, None]), 3, rank)
            order = np.lexsort((np.broadcast_to(cols, rank.shape), -score, rank))[:, :top]
            mine = np.sort(np.where(np.take_along_axis(rank, order, 1) < 3, order, 1 << 30), 1)
            out[rows, g] = -1
            out[rows, g, :mine.shape[1]] = np.where(mine < 1 << 30, mine, -1)
    return out


def attention(case, q, H, selected, every=1):
    """(result, bound) as tests.paged_ref.attention has them, over the positions of the chosen pages; of each `every`-th row of a sequence alone, where that is more than 1."""
    k, v = case.values("k"), case.values("v")
    out, tol = np.zeros((case.rows, H, case.hd)), np.zeros((case.rows, H, case.hd))
    rep = H // case.KV
    for b, (n, l) in enumerate(zip(case.news, case.lens)):
        for i in range(0, n, every):
            p, r = l - n + i, case.starts[b] + i
            for g in range(case.KV):
                j = np.concatenate([np.arange(c * case.page, (c + 1) * case.page) for c in selected[r, g] if 0 <= c < case.table.shape[1]] + [np.zeros(0, int)]).astype(int)
                j = j[j <= p]
                ids, slots = np.zeros(0, int), np.zeros(0, int)
                if j.size:
                    ids = case.table[b, j // case.page]
                    j, ids = j[(ids >= 0) & (ids < case.n_pages)], ids[(ids >= 0) & (ids < case.n_pages)]
                    slots = j % case.page
                if not j.size:
                    continue
                kk, vv = k[ids, g, slots], v[ids, g, slots]
                for h in range(g * rep, (g + 1) * rep):
                    x = q[r, h].astype(np.float64)
                    with np.errstate(invalid="ignore", over="ignore"):
                        s = kk @ x / np.sqrt(case.hd)
                        w = np.exp(s - s.max())
                        w /= w.sum()
                        out[r, h] = w @ vv
                        A = w @ np.abs(vv)
                        E = U32 * (case.hd * (np.abs(kk) @ np.abs(x)).max() / np.sqrt(case.hd) + 8 * np.abs(s).max() + 16)
                        tol[r, h] = U16 * np.abs(out[r, h]) + (U16 + 4 * E + U32 * j.size) * A + 2.0 ** -25 * (j.size * np.abs(vv).max(0) + 1)
    return out, tol
