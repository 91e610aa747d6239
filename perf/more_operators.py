"""What the speed of a serving step's further operators is measured on, beside those of `perf/operators.py`.

* `sample`: a token for every row of logits by temperature, top-k, top-p and min-p from given random numbers, and the probability that it had among those that
  were left (`jsgrad_hip_sample_rows`).
* `copy`: pages of all layers copied to other pages, where a prompt gets several answers or a pool is packed (`jsgrad_hip_paged_copy`).
* `norm`: the new rows of a ragged batch, q and k normed per head and rotated, and written into the pages (`jsgrad_hip_paged_write_norm`); int8 rows are read
  back as the values that the codes stand for (`jsgrad_hip_paged_read`).
* `sparse`: the bounds of the pages that the new rows touched, the pages that every row's queries choose by them, and attention over these
  (`jsgrad_hip_paged_bounds`, `jsgrad_hip_paged_select`, `jsgrad_hip_attn_selected`).

Head shapes are those of `denograd_amd.synthetic.CONFIGS`: 32 query and 8 kv heads, of 64 (1B) or 128 (8B), and a few others that the calls take;
vocabularies are theirs and generic ones.  A batch is described as in `perf/operators.py`: `seqs` sequences with `new` rows each and lengths that fall from
`length` by the share `ragged`.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False


def listed() -> list[dict]:
    return [
        # one conversation: the settings that a chat has, where only latency counts
        {"name": "sample-1x128256-f16", "kind": "sample", "rows": 1, "n": 128256, "act": "f16", "settings": "usual", "pad": 0},
        # a serving step's sixteen sequences, each with its caller's own settings, greedy ones among them
        {"name": "sample-16x128256-f16", "kind": "sample", "rows": 16, "n": 128256, "act": "f16", "settings": "mixed", "pad": 0},
        # a small odd vocabulary in float, rows inside wider ones, drawn from all of it
        {"name": "sample-37x50257-f32", "kind": "sample", "rows": 37, "n": 50257, "act": "f32", "settings": "whole", "pad": 7},
        # the largest: many answers sampled at once, from the smallest set that holds 95 % of the mass
        {"name": "sample-256x128256-f16", "kind": "sample", "rows": 256, "n": 128256, "act": "f16", "settings": "nucleus", "pad": 0},
        # three more answers to one prompt of the 1B model: the begun last page of each, in sixteen layers
        {"name": "copy-3x37-f16", "kind": "copy", "pages": "f16", "layers": 16, "kv": 8, "hd": 64, "page": 64, "pool": 64, "moves": 3, "held": 37},
        # the 8B model's pool packed after an hour of serving
        {"name": "copy-160-int8", "kind": "copy", "pages": "int8", "layers": 32, "kv": 8, "hd": 128, "page": 64, "pool": 352, "moves": 160, "held": 64},
        # one token of one conversation
        {"name": "norm-1x1-f16", "kind": "norm", "pages": "f16", "heads": 32, "kv": 8, "hd": 128, "page": 64, "seqs": 1, "new": 1, "length": 517, "ragged": 0.0},
        # the next message of sixteen conversations of different lengths
        {"name": "norm-16x57-int8", "kind": "norm", "pages": "int8", "heads": 32, "kv": 8, "hd": 64, "page": 32, "seqs": 16, "new": 57, "length": 1500, "ragged": 0.8},
        # sixteen long prompts at once
        {"name": "norm-16x2048-f16", "kind": "norm", "pages": "f16", "heads": 32, "kv": 8, "hd": 128, "page": 64, "seqs": 16, "new": 2048, "length": 2048, "ragged": 0.0},
        # one token behind a long document
        {"name": "sparse-1x1-33000-f16", "kind": "sparse", "pages": "f16", "heads": 32, "kv": 8, "hd": 128, "page": 64, "seqs": 1, "new": 1, "length": 33000, "ragged": 0.0,
         "first": 1, "recent": 2, "top": 32},
        # a step of sixteen long conversations of very different lengths
        {"name": "sparse-16x1-int8", "kind": "sparse", "pages": "int8", "heads": 32, "kv": 8, "hd": 128, "page": 32, "seqs": 16, "new": 1, "length": 32768, "ragged": 0.9,
         "first": 1, "recent": 4, "top": 64},
        # the largest: a part of a long document's prompt
        {"name": "sparse-1x2048-f16", "kind": "sparse", "pages": "f16", "heads": 32, "kv": 8, "hd": 64, "page": 64, "seqs": 1, "new": 2048, "length": 16384, "ragged": 0.0,
         "first": 1, "recent": 2, "top": 16},
    ]


def _log(rng, lo: int, hi: int) -> int:
    """A whole number between lo and hi, even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng) -> dict:
    most = {}
    for c in listed():
        w = work(c)
        most[c["kind"]] = [max(a, b) for a, b in zip(most.get(c["kind"], [0.0, 0.0]), (w["bytes"], w["flops"]))]
    while True:
        kind = rng.choice(["sample", "copy", "norm", "sparse", "sparse"])
        heads, kv = rng.choice([(32, 8), (32, 8), (16, 8), (12, 4), (16, 2), (8, 8), (64, 8)])
        pages, hd, page = rng.choice(["f16", "int8"]), rng.choice([64, 128]), rng.choice([16, 32, 64, 128, 256])
        if kind == "sample":
            case = {"kind": kind, "rows": _log(rng, 1, 256), "n": _log(rng, 600, 262144), "act": rng.choice(["f16", "f16", "f32"]),
                    "settings": rng.choice(["usual", "mixed", "mixed", "whole", "nucleus"]), "pad": rng.choice([0, 0, rng.randint(1, 300)])}
        elif kind == "copy":
            pool = _log(rng, 8, 700)
            case = {"kind": kind, "pages": pages, "layers": rng.choice([2, 16, 32]), "kv": kv, "hd": hd, "page": page, "pool": pool, "moves": _log(rng, 1, pool // 2),
                    "held": rng.choice([page, rng.randint(1, page)])}
            if _page_bytes(case) * case["layers"] * pool > 2e9:
                continue
        else:
            case = {"kind": kind, "pages": pages, "heads": heads, "kv": kv, "hd": hd, "page": page, "seqs": _log(rng, 1, 64), "ragged": rng.choice([0.0, rng.uniform(0.1, 0.9)])}
            case["new"] = rng.choice([1, _log(rng, 2, 2048)])
            case["length"] = case["new"] + rng.choice([0, _log(rng, 1, 32768 if kind == "sparse" else 8192)])
            if kind == "sparse":
                case["first"], case["recent"] = rng.choice([0, 1, 2]), rng.choice([1, 2, 4])
                case["top"] = case["first"] + case["recent"] + _log(rng, 1, 64)
                if case["top"] * page > 8192 or case["seqs"] * case["new"] > 4096:
                    continue
            if case["length"] * case["seqs"] > 300000:
                continue
        w = work(case)
        if w["bytes"] <= most[kind][0] and w["flops"] <= most[kind][1]:
            return case


# ---- the batch of a case

def _batch(case: dict) -> tuple[list[int], list[int]]:
    """New rows and length of every sequence, in an order that is not sorted."""
    n, top = case["seqs"], case["length"]
    news, lens = [case["new"]] * n, []
    for i in range(n):
        at = (i * 7) % n if n % 7 else i
        lens.append(max(news[i], int(top * (1.0 - case["ragged"] * at / max(1, n - 1))) if n > 1 else top))
    return news, lens


def _page_bytes(case: dict) -> float:
    """Bytes of a page of one layer: K and V and, of int8, their scales."""
    return 2.0 * case["kv"] * case["page"] * (case["hd"] * 2 if case["pages"] == "f16" else case["hd"] + 4)


def work(case: dict) -> dict:
    if case["kind"] == "sample":
        return {"bytes": float(case["rows"] * case["n"] * (2 if case["act"] == "f16" else 4) + 28 * case["rows"]), "flops": 2.0 * case["rows"] * case["n"]}
    if case["kind"] == "copy":
        return {"bytes": 2.0 * case["moves"] * case["layers"] * _page_bytes(case) * case["held"] / case["page"] + 12 * case["moves"], "flops": 0.0}
    H, KV, D, P = case["heads"], case["kv"], case["hd"], case["page"]
    news, lens = _batch(case)
    rows = sum(news)
    held = KV * (D if case["pages"] == "f16" else D / 2 + 2) * 2          # bytes of one position's K, or of its V
    plan = 4 * (2 * case["seqs"] + 1)
    if case["kind"] == "norm":
        # q, k and v in, q and the cache rows out, int8 ones once more in and out as fp16; cos and sin of every position
        back = 2 * held + 4 * KV * D if case["pages"] == "int8" else 0
        return {"bytes": rows * (2 * (H + 2 * KV) * D + 2 * H * D + 2 * held + back + 2 * D) + plan, "flops": rows * ((H + KV) * 7.0 * D)}
    total = float(rows * 4 * H * D + rows * KV * case["top"] * 4 + plan)
    flops = 0.0
    for n, l in zip(news, lens):
        pages = -(-l // P)
        touched = pages - (l - n) // P
        total += touched * (P * held + KV * (2 * D + 4)) + pages * KV * (2 * D + 4)
        # a sequence's positions are read once each, at most as many as its rows choose
        total += min(l, n * case["top"] * P) * 2 * held
        for p in (range(l - n, l) if n <= 64 else range(l - n, l, max(1, n // 64))):
            own_pages = p // P + 1
            keys = (p + 1) if own_pages <= case["top"] else (case["top"] - 1) * P + p % P + 1
            flops += (4.0 * D * H * keys + (4.0 * D * H * own_pages if own_pages > case["top"] else 0.0)) * (n / len(range(l - n, l, max(1, n // 64))) if n > 64 else 1.0)
    return {"bytes": total, "flops": flops}


def _rng(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed)


def _settings(case: dict, g: torch.Generator):
    """temperature, top_k, top_p and min_p of every row."""
    n = case["rows"]
    if case["settings"] == "usual":
        rows = [(0.7, 50, 0.9, 0.0)] * n
    elif case["settings"] == "whole":
        rows = [(1.0, 0, 1.0, 0.0)] * n
    elif case["settings"] == "nucleus":
        rows = [(0.8, 0, 0.95, 0.0)] * n
    else:
        pick = lambda values: [values[i] for i in torch.randint(len(values), (n,), generator=g, device="cuda").tolist()]
        rows = list(zip(pick([0.0, 0.3, 0.7, 1.0, 1.3]), pick([0, 1, 20, 50, 200, 1000]), pick([1.0, 0.95, 0.9, 0.5]), pick([0.0, 0.0, 0.02, 0.1])))
    f = lambda i, t: torch.tensor([r[i] for r in rows], dtype=t, device="cuda")
    return f(0, torch.float32), f(1, torch.int32), f(2, torch.float32), f(3, torch.float32)


def _rows(g, n: int, heads: int, hd: int, keys: bool) -> torch.Tensor:
    """Rows as a projection makes them: keys have a few channels that are several times as large as the others."""
    x = torch.randn(n, heads, hd, generator=g, device="cuda")
    if keys:
        x *= 1.0 + 3.0 * (torch.rand(heads, hd, generator=g, device="cuda") < 0.06)
    return x.half()


def _pool(g, n_pages: int, KV: int, P: int, D: int, keys: bool, int8: bool):
    """A pool of rows and, of int8, their scales."""
    x = _rows(g, n_pages * P, KV, D, keys).reshape(n_pages, P, KV, D).transpose(1, 2).contiguous()
    if not int8:
        return x, None
    scale = x.abs().amax(-1).float() / 127.0
    scale = torch.where(scale == 0, torch.ones_like(scale), scale)
    return torch.round(x.float() / scale[..., None]).to(torch.int8), scale


def prepare(case: dict, seed: int) -> dict:
    g = _rng(seed)
    s = {"case": dict(case)}
    if case["kind"] == "sample":
        rows, n = case["rows"], case["n"]
        # most of a vocabulary far below a few hundred entries that the model thinks of; a third of the rows with a grammar that forbids nine of ten
        x = 2.0 * torch.randn(rows, n + case["pad"], generator=g, device="cuda")
        x += (torch.rand(x.shape, generator=g, device="cuda") < 0.002) * 9.0 * torch.rand(x.shape, generator=g, device="cuda")
        x[2::3] = torch.where(torch.rand(x[2::3].shape, generator=g, device="cuda") < 0.9, -math.inf, x[2::3])
        s["logits"] = x.half() if case["act"] == "f16" else x
        s["temperature"], s["top_k"], s["top_p"], s["min_p"] = _settings(case, g)
        s["uniforms"] = torch.rand(rows, generator=g, device="cuda")
        s["tokens"], s["probs"] = torch.zeros(rows, dtype=torch.int32, device="cuda"), torch.zeros(rows, device="cuda")
        return s
    int8 = case["pages"] == "int8"
    if case["kind"] == "copy":
        L, KV, D, P, n = case["layers"], case["kv"], case["hd"], case["page"], case["pool"]
        # K and V of every layer, a pool each
        if int8:
            s["held"] = {"rows": torch.randint(-127, 128, (2 * L, n, KV, P, D), generator=g, device="cuda", dtype=torch.int8), "scales": torch.rand(2 * L, n, KV, P, generator=g, device="cuda") * 0.1}
        else:
            s["held"] = {"rows": torch.randn(2 * L, n, KV, P, D, generator=g, device="cuda", dtype=torch.float16)}
        s["pools"] = [pool for held in s["held"].values() for pool in held]
        order = torch.randperm(n, generator=g, device="cuda")[:2 * case["moves"]].int()
        s["moves"] = torch.stack([order[0::2], order[1::2], torch.full_like(order[0::2], case["held"])], 1).contiguous()
        return s
    H, KV, D, P = case["heads"], case["kv"], case["hd"], case["page"]
    news, lens = _batch(case)
    rows, most = sum(news), max(lens)
    held = [-(-l // P) for l in lens]
    width, n_pages = -(-most // P), sum(held) + 3
    # the pages of every sequence lie anywhere in the pool, as they do after an hour of serving; entries behind a sequence's end hold -1
    order = torch.randperm(n_pages, generator=g, device="cuda").int()
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(held):
        table[b, :n] = order[at:at + n]
        at += n
    starts = [0]
    for n in news:
        starts.append(starts[-1] + n)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    s.update(table=table, row_starts=i32(starts), lengths=i32(lens), rows=rows)
    if case["kind"] == "norm":
        s["pages_k"], s["pages_v"] = (torch.zeros(n_pages, KV, P, D, dtype=torch.int8 if int8 else torch.float16, device="cuda") for _ in range(2))
        s["scales_k"], s["scales_v"] = ((torch.ones(n_pages, KV, P, device="cuda") for _ in range(2)) if int8 else (None, None))
        s["q"], s["k"], s["v"] = _rows(g, rows, H, D, False), _rows(g, rows, KV, D, True), _rows(g, rows, KV, D, False)
        s["q_weight"], s["k_weight"] = ((1.0 + 0.3 * torch.randn(D, generator=g, device="cuda")).half() for _ in range(2))
        angle = torch.outer(torch.arange(width * P, device="cuda", dtype=torch.float64), 500000.0 ** (-torch.arange(0, D, 2, device="cuda", dtype=torch.float64) / D))
        s["rope"] = torch.stack([angle.cos(), angle.sin()], -1).half()
        s["q_out"], s["k_out"], s["v_out"] = torch.zeros_like(s["q"]), torch.zeros_like(s["k"]), torch.zeros_like(s["v"])
        return s
    s["pages_k"], s["scales_k"] = _pool(g, n_pages, KV, P, D, True, int8)
    s["pages_v"], s["scales_v"] = _pool(g, n_pages, KV, P, D, False, int8)
    s["q"] = _rows(g, rows, H, D, False)
    s["out"] = torch.zeros_like(s["q"])
    s["selected"] = torch.zeros(rows, KV, case["top"], dtype=torch.int32, device="cuda")
    # the pages that the new rows are on, and the bounds of all the others from the steps before
    touched = [(b, i) for b, (n, l) in enumerate(zip(news, lens)) for i in range((l - n) // P, -(-l // P))]
    s["touched"] = torch.tensor(touched, dtype=torch.long, device="cuda").reshape(-1, 2)
    every = [(b, i) for b, l in enumerate(lens) for i in range(-(-l // P))]
    s["bounds"] = torch.zeros(n_pages, KV, 2, D, dtype=torch.int8, device="cuda")
    s["bound_scales"] = torch.ones(n_pages, KV, device="cuda")
    every = torch.tensor(every, dtype=torch.long, device="cuda")
    for part in every.split(4096):
        _bounds(s, part)
    s["bounds"][table[s["touched"][:, 0], s["touched"][:, 1]].long()] = 0
    return s


# ---- the framework's calls

_WORKSPACE: dict = {}
EPS = 1e-5


def _workspace(key, nbytes: int):
    """One for every step of a server, or every layer of a model."""
    from denograd_amd.tensor import Tensor
    if key not in _WORKSPACE:
        _WORKSPACE[key] = Tensor.zeros((max(1, nbytes),), "uint8")
    return _WORKSPACE[key].ptr


def _own(s: dict):
    from denograd_amd import ffi
    from denograd_amd.device import Device
    from denograd_amd.ffi import check
    case, ptr = s["case"], (lambda t: None if t is None else t.data_ptr())
    lib = ffi.load()
    if "ready" not in s:
        Device.get("HIP").init()
        s["ready"] = True
        if case["kind"] == "copy":
            pools = []
            for t in s["pools"]:
                pools.append(ffi.Pool(ptr(t), case["kv"], case["page"], t.element_size() * (case["hd"] if t.dim() == 4 else 1)))
            s["host_pools"] = (ffi.Pool * len(pools))(*pools)
        elif case["kind"] != "sample":
            s["desc"] = ffi.PagesDesc(ffi.W_I8 if case["pages"] == "int8" else ffi.W_F16, s["pages_k"].shape[0], case["page"], case["kv"], case["hd"], s["table"].shape[1],
                                      ptr(s["pages_k"]), ptr(s["pages_v"]), ptr(s["scales_k"]), ptr(s["scales_v"]), ptr(s["table"]))
    if case["kind"] == "sample":
        ws = _workspace(("sample", case["rows"], case["n"]), lib.jsgrad_hip_sample_rows_workspace_bytes(case["rows"], case["n"]))
        check(lib.jsgrad_hip_sample_rows_ordered(ptr(s["logits"]), case["rows"], case["n"], case["n"] + case["pad"], ffi.F16 if case["act"] == "f16" else ffi.F32, ptr(s["temperature"]),
                                                 ptr(s["top_k"]), ptr(s["top_p"]), ptr(s["min_p"]), ffi.MIN_P_LAST, ptr(s["uniforms"]), ptr(s["tokens"]), ptr(s["probs"]), ws))
        return {"tokens": s["tokens"], "probs": s["probs"]}
    if case["kind"] == "copy":
        check(lib.jsgrad_hip_paged_copy(s["host_pools"], len(s["host_pools"]), case["pool"], ptr(s["moves"]), case["moves"]))
        return s["held"]
    batch = (s["desc"], ptr(s["row_starts"]), ptr(s["lengths"]), case["seqs"], s["rows"])
    if case["kind"] == "norm":
        check(lib.jsgrad_hip_paged_write_norm(*batch, ptr(s["q"]), ptr(s["k"]), ptr(s["v"]), ptr(s["q_weight"]), ptr(s["k_weight"]), EPS, ptr(s["rope"]), s["rope"].shape[0],
                                              ptr(s["q_out"]), case["heads"]))
        if case["pages"] == "f16":
            return {"q": s["q_out"], "k": s["pages_k"], "v": s["pages_v"]}
        check(lib.jsgrad_hip_paged_read(*batch, ptr(s["k_out"]), ptr(s["v_out"])))
        return {"q": s["q_out"], "k": s["k_out"], "v": s["v_out"]}
    H, KV, D = case["heads"], case["kv"], case["hd"]
    ws = _workspace(("attend", H, KV, D), lib.jsgrad_hip_attn_selected_workspace_bytes(H, KV, D))
    check(lib.jsgrad_hip_paged_bounds(*batch, ptr(s["bounds"]), ptr(s["bound_scales"])))
    check(lib.jsgrad_hip_paged_select(*batch, ptr(s["q"]), H, ptr(s["bounds"]), ptr(s["bound_scales"]), case["first"], case["recent"], case["top"], ptr(s["selected"])))
    check(lib.jsgrad_hip_attn_selected(*batch, ptr(s["q"]), ptr(s["out"]), H, ptr(s["selected"]), case["top"], ws))
    return {"bounds": s["bounds"], "scales": s["bound_scales"], "selected": s["selected"], "out": s["out"]}


# ---- the plain form

def _sample(s: dict) -> dict:
    """In 64 bits: a token changes where a sum's rounding reaches a border between two of 128256."""
    x = s["logits"][:, :s["case"]["n"]].double()
    x = torch.where(torch.isnan(x), -math.inf, x)
    col = lambda name: s[name].double().unsqueeze(1)
    top, order = torch.sort(x, dim=1, descending=True, stable=True)
    greedy = col("temperature") < 1e-6
    w = ((top - top[:, :1]) / torch.where(greedy, 1.0, col("temperature"))).exp()
    w = torch.where(top == top[:, :1], 1.0, w)
    rank = torch.arange(x.shape[1], device="cuda")
    k = s["top_k"].unsqueeze(1)
    w = torch.where((rank < k) | (k <= 0), w, 0.0)
    before = w.cumsum(1) - w
    keep = (before < col("top_p") * w.sum(1, keepdim=True)) | (rank == 0) | (col("top_p") >= 1.0)
    w = torch.where(keep & (w >= col("min_p").clamp(max=1.0)), w, 0.0)
    w = torch.zeros_like(w).scatter_(1, order, w)
    run = w.cumsum(1)
    drawn = (run > col("uniforms") * run[:, -1:]).to(torch.uint8).argmax(1)
    none = torch.isneginf(top[:, 0])
    s["tokens"].copy_(torch.where(none, -1, torch.where(greedy[:, 0], order[:, 0], drawn)))
    s["probs"].copy_(torch.where(none, 0.0, torch.where(greedy[:, 0], 1.0, w.gather(1, drawn[:, None])[:, 0] / run[:, -1])))
    return {"tokens": s["tokens"], "probs": s["probs"]}


def _places(s: dict):
    """(sequence, position) of every row of the batch, and the page and slot that hold it."""
    starts, lens = s["row_starts"].long(), s["lengths"].long()
    row = torch.arange(s["rows"], device="cuda")
    b = torch.searchsorted(starts, row, right=True) - 1
    pos = lens[b] - starts[b + 1] + row
    P = s["case"]["page"]
    return b, pos, s["table"][b, pos // P].long(), pos % P


def _gather(pages: torch.Tensor, scales, page: torch.Tensor, slot: torch.Tensor) -> torch.Tensor:
    """Rows [..., KV, HD] in 32 bits of the places given."""
    kv = torch.arange(pages.shape[1], device="cuda")
    x = pages[page[..., None], kv, slot[..., None]].float()
    return x if scales is None else x * scales[page[..., None], kv, slot[..., None]][..., None]


def _norm(s: dict):
    case = s["case"]
    _, pos, page, slot = _places(s)
    kv = torch.arange(case["kv"], device="cuda")
    c, n = s["rope"][pos][:, None].float().unbind(-1)

    def turned(x, weight):
        x = x.float()
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.float()
        e, o = x[..., 0::2], x[..., 1::2]
        return torch.stack([e * c - o * n, e * n + o * c], -1).reshape(x.shape)

    s["q_out"].copy_(turned(s["q"], s["q_weight"]))
    for name, x in (("k", turned(s["k"], s["k_weight"])), ("v", s["v"].float())):
        if case["pages"] == "int8":
            scale = x.abs().amax(-1) / 127.0
            scale = torch.where(scale == 0, torch.ones_like(scale), scale)
            s["scales_" + name][page[:, None], kv, slot[:, None]] = scale
            x = torch.round(x / scale[..., None])
        s["pages_" + name][page[:, None], kv, slot[:, None]] = x.to(s["pages_" + name].dtype)
    if case["pages"] == "f16":
        return {"q": s["q_out"], "k": s["pages_k"], "v": s["pages_v"]}
    for name in ("k", "v"):
        s[name + "_out"].copy_(_gather(s["pages_" + name], s["scales_" + name], page, slot))
    return {"q": s["q_out"], "k": s["k_out"], "v": s["v_out"]}


def _step(top: torch.Tensor) -> torch.Tensor:
    """The smallest power of two s with top <= 127 s; 1 where top is 0."""
    f, e = torch.frexp(top)                                   # top = f * 2^e, 1/2 <= f < 1
    return torch.where(top == 0, 1.0, torch.ldexp(torch.ones_like(top), e - 7 + (f > 127.0 / 128.0).int()))


def _bounds(s: dict, places: torch.Tensor) -> None:
    """Bounds of the keys of the pages at (sequence, page of it)."""
    b, i = places[:, 0], places[:, 1]
    P, ids = s["case"]["page"], s["table"][places[:, 0], places[:, 1]].long()
    k = s["pages_k"][ids].float()
    if s["scales_k"] is not None:
        k = k * s["scales_k"][ids][..., None]
    there = (i[:, None] * P + torch.arange(P, device="cuda") < s["lengths"].long()[b, None])[:, None, :, None]
    lo, hi = k.masked_fill(~there, math.inf).amin(2), k.masked_fill(~there, -math.inf).amax(2)
    step = _step(torch.maximum(lo.abs(), hi.abs()).amax(-1))
    s["bounds"][ids] = torch.stack([torch.floor(lo / step[..., None]), torch.ceil(hi / step[..., None])], 2).to(torch.int8)
    s["bound_scales"][ids] = step


def _sparse(s: dict):
    case = s["case"]
    H, KV, D, P, top = case["heads"], case["kv"], case["hd"], case["page"], case["top"]
    R, width = H // KV, s["table"].shape[1]
    for part in s["touched"].split(4096):
        _bounds(s, part)
    seq, pos, _, _ = _places(s)
    step = max(1, min(s["rows"], int(2.5e8 // max(width * KV * 2 * D, top * P * KV * D))))
    for r0 in range(0, s["rows"], step):
        r = slice(r0, min(s["rows"], r0 + step))
        n, p = pos[r].shape[0], pos[r]
        q = s["q"][r].float().reshape(n, KV, R, D)
        code = torch.round(q / _step(q.abs().amax((-1, -2)))[..., None, None])
        ids = s["table"][seq[r]].long()                       # [n, width]
        at = torch.arange(width, device="cuda")
        last = (p // P)[:, None]
        there = (ids >= 0) & (at <= last)
        held = s["bounds"][ids.clamp(min=0)].float()          # [n, width, KV, 2, D]
        # sums of whole numbers below 2^24 are exact in 32 bits; positive codes meet the upper bounds, negative ones the lower
        lo, hi = (held[:, :, :, i].permute(0, 2, 3, 1).contiguous() for i in (0, 1))
        score = (torch.matmul(code.clamp(min=0), hi) + torch.matmul(code.clamp(max=0), lo)).amax(2)
        score = score * s["bound_scales"][ids.clamp(min=0)].transpose(1, 2)
        always = (at < case["first"]) | (at > last - case["recent"])
        score = score.masked_fill(always[:, None], math.inf).masked_fill(~there[:, None], -math.inf)
        best = torch.sort(score, dim=-1, descending=True, stable=True)
        n_top = min(top, width)
        chosen = torch.where(torch.isneginf(best.values[..., :n_top]), width, best.indices[..., :n_top]).sort(-1).values
        s["selected"][r] = -1
        s["selected"][r, :, :n_top] = torch.where(chosen == width, -1, chosen).int()
        # their positions
        key = (chosen[..., None] * P + torch.arange(P, device="cuda")).reshape(n, KV, n_top * P)
        seen = (chosen < width)[..., None].expand(n, KV, n_top, P).reshape(key.shape) & (key <= p[:, None, None])
        page = ids.gather(1, chosen.clamp(max=width - 1).reshape(n, -1)).reshape(n, KV, n_top, 1).expand(n, KV, n_top, P).reshape(key.shape).clamp(min=0)
        kv = torch.arange(KV, device="cuda")[:, None]

        def rows(name):
            x = s["pages_" + name][page, kv, key % P].float()
            return x if s["scales_" + name] is None else x * s["scales_" + name][page, kv, key % P][..., None]

        x = torch.matmul(q, rows("k").transpose(-1, -2).contiguous()).mul_(1.0 / math.sqrt(D)).masked_fill_(~seen[:, :, None], -math.inf)
        x = x.sub_(x.amax(-1, keepdim=True).clamp(min=-3e38)).exp_()
        x = x.div_(x.sum(-1, keepdim=True).clamp(min=1e-37))
        s["out"][r] = torch.matmul(x, rows("v")).reshape(n, H, D).half()
    return {"bounds": s["bounds"], "scales": s["bound_scales"], "selected": s["selected"], "out": s["out"]}


def run(s: dict):
    if own:
        return _own(s)
    kind = s["case"]["kind"]
    if kind == "sample":
        return _sample(s)
    if kind == "norm":
        return _norm(s)
    if kind == "sparse":
        return _sparse(s)
    src, dst, held = s["moves"][:, 0].long(), s["moves"][:, 1].long(), s["case"]["held"]
    for pool in s["pools"]:
        pool[dst, :, :held] = pool[src, :, :held]
    return s["held"]


# ---- in 64 bits, row by row

def _exact_sample(s: dict) -> dict:
    out, probs = [], []
    x = s["logits"][:, :s["case"]["n"]].cpu().numpy().astype(np.float64)
    T, K, P, M, U = (s[n].cpu().numpy().astype(np.float64) for n in ("temperature", "top_k", "top_p", "min_p", "uniforms"))
    for r in range(x.shape[0]):
        v = np.where(np.isnan(x[r]), -np.inf, x[r])
        best = int(np.argmax(v))
        if v[best] == -np.inf or T[r] < 1e-6:
            out.append(-1 if v[best] == -np.inf else best)
            probs.append(0.0 if v[best] == -np.inf else 1.0)
            continue
        with np.errstate(invalid="ignore"):
            w = np.where(v == v[best], 1.0, np.exp((v - v[best]) / T[r]))
        order = np.argsort(-v, kind="stable")
        if K[r] > 0:
            order = order[:int(K[r])]
        if P[r] < 1.0:
            mass = np.cumsum(w[order])
            order = order[:1 + int(np.count_nonzero(mass[:-1] < P[r] * mass[-1]))]
        order = np.sort(order[w[order] >= min(M[r], 1.0)])
        run_ = np.cumsum(w[order])
        out.append(int(order[np.searchsorted(run_, U[r] * run_[-1], side="right")]))
        probs.append(w[out[-1]] / run_[-1])
    return {"tokens": torch.tensor(out, dtype=torch.int32, device="cuda"), "probs": torch.tensor(probs, dtype=torch.float64, device="cuda")}


def _exact_norm(s: dict, news, lens):
    pos = torch.cat([torch.arange(l - m, l, device="cuda") for m, l in zip(news, lens)])
    cos, sin = s["rope"][pos].double().unbind(-1)
    turn = torch.complex(cos, sin).unsqueeze(1)

    def turned(x, weight):
        x = x.double()
        x = x / (x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * weight.double()
        return torch.view_as_real(torch.view_as_complex(x.reshape(*x.shape[:-1], -1, 2).contiguous()) * turn).reshape(x.shape)

    out = {"q": turned(s["q"], s["q_weight"]), "k": turned(s["k"], s["k_weight"]), "v": s["v"].double()}
    if s["case"]["pages"] == "int8":
        for n in ("k", "v"):
            most = out[n].abs().amax(-1, keepdim=True).clamp(min=1e-300)
            out[n] = torch.round(out[n] * (127.0 / most)) * (most / 127.0)
        return out
    P = s["case"]["page"]
    for n in ("k", "v"):
        rows, out[n], at = out[n], s["pages_" + n].double(), 0
        for b, (m, l) in enumerate(zip(news, lens)):
            for p in range(l - m, l):
                if p == l - m or p % P == 0:
                    end = min(l, (p // P + 1) * P)
                    out[n][int(s["table"][b, p // P]), :, p % P:p % P + end - p] = rows[at:at + end - p].transpose(0, 1)
                    at += end - p
    return out


def _exact_sparse(s: dict, news, lens):
    case = s["case"]
    H, KV, D, P, top = case["heads"], case["kv"], case["hd"], case["page"], case["top"]
    bounds, scales = s["bounds"].clone(), s["bound_scales"].clone()
    selected, out = torch.full_like(s["selected"], -1), torch.zeros(s["rows"], H, D, dtype=torch.float64, device="cuda")
    table = s["table"].tolist()

    def values(name, ids):                                    # [KV, positions, D]; a row of int8 codes is the float product code * scale
        if s["scales_" + name] is None:
            return torch.cat([s["pages_" + name][i] for i in ids], 1).double()
        return torch.cat([s["pages_" + name][i].float() * s["scales_" + name][i][..., None] for i in ids], 1).double()

    def step_of(x):                                           # smallest power of two that 127 times is x and more
        e = torch.ceil(torch.log2((x / 127.0).clamp(min=1e-300)))
        e = torch.where(127.0 * torch.exp2(e - 1) >= x, e - 1, e)
        e = torch.where(127.0 * torch.exp2(e) < x, e + 1, e)
        return torch.where(x == 0, 1.0, torch.exp2(e))

    at = 0
    for b, (m, l) in enumerate(zip(news, lens)):
        n_pages = -(-l // P)
        ids = table[b][:n_pages]
        k, v = values("k", ids), values("v", ids)
        first_touched = (l - m) // P
        for i in range(first_touched, n_pages):
            mine = k[:, i * P:min(l, (i + 1) * P)]
            low, high = mine.min(1).values, mine.max(1).values
            st = step_of(torch.maximum(-low, high).amax(-1))
            bounds[ids[i], :, 0] = torch.floor(low / st[:, None]).to(torch.int8)
            bounds[ids[i], :, 1] = torch.ceil(high / st[:, None]).to(torch.int8)
            scales[ids[i]] = st.float()
        box, unit = torch.stack([bounds[i] for i in ids]).double(), torch.stack([scales[i] for i in ids]).double()     # [pages, KV, 2, D], [pages, KV]
        per = max(1, int(1.5e8 // (n_pages * D * H)))
        for r in range(0, m, per):
            rows = min(per, m - r)
            q = s["q"][at + r:at + r + rows].double().reshape(rows, KV, H // KV, D)
            code = torch.round(q / step_of(q.abs().amax((2, 3)))[..., None, None])
            p = torch.arange(l - m + r, l - m + r + rows, device="cuda")
            page = torch.arange(n_pages, device="cuda")
            for g in range(KV):
                c = code[:, g, :, None]                       # [rows, heads, 1, D]
                sc = torch.maximum(c * box[:, g, 0], c * box[:, g, 1]).sum(-1).amax(1) * unit[:, g]
                sc = torch.where((page < case["first"]) | (page > (p // P)[:, None] - case["recent"]), 1e300, sc)
                sc = torch.where(page > (p // P)[:, None], -1e300, sc)
                rank = torch.sort(-sc, dim=1, stable=True).indices
                place = torch.empty_like(rank).scatter_(1, rank, page.expand_as(rank).contiguous())
                chosen = (place < top) & (page <= (p // P)[:, None])
                slot = chosen.cumsum(1) - 1
                where = chosen.nonzero()
                selected[at + r + where[:, 0], g, slot[where[:, 0], where[:, 1]]] = where[:, 1].int()
                seen = chosen.repeat_interleave(P, 1)[:, :l] & (torch.arange(l, device="cuda") <= p[:, None])
                x = torch.matmul(q[:, g].reshape(-1, D), k[g, :l].t().contiguous()).reshape(rows, H // KV, l) / math.sqrt(D)
                x = torch.softmax(x.masked_fill(~seen[:, None], -math.inf), -1)
                out[at + r:at + r + rows, g * (H // KV):(g + 1) * (H // KV)] = torch.matmul(x.reshape(-1, l), v[g, :l]).reshape(rows, H // KV, D)
        at += m
    return {"bounds": bounds, "scales": scales, "selected": selected, "out": out}


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    if case["kind"] == "sample":
        return _exact_sample(s)
    if case["kind"] == "copy":
        out = {name: t.clone() for name, t in s["held"].items()}
        for a, b, n in s["moves"].tolist():
            for t in out.values():
                t[:, b, :, :n] = t[:, a, :, :n]
        return out
    news, lens = _batch(case)
    return _exact_norm(s, news, lens) if case["kind"] == "norm" else _exact_sparse(s, news, lens)
