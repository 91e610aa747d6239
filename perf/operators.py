"""What the speed of the paged KV cache is measured on: the three calls that a server makes of it per layer.

* `write`: the new rows of a ragged batch are rotated and written into the pages, in fp16 or quantised to int8, and what was written is read
  back (`jsgrad_hip_paged_write`, `jsgrad_hip_paged_read`): the rotated queries and the cache rows as the values that the codes stand for.
* `read`: whole sequences come out of the pages as contiguous rows (`jsgrad_hip_paged_read`).
* `attn`: the queries of a ragged batch over the pages, one new token per sequence or a chunk of them, over everything before them or over a
  sliding window and a few first tokens (`jsgrad_hip_attn_paged`).

A batch is described by `seqs` sequences with `new` rows each and lengths around `length`; `ragged` spreads the lengths (and with `chunk` the
first sequence alone has that many new rows, the others one: a prompt that joins a batch of running sequences).  Head shapes are those of
`denograd_amd.synthetic.CONFIGS`: 32 query and 8 kv heads, of 64 (1B) or 128 (8B), and a few others that the calls take.
"""
from __future__ import annotations

import math

import torch

own = False


def listed() -> list[dict]:
    return [
        # one conversation with the 1B model: one new token, where only latency counts
        {"name": "write-1x1-int8", "kind": "write", "pages": "int8", "heads": 32, "kv": 8, "hd": 64, "page": 64, "seqs": 1, "new": 1, "length": 517, "ragged": 0.0},
        # the next message of sixteen conversations of different lengths
        {"name": "write-16x57-f16", "kind": "write", "pages": "f16", "heads": 32, "kv": 8, "hd": 128, "page": 16, "seqs": 16, "new": 57, "length": 1500, "ragged": 0.8},
        # sixteen long prompts at once
        {"name": "write-16x2048-int8", "kind": "write", "pages": "int8", "heads": 32, "kv": 8, "hd": 128, "page": 64, "seqs": 16, "new": 2048, "length": 2048, "ragged": 0.0},
        # a prompt's cache rows taken out, to be kept for the next conversation that begins like it
        {"name": "read-1x371-f16", "kind": "read", "pages": "f16", "heads": 32, "kv": 8, "hd": 64, "page": 64, "seqs": 1, "new": 371, "length": 371, "ragged": 0.0},
        # sixteen sequences moved out of the way, as they are when a server runs out of pages
        {"name": "read-16x2304-int8", "kind": "read", "pages": "int8", "heads": 32, "kv": 8, "hd": 128, "page": 32, "seqs": 16, "new": 2304, "length": 2304, "ragged": 0.0},
        # one token of one conversation with the 1B model
        {"name": "attn-1x1-f16", "kind": "attn", "pages": "f16", "heads": 32, "kv": 8, "hd": 64, "page": 64, "seqs": 1, "new": 1, "length": 517, "ragged": 0.0, "window": 0, "sinks": 0},
        # a serving step of the 8B model: sixteen sequences of very different lengths
        {"name": "attn-16x1-int8", "kind": "attn", "pages": "int8", "heads": 32, "kv": 8, "hd": 128, "page": 64, "seqs": 16, "new": 1, "length": 4352, "ragged": 0.9, "window": 0, "sinks": 0},
        # three whole books in the context, one token each
        {"name": "attn-3x1-65000-f16", "kind": "attn", "pages": "f16", "heads": 32, "kv": 8, "hd": 128, "page": 128, "seqs": 3, "new": 1, "length": 65000, "ragged": 0.3, "window": 0, "sinks": 0},
        # the next message of a conversation
        {"name": "attn-1x57-f16", "kind": "attn", "pages": "f16", "heads": 32, "kv": 8, "hd": 128, "page": 16, "seqs": 1, "new": 57, "length": 1081, "ragged": 0.0, "window": 0, "sinks": 0},
        # a prompt that joins thirty running sequences
        {"name": "attn-512+30-int8", "kind": "attn", "pages": "int8", "heads": 32, "kv": 8, "hd": 128, "page": 64, "seqs": 31, "new": 1, "chunk": 512, "length": 2304, "ragged": 0.7, "window": 0, "sinks": 0},
        # a long document read with a window of 1024 and four first tokens
        {"name": "attn-1x8192-window-f16", "kind": "attn", "pages": "f16", "heads": 32, "kv": 8, "hd": 64, "page": 64, "seqs": 1, "new": 8192, "length": 8192, "ragged": 0.0, "window": 1024, "sinks": 4},
        # the largest: sixteen long prompts at once, over an int8 cache
        {"name": "attn-16x2048-int8", "kind": "attn", "pages": "int8", "heads": 32, "kv": 8, "hd": 128, "page": 64, "seqs": 16, "new": 2048, "length": 2048, "ragged": 0.0, "window": 0, "sinks": 0},
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
        kind = rng.choice(["write", "read", "attn", "attn", "attn"])
        heads, kv = rng.choice([(32, 8), (32, 8), (16, 8), (12, 4), (16, 2), (8, 8), (64, 8)])
        case = {"kind": kind, "pages": rng.choice(["f16", "int8"]), "heads": heads, "kv": kv, "hd": rng.choice([64, 128]), "page": rng.choice([16, 32, 64, 128, 256]),
                "seqs": _log(rng, 1, 64), "ragged": rng.choice([0.0, rng.uniform(0.1, 0.9)])}
        if kind == "attn":
            case["new"] = rng.choice([1, 1, _log(rng, 2, 4096)])
            case["length"] = case["new"] + rng.choice([0, _log(rng, 1, 32768)])
            if case["new"] == 1 and rng.random() < 0.25:
                case["chunk"] = min(case["length"], _log(rng, 16, 1024))
            case["window"] = rng.choice([0, 0, _log(rng, 1, 4096)])
            case["sinks"] = rng.choice([0, 4, rng.randint(1, 130)]) if case["window"] else 0
        elif kind == "write":
            case["new"] = rng.choice([1, _log(rng, 2, 2048)])
            case["length"] = case["new"] + rng.choice([0, _log(rng, 1, 8192)])
        else:
            case["length"] = case["new"] = _log(rng, 1, 4096)
        if case["length"] * case["seqs"] > 300000:
            continue
        if _plain_values(case) > 2.2e9:                       # scores of the plain form, which fills the batch up to its longest
            continue
        w = work(case)
        if w["bytes"] <= most[kind][0] and w["flops"] <= most[kind][1]:
            return case


# ---- the batch of a case

def _batch(case: dict) -> tuple[list[int], list[int]]:
    """New rows and length of every sequence: lengths fall evenly from `length` by the share `ragged`, in an order that is not sorted."""
    n, top = case["seqs"], case["length"]
    news = [case["new"]] * n
    if "chunk" in case:
        news[0] = case["chunk"]
    lens = []
    for i in range(n):
        at = (i * 7) % n if n % 7 else i
        lens.append(max(news[i], int(top * (1.0 - case["ragged"] * at / max(1, n - 1))) if n > 1 else top))
    return news, lens


def _plain_values(case: dict) -> float:
    news, lens = _batch(case)
    return float(case["seqs"]) * case["heads"] * max(news) * max(lens) if case["kind"] == "attn" else 0.0


def _seen(case: dict, new: int, length: int) -> tuple[int, int]:
    """(visible pairs of a row and a key, keys that some row sees) of one sequence and one head."""
    w, s = case["window"], case["sinks"]
    first = length - new
    if not w:
        return (first + 1 + length) * new // 2, length
    pairs = 0
    for p in range(first, length):
        lo = max(0, p - w + 1)
        pairs += p + 1 - lo + min(s, lo)
    lo = max(0, first - w + 1)
    return pairs, length - lo + min(s, lo)


def work(case: dict) -> dict:
    H, KV, D = case["heads"], case["kv"], case["hd"]
    news, lens = _batch(case)
    rows = sum(news)
    held = KV * (D if case["pages"] == "f16" else D / 2 + 2) * 2          # bytes of one position's K, or of its V
    plan = 4 * (2 * case["seqs"] + 1)
    if case["kind"] == "write":
        # q, k and v in, q and the cache rows out, and those once more in and out as fp16; cos and sin of every position
        return {"bytes": rows * (2 * (H + 2 * KV) * D + 2 * H * D + 4 * held + 4 * KV * D + 2 * D) + plan, "flops": 3.0 * rows * (H + KV) * D}
    if case["kind"] == "read":
        return {"bytes": rows * (2 * held + 4 * KV * D) + plan, "flops": float(rows * 2 * KV * D)}
    seen = [_seen(case, n, l) for n, l in zip(news, lens)]
    return {"bytes": rows * 4 * H * D + sum(k for _, k in seen) * 2 * held + plan, "flops": 4.0 * D * H * sum(p for p, _ in seen)}


def _rng(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed)


def _rows(g, n: int, heads: int, hd: int, keys: bool) -> torch.Tensor:
    """Rows as a projection makes them: keys have a few channels that are several times as large as the others."""
    x = torch.randn(n, heads, hd, generator=g, device="cuda")
    if keys:
        x *= 1.0 + 3.0 * (torch.rand(heads, hd, generator=g, device="cuda") < 0.06)
    return x.half()


def prepare(case: dict, seed: int) -> dict:
    g = _rng(seed)
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
    int8 = case["pages"] == "int8"
    s = {"case": dict(case), "table": table, "row_starts": i32(starts), "lengths": i32(lens), "rows": rows, "most": most, "most_new": max(news)}
    if case["kind"] == "write":
        s["pages_k"], s["pages_v"] = (torch.zeros(n_pages, KV, P, D, dtype=torch.int8 if int8 else torch.float16, device="cuda") for _ in range(2))
        s["scales_k"], s["scales_v"] = ((torch.ones(n_pages, KV, P, device="cuda") for _ in range(2)) if int8 else (None, None))
        s["q"], s["k"], s["v"] = _rows(g, rows, H, D, False), _rows(g, rows, KV, D, True), _rows(g, rows, KV, D, False)
        angle = torch.outer(torch.arange(width * P, device="cuda", dtype=torch.float64), 500000.0 ** (-torch.arange(0, D, 2, device="cuda", dtype=torch.float64) / D))
        s["rope"] = torch.stack([angle.cos(), angle.sin()], -1).half()
        s["q_out"], s["k_out"], s["v_out"] = torch.zeros_like(s["q"]), torch.zeros_like(s["k"]), torch.zeros_like(s["v"])
        return s
    for name in ("k", "v"):
        x = _rows(g, n_pages * P, KV, D, name == "k").reshape(n_pages, P, KV, D).transpose(1, 2).contiguous()
        s["scales_" + name] = None
        if int8:
            scale = x.abs().amax(-1).float() / 127.0
            s["scales_" + name] = torch.where(scale == 0, torch.ones_like(scale), scale)
            x = torch.round(x.float() / s["scales_" + name][..., None]).to(torch.int8)
        s["pages_" + name] = x
    if case["kind"] == "attn":
        s["q"] = _rows(g, rows, H, D, False)
        s["out"] = torch.zeros_like(s["q"])
    else:
        s["k_out"], s["v_out"] = (torch.zeros(rows, KV, D, dtype=torch.float16, device="cuda") for _ in range(2))
    return s


# ---- the framework's calls

_WORKSPACE: dict = {}


def _own(s: dict):
    from denograd_amd import ffi
    from denograd_amd.device import Device
    from denograd_amd.ffi import check
    from denograd_amd.tensor import Tensor
    case, ptr = s["case"], (lambda t: None if t is None else t.data_ptr())
    lib = ffi.load()
    if "desc" not in s:
        Device.get("HIP").init()
        s["desc"] = ffi.PagesDesc(ffi.W_I8 if case["pages"] == "int8" else ffi.W_F16, s["pages_k"].shape[0], case["page"], case["kv"], case["hd"], s["table"].shape[1],
                                  ptr(s["pages_k"]), ptr(s["pages_v"]), ptr(s["scales_k"]), ptr(s["scales_v"]), ptr(s["table"]))
    batch = (s["desc"], ptr(s["row_starts"]), ptr(s["lengths"]), case["seqs"], s["rows"])
    if case["kind"] == "attn":
        shape = (case["heads"], case["kv"], case["hd"])
        if shape not in _WORKSPACE:                           # one for every layer of a model
            _WORKSPACE[shape] = Tensor.zeros((lib.jsgrad_hip_attn_paged_workspace_bytes(*shape),), "uint8")
        check(lib.jsgrad_hip_attn_paged(*batch, ptr(s["q"]), ptr(s["out"]), case["heads"], case["window"], case["sinks"], _WORKSPACE[shape].ptr))
        return s["out"]
    if case["kind"] == "write":
        check(lib.jsgrad_hip_paged_write(*batch, ptr(s["q"]), ptr(s["k"]), ptr(s["v"]), ptr(s["rope"]), s["rope"].shape[0], ptr(s["q_out"]), case["heads"]))
    check(lib.jsgrad_hip_paged_read(*batch, ptr(s["k_out"]), ptr(s["v_out"])))
    return {"q": s["q_out"], "k": s["k_out"], "v": s["v_out"]} if case["kind"] == "write" else {"k": s["k_out"], "v": s["v_out"]}


# ---- the plain form

def _places(s: dict):
    """(sequence, position) of every row of the batch, and the page and slot that hold it."""
    starts, lens = s["row_starts"].long(), s["lengths"].long()
    row = torch.arange(s["rows"], device="cuda")
    b = torch.searchsorted(starts, row, right=True) - 1
    pos = lens[b] - starts[b + 1] + row
    P = s["case"]["page"]
    return b, pos, s["table"][b, pos // P].long(), pos % P


def _rotate(x: torch.Tensor, cs: torch.Tensor) -> torch.Tensor:
    x, c, n = x.float(), cs[:, None, :, 0].float(), cs[:, None, :, 1].float()
    e, o = x[..., 0::2], x[..., 1::2]
    return torch.stack([e * c - o * n, e * n + o * c], -1).reshape(x.shape)


def _gather(pages: torch.Tensor, scales, page: torch.Tensor, slot: torch.Tensor) -> torch.Tensor:
    """Rows [..., KV, HD] in 32 bits of the places given."""
    kv = torch.arange(pages.shape[1], device="cuda")
    x = pages[page[..., None], kv, slot[..., None]].float()
    return x if scales is None else x * scales[page[..., None], kv, slot[..., None]][..., None]


def run(s: dict):
    if own:
        return _own(s)
    case = s["case"]
    if case["kind"] == "write":
        _, pos, page, slot = _places(s)
        kv = torch.arange(case["kv"], device="cuda")
        cs = s["rope"][pos]
        s["q_out"].copy_(_rotate(s["q"], cs))
        for name, x in (("k", _rotate(s["k"], cs)), ("v", s["v"].float())):
            if case["pages"] == "int8":
                scale = x.abs().amax(-1) / 127.0
                scale = torch.where(scale == 0, torch.ones_like(scale), scale)
                s["scales_" + name][page[:, None], kv, slot[:, None]] = scale
                x = torch.round(x / scale[..., None])
            s["pages_" + name][page[:, None], kv, slot[:, None]] = x.to(s["pages_" + name].dtype)
    if case["kind"] != "attn":
        _, _, page, slot = _places(s)
        for name in ("k", "v"):
            s[name + "_out"].copy_(_gather(s["pages_" + name], s["scales_" + name], page, slot))
        return {"q": s["q_out"], "k": s["k_out"], "v": s["v_out"]} if case["kind"] == "write" else {"k": s["k_out"], "v": s["v_out"]}

    # the batch filled up to its longest sequence and its most new rows
    B, H, KV, D, P, L, N = case["seqs"], case["heads"], case["kv"], case["hd"], case["page"], s["most"], s["most_new"]
    b, pos, _, _ = _places(s)
    at = torch.arange(s["rows"], device="cuda") - s["row_starts"].long()[b]
    q = torch.zeros(B, N, H, D, device="cuda")
    q[b, at] = s["q"].float()
    p_q = torch.full((B, N), -1, dtype=torch.long, device="cuda")
    p_q[b, at] = pos
    j = torch.arange(L, device="cuda")
    page = s["table"].long().clamp(min=0)[:, j // P]
    k = _gather(s["pages_k"], s["scales_k"], page, (j % P).expand(B, L)).permute(0, 2, 3, 1).contiguous()      # [B, KV, HD, L]
    v = _gather(s["pages_v"], s["scales_v"], page, (j % P).expand(B, L)).permute(0, 2, 1, 3).contiguous()      # [B, KV, L, HD]
    q = q.reshape(B, N, KV, H // KV, D).permute(0, 2, 3, 1, 4).reshape(B, KV, H // KV * N, D)
    seen = j <= p_q[..., None]
    if case["window"]:
        seen = seen & ((j > p_q[..., None] - case["window"]) | (j < case["sinks"]))
    x = torch.matmul(q, k).reshape(B, KV, H // KV, N, L).mul_(1.0 / math.sqrt(D)).masked_fill_(~seen[:, None, None], -math.inf)
    x = x.sub_(x.amax(-1, keepdim=True).clamp(min=-3e38)).exp_()
    x = x.div_(x.sum(-1, keepdim=True).clamp(min=1e-37))
    o = torch.matmul(x.reshape(B, KV, H // KV * N, L), v).reshape(B, H, N, D)
    s["out"].copy_(o[b, :, at])
    return s["out"]


# ---- in 64 bits, sequence by sequence

def _rows_of(s: dict, name: str, b: int, lo: int, hi: int) -> torch.Tensor:
    """Positions [lo, hi) of sequence b as [KV, positions, HD]."""
    P = s["case"]["page"]
    first = lo // P
    ids = s["table"][b, first:-(-hi // P)].tolist()
    x = torch.cat([s["pages_" + name][i] for i in ids], 1).double()
    if s["scales_" + name] is not None:
        x = x * torch.cat([s["scales_" + name][i] for i in ids], 1).double().unsqueeze(-1)
    return x[:, lo - first * P:hi - first * P]


def _turned(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    z = torch.view_as_complex(x.double().reshape(*x.shape[:-1], -1, 2).contiguous()) * torch.complex(cos, sin).unsqueeze(1)
    return torch.view_as_real(z).reshape(x.shape)


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    news, lens = _batch(case)
    H, KV, D = case["heads"], case["kv"], case["hd"]
    if case["kind"] == "read":
        return {n: torch.cat([_rows_of(s, n, b, l - m, l).transpose(0, 1) for b, (m, l) in enumerate(zip(news, lens))]) for n in ("k", "v")}
    if case["kind"] == "write":
        pos = torch.cat([torch.arange(l - m, l, device="cuda") for m, l in zip(news, lens)])
        cos, sin = s["rope"][pos].double().unbind(-1)
        out = {"q": _turned(s["q"], cos, sin), "k": _turned(s["k"], cos, sin), "v": s["v"].double()}
        if case["pages"] == "int8":
            for n in ("k", "v"):
                top = out[n].abs().amax(-1, keepdim=True).clamp(min=1e-300)
                out[n] = torch.round(out[n] * (127.0 / top)) * (top / 127.0)
        return out
    out, at = [], 0
    for b, (m, l) in enumerate(zip(news, lens)):
        k, v = _rows_of(s, "k", b, 0, l), _rows_of(s, "v", b, 0, l)
        q = s["q"][at:at + m].double().transpose(0, 1)         # [H, rows, HD]
        at += m
        per = max(1, int(2e8 // (H // KV * l)))               # rows at a time
        o = torch.empty(H, m, D, dtype=torch.float64, device="cuda")
        for g in range(KV):
            for r in range(0, m, per):
                mine = q[g * (H // KV):(g + 1) * (H // KV), r:r + per]
                p = torch.arange(l - m + r, l - m + r + mine.shape[1], device="cuda").unsqueeze(1)
                j = torch.arange(l, device="cuda")
                hidden = j > p
                if case["window"]:
                    hidden |= (j <= p - case["window"]) & (j >= case["sinks"])
                x = (mine.reshape(-1, D) @ k[g].t().contiguous()).reshape(H // KV, -1, l) / math.sqrt(D)
                w = torch.softmax(x.masked_fill(hidden, -math.inf), -1)
                o[g * (H // KV):(g + 1) * (H // KV), r:r + per] = (w.reshape(-1, l) @ v[g]).reshape(H // KV, -1, D)
        out.append(o.transpose(0, 1))
    return torch.cat(out)
