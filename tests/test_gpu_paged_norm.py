"""Rows written into pages behind a norm of queries and keys per head, against float64, and models that have such norms."""
import numpy as np
import pytest

from denograd_amd import synthetic
from denograd_amd.ffi import check
from denograd_amd.llama import convert_from_huggingface
from denograd_amd.llama3 import Llama3
from denograd_amd.paged import PagedCache
from denograd_amd.tensor import Tensor
from tests.paged_ref import U16, U32, Case
from tests.test_gpu_paged import rope_table

pytestmark = pytest.mark.gpu
EPS = 1e-5


def normed(x, w, eps=EPS):
    x = x.astype(np.float64)
    return x / np.sqrt((x * x).sum(-1, keepdims=True) / x.shape[-1] + eps) * w.astype(np.float64)


def rotated(x, cs):
    c, s = cs[:, None, :, 0].astype(np.float64), cs[:, None, :, 1].astype(np.float64)
    e, o = x[..., 0::2], x[..., 1::2]
    return np.stack([e * c - o * s, e * s + o * c], -1).reshape(x.shape)


def slack(x, cs, hd):
    """What float steps may be off by, before the last rounding.  The sum of hd squares, positive, comes in hd roundings at most, the mean, eps, root and quotient in one each: the factor is off by
    U32 (hd / 2 + 4) of itself, the two products by U32 each; a rotation adds two products of which each and the sum are rounded: 2 U32 of |e c| + |o s|."""
    m = rotated(np.abs(x), np.abs(cs) * np.array([1, -1]))    # |e c| + |o s| and, of the odd ones, a sum with another sign
    m = np.maximum(np.abs(m), rotated(np.abs(x), np.abs(cs)))
    return U32 * (hd / 2 + 9) * m


@pytest.mark.parametrize("kind,hd,H,KV,page,news,lens,rope", [
    ("float16", 64, 4, 2, 16, [1], [1], True), ("int8", 64, 4, 2, 16, [1], [40], True), ("float16", 128, 32, 8, 64, [5, 0, 17, 1], [5, 9, 200, 64], True),
    ("int8", 128, 32, 8, 64, [5, 0, 17, 1], [5, 9, 200, 64], True), ("int8", 128, 3, 1, 32, [33], [97], False), ("float16", 64, 7, 7, 256, [2] * 9, [2, 3, 255, 256, 257, 258, 600, 4, 5], False),
    ("int8", 64, 24, 8, 128, [1] * 70, list(range(1, 71)), True), ("float16", 128, 64, 8, 16, [700, 3], [700, 1000], True),
])
def test_rows_normed_rotated_and_written(hip, kind, hd, H, KV, page, news, lens, rope):
    rng = np.random.default_rng(hd + H + page + len(news))
    c = Case(rng, kind, hd, KV, page, news, lens, extra_rows=2).device()
    n = int(c.starts[-1])
    q, k, v = (rng.standard_normal((c.rows, h, hd)).astype(np.float16) for h in (H, KV, KV))
    k *= np.float16(30)
    q[0, 0] = 0                                               # a row of zeros stays one
    q[-3, -1] *= np.float16(2.0 ** -14)                       # eps is most of the mean: halves below the normal ones among them
    k[0, -1] = 6e4                                            # squares beyond a half's range
    wq, wk = ((1 + 0.3 * rng.standard_normal(hd)).astype(np.float16) for _ in range(2))
    cs = rope_table(c.width * page, hd, rng)
    tq, tk, tv, tc, to, twq, twk = Tensor(q), Tensor(k), Tensor(v), Tensor(cs), Tensor.full(q.shape, 7.0, "float16"), Tensor(wq), Tensor(wk)
    check(hip.jsgrad_hip_paged_write_norm(*c.batch, tq.ptr, tk.ptr, tv.ptr, twq.ptr, twk.ptr, EPS, tc.ptr if rope else None, cs.shape[0] if rope else 0, to.ptr, H))
    pos = np.concatenate([np.arange(l - m, l) for m, l in zip(news, lens)])
    turn = cs[pos] if rope else np.broadcast_to(np.array([1, 0], np.float16), cs[pos].shape)
    place = [c.places(b, l - m, l) for b, (m, l) in enumerate(zip(news, lens))]
    ids, slots = (np.concatenate([p[i] for p in place]) for i in (0, 1))
    xq, xk = normed(q[:n], wq), normed(k[:n], wk)
    want_q, want_k = rotated(xq, turn), rotated(xk, turn)
    eq, ek = slack(xq, turn, hd), slack(xk, turn, hd)
    got = to.numpy()
    assert np.all(np.abs(got[:n].astype(np.float64) - want_q) <= U16 * np.abs(want_q) + eq * (1 + U16) + 2.0 ** -25) and np.all(got[n:] == 7)
    for name, want, off in (("k", want_k, ek), ("v", v[:n].astype(np.float64), 0)):
        pool = c.t[name].numpy()[ids, :, slots].astype(np.float64)
        if kind == "float16":
            assert np.all(np.abs(pool - want) <= U16 * np.abs(want) + off * (1 + U16) + (2.0 ** -25 if name == "k" else 0))
        else:
            s, top = c.t["s" + name].numpy()[ids, :, slots].astype(np.float64), np.abs(want).max(-1)
            reach = np.max(np.broadcast_to(off, want.shape), -1) / 127 + 2 * U32 * top / 127
            assert np.all(np.abs(s - np.where(top == 0, 1, top / 127)) <= reach)
            assert np.all(np.abs(pool * s[..., None] - want) <= s[..., None] * (0.5 + 2 * 127 * U32) + off)


def test_q_alone_in_place_and_none(hip):
    """q_out may be q; without q only k and v are written."""
    rng = np.random.default_rng(3)
    for with_q in (True, False):
        c = Case(rng, "float16", 64, 2, 16, [3, 1], [3, 20]).device()
        q, k, v = (rng.standard_normal((c.rows, h, 64)).astype(np.float16) for h in (4, 2, 2))
        w = np.ones(64, np.float16)
        t = [Tensor(x) for x in (q, k, v, w)]
        check(hip.jsgrad_hip_paged_write_norm(*c.batch, t[0].ptr if with_q else None, t[1].ptr, t[2].ptr, t[3].ptr if with_q else None, t[3].ptr, EPS, None, 0, t[0].ptr if with_q else None,
                                              4 if with_q else 0))
        want = normed(q, w) if with_q else q.astype(np.float64)
        assert np.all(np.abs(t[0].numpy().astype(np.float64) - want) <= (U16 + U32 * 41) * np.abs(want) + 2.0 ** -25)
        ids, slots = (np.concatenate(x) for x in zip(*(c.places(b, l - m, l) for b, (m, l) in enumerate(zip(c.news, c.lens)))))
        assert np.all(np.abs(c.t["k"].numpy()[ids, :, slots].astype(np.float64) - normed(k, w)) <= (U16 + U32 * 41) * np.abs(normed(k, w)) + 2.0 ** -25)


def test_a_row_that_is_not_finite(hip):
    """The row of a head that holds it is not a number, and no other."""
    rng = np.random.default_rng(4)
    c = Case(rng, "int8", 64, 2, 16, [4], [4]).device()
    q, k, v = (rng.standard_normal((4, h, 64)).astype(np.float16) for h in (4, 2, 2))
    k[1, 0, 5], k[2, 1, 9], q[3, 2, 0] = np.nan, np.inf, -np.inf
    w = np.ones(64, np.float16)
    t = [Tensor(x) for x in (q, k, v, w)]
    check(hip.jsgrad_hip_paged_write_norm(*c.batch, t[0].ptr, t[1].ptr, t[2].ptr, t[3].ptr, t[3].ptr, EPS, None, 0, t[0].ptr, 4))
    s = c.t["sk"].numpy()[c.table[0, 0], :, :4].T
    assert np.isnan(s[1, 0]) and np.isnan(s[2, 1]) and np.isfinite(s).sum() == 6
    got = t[0].numpy()
    assert np.isnan(got[3, 2]).any() and np.isfinite(np.delete(got.reshape(16, 64), 14, 0)).all()


def qk_model(**more):
    cfg = synthetic.config("tiny16", max_context=256, qk_norm=True, **more)
    sd = synthetic.random_state_dict(cfg, seed=3, std=0.05)
    rng = np.random.default_rng(9)
    for k in sd:
        if "q_norm" in k or "k_norm" in k:
            sd[k] = (1 + 0.3 * rng.standard_normal(sd[k].shape)).astype(np.float16)
    return cfg, sd, Llama3.from_config(cfg).load_weights(sd)


def test_a_model_with_norms_of_queries_and_keys(hip):
    """One layer by hand: the block's input, normed, through wq and wk in float64, normed per head and rotated, is what the pages hold, within the rounding of wk's result (U16, and the float sums of
    256 products, of the values that are normed)."""
    cfg, sd, llm = qk_model()
    m = llm.model
    cache = PagedCache(2, 2, 64, 16, 16)
    s = cache.add()
    toks = np.random.default_rng(1).integers(0, cfg["vocab_size"], 21).astype(np.int32)
    m.forward_paged(cache, [s], [toks])
    x = sd["tok_embeddings.weight"][toks].astype(np.float64)
    xn = x / np.sqrt((x * x).mean(-1, keepdims=True) + cfg["norm_eps"])
    k = (xn @ sd["layers.0.attention.wk.weight"].astype(np.float64).T).reshape(21, 2, 64)
    angle = np.outer(np.arange(21), cfg["rope_theta"] ** (-np.arange(0, 64, 2) / 64))
    want = rotated(normed(k, sd["layers.0.attention.k_norm.weight"], cfg["norm_eps"]), np.stack([np.cos(angle), np.sin(angle)], -1))
    got = cache.pools[0].numpy()[0][cache.pages[s]].transpose(0, 2, 1, 3).reshape(-1, 2, 64)[:21]
    assert np.abs(got - want).max() <= 8 * U16 * np.abs(want).max()
    # pieces, single tokens and a batch beside others end where the whole prompt does
    whole = m._paged.logits.numpy()[0].astype(np.float64)
    t = cache.add()
    for a, b in ((0, 7), (7, 8), (8, 20), (20, 21)):
        m.forward_paged(cache, [t], [toks[a:b]])
    assert np.abs(m._paged.logits.numpy()[0] - whole).max() <= 1e-2 * np.abs(whole).max()
    assert llm.generate_paged([toks, toks[:3]], 4, dtype="int8").shape == (2, 4)
    # the norms are in the result at all
    plain = Llama3.from_config(dict(cfg, qk_norm=False)).load_weights(sd)
    p = cache.add()
    plain.model.forward_paged(cache, [p], [toks])
    assert np.abs(plain.model._paged.logits.numpy()[0] - whole).max() > 0.05 * np.abs(whole).max()
    for call in (lambda: m.forward(np.array([[1]]), 0), lambda: m.forward_rows(np.array([[1, 2]]), 0), lambda: m.logits):
        with pytest.raises(NotImplementedError, match="paged"):
            call()


def test_norm_arguments_of_the_batch(hip):
    from denograd_amd.nn import RMSNorm
    cache = PagedCache(1, 2, 64, 4, 16)
    batch = cache.begin([cache.add()], [2])
    k, q = Tensor.zeros((2, 2, 64), "float16"), Tensor.zeros((2, 4, 64), "float16")
    a, b, short = RMSNorm(64, 1e-5), RMSNorm(64, 1e-6), RMSNorm(32, 1e-5)
    a.weight, b.weight, short.weight = Tensor.ones((64,), "float16"), Tensor.ones((64,), "float16"), Tensor.ones((32,), "float16")
    for bad in (dict(q_norm=a), dict(k_norm=a), dict(q_norm=a, k_norm=b), dict(q_norm=short, k_norm=a)):
        with pytest.raises(ValueError, match="norms of q and k"):
            batch.write(0, k, k, q, None, 4, **bad)
    batch.write(0, k, k, q, None, 4, q_norm=a, k_norm=a)
    batch.write(0, k, k, k_norm=a)


def test_a_checkpoint_with_norms_in_rotate_half_order(hip):
    """Features of a head come interleaved, and so do the weights of its norm: the norm of permuted rows is the permuted norm."""
    rng = np.random.default_rng(2)
    w = rng.standard_normal(64).astype(np.float16)
    out = convert_from_huggingface({"model.layers.0.self_attn.q_norm.weight": w, "model.layers.0.self_attn.k_norm.weight": w}, 1, 4, 2)
    for x in "qk":
        got = out[f"layers.0.attention.{x}_norm.weight"].numpy()
        assert np.array_equal(got, np.stack([w[:32], w[32:]], -1).reshape(-1))
    kept = convert_from_huggingface({"model.layers.0.self_attn.q_norm.weight": w}, 1, 4, 2, permute_layers=False)
    assert np.array_equal(kept["layers.0.attention.q_norm.weight"].numpy(), w)


@pytest.mark.parametrize("hd", [64, 128])
def test_codes_are_the_nearest_whole_numbers(hip, hd):
    """Of v, whose rows are not changed: to 127 x / max |x| in 64 bits (three roundings of 2^-53 there, of at most 127); halves have many quotients in the middle between two."""
    rng = np.random.default_rng(hd)
    c = Case(rng, "int8", hd, 8, 64, [2000], [2000]).device()
    v = rng.standard_normal((2000, 8, hd)).astype(np.float16)
    v[::3] = (v[::3] * 16).round() / 16                       # few values: ties in most rows
    v[0, 0], v[1, 1] = 0, 6e-8
    k, tv, w = Tensor(rng.standard_normal((2000, 8, hd)).astype(np.float16)), Tensor(v), Tensor(np.ones(hd, np.float16))
    check(hip.jsgrad_hip_paged_write_norm(*c.batch, None, k.ptr, tv.ptr, None, w.ptr, EPS, None, 0, None, 0))
    ids, slots = c.places(0, 0, 2000)
    codes = c.t["v"].numpy()[ids, :, slots].astype(np.float64)
    most = np.abs(v.astype(np.float64)).max(-1, keepdims=True)
    exact = 127 * v.astype(np.float64) / np.where(most == 0, 1, most)
    assert np.all(np.abs(codes - exact) <= 0.5 + 4 * 127 * 2.0 ** -53)
