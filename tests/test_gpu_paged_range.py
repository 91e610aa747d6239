"""Attention over a paged cache where the keys with the largest weights have values of zero: what is left of the result comes from weights that are small beside them.

Bound of one element, as tests/paged_ref.py has it but for what fp16's normal numbers do not hold.  The weights are rounded to fp16 times a power of two that puts the largest of a
row at 2^8 and more (int8: the largest product of a weight and its row's scale of V, among the rows that are not zeros), so that one below 2^-14 is off by 2^-25, twice where
it is scaled down afterwards: 2^-32 of the largest.  With n keys that is 2^-32 n max |V| for fp16 pages, and 2^-32 n max (w |V|) for int8 ones, whose largest code is 127."""
import numpy as np
import pytest

from tests.paged_ref import U16, U32, Case
from tests.test_gpu_paged import in_chunks, padded, run_attention

pytestmark = pytest.mark.gpu


def reference(c, q, H):
    k, v = c.values("k"), c.values("v")
    out, tol = np.zeros((c.rows, H, c.hd)), np.zeros((c.rows, H, c.hd))
    rep = H // c.KV
    for b, (n, l) in enumerate(zip(c.news, c.lens)):
        ids, slots = c.places(b, 0, l)
        for i in range(n):
            seen, r = l - n + i + 1, c.starts[b] + i
            kk, vv = k[ids[:seen], :, slots[:seen]], v[ids[:seen], :, slots[:seen]]
            for h in range(H):
                g, x = h // rep, q[r, h].astype(np.float64)
                s = kk[:, g] @ x / np.sqrt(c.hd)
                w = np.exp(s - s.max())
                w /= w.sum()
                out[r, h] = w @ vv[:, g]
                size = np.abs(vv[:, g])
                A = w @ size
                E = U32 * (c.hd * (np.abs(kk[:, g]) @ np.abs(x)).max() / np.sqrt(c.hd) + 8 * np.abs(s).max() + 16)
                largest = (w * size.max(-1)).max() if c.kind == "int8" else size.max()
                tol[r, h] = U16 * np.abs(out[r, h]) + 2.0 ** -25 + (U16 + 4 * E + U32 * seen) * A + 2.0 ** -32 * seen * (largest + A)
    return out, tol


def case(kind, hd, news, lens, above, size, at):
    """The key at every position of `at` has scores `above` (in powers of two) higher than the others', and values of zero; the others' are size / 4 to size / 2."""
    rng = np.random.default_rng(hd + lens[0] + above)
    KV, H = 2, 4
    c = Case(rng, kind, hd, KV, 16, news, lens)
    u = rng.choice([-1.0, 1.0], hd)
    a = np.sqrt(above * np.log(2) / np.sqrt(hd))
    k = 0.05 * rng.standard_normal(c.k.shape)
    v = size * rng.uniform(0.25, 0.5, c.v.shape)
    for b, l in enumerate(lens):
        ids, slots = c.places(b, 0, l)
        mine = [p for p in at if p < l]
        k[ids[mine], :, slots[mine]], v[ids[mine], :, slots[mine]] = a * u, 0
    c = Case(np.random.default_rng(hd + lens[0] + above), kind, hd, KV, 16, news, lens, k=k.astype(np.float16), v=v.astype(np.float16))
    q = (a * u + 0.05 * rng.standard_normal((c.rows, H, hd))).astype(np.float16)
    return c, q, H


SHAPES = [(64, [1, 1], [400, 1500]), (128, [2, 1], [300, 1100]), (64, [70, 1], [400, 33]), (128, [90], [500])]
ZEROS = [(0, 0.5, range(0, 4000, 3)), (0, 1e-5, [0, 100, 101]), (17, 0.5, [7]), (20, 1.0, [0]), (20, 1.0, [299]), (24, 60.0, [1, 77]), (28, 1000.0, [0])]


def check_case(hip, c, q, H, chunks):
    n = int(c.starts[-1])
    if chunks:
        q = padded(in_chunks(c, H), q)
    else:
        c.device()
    ref, tol = reference(c, q, H)
    got = run_attention(hip, c, q, H, 0, 0, times=2)
    off = np.abs(got[:n].astype(np.float64) - ref[:n])
    assert np.all(off <= tol[:n]), (np.argwhere(~(off <= tol[:n]))[:4], got[:n][~(off <= tol[:n])][:4], ref[:n][~(off <= tol[:n])][:4])


@pytest.mark.parametrize("kind", ["float16", "int8"])
@pytest.mark.parametrize("above,size,at", ZEROS)
@pytest.mark.parametrize("hd,news,lens", SHAPES)
def test_values_of_zero_at_the_largest_weights(hip, kind, hd, news, lens, above, size, at):
    check_case(hip, *case(kind, hd, news, lens, above, size, at), chunks=False)


@pytest.mark.parametrize("kind", ["float16", "int8"])
@pytest.mark.parametrize("above,size,at", ZEROS)
@pytest.mark.parametrize("hd,news,lens", SHAPES[2:])
def test_values_of_zero_at_the_largest_weights_in_chunks(hip, kind, hd, news, lens, above, size, at):
    check_case(hip, *case(kind, hd, news, lens, above, size, at), chunks=True)


@pytest.mark.parametrize("chunks", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
def test_zero_codes_under_any_scale_and_scales_near_zero(hip, hd, chunks):
    """A caller's own int8 pages: zero codes are zeros under the largest and the smallest scale, and under 0; codes under scales from 1e-38 to 1e-25 are zeros as fp16 results show them."""
    c, q, H = case("int8", hd, [70], [400], 5, 0.5, list(range(0, 400, 7)))
    ids, slots = c.places(0, 0, 400)
    for i, p in enumerate(range(0, 400, 7)):
        c.sv[ids[p], :, slots[p]] = [3e38, 1e-38, 0.0, 1.0, 1e-25, 65504.0][i % 6]
    for i, p in enumerate(range(1, 400, 49)):
        c.sv[ids[p], :, slots[p]] = [1e-38, 1e-30, 1e-25, 0.0][i % 4]
    check_case(hip, c, q, H, chunks)


@pytest.mark.parametrize("kind", ["float16", "int8"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("chunks", [False, True])
def test_the_largest_weight_of_a_row_is_not_rounded(hip, kind, hd, chunks):
    """As with the contiguous cache.  Bound of one element: U16 |out| for the result; U16 w |V| for every key but the one with the largest weight (int8: weight times scale of V) and, as the
    sum may be of the weights before or after their rounding, U16 w |out| for the same keys; scores are sums of four products, all others being zeros, so that
    E = U32 (4 S + 8 max |s| + 16), twice for weights and sum each; float sums over n keys."""
    rng = np.random.default_rng(hd)
    KV, H, news, lens = 2, 8, [150], [190]
    c = Case(rng, kind, hd, KV, 64, news, lens)
    q = np.zeros((c.rows, H, hd))
    q[..., 3::hd // 4] = 3 * np.sqrt(hd) / 2 * rng.standard_normal((c.rows, H, 4))
    q = q.astype(np.float16)
    got = run_attention(hip, *((lambda d: (d, padded(d, q)))(in_chunks(c, H)) if chunks else (c.device(), q)), H, 0, 0)
    k, v = c.values("k"), c.values("v")
    ids, slots = c.places(0, 0, lens[0])
    worst = 0.0
    for i in range(news[0]):
        n = lens[0] - news[0] + i + 1
        for h in range(H):
            g, x = h // (H // KV), q[i, h].astype(np.float64)
            kk, vv = k[ids[:n], g, slots[:n]], v[ids[:n], g, slots[:n]]
            s = kk @ x / np.sqrt(hd)
            w = np.exp(s - s.max())
            w /= w.sum()
            out, A = w @ vv, w @ np.abs(vv)
            E = U32 * (4 * (np.abs(kk) @ np.abs(x)).max() / np.sqrt(hd) + 8 * np.abs(s).max() + 16)
            top = (w * c.sv[ids[:n], g, slots[:n]] if kind == "int8" else w).argmax()
            others = A - w[top] * np.abs(vv[top]) + (1 - w[top]) * np.abs(out)
            tol = U16 * (np.abs(out) + others) + 2.0 ** -25 + (4 * E + U32 * n) * (A + np.abs(out)) + 2.0 ** -32 * n
            worst = max(worst, (np.abs(got[i, h] - out) / tol).max())
    assert worst <= 1, worst
