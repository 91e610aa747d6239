"""Tokens of one to three rows of up to 2^20 logits: as many parts, and groups of them, as a row ever has; against float64."""
import numpy as np
import pytest

from denograd_amd import ffi
from tests.sample_ref import sample
from tests.test_gpu_sample_rows import agree, logits
from tests.test_gpu_sample_rows_order import agree as agree_last

pytestmark = pytest.mark.gpu

# candidates of the first few, borders by number, by mass and by both, the whole vocabulary, the greedy token
SETTINGS = [(0.7, 50, 0.9, 0.0), (1.0, 256, 1.0, 1e-4), (1.3, 257, 0.95, 1e-3), (1.0, 0, 0.9, 0.0), (0.8, 70000, 1.0, 0.0), (1.5, 200000, 0.999, 1e-5), (1.0, 0, 1.0, 0.0), (0.0, 0, 1.0, 0.0)]


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("rows,n", [(1, 262145), (2, 270000), (3, 270000), (1, 524288), (1, 524289), (2, (1 << 20) - 1), (1, (1 << 20) - 1), (1, 1 << 20), (2, 1 << 20)])
def test_long_rows(hip, rows, n, dtype):
    rng = np.random.default_rng(rows + n)
    x = logits(rng, rows, n, dtype)
    x[0, n - 1] = x[0].max() + 1                              # in the last part, and the last entry of the row
    for i in range(0, len(SETTINGS), rows):
        T, k, p, m = (np.array([SETTINGS[(i + r) % len(SETTINGS)][j] for r in range(rows)]) for j in range(4))
        args = dict(temperature=T, top_k=k, top_p=p, min_p=m, uniforms=np.where(rng.random(rows) < 0.2, 1 - 2.0 ** -24, rng.random(rows)))
        agree(hip, x, **args)
        if m.any():
            agree_last(hip, x, **args)


@pytest.mark.parametrize("n", [524289, 1 << 20])
def test_long_rows_that_are_flat_or_masked(hip, n):
    """More candidates than a list, in every part; and all but a few entries masked."""
    rng = np.random.default_rng(n)
    flat = np.zeros((1, n), np.float16)
    masked = np.full((1, n), -np.inf, np.float32)
    at = np.sort(rng.choice(n, 300, replace=False))
    masked[0, at] = rng.standard_normal(300)
    few = rng.integers(0, 3, (1, n)).astype(np.float32)
    for x in (flat, masked, few):
        for T, k, p, m in ((0.7, 50, 0.9, 0.0), (1.0, 299, 0.5, 0.1), (1.0, 0, 0.25, 0.0), (1.0, 1000, 1.0, 0.0), (1.0, 0, 1.0, 0.0)):
            agree(hip, x, temperature=[T], top_k=[k], top_p=[p], min_p=[m], uniforms=[float(rng.integers(0, 8)) / 8])


def test_the_last_group_counts(hip):
    """The first top_k of a row are its last entries, one to a group of the last parts."""
    n = 1 << 20
    x = np.full((1, n), -20.0, np.float16)
    x[0, n - 200 * 512::512] = np.linspace(1, 4, 200).astype(np.float16)
    for u in (0.0, 0.3, 0.999):
        agree(hip, x, temperature=[1.0], top_k=[200], top_p=[1.0], min_p=[0.0], uniforms=[u])
        assert sample(x[0], 1.0, 200, u=u)[0] >= n - 200 * 512
    assert ffi.load().jsgrad_hip_sample_rows_workspace_bytes(1, n) > ffi.load().jsgrad_hip_sample_rows_workspace_bytes(1, n // 2)
