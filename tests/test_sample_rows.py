"""Refusals of jsgrad_hip_sample_rows and RowSampler, and the shares of a total that borders are made of; without a GPU."""
import os
import subprocess

import numpy as np
import pytest

from denograd_amd import ffi
from denograd_amd.sampling import RowSampler

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("change,match", [
    (dict(logits=None), "null"), (dict(uniforms=None), "null"), (dict(tokens=None), "null"), (dict(workspace=None), "null"), (dict(act=2), "dtype"), (dict(rows=0), "rows"), (dict(rows=65536), "rows"),
    (dict(n=0), "logits"), (dict(n=(1 << 20) + 1), "logits"), (dict(stride=99), "stride"), (dict(stride=1 << 40), "stride"), (dict(logits=4097), "aligned"), (dict(act=0, logits=4098), "aligned"),
    (dict(top_k=4098), "4-byte"), (dict(tokens=4097), "4-byte"), (dict(probs=4098), "4-byte"), (dict(workspace=4104), "workspace"),
])
def test_refusals(change, match):
    lib = ffi.load()
    args = dict(logits=4096, rows=2, n=100, stride=100, act=1, temperature=4096, top_k=4096, top_p=4096, min_p=4096, uniforms=4096, tokens=4096, probs=4096, workspace=4096)
    args.update(change)
    assert lib.jsgrad_hip_sample_rows(*args.values()) != 0
    assert match in lib.jsgrad_hip_last_error().decode()
    assert lib.jsgrad_hip_sample_rows_workspace_bytes(0, 5) == lib.jsgrad_hip_sample_rows_workspace_bytes(5, 0) == 0 < lib.jsgrad_hip_sample_rows_workspace_bytes(1, 1)


@pytest.mark.parametrize("bad", [dict(temperature=-1), dict(temperature=np.nan), dict(temperature=np.inf), dict(top_k=-1), dict(top_p=1.1), dict(top_p=-0.1), dict(min_p=2), dict(min_p=np.nan),
                                 dict(top_p=[0.5, 0.6], min_p=[0, 0, 0]), dict(temperature=[]), dict(top_p=[[0.5]])])
def test_settings_that_are_refused(bad):
    with pytest.raises(ValueError):
        RowSampler(**bad)


def test_shares_of_a_total_are_exact(tmp_path):
    """floor and ceiling of f * z against Python's whole numbers and fractions."""
    from fractions import Fraction
    rng = np.random.default_rng(0)
    f = np.concatenate([rng.random(300), 2.0 ** -rng.uniform(0, 149, 300), [0, 0.5, 0.25, 1 - 2.0 ** -24, 2.0 ** -149, 2.0 ** -126, 2.0 ** -23]]).astype(np.float32)
    z = np.concatenate([rng.integers(1, 1 << 62, f.size - 3), [1, 1 << 62, 1 << 42]]).astype(np.uint64)
    z[::7] = np.uint64(1) << rng.integers(0, 62, z[::7].size).astype(np.uint64)
    src = tmp_path / "share.cpp"
    src.write_text(f'#include "{ROOT}/denograd_amd/csrc/sample_rows.h"\n#include <stdio.h>\n'
                   'int main() { unsigned b; unsigned long long z; while (scanf("%u %llu", &b, &z) == 2)\n'
                   '  printf("%llu %llu\\n", (unsigned long long)jsg::sample_share(b, z, false), (unsigned long long)jsg::sample_share(b, z, true)); }\n')
    subprocess.run(["g++", "-O2", "-o", str(tmp_path / "share"), str(src)], check=True)
    lines = "".join(f"{b} {v}\n" for b, v in zip(f.view(np.uint32), z))
    out = subprocess.run([str(tmp_path / "share")], input=lines, capture_output=True, text=True, check=True).stdout.split()
    for i, (a, b) in enumerate(zip(f, z)):
        exact = Fraction(float(a)) * int(b)
        assert int(out[2 * i]) == exact.__floor__() and int(out[2 * i + 1]) == exact.__ceil__()
