"""Refusals of jsgrad_hip_sample_rows_ordered, and of what takes min-p in either place; without a GPU."""
import numpy as np
import pytest

from denograd_amd import ffi
from denograd_amd.sampling import RowSampler


@pytest.mark.parametrize("change,match", [(dict(order=2), "order 2"), (dict(order=-1), "order -1"), (dict(logits=None), "null"), (dict(uniforms=None), "null"), (dict(min_p=4098), "4-byte"), (dict(n=0), "logits"),
                                          (dict(stride=99), "stride")])
def test_refusals(change, match):
    lib = ffi.load()
    args = dict(logits=4096, rows=2, n=100, stride=100, act=1, temperature=4096, top_k=4096, top_p=4096, min_p=4096, order=ffi.MIN_P_LAST, uniforms=4096, tokens=4096, probs=4096, workspace=4096)
    args.update(change)
    assert lib.jsgrad_hip_sample_rows_ordered(*args.values()) != 0
    said = lib.jsgrad_hip_last_error().decode()
    assert match in said and "_ordered" in said


def test_settings():
    assert RowSampler().order == ffi.MIN_P_FIRST and RowSampler(min_p=0.1, min_p_last=True).order == ffi.MIN_P_LAST
    with pytest.raises(ValueError):
        RowSampler(min_p=np.nan, min_p_last=True)
