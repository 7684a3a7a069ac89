"""oracle/quant_pages.py at the ends of fp16's range."""

import numpy as np
import pytest

from oracle import quant_pages as oq


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("group", [32, 64])
def test_oracle_holds_what_fp16_holds(bits, group):
    rng = np.random.default_rng(0)
    lo, hi = np.sort(rng.uniform(-65504, 65504, (2, 4000)), 0)
    lo[:1000], hi[500:1500] = -65504, 65504
    x = (lo[:, None] + (hi - lo)[:, None] * rng.random((4000, group))).astype(np.float16)
    x[:, 0], x[:, 1] = lo, hi
    codes, s, b = oq.quantise(x, bits, group)
    top = s.astype(np.float64) * (2**bits - 1) + b.astype(np.float64)
    assert top.max() <= 65504 and np.isfinite(b).all() and codes.max() <= 2**bits - 1
    assert (np.abs(oq.value(codes, s, b) - x.astype(np.float64)) <= s.astype(np.float64) / 2).all()
    assert (x.max(-1) > top[:, 0]).any()  # the scale below was taken somewhere
