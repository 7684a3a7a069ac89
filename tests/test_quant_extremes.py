"""What needs no GPU: oracle/quant_pages.py at the ends of fp16's range, PagedKVCache.read of pages that are not codes."""

import numpy as np
import pytest
import torch

from oracle import quant_pages as oq
from shardcompute_b200.parallel import PagedKVCache


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


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_read_of_a_cache_in_full(dtype):
    """The pages' own type, and zeros where there is no page: no other request's tokens."""
    c = PagedKVCache(num_layers=2, kv_heads=3, head_dim=64, n_pages=4, max_batch=2, max_len=64, dtype=dtype, device=torch.device("cpu"))
    g = torch.Generator().manual_seed(0)
    c.k.copy_(torch.randn(c.k.shape, generator=g))
    c.v.copy_(torch.randn(c.v.shape, generator=g))
    c.lens[1] = 50
    c.block_table[1] = torch.tensor([2, -1, 0, 4], dtype=torch.int32)  # no page; a page past the pool
    for got, held in zip(c.read(1, 1), (c.k[1], c.v[1])):
        assert got.dtype is dtype and got.shape == (50, 3, 64)
        assert torch.equal(got[:16], held[2].transpose(0, 1)) and torch.equal(got[32:48], held[0].transpose(0, 1))
        assert (got[16:32] == 0).all() and (got[48:] == 0).all()
    assert [x.dtype for x in c.read(1, 1, torch.float16)] == [torch.float16] * 2
    assert [x.shape for x in c.read(0, 0)] == [(0, 3, 64)] * 2
