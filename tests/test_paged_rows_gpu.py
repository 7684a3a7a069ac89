"""The attention over a paged cache where a call's rows or pages are cut otherwise than usual."""

import math

import numpy as np
import pytest
import torch

from oracle import paged as op
from shardcompute_b200 import _lib as L
from tests.test_paged_gpu import attn_bound, check_attn, make_attn, run_attn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("prefix,new,rows", [(0, [3, 5, 2], 7), (77, [1, 1, 1], 2), (0, [9, 150, 70], 100), (300, [150, 150], 299),
                                             (5000, [1] * 40 + [4], 42), (40, [20, 0, 7], 20), (0, [4, 4], 1)])
def test_q_ends_before_the_last_request(cuda, rng, dtype, prefix, new, rows):
    """Fewer rows of q than were reserved: the rows that are there see what they see in the whole call."""
    hq, hkv, hd = 8, 2, 64
    d = make_attn(cuda, rng, dtype, hq, hkv, hd, 16, prefix, [n + 30 for n in new], new, pad=0)
    want, mass, dot, keys, tail = (x[:rows] for x in op.attention(d["q"].double().numpy(), d["k"].double().numpy(), d["v"].double().numpy(),
                                                                  d["start"], d["lens"], d["table"], d["ptab"], prefix, hq, 1 / math.sqrt(hd)))
    d["q"] = d["q"][:rows].contiguous()
    got = run_attn(cuda, d).double().cpu().numpy().reshape(want.shape)
    assert (np.abs(got - want) <= attn_bound(dtype, want, mass, dot, keys, tail, hd)).all()
    assert L.load().sc_prefix_attn_device_error(1) == 0


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("page,B,hkv", [(128, 40, 4), (256, 40, 4), (4096, 8, 2), (32768, 2, 1)])
def test_large_pages(cuda, rng, dtype, hd, page, B, hkv):
    """Pages of a tile of keys and more, up to the largest: a token each behind a prefix that ends inside a page, then a
    chunk behind it, and alone."""
    hq = 2 * hkv
    prefix = 3000
    lens = [1, page // 2 + 1] + [int(x) for x in rng.integers(1, min(page, 600), B - 2)]
    check_attn(cuda, dtype, make_attn(cuda, rng, dtype, hq, hkv, hd, page, prefix, lens, [1] * B), hq)
    for prefix, n, own in ((page + 3 if page < 1000 else 131, 700, 700), (0, 650, 901)):
        d = make_attn(cuda, rng, dtype, hq, hkv, hd, page, prefix, [own], [n])
        if page < 1000:  # a page that is not there, in the prefix or among the chunk's own
            (d["ptab"] if prefix else d["table"][0])[1] = -1
        check_attn(cuda, dtype, d, hq)
