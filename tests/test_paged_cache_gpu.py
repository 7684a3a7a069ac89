"""PagedKVCache: what a serving loop counts on between its calls."""

import pytest
import torch

from shardcompute_b200 import _lib as L
from shardcompute_b200 import ops
from shardcompute_b200.parallel import PagedKVCache

pytestmark = pytest.mark.gpu


def test_a_truncation_does_not_cover_a_refused_reservation(cuda):
    cache = PagedKVCache(1, 1, 64, n_pages=4, max_batch=2, max_len=64, max_tokens=100, device=cuda)
    cache.reserve([20, 0])
    cache.check()
    cache.reserve([20, 33])  # two pages left, four needed
    cache.truncate([20, 0])
    assert int(cache.status) == 1 and int(cache.truncate_status) == 0
    with pytest.raises(ValueError, match="reserve: not enough free pages"):
        cache.check()
    assert cache.lens.tolist() == [20, 0] and int(cache.free_count) == 2
    cache.reserve([0, 32])
    cache.check()
    cache.free_count.fill_(3)  # as if a page had been given back already
    cache.truncate([0, 0])
    cache.reserve([0, 0])
    with pytest.raises(ValueError, match="truncate: no room"):
        cache.check()


def test_check_reports_an_attention_that_gave_up(cuda, monkeypatch):
    """The word that a kernel raises when a bounded wait runs out, here by a stand-in for its reader."""
    cache = PagedKVCache(1, 1, 64, n_pages=4, max_batch=2, max_len=64, device=cuda)
    assert ops.prefix_attn_device_error() == 0
    cache.check()
    asked = []
    monkeypatch.setattr(L.load(), "sc_prefix_attn_device_error", lambda reset: asked.append(reset) or 1)
    with pytest.raises(RuntimeError, match="bounded wait"):
        cache.check()
    assert asked == [1]
