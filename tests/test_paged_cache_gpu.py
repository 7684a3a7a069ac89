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


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_captured_steps_of_a_model(cuda, dtype):
    """reserve, the model on rows padded to a fixed number, truncate: captured once and replayed over ragged steps, some
    refused, against the same calls made one by one.  The same kernels on the same values: the same bits."""
    import asyncio

    import numpy as np

    from oracle import sharder as osh
    from oracle import synth
    from shardcompute_b200.model.config import ModelConfig
    from shardcompute_b200.parallel import ParallelTransformer, RankWeights

    shape = synth.tiny_shape()
    cfg = ModelConfig.from_dict(synth.model_config_dict(shape))
    model = ParallelTransformer.from_config(cfg, 1, 0, None)
    model.load_rank_weights(RankWeights.from_shard(cfg, osh.shard_weights(synth.checkpoint(shape, seed=0), 1, 0), 1, 0, shape.bits, shape.group_size,
                                                   cuda))
    B, T, gen = 4, 24, np.random.default_rng(3)
    run = lambda ids, past: asyncio.run(model.forward(ids, past_key_values=past))[0]  # noqa: E731
    caches = [PagedKVCache(cfg.num_layers, cfg.kv_heads, cfg.head_dim, 14, B, 64, max_prefix=64, max_tokens=T, dtype=dtype, device=cuda)
              for _ in range(2)]
    for c in caches:
        c.reserve([20, 0, 0, 0])
        run(torch.arange(T, device=cuda)[None] % shape.vocab_size, c.layers())
        c.check()
        c.share_prefix(0)
    ids = torch.zeros(1, T, dtype=torch.long, device=cuda)
    new, keep = (torch.zeros(B, dtype=torch.int32, device=cuda) for _ in range(2))

    def step(c):
        c.reserve(new)
        logits = run(ids, c.layers())
        c.truncate(keep)
        return logits

    keep.fill_(64)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(caches[1])  # no tokens
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        logits = step(caches[1])

    lens, refused = np.zeros(B, int), 0
    for n, (add, cut) in enumerate([([5, 1, 9, 0], 0), ([1, 1, 1, 1], 0), ([6, 6, 6, 6], 2), ([20, 0, 0, 4], 0), ([1, 1, 0, 1], 0), ([24, 24, 24, 24], 0),
                                    ([0, 0, 0, 0], 0), ([1, 2, 3, 4], 1)]):
        fits = sum(add) <= T
        refused += not fits
        lens = np.maximum(lens + (np.array(add) - np.minimum(cut, add) if fits else 0), 0)
        ids.copy_(torch.from_numpy(gen.integers(0, shape.vocab_size, (1, T))))
        new.copy_(torch.tensor(add))
        keep.copy_(torch.from_numpy(lens))
        if n == 4:  # more positions than so far: the model's rotary tables grow
            run(torch.zeros(1, 1, dtype=torch.long, device=cuda), model.new_cache(1, 600))
        want = step(caches[0])
        graph.replay()
        rows = sum(add) if fits else 0
        assert torch.equal(logits[0, :rows], want[0, :rows]) and bool(torch.isfinite(logits).all())
        for name in ("lens", "free_count", "block_table", "status", "truncate_status"):
            assert torch.equal(getattr(caches[0], name), getattr(caches[1], name)), name
        assert caches[1].lens.tolist() == lens.tolist()
        if fits:
            caches[1].check()
        else:
            with pytest.raises(ValueError, match="rows"):
                caches[1].check()
    assert refused == 1
