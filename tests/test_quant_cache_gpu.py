"""PagedKVCache in 8 or 4 bits under a model, and read back."""

import asyncio

import numpy as np
import pytest
import torch

from oracle import sharder as osh
from oracle import synth
from shardcompute_b200 import ops
from shardcompute_b200.model.config import ModelConfig
from shardcompute_b200.parallel import PagedKVCache, ParallelTransformer, RankWeights

pytestmark = pytest.mark.gpu


def tiny_model(cuda):
    shape = synth.tiny_shape()
    cfg = ModelConfig.from_dict(synth.model_config_dict(shape))
    model = ParallelTransformer.from_config(cfg, 1, 0, None)
    model.load_rank_weights(RankWeights.from_shard(cfg, osh.shard_weights(synth.checkpoint(shape, seed=0), 1, 0), 1, 0, shape.bits, shape.group_size, cuda))
    return shape, cfg, lambda ids, past: asyncio.run(model.forward(ids, past_key_values=past))[0][0]


def make(cfg, cuda, **kw):
    return PagedKVCache(cfg.num_layers, cfg.kv_heads, cfg.head_dim, 24, 3, 64, page_size=16, max_prefix=64, max_tokens=48, device=cuda, **kw)


def rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


@pytest.mark.parametrize("bits,group", [(8, 32), (8, 64), (4, 32)])
def test_model_over_codes(cuda, bits, group):
    """A shared prefix, ragged chunks, single tokens, rejected drafts, a request that ends, over a cache in codes and over one in
    fp32.  8 bits: a key or value is off by at most half a step, a 510th of its group's range, which is some six times its
    rms: 1.2e-2, for keys and values of two layers 4.7e-2 at most, and seldom all one way.  (4 bits: sixteen times that says
    nothing; the values are finite and the keys and values of the first layer within half a step.)"""
    shape, cfg, run = tiny_model(cuda)
    gen = np.random.default_rng(5)
    words = lambda n: gen.integers(0, shape.vocab_size, n).tolist()  # noqa: E731
    quant, full = make(cfg, cuda, bits=bits, group_size=group), make(cfg, cuda)
    held = sum(p.data.numel() for p in quant.pages)  # a token's bits and 4 bytes a group, against 4 bytes a value
    assert held == full.k.numel() * 2 // group * (group * bits // 8 + 4)

    def step(tokens):
        outs = []
        for c in (quant, full):
            c.reserve([len(t) for t in tokens])
            c.check()
            outs.append(run(torch.tensor([sum(tokens, [])], device=cuda), c.layers()))
        assert torch.isfinite(outs[0]).all()
        if bits == 8:
            assert rel(*outs) <= 4.7e-2

    step([words(21), [], []])
    for c in (quant, full):
        c.share_prefix(0)
    for new_n, keep in [((5, 1, 9), (5, 1, 9)), ((1, 1, 1), (6, 2, 10)), ((4, 0, 3), (8, 2, 10)), ((1, 1, 1), (9, 0, 11)), ((2, 17, 1), (11, 17, 12))]:
        step([words(n) for n in new_n])
        for c in (quant, full):
            c.truncate(keep)
            c.check()
            assert c.lens.tolist() == list(keep)
        for b in range(3):
            for (a, w), heads in ((x, cfg.kv_heads) for x in zip(quant.read(0, b, torch.float32), full.read(0, b, torch.float32))):
                assert a.shape == w.shape == (keep[b], heads, cfg.head_dim)
                if keep[b]:
                    g = w.unflatten(-1, (-1, group))
                    half = (g.amax(-1) - g.amin(-1)) / (2**bits - 1) / 2
                    # the step is rounded up by up to 2^-10 (and the bias down); the fp32 cache's own keys differ by a rounding
                    limit = half * (1 + 2.0**-9) + g.abs().amax(-1) * 2.0**-10
                    assert ((a - w).unflatten(-1, (-1, group)).abs().amax(-1) <= limit).all()
    for c in (quant, full):
        c.truncate([0, 0, 0])
        c.release_prefix()
        c.check()
    assert int(quant.free_count) == 24
    with pytest.raises(IndexError):
        quant.read(0, 3)


@pytest.mark.parametrize("bits", [8, 4])
def test_a_layer_makes_the_operators_calls(cuda, bits, monkeypatch):
    """The attention layer's outputs are those of the operators on its projections: the same bits."""
    shape, cfg, run = tiny_model(cuda)
    a, b = make(cfg, cuda, bits=bits), make(cfg, cuda, bits=bits)
    ids = torch.arange(20, device=cuda)[None] % shape.vocab_size
    for c in (a, b):
        c.reserve([13, 0, 7])
    first = run(ids, a.layers())
    seen = []
    real = ops.paged_rope_append_q, ops.prefix_attn_q
    monkeypatch.setattr(ops, "paged_rope_append_q", lambda *args: seen.append("append") or real[0](*args))
    monkeypatch.setattr(ops, "prefix_attn_q", lambda *args, **kw: seen.append("attn") or real[1](*args, **kw))
    assert torch.equal(first, run(ids, b.layers())) and seen == ["append", "attn"] * cfg.num_layers
    for p, q in zip(a.pages, b.pages):
        assert torch.equal(p.data, q.data)


@pytest.mark.parametrize("bits", [8, 4])
def test_captured_steps(cuda, bits):
    """reserve, model, truncate captured once and replayed over ragged steps against the same calls one by one: the same bits."""
    shape, cfg, run = tiny_model(cuda)
    B, T, gen = 3, 24, np.random.default_rng(3)
    caches = [PagedKVCache(cfg.num_layers, cfg.kv_heads, cfg.head_dim, 14, B, 64, max_prefix=64, max_tokens=T, bits=bits, group_size=32, device=cuda)
              for _ in range(2)]
    for c in caches:
        c.reserve([20, 0, 0])
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
        step(caches[1])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        logits = step(caches[1])
    lens = np.zeros(B, int)
    for add, cut in [([5, 1, 9], 0), ([1, 1, 1], 0), ([6, 6, 6], 2), ([0, 20, 4], 0), ([24, 24, 24], 0), ([0, 0, 0], 0), ([1, 2, 3], 1)]:
        fits = sum(add) <= T
        lens = np.maximum(lens + (np.array(add) - np.minimum(cut, add) if fits else 0), 0)
        ids.copy_(torch.from_numpy(gen.integers(0, shape.vocab_size, (1, T))))
        new.copy_(torch.tensor(add))
        keep.copy_(torch.from_numpy(lens))
        want = step(caches[0])
        graph.replay()
        rows = sum(add) if fits else 0
        assert torch.equal(logits[:rows], want[:rows]) and bool(torch.isfinite(logits).all())
        for name in ("lens", "free_count", "block_table", "status", "truncate_status"):
            assert torch.equal(getattr(caches[0], name), getattr(caches[1], name)), name
        for p, q in zip(caches[0].pages, caches[1].pages):
            assert torch.equal(p.data, q.data)
        assert caches[1].lens.tolist() == lens.tolist()
