"""The paged cache's refusals, which need no GPU: the C entries return before any launch, the tensor functions raise."""

import numpy as np
import pytest
import torch

from oracle import paged as op
from shardcompute_b200 import _lib as L
from shardcompute_b200 import ops

A = 1 << 20  # an address that no refused call reads
I31 = 2**31 - 1


def reserve(**kw):
    a = dict(lens=A, new=A, B=4, prefix=None, table=A, blocks=8, free=A, n_free=100, count=A, page=16, rows=10, kv=A, starts=A, slots=A,
             pos=A, left=A, status=A)
    a.update(kw)
    return L.load().sc_paged_reserve(a["lens"], a["new"], a["B"], a["prefix"], a["table"], a["blocks"], a["free"], a["n_free"], a["count"],
                                     a["page"], a["rows"], a["kv"], a["starts"], a["slots"], a["pos"], a["left"], a["status"], None)


@pytest.mark.parametrize("kw", [dict(B=0), dict(B=16385), dict(B=-1), dict(blocks=0), dict(n_free=0), dict(rows=0), dict(page=0),
                                dict(page=1 << 26), dict(blocks=I31)])
def test_reserve_refuses_shapes(kw):
    assert reserve(**kw) == L.SC_ERR_SHAPE


@pytest.mark.parametrize("name", ["lens", "new", "table", "free", "count", "kv", "starts", "slots", "pos", "left", "status"])
def test_reserve_refuses_null(name):
    assert reserve(**{name: None}) == L.SC_ERR_ARG


def truncate(**kw):
    a = dict(lens=A, keep=A, B=4, table=A, blocks=8, free=A, n_free=100, count=A, page=16, out=A, left=A, status=A)
    a.update(kw)
    return L.load().sc_paged_truncate(a["lens"], a["keep"], a["B"], a["table"], a["blocks"], a["free"], a["n_free"], a["count"], a["page"],
                                      a["out"], a["left"], a["status"], None)


@pytest.mark.parametrize("kw", [dict(B=0), dict(B=16385), dict(blocks=0), dict(n_free=0), dict(page=0), dict(page=1 << 26)])
def test_truncate_refuses_shapes(kw):
    assert truncate(**kw) == L.SC_ERR_SHAPE


@pytest.mark.parametrize("name", ["lens", "keep", "table", "free", "count", "out", "left", "status"])
def test_truncate_refuses_null(name):
    assert truncate(**{name: None}) == L.SC_ERR_ARG


def append(**kw):
    a = dict(qkv=A, dt=L.SC_F32, rows=4, end=A, slots=A, pos=A, cos=A, sin=A, max_pos=64, hq=8, hkv=2, hd=64, q=A, k=A, v=A, cdt=L.SC_F16,
             pages=10, page=16)
    a.update(kw)
    return L.load().sc_paged_rope_append(a["qkv"], a["dt"], a["rows"], a["end"], a["slots"], a["pos"], a["cos"], a["sin"], a["max_pos"],
                                         a["hq"], a["hkv"], a["hd"], a["q"], a["k"], a["v"], a["cdt"], a["pages"], a["page"], None)


@pytest.mark.parametrize("kw,code", [(dict(rows=0), L.SC_ERR_SHAPE), (dict(hq=0), L.SC_ERR_SHAPE), (dict(hd=12), L.SC_ERR_SHAPE),
                                     (dict(hd=0), L.SC_ERR_SHAPE), (dict(max_pos=0), L.SC_ERR_SHAPE), (dict(pages=I31), L.SC_ERR_SHAPE),
                                     (dict(hq=1 << 22), L.SC_ERR_SHAPE), (dict(dt=L.SC_I32), L.SC_ERR_ARG), (dict(cdt=L.SC_U8), L.SC_ERR_ARG),
                                     (dict(qkv=A + 4), L.SC_ERR_ARG), (dict(k=A + 8), L.SC_ERR_ARG), (dict(cos=A + 4), L.SC_ERR_ARG),
                                     (dict(v=None), L.SC_ERR_ARG), (dict(end=None), L.SC_ERR_ARG), (dict(pos=None), L.SC_ERR_ARG)])
def test_append_refuses(kw, code):
    assert append(**kw) == code


def attn(**kw):
    a = dict(q=A, k=A, v=A, dt=L.SC_F16, T=4, starts=A, lens=A, table=A, B=4, blocks=8, ptab=A, plen=A, pblocks=4, hq=8, hkv=2, hd=128,
             pages=100, page=16, scale=0.1, out=A, ws=A, wb=1 << 40)
    a.update(kw)
    return L.load().sc_prefix_attn(a["q"], a["k"], a["v"], a["dt"], a["T"], a["starts"], a["lens"], a["table"], a["B"], a["blocks"], a["ptab"],
                                   a["plen"], a["pblocks"], a["hq"], a["hkv"], a["hd"], a["pages"], a["page"], a["scale"], a["out"], a["ws"],
                                   a["wb"], None)


@pytest.mark.parametrize("kw,code", [(dict(hd=96), L.SC_ERR_UNSUPPORTED), (dict(hd=256), L.SC_ERR_UNSUPPORTED), (dict(page=8), L.SC_ERR_UNSUPPORTED),
                                     (dict(page=48), L.SC_ERR_UNSUPPORTED), (dict(page=1 << 16), L.SC_ERR_UNSUPPORTED), (dict(T=0), L.SC_ERR_SHAPE),
                                     (dict(B=0), L.SC_ERR_SHAPE), (dict(B=65536), L.SC_ERR_SHAPE), (dict(blocks=0), L.SC_ERR_SHAPE),
                                     (dict(pages=0), L.SC_ERR_SHAPE), (dict(hq=7), L.SC_ERR_SHAPE), (dict(hkv=0), L.SC_ERR_SHAPE),
                                     (dict(hq=1), L.SC_ERR_SHAPE), (dict(pages=1 << 27), L.SC_ERR_SHAPE), (dict(T=1 << 29), L.SC_ERR_SHAPE),
                                     (dict(blocks=1 << 28), L.SC_ERR_SHAPE), (dict(pblocks=1 << 28), L.SC_ERR_SHAPE), (dict(dt=L.SC_I32), L.SC_ERR_ARG),
                                     (dict(scale=0.0), L.SC_ERR_ARG), (dict(scale=-1.0), L.SC_ERR_ARG), (dict(scale=float("nan")), L.SC_ERR_ARG),
                                     (dict(scale=float("inf")), L.SC_ERR_ARG), (dict(ptab=None), L.SC_ERR_ARG), (dict(pblocks=0), L.SC_ERR_ARG),
                                     (dict(q=None), L.SC_ERR_ARG), (dict(out=None), L.SC_ERR_ARG), (dict(q=A + 2), L.SC_ERR_ARG),
                                     (dict(v=A + 8), L.SC_ERR_ARG), (dict(ws=A + 4), L.SC_ERR_ARG), (dict(blocks=4096, wb=16), L.SC_ERR_WORKSPACE),
                                     (dict(blocks=4096, ws=None), L.SC_ERR_WORKSPACE)])
def test_attn_refuses(kw, code):
    assert attn(**kw) == code
    assert L.last_error()


def test_workspace_is_bounded():
    """Scratch stays a small multiple of the output, whatever the batch."""
    for T, B in [(1, 1), (1, 4096), (256, 256), (16384, 1), (16384, 64), (100000, 1000)]:
        for dt in (torch.float16, torch.float32):
            n = ops.prefix_attn_workspace_bytes(T, B, 32, 8, 128, 4096, 4096, 16, dt)
            assert 0 <= n <= 64 * max(T, 148) * 32 * 130 * 4
    assert L.load().sc_prefix_attn_workspace_bytes(4, 4, 7, 2, 128, 8, 8, 16, 0) == 0


def test_workspace_of_long_chunks():
    """Chunks that fill the machine need none, until a share of the keys would pass 131072: then one result more per row."""
    bytes_of = lambda blocks, dt: ops.prefix_attn_workspace_bytes(16384, 1, 32, 8, 128, blocks, 16, 16, dt)  # noqa: E731
    for dt in (torch.float16, torch.float32):
        assert bytes_of(1000, dt) == 0
    assert bytes_of(8192 - 16, torch.float16) == 0
    assert bytes_of(8192, torch.float16) == 2 * 16384 * 32 * 130 * 4


def test_cpu_tensors_are_refused():
    z = torch.zeros(4, dtype=torch.int32)
    t = torch.zeros(4, 2, dtype=torch.int32)
    pool = torch.zeros(2, 1, 16, 64)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.paged_reserve(z, z, t, z, z[:1], 16, max_tokens=4)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.paged_truncate(z, z, t, z, z[:1], 16)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.paged_rope_append(torch.zeros(1, 192), z, z, z, torch.zeros(4, 32), torch.zeros(4, 32), torch.zeros(1, 64), pool, pool)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.prefix_attn(torch.zeros(4, 64), pool, pool, torch.zeros(5, dtype=torch.int32), z, t)


def test_pools_are_checked_before_the_device():
    pool, z = torch.zeros(2, 1, 16, 64), torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError, match="pages"):
        ops.prefix_attn(torch.zeros(4, 64), pool[0], pool[0], z, z, z)
    with pytest.raises(ValueError, match="pages"):
        ops.prefix_attn(torch.zeros(4, 64), pool, pool.double(), z, z, z)
    with pytest.raises(ValueError, match="pages"):
        ops.prefix_attn(torch.zeros(4, 64), pool.int(), pool.int(), z, z, z)


# ------------------------------------------------------------------------------------------------ the oracle itself

def test_oracle_reserve_then_truncate_gives_every_page_back():
    rng = np.random.default_rng(0)
    B, page, n_pages = 6, 4, 60
    free, count = rng.permutation(n_pages), n_pages
    table, lens = np.full((B, 12), -1), np.zeros(B, np.int64)
    for _ in range(20):
        new = rng.integers(0, 4, B)
        st, table, lens, start, slots, pos, count = op.reserve(lens, new, table, free, count, page, 100)
        assert st == 0 and len(set(slots.tolist())) == len(slots) == new.sum() == start[-1]
        st, lens, free, count = op.truncate(lens, np.where(rng.random(B) < 0.3, 0, lens - rng.integers(0, 3, B)), table, free, count, page)
        assert st == 0
        live = [int(x) for b in range(B) for x in table[b, : -(-lens[b] // page)]]
        assert sorted(live + free[:count].tolist()) == list(range(n_pages))


def test_oracle_attention_against_a_plain_softmax():
    rng = np.random.default_rng(1)
    k, v, q = rng.standard_normal((3, 1, 16, 8)), rng.standard_normal((3, 1, 16, 8)), rng.standard_normal((2, 2 * 8))
    out, *_ = op.attention(q, k, v, [0, 2], [20], np.array([[2, 0]]), np.array([1]), 5, 2, 0.5)
    keys, vals = np.concatenate([k[1, 0, :5], k[2, 0], k[0, 0, :4]]), np.concatenate([v[1, 0, :5], v[2, 0], v[0, 0, :4]])
    for i in range(2):
        for h in range(2):
            s = keys[: 24 + i] @ q[i].reshape(2, 8)[h] * 0.5
            w = np.exp(s) / np.exp(s).sum()
            assert np.allclose(out[i, h], w @ vals[: 24 + i])
