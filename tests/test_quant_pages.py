"""The paged cache in 8 or 4 bits, without a GPU: what its operators refuse, and the oracle's own layout and rounding."""

import numpy as np
import pytest
import torch

from oracle import quant_pages as oq
from shardcompute_b200 import _lib as L
from shardcompute_b200 import ops

A = 1 << 20  # an address that no refused call reads
I31 = 2**31 - 1
KINDS = [(hd, bits, group) for hd in (64, 128) for bits in (4, 8) for group in (32, 64)]


def test_page_bytes():
    for hd, bits, group in KINDS:
        for page in (16, 48, 128):
            assert ops.quant_page_bytes(page, hd, bits, group) == page // 16 * oq.block_bytes(hd, bits, group)
    for page, hd, bits, group in [(8, 128, 4, 64), (24, 128, 4, 64), (0, 128, 4, 64), (16, 96, 4, 64), (16, 128, 2, 64), (16, 128, 4, 128)]:
        assert L.load().sc_quant_page_bytes(page, hd, bits, group) == 0
        with pytest.raises(ValueError, match="unsupported"):
            ops.quant_page_bytes(page, hd, bits, group)


def append(**kw):
    a = dict(qkv=A, dt=L.SC_F32, rows=4, end=A, slots=A, pos=A, cos=A, sin=A, max_pos=64, hq=8, hkv=2, hd=64, q=A, pages=A, bits=4, group=64, n=10, page=16)
    a.update(kw)
    return L.load().sc_paged_rope_append_q(a["qkv"], a["dt"], a["rows"], a["end"], a["slots"], a["pos"], a["cos"], a["sin"], a["max_pos"], a["hq"],
                                           a["hkv"], a["hd"], a["q"], a["pages"], a["bits"], a["group"], a["n"], a["page"], None)


@pytest.mark.parametrize("kw,code", [(dict(rows=0), L.SC_ERR_SHAPE), (dict(hq=0), L.SC_ERR_SHAPE), (dict(hkv=0), L.SC_ERR_SHAPE),
                                     (dict(n=0), L.SC_ERR_SHAPE), (dict(max_pos=0), L.SC_ERR_SHAPE), (dict(n=I31), L.SC_ERR_SHAPE),
                                     (dict(hq=1 << 22), L.SC_ERR_SHAPE), (dict(hkv=1 << 30), L.SC_ERR_SHAPE), (dict(hd=96), L.SC_ERR_UNSUPPORTED),
                                     (dict(bits=3), L.SC_ERR_UNSUPPORTED), (dict(group=16), L.SC_ERR_UNSUPPORTED), (dict(page=8), L.SC_ERR_UNSUPPORTED),
                                     (dict(page=40), L.SC_ERR_UNSUPPORTED), (dict(dt=L.SC_I32), L.SC_ERR_ARG), (dict(qkv=A + 4), L.SC_ERR_ARG),
                                     (dict(q=A + 2), L.SC_ERR_ARG), (dict(pages=A + 8), L.SC_ERR_ARG), (dict(cos=A + 4), L.SC_ERR_ARG)]
                         + [({name: None}, L.SC_ERR_ARG) for name in ("qkv", "end", "slots", "pos", "cos", "sin", "q", "pages")])
def test_append_refuses(kw, code):
    assert append(**kw) == code and L.last_error()


def read(**kw):
    a = dict(pages=A, bits=4, group=64, n=10, page=16, hkv=2, hd=64, slots=A, rows=4, end=A, k=A, v=A, dt=L.SC_F16)
    a.update(kw)
    return L.load().sc_paged_read_q(a["pages"], a["bits"], a["group"], a["n"], a["page"], a["hkv"], a["hd"], a["slots"], a["rows"], a["end"], a["k"],
                                    a["v"], a["dt"], None)


@pytest.mark.parametrize("kw,code", [(dict(rows=0), L.SC_ERR_SHAPE), (dict(hkv=0), L.SC_ERR_SHAPE), (dict(n=0), L.SC_ERR_SHAPE),
                                     (dict(n=I31), L.SC_ERR_SHAPE), (dict(hkv=1 << 22), L.SC_ERR_SHAPE), (dict(hd=32), L.SC_ERR_UNSUPPORTED),
                                     (dict(bits=16), L.SC_ERR_UNSUPPORTED), (dict(group=128), L.SC_ERR_UNSUPPORTED), (dict(page=0), L.SC_ERR_UNSUPPORTED),
                                     (dict(dt=L.SC_U8), L.SC_ERR_ARG), (dict(k=A + 2), L.SC_ERR_ARG), (dict(pages=None), L.SC_ERR_ARG),
                                     (dict(slots=None), L.SC_ERR_ARG), (dict(k=None), L.SC_ERR_ARG), (dict(v=None), L.SC_ERR_ARG)])
def test_read_refuses(kw, code):
    assert read(**kw) == code and L.last_error()


def attn(**kw):
    a = dict(q=A, pages=A, bits=4, group=64, T=4, starts=A, lens=A, table=A, B=4, blocks=8, ptab=A, plen=A, pblocks=4, hq=8, hkv=2, hd=128,
             n=100, page=16, scale=0.1, out=A, ws=A, wb=1 << 40)
    a.update(kw)
    return L.load().sc_prefix_attn_q(a["q"], a["pages"], a["bits"], a["group"], a["T"], a["starts"], a["lens"], a["table"], a["B"], a["blocks"],
                                     a["ptab"], a["plen"], a["pblocks"], a["hq"], a["hkv"], a["hd"], a["n"], a["page"], a["scale"], a["out"],
                                     a["ws"], a["wb"], None)


@pytest.mark.parametrize("kw,code", [(dict(hd=96), L.SC_ERR_UNSUPPORTED), (dict(bits=5), L.SC_ERR_UNSUPPORTED), (dict(group=128), L.SC_ERR_UNSUPPORTED),
                                     (dict(page=8), L.SC_ERR_UNSUPPORTED), (dict(page=48), L.SC_ERR_UNSUPPORTED), (dict(page=1 << 16), L.SC_ERR_UNSUPPORTED),
                                     (dict(T=0), L.SC_ERR_SHAPE), (dict(B=0), L.SC_ERR_SHAPE), (dict(B=65536), L.SC_ERR_SHAPE),
                                     (dict(blocks=0), L.SC_ERR_SHAPE), (dict(n=0), L.SC_ERR_SHAPE), (dict(hq=7), L.SC_ERR_SHAPE),
                                     (dict(hkv=0), L.SC_ERR_SHAPE), (dict(n=1 << 27), L.SC_ERR_SHAPE), (dict(T=1 << 29), L.SC_ERR_SHAPE),
                                     (dict(blocks=1 << 28), L.SC_ERR_SHAPE), (dict(pblocks=1 << 28), L.SC_ERR_SHAPE), (dict(scale=0.0), L.SC_ERR_ARG),
                                     (dict(scale=-1.0), L.SC_ERR_ARG), (dict(scale=float("nan")), L.SC_ERR_ARG), (dict(scale=float("inf")), L.SC_ERR_ARG),
                                     (dict(scale=6e28), L.SC_ERR_ARG), (dict(ptab=None), L.SC_ERR_ARG), (dict(pblocks=0), L.SC_ERR_ARG),
                                     (dict(q=None), L.SC_ERR_ARG), (dict(pages=None), L.SC_ERR_ARG), (dict(out=None), L.SC_ERR_ARG),
                                     (dict(q=A + 2), L.SC_ERR_ARG), (dict(pages=A + 8), L.SC_ERR_ARG), (dict(ws=A + 4), L.SC_ERR_ARG),
                                     (dict(blocks=4096, wb=16), L.SC_ERR_WORKSPACE), (dict(blocks=4096, ws=None), L.SC_ERR_WORKSPACE)])
def test_attn_refuses(kw, code):
    assert attn(**kw) == code and L.last_error()


def test_attn_workspace_is_bounded():
    for T, B in [(1, 1), (1, 4096), (256, 256), (16384, 1), (16384, 64), (100000, 1000)]:
        for bits, group in [(4, 64), (8, 32)]:
            n = ops.prefix_attn_q_workspace_bytes(T, B, 32, 8, 128, 4096, 4096, 16, bits, group)
            assert 0 <= n <= 64 * max(T, 148) * 32 * 130 * 4
    assert L.load().sc_prefix_attn_q_workspace_bytes(4, 4, 7, 2, 128, 4, 64, 8, 8, 16) == 0
    assert L.load().sc_prefix_attn_q_workspace_bytes(4, 4, 8, 2, 96, 4, 64, 8, 8, 16) == 0


def test_tensors_are_checked():
    z, t = torch.zeros(4, dtype=torch.int32), torch.zeros(4, 2, dtype=torch.int32)
    pool = ops.quant_pages(2, 1, 16, 64, device=torch.device("cpu"))
    tab, q = torch.zeros(4, 32), torch.zeros(4, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.paged_rope_append_q(torch.zeros(1, 192), z, z, z, tab, tab, q[:1], pool)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.paged_read_q(pool, z)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.prefix_attn_q(q, pool, torch.zeros(5, dtype=torch.int32), z, t)
    for bad in (pool._replace(data=pool.data[..., :-16]), pool._replace(data=pool.data[0]), pool._replace(data=pool.data.view(torch.int8)),
                pool._replace(bits=8), pool._replace(head_dim=128), pool._replace(page_size=32)):
        with pytest.raises(ValueError, match="pages"):
            ops.prefix_attn_q(q, bad, z, z, t)
        with pytest.raises(ValueError, match="pages"):
            ops.paged_read_q(bad, z)
        with pytest.raises(ValueError, match="pages"):
            ops.paged_rope_append_q(torch.zeros(1, 192), z, z, z, tab, tab, q[:1], bad)
    with pytest.raises(ValueError, match="together"):
        ops.paged_read_q(pool, z, k_out=torch.zeros(4, 1, 64))
    with pytest.raises(ValueError, match="float16 or float32"):
        ops.paged_read_q(pool, z, dtype=torch.float64)


# ------------------------------------------------------------------------------------------------ the oracle itself

@pytest.mark.parametrize("hd,bits,group", KINDS)
def test_layout_gives_every_bit_one_place(hd, bits, group):
    seen = np.zeros(oq.block_bytes(hd, bits, group) * 8, int)
    for side in (0, 1):
        for tok in range(16):
            for d in range(hd):
                byte, shift = oq.place(side, tok, d, hd, bits, group)
                seen[byte * 8 + shift:byte * 8 + shift + bits] += 1
            for g in range(hd // group):
                at = oq.meta_place(side, tok, g, hd, bits, group)
                seen[at * 8:at * 8 + 32] += 1
    assert (seen == 1).all()


@pytest.mark.parametrize("hd,bits,group", KINDS)
def test_oracle_quantises_within_half_a_step(hd, bits, group):
    rng = np.random.default_rng(0)
    for scale, shift in [(1.0, 0.0), (1e-4, 0.0), (3000.0, 100.0), (1e-3, 50.0), (0.0, 1.3)]:
        x = (rng.standard_normal((3, 2, 16, hd)) * scale + shift).astype(np.float32)
        codes, s, b = oq.quantise(x, bits, group)
        step = np.repeat(s.astype(np.float64), group, -1)
        assert (np.abs(oq.value(codes, s, b) - x) <= step / 2 * (1 + 2.0**-40)).all() or scale == 0.0
        assert codes.min() >= 0 and codes.max() <= 2**bits - 1
        data = oq.fill(x, x[::-1], bits, group)
        k, v = oq.values(data, hd, 16, bits, group)
        assert np.array_equal(k, oq.value(codes, s, b)) and np.array_equal(v, oq.value(codes, s, b)[::-1])
        one = np.zeros_like(data)
        for slot in range(48):
            for side, y in ((0, x), (1, x[::-1])):
                c1, s1, b1 = oq.quantise(y[slot // 16, :, slot % 16], bits, group)
                oq.put(one, slot, 16, side, c1, s1, b1, bits, group)
        assert np.array_equal(one, data)


def test_floor16():
    x = np.array([0.0, 1e-9, -1e-9, 1.0, 1.0004, -1.0004, 65504.0, 70000.0, -70000.0, 2.0**-24, -(2.0**-24)])
    assert oq.floor16(x).tolist() == [0.0, 0.0, -(2.0**-24), 1.0, 1.0, -1.0009765625, 65504.0, 65504.0, -np.inf, 2.0**-24, -(2.0**-24)]


# ------------------------------------------------------------------------------------------------ the cache class

def test_cache_in_codes():
    from shardcompute_b200.parallel import PagedKVCache

    a = dict(num_layers=2, kv_heads=3, head_dim=64, n_pages=4, max_batch=2, max_len=64, device=torch.device("cpu"))
    for bits, group in [(4, 32), (8, 64)]:
        c = PagedKVCache(**a, bits=bits, group_size=group)
        assert c.k is None and c.v is None and [layer.pages.data.shape for layer in c.layers()] == [(4, 3, oq.block_bytes(64, bits, group))] * 2
        assert all(layer.pages.bits == bits and layer.pages.group_size == group for layer in c.layers())
        c.check()
    for kw in (dict(bits=2), dict(bits=16), dict(bits=4, group_size=128), dict(bits=8, group_size=16)):
        with pytest.raises(ValueError, match="unsupported"):
            PagedKVCache(**a, **kw)
    full = PagedKVCache(**a)
    assert all(layer.pages is None for layer in full.layers())
    full.block_table[1, 0], full.lens[1] = 2, 3
    full.k[1, 2, :, :3] = torch.arange(3.0).view(1, 3, 1)
    k, v = full.read(1, 1, torch.float32)
    assert k.shape == (3, 3, 64) and k[:, 0, 0].tolist() == [0.0, 1.0, 2.0] and (v == 0).all()
