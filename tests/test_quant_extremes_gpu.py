"""The paged cache in 8 or 4 bits where values, queries and scales stand out, against oracle/quant_pages.py."""

import math

import numpy as np
import pytest
import torch

from oracle import quant_pages as oq
from shardcompute_b200 import _lib as L
from shardcompute_b200 import ops
from shardcompute_b200.parallel import PagedKVCache
from tests.test_quant_pages_gpu import attn_bound, i32, make_attn, pool, run_attn

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------ values that are not finite

@pytest.mark.parametrize("bad", [np.inf, -np.inf, 1e7], ids=["inf", "-inf", "1e7"])
@pytest.mark.parametrize("hd,bits,group", [(128, 4, 64), (128, 8, 32), (64, 4, 32)])
@pytest.mark.parametrize("longest", [700, 20000], ids=["clusters", "line"])
def test_a_group_that_is_not_finite_leaves_the_others(cuda, rng, longest, hd, bits, group, bad):
    """A value of v that is not finite (or past what a group can hold) makes its group's dims NaN in the rows that see it; the other
    groups' dims of these rows, and all of the others, are what they are without it, within the bound of finite values."""
    hq, hkv, lens, new = 4, 2, [longest, 90, 50], [1, 4, 1]
    d = make_attn(rng, hq, hkv, hd, 16, bits, group, 0, lens, new, dirty=False)
    assert (ops.prefix_attn_q_workspace_bytes(8, 3, hq, hkv, hd, d["table"].shape[1], 0, 16, bits, group) == 0) == (longest == 700)
    # through the append: token 333 of the first request, the last but one of the second, in head 1, dim 5
    pages, at = pool(d, cuda), [(0, 333), (1, 88)]
    slots = [int(d["table"][b, t // 16]) * 16 + t % 16 for b, t in at]
    x = np.zeros((2, 1 + 2 * hkv, hd), np.float32)
    x[:, 1:] = rng.standard_normal((2, 2 * hkv, hd))
    x[:, 1 + hkv + 1, 5] = bad
    one = torch.ones(4, hd // 2, device=cuda)
    ops.paged_rope_append_q(torch.from_numpy(x.reshape(2, -1)).to(cuda), i32([0, 2], cuda), i32(slots, cuda), i32([0, 0], cuda), one, one * 0,
                            torch.empty(2, hd, dtype=torch.float16, device=cuda), pages)
    d["data"] = pages.data.cpu().numpy()
    got = run_attn(cuda, d, with_prefix=False)[:6].double().cpu().numpy().reshape(6, hq, hd)
    # the oracle on the same bytes with zeros in that group: the other dims do not depend on it
    finite = d["data"].copy()
    for s in slots:
        m = s % 16
        base = oq.meta_place(1, m, 0, hd, bits, group)
        held = finite[s // 16, 1, base:base + 4].view(np.float16)
        assert np.isnan(held[1])  # what the append writes of such a group
        finite[s // 16, 1, base:base + 4] = 0
    want, mass, dot, keys, tail = oq.attention(d["q"].double().numpy(), finite, d["start"], d["lens"], d["table"], d["ptab"], 0, hq, hd, 16, bits,
                                               group, 1 / math.sqrt(hd))
    sees = np.zeros(got.shape, bool)
    sees[[0, 3, 4], 2:, :group] = True  # heads 2, 3 are of kv head 1; of the second request's rows the last two see token 88
    assert np.array_equal(np.isnan(got), sees)
    err, bound = np.abs(got - want), attn_bound(want, mass, dot, keys, tail, hd)
    assert (err[~sees] <= bound[~sees]).all(), np.nanmax(np.where(sees, 0, err / bound))
    assert L.load().sc_prefix_attn_device_error(1) == 0


# ------------------------------------------------------------------------------------------------ queries with a dim that stands out

@pytest.mark.parametrize("bits,hd,group", [(4, 128, 64), (4, 128, 32), (4, 64, 64), (8, 128, 64), (8, 64, 32)])
@pytest.mark.parametrize("large", [2000.0, 20000.0])
@pytest.mark.parametrize("drafts", [False, True])
def test_scores_beside_a_dim_that_stands_out(cuda, rng, drafts, large, bits, hd, group):
    """Two tokens a request whose scores are equal, though their codes differ: q is the same over eight dims, over which both tokens'
    codes have one sum.  One dim of q is far larger than the rest, over a code of 1 in both; each head has another such dim, so that every
    place of a code in its word is met.  The second token's value is 1, the first one's 0, so that the output is 1 / (1 + exp(-x)), x the
    difference of the scores.  S adds 16 dims at a time to an fp32 sum, off by less than 2^-23 of the largest product that may stand there,
    2^bits max |q|: hd / 16 of that, which the scale makes 2 here."""
    B, hq, most = 32, 8, 2**bits - 1
    limit = hd / 16 * 2.0**-23 * 2**bits * large
    codes = rng.integers(1, most + 1, (B, 2, hd // 8, 8))
    for a, c in ((codes[b, 0, g], codes[b, 1, g]) for b in range(B) for g in range(hd // 8)):
        while a.sum() != c.sum():
            i = rng.integers(0, 8)
            c[i] = min(max(c[i] + np.sign(a.sum() - c.sum()), 1), most)
    codes[:, :, 0] = 1
    assert (codes[:, 0].sum(-1) == codes[:, 1].sum(-1)).all() and (codes[:, 0] != codes[:, 1]).any()
    data, n = np.zeros((B, 1, oq.block_bytes(hd, bits, group)), np.uint8), hd // group
    one, zero = np.ones((1, n), np.float16), np.zeros((1, n), np.float16)
    for b in range(B):
        for t in (0, 1):
            oq.put(data, 16 * b + t, 16, 0, codes[b, t].reshape(1, hd), one, zero, bits, group)
            oq.put(data, 16 * b + t, 16, 1, np.full((1, hd), t), one, zero, bits, group)
    T = 3 * B if drafts else B  # tiles of 16 rows; the first two of a draft's three tokens see one token or none
    q = np.repeat(rng.standard_normal((T, hq, hd // 8)), 8, -1)
    q[..., :8] = 0.0
    q[:, np.arange(hq), np.arange(hq)] = large
    pages = ops.QuantPages(torch.from_numpy(data).to(cuda), hd, 16, bits, group)
    out = ops.prefix_attn_q(torch.from_numpy(q.reshape(T, -1)).half().to(cuda), pages, i32(np.arange(B + 1) * (T // B), cuda), i32([2] * B, cuda),
                            i32(np.arange(B)[:, None], cuda), scale=2.0 / limit)
    got = out.double().cpu().numpy().reshape(B, -1, hq, hd)[:, -1]
    # the weights' rounding to fp16 and the output's: 3 2^-11 of a value, 8e-3 of x
    assert (np.abs(np.log(got / (1 - got))) <= 2.008).all(), (got.min(), got.max())


# ------------------------------------------------------------------------------------------------ the ends of fp16's range

@pytest.mark.parametrize("src", [torch.float16, torch.float32])
@pytest.mark.parametrize("hd,bits,group", [(128, 4, 64), (128, 8, 64), (64, 4, 32), (64, 8, 32)])
def test_what_fp16_holds_is_held(cuda, rng, hd, bits, group, src):
    """Groups up to +-65504: codes, scales and biases as the oracle's, every value at most half a step off, and finite as fp16."""
    ends = [(0, 65504), (-65504, 65504), (1, 65504), (-65504, 0), (65504, 65504), (-65504, -65504), (65472, 65504), (-3, 65504), (30000, 65504),
            (-65504, 65472), (1e-3, 65504), (-40000, 60000)]
    rows, hkv = len(ends), 2
    x = np.stack([lo + (hi - lo) * rng.random((hkv, hd // group, group)) for lo, hi in ends])
    x[..., 0], x[..., 1] = np.array(ends)[:, :1, None], np.array(ends)[:, 1:, None]
    x = torch.from_numpy(x.reshape(rows, hkv, hd)).float().clamp(-65504, 65504).to(src)
    pages, one, at = ops.quant_pages(1, hkv, 16, hd, bits, group, cuda), torch.ones(16, hd // 2, device=cuda), i32(np.arange(rows), cuda)
    qkv = torch.cat([x.new_zeros(rows, 1, hd), x, x], 1).reshape(rows, -1).to(cuda)
    ops.paged_rope_append_q(qkv, i32([0, rows], cuda), at, at, one, one * 0, torch.empty(rows, hd, dtype=torch.float16, device=cuda), pages)
    want, s, b = oq.quantise(x.float().numpy(), bits, group)
    assert np.isfinite(b).all()
    for codes, scales, biases in oq.take(pages.data.cpu().numpy(), hd, 16, bits, group):
        assert np.array_equal(codes[0, :, :rows].swapaxes(0, 1), want)
        assert np.array_equal(scales[0, :, :rows].swapaxes(0, 1), s) and np.array_equal(biases[0, :, :rows].swapaxes(0, 1), b)
    for v in ops.paged_read_q(pages, at, dtype=torch.float32):
        # s / 2, and the rounding of s c + b to fp32
        limit = np.repeat(s.astype(np.float64), group, -1) / 2 + 2.0**-24 * 65536
        assert (np.abs(v.double().cpu().numpy() - x.double().numpy()) <= limit).all()
    assert all(bool(torch.isfinite(v).all()) for v in ops.paged_read_q(pages, at))
    # a row that sees all of it, by few rows and by many
    for new in (1, 80):
        q = torch.from_numpy(rng.standard_normal((new, 2 * hkv * hd)) * 1e-4).half()
        table, start, lens = np.zeros((1, 1), np.int32), [0, new], [rows]
        out = ops.prefix_attn_q(q.to(cuda), pages, i32(start, cuda), i32(lens, cuda), i32(table, cuda))
        assert torch.isfinite(out[-1]).all()


def test_append_past_fp16s_range(cuda):
    """A value past +-65504 in fp32 makes its group NaN, the last one within it does not."""
    hd, values = 64, [65504.0, 65505.0, -65504.0, -65505.0, 1e6]
    x = torch.zeros(len(values), 3, hd)
    x[:, 2, 7] = torch.tensor(values)
    for bits in (4, 8):
        pages, one, at = ops.quant_pages(1, 1, 16, hd, bits, 32, cuda), torch.ones(16, hd // 2, device=cuda), i32(np.arange(len(values)), cuda)
        ops.paged_rope_append_q(x.reshape(len(values), -1).to(cuda), i32([0, len(values)], cuda), at, at, one, one * 0,
                                torch.empty(len(values), hd, dtype=torch.float16, device=cuda), pages)
        k, v = ops.paged_read_q(pages, at)
        assert torch.isfinite(k).all() and torch.isfinite(v[..., 32:]).all()
        assert v[:, 0, :32].isnan().all(-1).tolist() == [False, True, False, True, True] == v[:, 0, :32].isnan().any(-1).tolist()


# ------------------------------------------------------------------------------------------------ PagedKVCache.read

@pytest.mark.parametrize("kind", [dict(bits=8), dict(bits=4, group_size=32), dict(dtype=torch.float16), dict(dtype=torch.float32)],
                         ids=["8", "4", "f16", "f32"])
def test_read_without_a_page(cuda, kind):
    """In codes and in full alike: zeros where the table has no page, the pages' own type unless another is asked for."""
    c = PagedKVCache(num_layers=1, kv_heads=2, head_dim=64, n_pages=4, max_batch=2, max_len=64, max_tokens=40, device=cuda, **kind)
    c.reserve([40, 0])
    for pool_ in ([p.data for p in c.pages] if c.pages else [c.k, c.v]):
        pool_.fill_(60 if c.pages else 3.0)
    c.block_table[0, 1] = -1
    for x in c.read(0, 0):
        assert x.dtype is kind.get("dtype", torch.float16) and x.shape == (40, 2, 64)
        assert (x[16:32] == 0).all() and (x[:16] != 0).all() and (x[32:] != 0).all()
