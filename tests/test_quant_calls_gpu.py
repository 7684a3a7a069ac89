"""The operators over pages in 8 or 4 bits as calls meet them: many rows from fp16, drafts in clusters, tables far wider than the lengths,
PagedKVCache with room for much longer requests than it holds."""

import math

import numpy as np
import pytest
import torch

from oracle import quant_pages as oq
from shardcompute_b200 import ops
from shardcompute_b200.parallel import PagedKVCache
from tests.test_quant_many_rows_gpu import FP16, bounds, check, oracle, plan_of
from tests.test_quant_pages_gpu import KINDS, check_append, make_attn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd,bits,group", KINDS)
def test_append_of_many_rows_in_fp16(cuda, rng, hd, bits, group):
    """Slots and positions that are none, rows behind the last, every head layout's items beside one another in a warp."""
    for hq, hkv, page, rows in ((4, 2, 16, 130), (1, 3, 32, 64), (7, 1, 48, 33)):
        check_append(cuda, rng, "f16", hq, hkv, hd, page, bits, group, rows)


@pytest.mark.parametrize("hd,bits,group", KINDS)
@pytest.mark.parametrize("B,hq,hkv,own,prefix", [(16, 8, 2, 400, 300), (8, 8, 2, 700, 0), (4, 32, 8, 900, 200)])
def test_drafts_in_clusters(cuda, rng, hd, bits, group, B, hq, hkv, own, prefix):
    """Tiles of 16 rows, two and more a request, over keys that several CTAs share."""
    new = [4] + [int(x) for x in rng.integers(3, 9, B - 1)]
    lens = [n + int(rng.integers(0, own)) for n in new]
    lens[0] = own
    d = make_attn(rng, hq, hkv, hd, 16, bits, group, prefix, lens, new)
    plan = plan_of(d, hq)
    assert plan.cluster >= 2 and len(d["q"]) * (hq // hkv) > 8 * B
    check(cuda, d, hq, "few")


def widened(d, own, prefix):
    """The same call with tables that could hold `own` and `prefix` tokens."""
    page = d["kind"][1]
    table, ptab = np.full((len(d["lens"]), own // page), -1, np.int32), np.full(prefix // page, -1, np.int32)
    table[:, :d["table"].shape[1]], ptab[:len(d["ptab"])] = d["table"], d["ptab"]
    return dict(d, table=table, ptab=ptab)


@pytest.mark.parametrize("hd,bits,group", [(128, 4, 64), (64, 8, 32)])
@pytest.mark.parametrize("B,own,prefix,new", [(48, 200, 3000, 1), (16, 300, 0, 1), (1, 40, 700, 1), (2, 200, 100, 3), (3, 400, 100, 150)])
def test_tables_far_wider_than_the_lengths(cuda, rng, hd, bits, group, B, own, prefix, new):
    """As a cache with room for 32768 tokens a request hands them over: another plan, the same answer."""
    lens = [own] + [new + int(x) for x in rng.integers(0, own - new, B - 1)]
    d = make_attn(rng, 8, 2, hd, 16, bits, group, prefix, lens, [new] * B, dirty=False)
    wide = widened(d, 32768, 32768 if prefix else 16)
    kind = plan_of(wide, 8).kind
    assert plan_of(wide, 8) != plan_of(d, 8)
    want = oracle(d, 8, kind)
    check(cuda, wide, 8, kind, prepared=want)


@pytest.mark.parametrize("bits,group", [(4, 64), (8, 32)])
@pytest.mark.parametrize("max_len,max_prefix", [(32768, 32768), (32768, 0), (96, 64)])
def test_a_cache_with_room_for_more(cuda, rng, bits, group, max_len, max_prefix):
    """reserve, append and attention through PagedKVCache: a prefix, chunks, single tokens, drafts, against float64 attention over the bytes
    that it holds by then."""
    hq, hkv, hd, B, T = 8, 2, 64, 5, 96
    c = PagedKVCache(1, hkv, hd, 64, B, max_len, max_prefix=max_prefix, max_tokens=T, device=cuda, bits=bits, group_size=group)
    pages = c.layers()[0].pages
    ang = torch.rand(min(c.max_positions, 400), hd // 2, device=cuda) * 6

    def step(new):
        st = c.reserve(new)
        c.check()
        q = torch.zeros(T, hq * hd, dtype=torch.float16, device=cuda)
        ops.paged_rope_append_q(torch.randn(T, (hq + 2 * hkv) * hd, device=cuda), st.q_start, st.slots, st.positions, ang.cos(), ang.sin(), q, pages)
        out = ops.prefix_attn_q(q, pages, st.q_start, st.kv_lens, c.block_table, c.prefix_table, c.prefix_len)
        plan = ops.prefix_attn_q_plan(T, B, hq, hkv, hd, c.block_table.shape[1], c.prefix_table.numel() if max_prefix else 0, 16, bits, group)
        rows, prefix = sum(new), int(c.prefix_len) if max_prefix else 0
        want, *parts = oq.attention(q[:rows].double().cpu().numpy(), pages.data.cpu().numpy(), st.q_start.tolist(), st.kv_lens.tolist(),
                                    c.block_table.cpu().numpy(), c.prefix_table.cpu().numpy() if max_prefix else [0], prefix, hq, hd, 16, bits, group,
                                    1 / math.sqrt(hd), fp16=FP16[plan.kind])
        each, whole = bounds(want, *parts, hd)
        err = np.abs(out[:rows].double().cpu().numpy().reshape(want.shape) - want)
        assert (err <= each).all() and (np.linalg.norm(err, axis=-1) <= whole).all()
        assert (out[rows:] == 0).all()

    if max_prefix:
        step([50, 0, 0, 0, 0])
        c.share_prefix(0)
    for new in ([20, 33, 1, 0, 40], [1, 1, 1, 1, 1], [3, 1, 5, 2, 1], [0, 0, 0, 1, 0]):
        step(new)
        c.truncate([max(int(n) - 1, 0) for n in c.lens])
        c.check()
