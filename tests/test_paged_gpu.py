"""The paged cache's operators against oracle/paged.py: bookkeeping exactly, the append to one rounding, the attention
within a bound that is derived from the number formats (attn_bound)."""

import math

import numpy as np
import pytest
import torch

from oracle import paged as op
from shardcompute_b200 import _lib as L
from shardcompute_b200 import ops

pytestmark = pytest.mark.gpu

DT = {"f16": torch.float16, "f32": torch.float32}


def i32(a, dev):
    return torch.from_numpy(np.ascontiguousarray(np.asarray(a, np.int32))).to(dev)


def scattered(rng, lens, page, extra=1, spare=20):
    """A block table over pages in random order, and the stack of the others."""
    blocks = [-(-int(n) // page) for n in lens]
    total = sum(blocks)
    ids = rng.permutation(total + spare).astype(np.int32)
    table = np.full((len(lens), max(blocks) + extra), -1, np.int32)
    at = 0
    for b, n in enumerate(blocks):
        table[b, :n] = ids[at:at + n]
        at += n
    free = np.full(total + spare, -1, np.int32)
    free[:spare] = ids[total:]
    return table, free, spare


# ------------------------------------------------------------------------------------------------ reserve

def check_reserve(cuda, lens, new, table, free, count, page, max_tokens, prefix, in_place=False):
    st, wtable, wkv, wstart, wslots, wpos, wcount = op.reserve(lens, new, table, free, count, page, max_tokens, prefix)
    tl, tt, tc = i32(lens, cuda), i32(table, cuda), i32([count], cuda)
    tf = i32(free, cuda)
    slots, pos = torch.full((max_tokens,), -9, dtype=torch.int32, device=cuda), torch.full((max_tokens,), -8, dtype=torch.int32, device=cuda)
    got = ops.paged_reserve(tl, i32(new, cuda), tt, tf, tc, page, prefix_len=i32([prefix], cuda), slots=slots, positions=pos,
                            kv_lens=tl if in_place else None, free_count_out=tc if in_place else None)
    assert int(got.status) == st
    assert np.array_equal(tt.cpu().numpy(), wtable)
    assert np.array_equal(got.kv_lens.cpu().numpy(), wkv)
    assert np.array_equal(got.q_start.cpu().numpy(), wstart)
    n = len(wslots)
    assert np.array_equal(slots[:n].cpu().numpy(), wslots) and (slots[n:] == -9).all()
    assert np.array_equal(pos[:n].cpu().numpy(), wpos) and (pos[n:] == -8).all()
    assert int(got.free_count) == wcount
    assert np.array_equal(tf.cpu().numpy(), free)
    if not in_place:
        assert np.array_equal(tl.cpu().numpy(), lens) and int(tc) == count
    return st


@pytest.mark.parametrize("B,page,max_len,max_new", [(1, 16, 0, 1), (1, 16, 15, 40), (7, 16, 100, 1), (33, 32, 64, 70), (600, 1, 9, 3),
                                                    (513, 128, 700, 300), (5000, 16, 40, 5)])
@pytest.mark.parametrize("in_place", [False, True])
def test_reserve(cuda, rng, B, page, max_len, max_new, in_place):
    lens, new = rng.integers(0, max_len + 1, B), rng.integers(0, max_new + 1, B)
    extra = -(-max_new // page) + 1
    table, free, count = scattered(rng, lens, page, extra=extra, spare=B * extra)
    assert check_reserve(cuda, lens, new, table, free, count, page, max(1, int(new.sum())) + int(rng.integers(0, 50)), 1234, in_place) == 0


def test_reserve_exact_fit_and_full_pages(cuda, rng):
    # lengths on page borders; exactly the last free page is taken; exactly max_tokens rows
    lens, new = np.array([16, 32, 0, 47]), np.array([1, 0, 16, 1])
    table, free, count = scattered(rng, lens, 16, extra=1, spare=2)
    assert check_reserve(cuda, lens, new, table, free, count, 16, 18, 0) == 0
    # nothing to reserve, no free page at all
    assert check_reserve(cuda, lens, np.zeros(4, int), table, free, 0, 16, 1, 0) == 0


@pytest.mark.parametrize("case", ["pages", "table", "tokens", "negative_len", "negative_new", "count", "huge", "many"])
@pytest.mark.parametrize("in_place", [False, True])
def test_reserve_refuses_on_the_device(cuda, rng, case, in_place):
    lens, new = np.array([16, 32, 0, 47]), np.array([1, 5, 16, 1])
    table, free, count = scattered(rng, lens, 16, extra=1, spare=8)
    rows, want = 40, {"pages": 1, "table": 2, "tokens": 4, "negative_len": 8, "negative_new": 8, "count": 16, "huge": 1 + 2 + 4, "many": 4 + 8}[case]
    if case == "pages":
        count = 2
    if case == "table":
        new[3] = 18
    if case == "tokens":
        rows = 22
    if case == "negative_len":
        lens[1] = -5
    if case == "negative_new":
        new[0] = -1
    if case == "count":
        count = 1000
    if case == "huge":  # the sum of the lengths passes 32 bits
        new[:] = 2**31 - 60
    if case == "many":
        new[:], rows = [-1, 5, 16, 17], 30
    assert check_reserve(cuda, lens, new, table, free, count, 16, rows, 0, in_place) == want


# ------------------------------------------------------------------------------------------------ truncate

def check_truncate(cuda, lens, keep, table, free, count, page, in_place=False):
    st, wlens, wfree, wcount = op.truncate(lens, keep, table, free, count, page)
    tl, tf, tc, tt = i32(lens, cuda), i32(free, cuda), i32([count], cuda), i32(table, cuda)
    got_lens, got_count, status = ops.paged_truncate(tl, i32(keep, cuda), tt, tf, tc, page, lens_out=tl if in_place else None,
                                                     free_count_out=tc if in_place else None)
    assert int(status) == st
    assert np.array_equal(got_lens.cpu().numpy(), wlens) and int(got_count) == wcount
    assert np.array_equal(tf.cpu().numpy(), wfree) and np.array_equal(tt.cpu().numpy(), table)
    return st


@pytest.mark.parametrize("B,page,max_len", [(1, 16, 1), (8, 16, 100), (700, 32, 90), (3000, 1, 7), (5000, 128, 300)])
@pytest.mark.parametrize("in_place", [False, True])
def test_truncate(cuda, rng, B, page, max_len, in_place):
    lens = rng.integers(0, max_len + 1, B)
    keep = np.where(rng.random(B) < 0.3, 0, lens - rng.integers(-3, 9, B))  # some negative, some past the length
    table, free, count = scattered(rng, lens, page)
    assert check_truncate(cuda, lens, keep, table, free, count, page, in_place) == 0


@pytest.mark.parametrize("case", ["twice", "table", "negative", "count"])
def test_truncate_refuses_on_the_device(cuda, rng, case):
    lens, keep = np.array([33, 16, 5]), np.array([0, 16, 0])
    table, free, count = scattered(rng, lens, 16, spare=3)
    want = {"twice": 1, "table": 2, "negative": 8, "count": 16}[case]
    if case == "twice":
        count = len(free) - 3
    if case == "table":
        lens[0] = 100
    if case == "negative":
        lens[2] = -1
    if case == "count":
        count = -1
    assert check_truncate(cuda, lens, keep, table, free, count, 16) == want


# ------------------------------------------------------------------------------------------------ append

@pytest.mark.parametrize("src,cache", [("f32", "f32"), ("f32", "f16"), ("f16", "f16"), ("f16", "f32")])
@pytest.mark.parametrize("hq,hkv,hd,page,rows", [(32, 8, 128, 16, 5), (4, 4, 64, 32, 67), (3, 1, 40, 1, 9), (6, 2, 8, 64, 1)])
def test_append(cuda, rng, src, cache, hq, hkv, hd, page, rows):
    pad, n_pages, max_pos = 3, -(-2 * rows // page) + 2, 300
    x = torch.from_numpy(rng.standard_normal((rows + pad, (hq + 2 * hkv) * hd)).astype(np.float32)).to(DT[src])
    pos = rng.integers(0, max_pos, rows + pad)
    slots = rng.permutation(n_pages * page)[:rows + pad]
    if rows > 4:  # not written: slots and positions that are none
        slots[0], slots[1], pos[2], pos[3] = -1, n_pages * page, max_pos, -1
    ang = rng.standard_normal((max_pos, hd // 2)) * 3
    cos, sin = np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)
    k0 = torch.from_numpy(rng.standard_normal((n_pages, hkv, page, hd))).to(DT[cache])
    v0 = torch.from_numpy(rng.standard_normal((n_pages, hkv, page, hd))).to(DT[cache])
    q0 = torch.full((rows + pad, hq * hd), 7.0, dtype=DT[cache])
    q, k, v = q0.to(cuda), k0.to(cuda), v0.to(cuda)
    ops.paged_rope_append(x.to(cuda), i32([0, rows // 2, rows], cuda), i32(slots, cuda), i32(pos, cuda), torch.from_numpy(cos).to(cuda),
                          torch.from_numpy(sin).to(cuda), q, k, v)
    h = x.double().numpy().reshape(rows + pad, hq + 2 * hkv, hd)
    there = (pos >= 0) & (pos < max_pos)
    cos1, sin1 = np.concatenate([cos, np.ones((1, hd // 2), np.float32)]), np.concatenate([sin, np.zeros((1, hd // 2), np.float32)])
    turned = op.rotate(h[:, : hq + hkv], np.where(there, pos, max_pos), cos1, sin1)
    wq, wk, wv = q0.double().numpy(), k0.double().numpy(), v0.double().numpy()
    wq[:rows] = turned[:rows, :hq].reshape(rows, -1)
    for t in range(rows):
        if there[t] and 0 <= slots[t] < n_pages * page:
            wk[slots[t] // page, :, slots[t] % page] = turned[t, hq:]
            wv[slots[t] // page, :, slots[t] % page] = h[t, hq + hkv:]
    # two fp32 products and their sum, each rounded (2^-24), then the cache's rounding
    size = np.abs(h[:, : hq + hkv]).max() * 2
    half_step = torch.finfo(DT[cache]).eps / 2 if cache == "f16" else 0.0
    tiny = 2.0**-25 if cache == "f16" else 0.0
    for got, want in ((q, wq), (k, wk)):
        assert (np.abs(got.double().cpu().numpy() - want) <= 3 * 2.0**-24 * size + (half_step * 1.001) * np.abs(want) + tiny).all()
    assert torch.equal(v.cpu(), torch.from_numpy(wv).to(DT[cache]))
    assert torch.equal(q[rows:].cpu(), q0[rows:])
    untouched = np.ones((n_pages, page), bool)
    for t in range(rows):
        if there[t] and 0 <= slots[t] < n_pages * page:
            untouched[slots[t] // page, slots[t] % page] = False
    u = torch.from_numpy(untouched)[:, None].expand(-1, hkv, -1)
    assert torch.equal(k.cpu()[u], k0[u])


def test_append_matches_rope_append(cuda, rng):
    """One request in pages against the contiguous cache: the same bits."""
    hq, hkv, hd, rows, page, max_pos = 8, 2, 64, 37, 16, 128
    qkv = torch.randn(rows, (hq + 2 * hkv) * hd, device=cuda)
    ang = torch.rand(max_pos, hd // 2, device=cuda) * 6
    cos, sin = ang.cos(), ang.sin()
    kc, vc = torch.zeros(1, hkv, 64, hd, device=cuda), torch.zeros(1, hkv, 64, hd, device=cuda)
    q1 = torch.empty(rows, hq * hd, device=cuda)
    ops.rope_append(qkv, 1, rows, hq, hkv, hd, torch.tensor([20], dtype=torch.int32, device=cuda), cos, sin, q1, kc, vc)
    kp, vp, q2 = torch.zeros(5, hkv, page, hd, device=cuda), torch.zeros(5, hkv, page, hd, device=cuda), torch.empty_like(q1)
    table = torch.tensor([4, 0, 2, 3], device=cuda)
    at = torch.arange(20, 20 + rows, device=cuda)
    slots = (table[at // page] * page + at % page).int()
    ops.paged_rope_append(qkv, i32([0, rows], cuda), slots, at.int(), cos, sin, q2, kp, vp)
    assert torch.equal(q1, q2)
    flat = lambda pool: pool[table].permute(1, 0, 2, 3).reshape(hkv, 64, hd)  # noqa: E731
    assert torch.equal(flat(kp), kc[0]) and torch.equal(flat(vp), vc[0])


# ------------------------------------------------------------------------------------------------ attention

def attn_bound(dtype, out, mass, dot, keys, tail, hd):
    """How far an output may be from float64.  With e = 2^-24 (a sum of fp32 products, each sum rounded or cut: 2 e), u
    the operands' own error, w_j the weights:
      score     ds = dot * (2 u + 2 (hd + 8) e) + 4 e dot     (products and sum; scaling and the difference to the maximum)
      weight    w_j (1 + 2 ds + 8 e + p): exp2 of it, p its rounding before the second product
      output    mass * (2 ds + 16 e + 2 p + u + 2 e (keys / 8 + 64)) for numerator and denominator, then its rounding
    fp16: u = 0, p = 2^-11, and weights below 2^-14 round to multiples of 2^-24: 2^-25 tail (tail = sum |v| / l).
    fp32: operands keep 2^-21, so u = p = 2^-21, and the output rounds by e."""
    e = 2.0**-24
    f16 = dtype == "f16"
    u, p = (0.0, 2.0**-11) if f16 else (2.0**-21, 2.0**-21)
    ds = (dot * (2 * u + 2 * (hd + 8) * e + 4 * e))[..., None]
    b = mass * (2 * ds + 16 * e + 2 * p + u + 2 * e * (keys[..., None] / 8 + 64))
    return b + (2.0**-25 * tail + 2.0**-11 * np.abs(out) * 1.01 + 2.0**-25 if f16 else e * np.abs(out) * 1.01 + 1e-30)


def make_attn(cuda, rng, dtype, hq, hkv, hd, page, prefix, lens, new, pad=2, dirty=True, scale_q=1.5):
    """Pools whose unused slots hold NaN and infinities, tables in random order, q."""
    B = len(lens)
    all_lens = list(lens) + [prefix]
    table, free, spare = scattered(rng, all_lens, page, spare=3)
    n_pages = len(free)
    k = rng.standard_normal((n_pages, hkv, page, hd)) + rng.standard_normal((1, hkv, 1, hd))
    v = rng.standard_normal((n_pages, hkv, page, hd)) + 0.3
    k, v = (torch.from_numpy(x).to(DT[dtype]) for x in (k, v))
    if dirty:
        used = np.zeros((n_pages, page), bool)
        for b, n in enumerate(all_lens):
            for i in range(n):
                used[table[b, i // page], i % page] = True
        u = torch.from_numpy(~used)[:, None, :].expand(-1, hkv, -1)
        k[u], v[u] = float("nan"), float("inf")
        v.view(-1)[::2] = torch.where(torch.isinf(v.view(-1)[::2]), torch.tensor(float("nan"), dtype=v.dtype), v.view(-1)[::2])
    rows = int(sum(new))
    q = torch.from_numpy(rng.standard_normal((rows + pad, hq * hd)) * scale_q).to(DT[dtype])
    start = np.concatenate([[0], np.cumsum(new)])
    ptab = table[B, : max(1, -(-prefix // page))] if prefix else np.zeros(1, np.int32)
    return dict(q=q, k=k, v=v, start=start, lens=np.array(lens), table=table[:B].copy(), ptab=ptab.copy(), prefix=prefix, pad=pad)


def run_attn(cuda, d, with_prefix=True, scale=None, workspace=None, out=None):
    if out is None:
        out = torch.full_like(d["q"], 5.0).to(cuda)
    pre = dict(prefix_table=i32(d["ptab"], cuda), prefix_len=i32([d["prefix"]], cuda)) if with_prefix else {}
    return ops.prefix_attn(d["q"].to(cuda), d["k"].to(cuda), d["v"].to(cuda), i32(d["start"], cuda), i32(d["lens"], cuda),
                           i32(d["table"], cuda), out=out, scale=scale, workspace=workspace, **pre)


def check_attn(cuda, dtype, d, hq, with_prefix=True, scale=None):
    hd = d["k"].shape[3]
    out = run_attn(cuda, d, with_prefix, scale)
    sc = 1 / math.sqrt(hd) if scale is None else scale
    want, mass, dot, keys, tail = op.attention(d["q"].double().numpy(), d["k"].double().numpy(), d["v"].double().numpy(), d["start"],
                                               d["lens"], d["table"], d["ptab"], d["prefix"] if with_prefix else 0, hq, sc)
    rows = int(d["start"][-1])
    got = out[:rows].double().cpu().numpy().reshape(want.shape)
    bound = attn_bound(dtype, want, mass, dot, keys, tail, hd)
    err = np.abs(got - want)
    assert np.isfinite(got).all()
    worst = np.unravel_index(np.argmax(err - bound), err.shape)
    assert (err <= bound).all(), (worst, got[worst], want[worst], bound[worst])
    assert (out[rows:] == 5.0).all()
    assert L.load().sc_prefix_attn_device_error(1) == 0
    return out


LAYOUTS = [(8, 2, 128), (4, 4, 64), (6, 1, 64), (24, 2, 128)]


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("hq,hkv,hd", LAYOUTS)
@pytest.mark.parametrize("page", [16, 64])
def test_attn_decode(cuda, rng, dtype, hq, hkv, hd, page):
    lens = [1, 16, 17, 5, 130, 64]
    d = make_attn(cuda, rng, dtype, hq, hkv, hd, page, 77, lens, [1] * 6)
    check_attn(cuda, dtype, d, hq)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("hq,hkv,hd", LAYOUTS)
@pytest.mark.parametrize("prefix", [0, 1, 16, 333])
def test_attn_ragged_chunks(cuda, rng, dtype, hq, hkv, hd, prefix):
    """Requests with no row, one row, drafts and chunks, with and without tokens before them."""
    new = [0, 1, 5, 37, 0, 16, 3]
    lens = [20, 1, 5, 60, 0, 16, 40]
    d = make_attn(cuda, rng, dtype, hq, hkv, hd, 16, prefix, lens, new)
    check_attn(cuda, dtype, d, hq)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("B,prefix,longest", [(1, 0, 1), (1, 2000, 700), (3, 5000, 40), (2, 0, 3001), (40, 129, 300)])
def test_attn_lengths(cuda, rng, dtype, B, prefix, longest):
    """From one token to many, few requests and many; values far apart in size."""
    lens = [longest] + [int(x) for x in rng.integers(1, longest + 1, B - 1)]
    d = make_attn(cuda, rng, dtype, 4, 1, 64, 32, prefix, lens, [1] * B)
    d["q"] *= torch.from_numpy(10.0 ** rng.integers(-3, 2, (d["q"].shape[0], 1))).to(d["q"].dtype)
    check_attn(cuda, dtype, d, 4)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("hq,hkv,hd", [(32, 4, 64), (64, 8, 128)])
@pytest.mark.parametrize("prefix,longest", [(1000, 60), (2900, 5)])
def test_attn_many_rows_many_tiles(cuda, rng, dtype, hq, hkv, hd, prefix, longest):
    """Several tiles of rows, each with several tiles of keys in one CTA, over and over: what one run leaves unordered
    shows in another."""
    new = [int(x) for x in rng.integers(1, 6, 16)]
    lens = [n + int(rng.integers(0, longest)) for n in new]
    d = make_attn(cuda, rng, dtype, hq, hkv, hd, 32, prefix, lens, new)
    out = check_attn(cuda, dtype, d, hq)
    for _ in range(8):
        assert torch.equal(out, run_attn(cuda, d))


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("hq,hkv,hd,page", [(32, 4, 64, 32), (24, 8, 128, 16)])
@pytest.mark.parametrize("prefix,longest", [(2900, 40), (1111, 700)])
def test_attn_shared_by_many_requests(cuda, rng, dtype, hq, hkv, hd, page, prefix, longest):
    """Batches large enough for the prefix to be taken once for all, with absent pages in it and in a request."""
    new = [int(x) for x in rng.integers(0, 6, 64)]
    lens = [n + int(rng.integers(0, longest)) for n in new]
    d = make_attn(cuda, rng, dtype, hq, hkv, hd, page, prefix, lens, new)
    check_attn(cuda, dtype, d, hq)
    d["ptab"][[0, len(d["ptab"]) - 1]] = [-1, len(d["k"]) + 5]
    d["table"][7, 0] = -3
    out = check_attn(cuda, dtype, d, hq)
    for _ in range(8):
        assert torch.equal(out, run_attn(cuda, d))


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("B,hq,hkv,hd", [(1, 8, 8, 128), (2, 6, 2, 64), (5, 8, 8, 128), (9, 16, 4, 64), (17, 8, 8, 128), (23, 5, 5, 64)])
@pytest.mark.parametrize("drafts", [False, True])
def test_attn_shares_joined(cuda, rng, dtype, B, hq, hkv, hd, drafts):
    """Few requests, whose keys several CTAs share: from two shares to eight, some without a key."""
    new = [int(x) for x in rng.integers(0, 8, B)] if drafts else [1] * B
    lens = [n + int(rng.integers(0, 2)) * int(rng.integers(0, 900)) for n in new]
    lens[0] = new[0] + 900
    for prefix in (0, 130):
        d = make_attn(cuda, rng, dtype, hq, hkv, hd, 16, prefix, lens, new)
        out = check_attn(cuda, dtype, d, hq)
        for _ in range(4):
            assert torch.equal(out, run_attn(cuda, d))


@pytest.mark.parametrize("hkv,hd,new,prefix,own,cut", [(4, 64, [1] * 48, 0, 16000, 2), (8, 128, [600], 16000, 600, 24), (8, 64, [600], 0, 16000, 24),
                                                       (4, 64, [1] * 128, 16000, 10, 24)])
def test_attn_long_rows_do_not_shrink(cuda, hkv, hd, new, prefix, own, cut):
    """fp32: the tensor cores cut their sums off towards zero, which must not add up over the keys.  With values above zero
    all of that is on one side, and the mean of out / exact - 1 shows it: at most 2^-23 for each of the `cut` sums that
    follow one another in the tensor cores.  The rest is rounded to nearest: 2^-24 for each of up to 1000 additions to a
    row's sum and to its weights', as a walk 2^-24 sqrt(1000) for a row, a fourteenth of that for the mean of 192 rows (the
    fewest here, 48 requests of 4 heads); four times it."""
    g = torch.Generator(device=cuda).manual_seed(7)
    B, page, G = len(new), 32, 4 if len(new) == 1 else 1 if prefix == 0 else 8
    per, pre = -(-own // page), -(-prefix // page)
    n_pages = B * per + pre
    k = torch.randn(n_pages, hkv, page, hd, device=cuda, generator=g)
    v = torch.rand(n_pages, hkv, page, hd, device=cuda, generator=g) + 0.5
    q = torch.randn(sum(new), hkv * G * hd, device=cuda, generator=g) * 0.25
    table = torch.arange(B * per, dtype=torch.int32, device=cuda).view(B, per)
    ptab = torch.arange(B * per, n_pages, dtype=torch.int32, device=cuda)
    start = np.concatenate([[0], np.cumsum(new)])
    kw = dict(prefix_table=ptab, prefix_len=i32([prefix], cuda)) if prefix else {}
    out = ops.prefix_attn(q, k, v, i32(start, cuda), i32([own] * B, cuda), table, **kw).view(-1, hkv, G, hd)
    total = 0.0
    for b in range(B):
        lo, hi = int(start[b]), int(start[b + 1])
        pos = torch.arange(own - (hi - lo), own, device=cuda)
        for h in range(hkv):
            flat = lambda x: torch.cat([x[ptab.long(), h].reshape(-1, hd)[:prefix], x[table[b].long(), h].reshape(-1, hd)[:own]]).double()
            s = q[lo:hi].view(-1, hkv, G, hd)[:, h].double() @ flat(k).T / math.sqrt(hd)
            s[..., prefix:].masked_fill_(torch.arange(own, device=cuda) > pos[:, None, None], float("-inf"))
            total += float((out[lo:hi, h].double() / (torch.softmax(s, -1) @ flat(v)) - 1).sum())
    assert abs(total / out.numel()) <= cut * 2.0**-23 + 4 * 2.0**-24 * math.sqrt(1000 / 192)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("new", [[1, 1, 1], [9, 40, 150]])
def test_attn_no_prefix_and_scale(cuda, rng, dtype, new):
    d = make_attn(cuda, rng, dtype, 8, 2, 64, 16, 0, [30, 200, 151], new)
    check_attn(cuda, dtype, d, 8, with_prefix=False, scale=0.3)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("prefix", [0, 50])
def test_attn_rows_that_see_nothing(cuda, rng, dtype, prefix):
    """More rows than tokens: the first ones see the prefix only, or nothing at all, and are zero."""
    d = make_attn(cuda, rng, dtype, 4, 2, 64, 16, prefix, [3, 0, 20], [7, 2, 20])
    out = check_attn(cuda, dtype, d, 4)
    if not prefix:
        assert (out[:4] == 0).all() and (out[7:9] == 0).all()


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("new", [[1, 1, 1], [5, 70, 33]])
def test_attn_absent_pages(cuda, rng, dtype, new):
    """Page ids outside the pool, in the prefix and among a request's own: their tokens are not seen."""
    d = make_attn(cuda, rng, dtype, 8, 2, 128, 16, 100, [40, 90, 33], new)
    d["ptab"][2], d["ptab"][5] = -1, 2**31 - 1
    d["table"][0, 0], d["table"][1, 3], d["table"][2, :] = d["k"].shape[0], -(2**31), -1
    check_attn(cuda, dtype, d, 8)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_attn_all_pages_absent(cuda, rng, dtype):
    d = make_attn(cuda, rng, dtype, 4, 2, 64, 16, 100, [40, 90], [1, 3])
    d["ptab"][:], d["table"][:] = -1, -1
    out = run_attn(cuda, d)
    assert (out[:4] == 0).all() and (out[4:] == 5.0).all()


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_attn_lengths_past_the_table(cuda, rng, dtype):
    """Lengths that the tables cannot hold are cut at the tables' ends."""
    d = make_attn(cuda, rng, dtype, 4, 2, 64, 16, 32, [32, 48], [1, 1], dirty=False)
    d["table"] = d["table"][:, :3]
    d["table"][0, 2] = d["table"][1, 2]
    full = dict(d, lens=np.array([48, 48]))
    over = dict(d, lens=np.array([4000, 2**31 - 1]), prefix=2**31 - 1)
    assert torch.equal(run_attn(cuda, full), run_attn(cuda, over))


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_attn_shared_page_and_same_request_twice(cuda, rng, dtype):
    """The same pages in two tables, and a prefix page that is also a request's own."""
    d = make_attn(cuda, rng, dtype, 4, 2, 64, 16, 64, [48, 48, 20], [1, 1, 4])
    d["table"][1] = d["table"][0]
    d["table"][2, 0] = d["ptab"][1]
    d["q"][1] = d["q"][0]
    out = check_attn(cuda, dtype, d, 4)
    assert torch.equal(out[0], out[1])


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_attn_not_finite_where_it_is_seen(cuda, rng, dtype):
    """A NaN in a request's own key reaches that request and no other."""
    d = make_attn(cuda, rng, dtype, 4, 2, 64, 16, 64, [48, 48, 20], [1, 1, 1])
    clean = run_attn(cuda, d)
    d["k"][d["table"][1, 1], 0, 3, 5] = float("nan")
    out = run_attn(cuda, d)
    assert torch.equal(out[[0, 2]], clean[[0, 2]])
    assert torch.isnan(out[1, : 2 * 64]).all() and torch.equal(out[1, 2 * 64:], clean[1, 2 * 64:])


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("hq,hkv,hd", [(4, 2, 64), (12, 2, 128)])
@pytest.mark.parametrize("new", [[3, 1, 5], [9, 150, 70]])
def test_attn_not_finite_where_it_is_hidden(cuda, rng, dtype, hq, hkv, hd, new):
    """Infinities and NaN in the keys and values of a chunk's later tokens: the rows before them are as without, the rows
    that see them are what the formula makes of it (fp32: not a number)."""
    lens = [n + 20 for n in new]
    d = make_attn(cuda, rng, dtype, hq, hkv, hd, 16, 40, lens, new, scale_q=0.3)
    v, k = d["v"], d["k"]

    def put(pool, b, back, h, col, what):  # the request's token `back` from its end
        i = lens[b] - back
        pool[d["table"][b, i // 16], h, i % 16, col] = what

    for b in range(3):
        if new[b] > 1:
            put(v, b, 1, 0, 3, float("nan"))
            put(v, b, 2, 1, 7, float("inf"))
            put(v, b, 1, 1, hd - 1, float("-inf"))
            put(v, b, new[b] - 1, 0, 11, float("-inf"))
            put(v, b, 1, 0, 11, float("inf"))
        if new[b] > 4:
            put(k, b, 1, 1, 5, float("nan"))
            put(v, b, new[b] // 2, 0, 40, float("nan"))
    out = run_attn(cuda, d)
    with np.errstate(invalid="ignore"):
        want, mass, dot, keys, tail = op.attention(d["q"].double().numpy(), k.double().numpy(), v.double().numpy(), d["start"], d["lens"],
                                                   d["table"], d["ptab"], d["prefix"], hq, 1 / math.sqrt(hd))
    got = out[: sum(new)].double().cpu().numpy().reshape(want.shape)
    fine = np.isfinite(want)
    assert 0 < (~fine).sum() < fine.size / 2
    if dtype == "f16":
        assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(got[np.isinf(want)], want[np.isinf(want)])
    else:
        assert np.array_equal(np.isfinite(got), fine)
    bound = attn_bound(dtype, want, np.where(fine, mass, 0), np.where(np.isfinite(dot), dot, 0), keys, np.where(fine, tail, 0), hd)
    assert (np.abs(got[fine] - want[fine]) <= bound[fine]).all()
    assert L.load().sc_prefix_attn_device_error(1) == 0


WIDE = ([(test_attn_ragged_chunks, (hq, hkv, hd, prefix)) for hq, hkv, hd in LAYOUTS for prefix in (0, 1, 333)]
        + [(test_attn_lengths, a) for a in [(1, 2000, 700), (3, 5000, 40), (2, 0, 3001), (40, 129, 300)]]
        + [(test_attn_no_prefix_and_scale, ([1, 1, 1],)), (test_attn_no_prefix_and_scale, ([9, 40, 150],)), (test_attn_rows_that_see_nothing, (0,)),
           (test_attn_rows_that_see_nothing, (50,)), (test_attn_absent_pages, ([1, 1, 1],)), (test_attn_absent_pages, ([5, 70, 33],)),
           (test_attn_all_pages_absent, ()), (test_attn_shared_page_and_same_request_twice, ()), (test_attn_not_finite_where_it_is_seen, ())]
        + [(test_attn_not_finite_where_it_is_hidden, (4, 2, 64, new)) for new in ([3, 1, 5], [9, 150, 70])]
        + [(test_attn_not_finite_where_it_is_hidden, (12, 2, 128, new)) for new in ([3, 1, 5], [9, 150, 70])])


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("which", ["table", "ptab"])
@pytest.mark.parametrize("case", range(len(WIDE)))
def test_attn_tables_with_room(cuda, rng, monkeypatch, dtype, which, case):
    """The same with tables that have room for 65536 more tokens: the call is cut for those, into other kernels and more
    shares, most of them without a key."""
    def roomy(*args, make=make_attn, **kw):
        d = make(*args, **kw)
        wide = 65536 // d["k"].shape[2]
        d[which] = np.concatenate([d[which], np.full(d[which].shape[:-1] + (wide,), -1, np.int32)], -1)
        return d

    monkeypatch.setitem(globals(), "make_attn", roomy)
    test, args = WIDE[case]
    test(cuda, rng, dtype, *args)


def test_attn_large_offsets(cuda):
    """Pages beyond 2^31 elements from the pool's start."""
    hkv, hd, page = 8, 128, 128
    n_pages = 2**31 // (hkv * page * hd) + 40
    k = torch.zeros(n_pages, hkv, page, hd, dtype=torch.float16, device=cuda)
    v = torch.zeros_like(k)
    ids = [n_pages - 1, n_pages - 20, 3]
    k[ids] = torch.randn(3, hkv, page, hd, device=cuda).half()
    v[ids] = torch.randn(3, hkv, page, hd, device=cuda).half()
    q = torch.randn(2, 16 * hd, device=cuda).half()
    args = (i32([0, 1, 2], cuda), i32([100, 120], cuda))
    far = ops.prefix_attn(q, k, v, *args, i32([[ids[1]], [ids[2]]], cuda), prefix_table=i32([ids[0]], cuda), prefix_len=i32([128], cuda))
    near = ops.prefix_attn(q, k[ids].contiguous(), v[ids].contiguous(), *args, i32([[1], [2]], cuda), prefix_table=i32([0], cuda), prefix_len=i32([128], cuda))
    assert torch.equal(far, near) and far.abs().sum() > 0


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_attn_matches_contiguous_flash_decode(cuda, rng, dtype):
    """Against the contiguous cache's kernel on the same values (fp32 cache there)."""
    hq, hkv, hd, page, Lmax, B = 8, 2, 128, 16, 256, 3
    kc = torch.randn(B, hkv, Lmax, hd, device=cuda).to(DT[dtype]).float()
    vc = torch.randn(B, hkv, Lmax, hd, device=cuda).to(DT[dtype]).float()
    q = torch.randn(B, hq * hd, device=cuda).to(DT[dtype])
    ref = torch.empty(B, hq * hd, device=cuda)
    ops.flash_decode(q.float(), kc, vc, i32([199], cuda), B, 1, hq, hkv, hd, 4, ref)
    nb = Lmax // page
    pool = lambda c: c.view(B, hkv, nb, page, hd).permute(0, 2, 1, 3, 4).reshape(B * nb, hkv, page, hd).to(DT[dtype]).contiguous()  # noqa: E731
    out = ops.prefix_attn(q, pool(kc), pool(vc), i32([0, 1, 2, 3], cuda), i32([200] * 3, cuda), torch.arange(B * nb, dtype=torch.int32, device=cuda).view(B, nb))
    # fp16: weights and output rounded by 2^-11 at most each; fp32: 2^-21 of three operands
    assert (out.float() - ref).abs().max() <= (2 * 2.0**-11 if dtype == "f16" else 2.0**-18) * vc.abs().max()


# ------------------------------------------------------------------------------------------------ used together

def test_serving_run_in_one_graph(cuda, rng):
    """Reserve, append and attend in a captured step, replayed over a ragged batch with drafts that are cut and requests
    that end, against contiguous copies of every request's tokens in float64."""
    hq, hkv, hd, page, B, max_blocks, P = 8, 2, 64, 16, 5, 8, 41
    n_pages, T, width = 40, 16, (hq + 2 * hkv) * hd
    g = torch.Generator(device=cuda).manual_seed(3)
    k = torch.full((n_pages, hkv, page, hd), float("nan"), dtype=torch.float32, device=cuda)
    v = k.clone()
    ang = torch.outer(torch.arange(256.0, device=cuda), 10.0 ** -torch.linspace(0, 3, hd // 2, device=cuda))
    cos, sin = ang.cos().contiguous(), ang.sin().contiguous()
    order = torch.from_numpy(rng.permutation(n_pages).astype(np.int32)).to(cuda)
    free, count = order.clone(), i32([n_pages], cuda)
    lens = torch.zeros(B, dtype=torch.int32, device=cuda)
    table = torch.full((B, max_blocks), -1, dtype=torch.int32, device=cuda)
    # the prefix is a request of its own: reserved and appended like any other, then its pages are the prefix's
    ptab = torch.full((1, 3), -1, dtype=torch.int32, device=cuda)
    st = ops.paged_reserve(i32([0], cuda), i32([P], cuda), ptab, free, count, page, max_tokens=P, free_count_out=count)
    pqkv = torch.randn(P, width, generator=g, device=cuda)
    pq = torch.empty(P, hq * hd, device=cuda)
    ops.paged_rope_append(pqkv, st.q_start, st.slots, st.positions, cos, sin, pq, k, v)
    plen = i32([P], cuda)

    new, keep, qkv = i32([0] * B, cuda), i32([0] * B, cuda), torch.zeros(T, width, device=cuda)
    q, out = torch.empty(T, hq * hd, device=cuda), torch.zeros(T, hq * hd, device=cuda)
    bufs = dict(kv_lens=lens, q_start=i32([0] * (B + 1), cuda), slots=i32([-1] * T, cuda), positions=i32([0] * T, cuda),
                free_count_out=count, status=i32([0], cuda))

    def step():
        s = ops.paged_reserve(lens, new, table, free, count, page, prefix_len=plen, **bufs)
        ops.paged_rope_append(qkv, s.q_start, s.slots, s.positions, cos, sin, q, k, v)
        ops.prefix_attn(q, k, v, s.q_start, s.kv_lens, table, prefix_table=ptab.view(-1), prefix_len=plen, out=out)
        ops.paged_truncate(lens, keep, table, free, count, page, lens_out=lens, free_count_out=count, status=bufs["status"])

    keep.fill_(10**6)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()  # no tokens yet
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()

    held = [np.zeros((0, width)) for _ in range(B)]  # every request's rows of qkv, as they are kept
    c64, s64 = cos.double().cpu().numpy(), sin.double().cpu().numpy()

    def turned(rows, at):
        x = rows.reshape(len(rows), hq + 2 * hkv, hd)
        return np.concatenate([op.rotate(x[:, : hq + hkv], at, c64, s64), x[:, hq + hkv:]], 1)

    pre = turned(pqkv.double().cpu().numpy(), np.arange(P))
    plan = [([3, 1, 5, 0, 7], None), ([1, 1, 1, 1, 1], None), ([4, 4, 0, 4, 4], [1, 2, 0, 4, 0]), ([1, 1, 1, 1, 1], [None, None, 0, None, None]),
            ([0, 9, 3, 1, 1], None), ([2, 2, 2, 2, 2], [0, None, None, 0, None]), ([5, 0, 0, 6, 1], None), ([1, 1, 1, 1, 1], None)]
    for new_n, cut in plan:
        total = sum(new_n)
        qkv.copy_(torch.randn(T, width, generator=g, device=cuda))
        new.copy_(i32(new_n, cuda))
        # cut: how many of the step's drafts stay (None: all); a request with 0 and no drafts ends
        kept = []
        for b in range(B):
            full = len(held[b]) + new_n[b]
            c = None if cut is None else cut[b]
            kept.append(full if c is None else (len(held[b]) + c if new_n[b] > 1 else 0))
        keep.copy_(i32(kept, cuda))
        graph.replay()
        assert int(bufs["status"]) == 0
        rows = qkv.double().cpu().numpy()
        got = out.double().cpu().numpy().reshape(T, hq, hd)
        at = 0
        for b in range(B):
            mine = np.concatenate([held[b], rows[at:at + new_n[b]]])
            x = np.concatenate([pre, turned(mine, P + np.arange(len(mine)))]) if len(mine) else pre
            for i in range(new_n[b]):
                n = P + len(held[b]) + i + 1
                for h in range(hq):
                    s = x[:n, hq + h // (hq // hkv)] @ x[n - 1, h] / math.sqrt(hd)
                    w = np.exp(s - s.max())
                    want = w @ x[:n, hq + hkv + h // (hq // hkv)] / w.sum()
                    # scores of size 30 at most, their operands rounded by 2^-24 and split to 2^-21: 30 * 4 * 2^-21 on every weight
                    assert np.abs(got[at + i, h] - want).max() <= 120 * 2.0**-21 * np.abs(x[:n, hq + hkv:]).max()
            at += new_n[b]
            held[b] = mine[: kept[b]]
        assert lens.tolist() == [len(x) for x in held]
        used = 3 + sum(-(-len(x) // page) for x in held)
        assert int(count) == n_pages - used
        live = [int(x) for b in range(B) for x in table[b, : -(-len(held[b]) // page)].tolist()] + ptab.view(-1).tolist()
        assert sorted(live + free[: int(count)].tolist()) == list(range(n_pages))  # every page held once or free


@pytest.mark.parametrize("dtype,tol", [("f32", 4e-4), ("f16", 4e-3)])
def test_model_over_a_paged_cache(cuda, dtype, tol):
    """A quantized model over the paged cache -- a shared prefix, ragged prompts, single tokens, drafts that are cut, a
    request that ends and one that takes its place -- against the same model over the contiguous cache, a request at a
    time.  fp32: the two attentions differ by d = 2^-19 (two operands and two weights split to 2^-21 each).  The layers round
    the MLP's inner values to fp16, where values that differ by d fall to different sides with probability d / 2^-11 and
    are then 2^-10 apart: 2^-10 sqrt(2^11 d) = 6e-5 after the first layer, and with that as d, 2^-10 sqrt(2^11 6e-5) = 3.4e-4
    after the second, the last.  fp16: keys, values, q, weights and outputs of the attention are rounded by up to 2^-11 each,
    five of them in two layers: 10 2^-11 = 4.9e-3 at most, and seldom all one way."""
    import asyncio

    from oracle import sharder as osh
    from oracle import synth
    from shardcompute_b200.model.config import ModelConfig
    from shardcompute_b200.parallel import PagedKVCache, ParallelTransformer, RankWeights

    shape = synth.tiny_shape()
    full = synth.checkpoint(shape, seed=0)
    cfg = ModelConfig.from_dict(synth.model_config_dict(shape))
    model = ParallelTransformer.from_config(cfg, 1, 0, None)
    model.load_rank_weights(RankWeights.from_shard(cfg, osh.shard_weights(full, 1, 0), 1, 0, shape.bits, shape.group_size, cuda))
    run = lambda ids, past: asyncio.run(model.forward(ids, past_key_values=past))[0][0]  # noqa: E731
    gen = np.random.default_rng(5)
    words = lambda n: gen.integers(0, shape.vocab_size, n).tolist()  # noqa: E731
    cache = PagedKVCache(cfg.num_layers, cfg.kv_heads, cfg.head_dim, 24, 3, 64, page_size=16, max_prefix=64, max_tokens=48, dtype=DT[dtype],
                         device=cuda)
    prefix = words(21)

    def step(tokens):
        """The new tokens of each request in, their logits out."""
        cache.reserve([len(t) for t in tokens])
        cache.check()
        ids = sum(tokens, [])
        out = run(torch.tensor([ids], device=cuda), cache.layers())
        return torch.split(out, [len(t) for t in tokens])

    def want(text):
        return run(torch.tensor([text], device=cuda), model.new_cache(1, 128))

    got = step([prefix, [], []])[0]
    assert rel(got, want(prefix)) <= tol
    cache.share_prefix(0)
    held = [[], [], []]
    for new_n, kept in [((5, 1, 9), None), ((1, 1, 1), None), ((4, 0, 3), (2, None, 0)), ((1, 1, 1), (None, "end", None)), ((2, 17, 1), None)]:
        tokens = [words(n) for n in new_n]
        outs = step(tokens)
        for b in range(3):
            if tokens[b]:
                ref = want(prefix + held[b] + tokens[b])[-len(tokens[b]):]
                assert rel(outs[b], ref) <= tol, (b, rel(outs[b], ref))
        keep = []
        for b in range(3):
            k = None if kept is None else kept[b]
            held[b] = [] if k == "end" else held[b] + (tokens[b] if k is None else tokens[b][:k])
            keep.append(len(held[b]))
        cache.truncate(keep)
        cache.check()
        assert cache.lens.tolist() == keep
    with pytest.raises(ValueError):
        cache.share_prefix(1)
    with pytest.raises(ValueError):
        cache.release_prefix()
    cache.truncate([0, 0, 0])
    cache.release_prefix()
    cache.check()
    assert int(cache.free_count) == 24 and sorted(cache.free_pages.tolist()) == list(range(24))
    cache.reserve([64, 64, 64])
    assert int(cache.status) == 4  # more rows than the cache was made for
    with pytest.raises(ValueError, match="rows"):
        cache.check()
    assert cache.lens.tolist() == [0, 0, 0]
    with pytest.raises(ValueError):
        run(torch.zeros(1, 49, dtype=torch.long, device=cuda), cache.layers())


def rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


def test_on_another_stream(cuda, rng):
    d = make_attn(cuda, rng, "f16", 8, 2, 128, 16, 500, [40, 90, 33], [1, 1, 1])
    first = run_attn(cuda, d)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        other = run_attn(cuda, d)
    s.synchronize()
    assert torch.equal(first, other)


def test_two_graphs_share_a_workspace(cuda, rng):
    """Two captured calls of other shapes with one workspace, replayed in turn on one stream."""
    a = make_attn(cuda, rng, "f16", 8, 2, 128, 16, 900, [40, 90, 33], [1, 1, 1])
    b = make_attn(cuda, rng, "f32", 4, 1, 64, 32, 3000, [700], [2])
    ws = torch.empty(64 << 20, dtype=torch.uint8, device=cuda)
    calls = []
    for d in (a, b):
        t = [d["q"].to(cuda), d["k"].to(cuda), d["v"].to(cuda), i32(d["start"], cuda), i32(d["lens"], cuda), i32(d["table"], cuda)]
        pre = dict(prefix_table=i32(d["ptab"], cuda), prefix_len=i32([d["prefix"]], cuda))
        want, out = ops.prefix_attn(*t, **pre), torch.zeros_like(t[0])
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            ops.prefix_attn(*t, out=out, workspace=ws, **pre)
        calls.append((graph, out, want, (t, pre)))  # what the graph reads stays alive
    for _ in range(3):
        for graph, out, _, _ in calls:
            out.zero_()
            graph.replay()
        for _, out, want, _ in calls:
            assert torch.equal(out, want)


def test_two_streams_at_once(cuda, rng):
    """Calls that overlap, each with the scratch it allocates."""
    d = [make_attn(cuda, rng, "f16", 8, 2, 128, 16, 4000, [40, 900, 33], [1, 1, 1]) for _ in range(2)]
    t = [[x["q"].to(cuda), x["k"].to(cuda), x["v"].to(cuda), i32(x["start"], cuda), i32(x["lens"], cuda), i32(x["table"], cuda)] for x in d]
    pre = [dict(prefix_table=i32(x["ptab"], cuda), prefix_len=i32([x["prefix"]], cuda)) for x in d]
    want = [ops.prefix_attn(*t[i], **pre[i]) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    for _ in range(10):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                outs[i].append(ops.prefix_attn(*t[i], **pre[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in outs[i])
