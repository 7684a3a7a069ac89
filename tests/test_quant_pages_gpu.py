"""The paged cache in 8 or 4 bits against oracle/quant_pages.py: codes, scales and biases exactly, values read back exactly, the
attention within a bound that is derived from the number formats (attn_bound)."""

import math

import numpy as np
import pytest
import torch

from oracle import quant_pages as oq
from shardcompute_b200 import _lib as L
from shardcompute_b200 import ops

pytestmark = pytest.mark.gpu

DT = {"f16": torch.float16, "f32": torch.float32}
KINDS = [(hd, bits, group) for hd in (64, 128) for bits in (4, 8) for group in (32, 64)]


def i32(a, dev):
    return torch.from_numpy(np.ascontiguousarray(np.asarray(a, np.int32))).to(dev)


def rotated(x, pos, cos, sin):
    """x [T, heads, hd] in fp32, every product and sum rounded: what the cache quantises."""
    half = x.shape[-1] // 2
    a, b = x[..., :half].astype(np.float32), x[..., half:].astype(np.float32)
    c, s = cos[pos][:, None], sin[pos][:, None]
    return np.concatenate([a * c - b * s, b * c + a * s], -1)


# ------------------------------------------------------------------------------------------------ append

def check_append(cuda, rng, src, hq, hkv, hd, page, bits, group, rows, pad=3, values=None):
    n_pages, max_pos = -(-2 * rows // page) + 2, 300
    x = rng.standard_normal((rows + pad, (hq + 2 * hkv) * hd)) if values is None else values(rng, (rows + pad, (hq + 2 * hkv) * hd))
    x = torch.from_numpy(x.astype(np.float32)).to(DT[src])
    pos, slots = rng.integers(0, max_pos, rows + pad), rng.permutation(n_pages * page)[:rows + pad]
    if rows > 4:  # not written: slots and positions that are none
        slots[0], slots[1], pos[2], pos[3] = -1, n_pages * page, max_pos, -1
    ang = rng.standard_normal((max_pos, hd // 2)) * 3
    cos, sin = np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)
    data0 = rng.integers(0, 256, (n_pages, hkv, ops.quant_page_bytes(page, hd, bits, group)), dtype=np.uint8)
    pages = ops.QuantPages(torch.from_numpy(data0).to(cuda), hd, page, bits, group)
    q = torch.full((rows + pad, hq * hd), 7.0, dtype=torch.float16, device=cuda)
    ops.paged_rope_append_q(x.to(cuda), i32([0, rows // 2, rows], cuda), i32(slots, cuda), i32(pos, cuda), torch.from_numpy(cos).to(cuda),
                            torch.from_numpy(sin).to(cuda), q, pages)
    h = x.float().numpy().reshape(rows + pad, hq + 2 * hkv, hd)
    there = (pos >= 0) & (pos < max_pos)
    cos1, sin1 = np.concatenate([cos, np.ones((1, hd // 2), np.float32)]), np.concatenate([sin, np.zeros((1, hd // 2), np.float32)])
    y = rotated(h[:, : hq + hkv], np.where(there, pos, max_pos), cos1, sin1)
    with np.errstate(over="ignore"):
        assert np.array_equal(q[:rows].cpu().numpy(), y[:rows, :hq].reshape(rows, -1).astype(np.float16))
    assert (q[rows:] == 7).all()
    # the oracle's codes put where they belong; everything else as it was
    want, sides = data0.copy(), (y[:, hq:], h[:, hq + hkv:])
    fits = [t for t in range(rows) if there[t] and 0 <= slots[t] < n_pages * page]
    for t in fits:
        for side, v in enumerate(sides):
            oq.put(want, slots[t], page, side, *oq.quantise(v[t], bits, group), bits, group)
    got = pages.data.cpu().numpy()
    tg, tw = oq.take(got, hd, page, bits, group), oq.take(want, hd, page, bits, group)
    for side in (0, 1):
        assert all(np.array_equal(tg[side][k], tw[side][k], equal_nan=True) for k in (1, 2))  # a zero's sign changes no s c + b
        assert np.array_equal(tg[side][0], tw[side][0])
    return pages, slots, q


@pytest.mark.parametrize("hd,bits,group", KINDS)
@pytest.mark.parametrize("src,hq,hkv,page,rows", [("f32", 4, 2, 16, 37), ("f16", 5, 1, 48, 1), ("f32", 1, 3, 64, 130)])
def test_append(cuda, rng, hd, bits, group, src, hq, hkv, page, rows):
    check_append(cuda, rng, src, hq, hkv, hd, page, bits, group, rows)


@pytest.mark.parametrize("values", [lambda r, n: r.standard_normal(n) * 1e-6, lambda r, n: r.standard_normal(n) * 9e3,
                                    lambda r, n: np.full(n, -0.37), lambda r, n: np.zeros(n), lambda r, n: 100 + r.standard_normal(n) * 1e-3,
                                    lambda r, n: r.standard_normal(n) * 10.0 ** r.integers(-9, 4, n)],
                         ids=["small", "large", "constant", "zero", "narrow", "wide"])
def test_append_values(cuda, rng, values):
    check_append(cuda, rng, "f32", 2, 2, 128, 16, 4, 64, 40, values=values)
    check_append(cuda, rng, "f32", 2, 2, 64, 16, 8, 32, 40, values=values)


@pytest.mark.parametrize("bits,group", [(4, 64), (8, 32)])
def test_append_next_to_the_border_of_two_codes(cuda, rng, bits, group):
    """Values of v at (c + 1/2) s + b, and up to three fp32 steps to either side: rounded as exact arithmetic rounds them."""
    rows, hd, most = 200, 128, 2**bits - 1

    def values(gen, shape):
        x = gen.standard_normal(shape).astype(np.float32).reshape(shape[0], -1, group)
        s = (np.abs(gen.standard_normal(x.shape[:2])) * 10.0 ** gen.integers(-3, 2, x.shape[:2])).astype(np.float16).astype(np.float64)[..., None]
        b = gen.standard_normal(x.shape[:2]).astype(np.float16).astype(np.float64)[..., None]
        near = (s * (gen.integers(0, most, x.shape) + 0.5) + b).astype(np.float32)
        for _ in range(3):
            near = np.nextafter(near, np.where(gen.random(x.shape) < 0.3, near, np.where(gen.random(x.shape) < 0.5, -np.inf, np.inf)).astype(np.float32))
        near[..., :1], near[..., 1:2] = b, s * most + b
        return near.reshape(shape)

    check_append(cuda, rng, "f32", 1, 1, hd, 16, bits, group, rows, values=values)


def test_append_of_what_is_not_finite(cuda, rng):
    """It shows in its own group of its own token and head, and nowhere else."""
    hd, hkv = 128, 2
    x = rng.standard_normal((6, (1 + 2 * hkv) * hd)).astype(np.float32)
    x[1, 3 * hd + 5], x[2, 3 * hd + 70], x[3, 4 * hd + 127], x[4, 3 * hd] = np.nan, np.inf, -np.inf, -1e5  # of v: not rotated
    pages = ops.quant_pages(1, hkv, 16, hd, 4, 64, cuda)
    slots, one = i32(np.arange(6), cuda), torch.ones(8, hd // 2, device=cuda)
    q = torch.zeros(6, hd, dtype=torch.float16, device=cuda)
    ops.paged_rope_append_q(torch.from_numpy(x).to(cuda), i32([0, 6], cuda), slots, slots, one, one * 0, q, pages)
    k, v = ops.paged_read_q(pages, slots, dtype=torch.float32)
    bad = ~torch.isfinite(v.view(6, hkv, 2, 64))
    want = torch.zeros(6, hkv, 2, dtype=torch.bool)
    want[1, 0, 0] = want[2, 0, 1] = want[3, 1, 1] = want[4, 0, 0] = True
    assert torch.equal(bad.any(-1).cpu(), want) and torch.equal(bad.all(-1).cpu(), want) and bool(torch.isfinite(k).all())
    # rows of a chunk: NaN in the group's dims from the token on that holds it; of k: everywhere
    rows = torch.randn(6, 2 * hd, device=cuda).half()
    table, lens = torch.zeros(1, 1, dtype=torch.int32, device=cuda), i32([6], cuda)
    out = ops.prefix_attn_q(rows, pages, i32([0, 6], cuda), lens, table).view(6, 2, 2, 64)
    assert torch.equal(out.isnan().all(-1).cpu(), want.cumsum(0) > 0) and torch.equal(out.isnan().any(-1).cpu(), want.cumsum(0) > 0)
    x[1:, hd + 70], x[1:, 3 * hd:] = np.inf, 1.0
    ops.paged_rope_append_q(torch.from_numpy(x).to(cuda), i32([0, 6], cuda), slots, slots, one, one * 0, q, pages)
    out = ops.prefix_attn_q(rows, pages, i32([0, 6], cuda), lens, table).view(6, 2, hd)
    assert out[1:, 0].isnan().all() and torch.isfinite(out[0]).all() and torch.isfinite(out[:, 1]).all()


def test_append_next_to_tokens_that_stay(cuda, rng):
    """Tokens share words of memory, not bytes: one written does not move its neighbours."""
    for hd, bits, group in KINDS:
        pages, slots, _ = check_append(cuda, rng, "f32", 1, 2, hd, 16, bits, group, 31, pad=0)
        before = [x.clone() for x in ops.paged_read_q(pages, i32(np.arange(48), cuda), dtype=torch.float32)]
        x, one = torch.randn(2, 5 * hd, device=cuda), torch.ones(4, hd // 2, device=cuda)
        two = [7, 20]
        ops.paged_rope_append_q(x, i32([0, 2], cuda), i32(two, cuda), i32([0, 1], cuda), one, one * 0, torch.empty(2, hd, dtype=torch.float16, device=cuda),
                                pages)
        after = ops.paged_read_q(pages, i32(np.arange(48), cuda), dtype=torch.float32)
        stay = [s for s in range(48) if s not in two]
        for a, b, lo in ((before[0], after[0], 1), (before[1], after[1], 3)):
            assert torch.equal(a[stay].view(torch.int32), b[stay].view(torch.int32))  # bits: slots never written hold NaN too
            assert (b[two] - x[:, lo * hd:(lo + 2) * hd].view(2, 2, hd)).abs().max() < 8 / (2**bits - 1)


# ------------------------------------------------------------------------------------------------ read

@pytest.mark.parametrize("hd,bits,group", KINDS)
@pytest.mark.parametrize("out", ["f16", "f32"])
def test_read(cuda, rng, hd, bits, group, out):
    page, n_pages, hkv = 32, 5, 3
    data = rng.integers(0, 256, (n_pages, hkv, ops.quant_page_bytes(page, hd, bits, group)), dtype=np.uint8)
    pages = ops.QuantPages(torch.from_numpy(data).to(cuda), hd, page, bits, group)
    slots = np.concatenate([rng.permutation(n_pages * page), [3, 3, -1, n_pages * page, 3]])
    k, v = ops.paged_read_q(pages, i32(slots, cuda), dtype=DT[out])
    for got, (c, s, b) in zip((k, v), oq.take(data, hd, page, bits, group)):
        c = c.reshape(n_pages, hkv, page, -1, group).astype(np.float64)
        # s c is exact in fp32, and so is the sum in float64 up to 2^-53: one rounding to fp32, one more to fp16
        with np.errstate(invalid="ignore", over="ignore"):
            want = (c * s.astype(np.float64)[..., None] + b.astype(np.float64)[..., None]).astype(np.float32).reshape(n_pages, hkv, page, hd)
            want = want.astype(np.float16) if out == "f16" else want
        there = (slots >= 0) & (slots < n_pages * page)
        want = np.where(there[:, None, None], want[np.where(there, slots, 0) // page, :, np.where(there, slots, 0) % page], 0)
        assert np.array_equal(got.cpu().numpy(), want, equal_nan=True)
    ko, vo = torch.full_like(k, 7.0), torch.full_like(v, 7.0)
    ops.paged_read_q(pages, i32(slots, cuda), q_start=i32([0, 4, 9], cuda), k_out=ko, v_out=vo)
    assert torch.equal(ko[:9].isnan(), k[:9].isnan()) and torch.equal(ko[:9].nan_to_num(), k[:9].nan_to_num()) and (ko[9:] == 7).all()
    assert torch.equal(vo[:9].nan_to_num(), v[:9].nan_to_num()) and (vo[9:] == 7).all()


# ------------------------------------------------------------------------------------------------ attention

def attn_bound(out, mass, dot, keys, tail, hd, rounded=False):
    """How far an output may be from float64.  With e = 2^-24 (a sum of fp32 products, each sum rounded or cut: 2 e), w_j the
    weights, sizes those of s c + |b|:
      score     ds = dot * (2 (hd + 8) e + 4 e)            (products and sums; scales, biases; the difference to the maximum)
      weight    w_j (1 + 2 ds + 8 e), times s, rounded to fp16: p = 2^-11, and steps of 2^-24 where the largest w s is 2^11
                or more: 2^-25 / 2^11 of that largest for every key, times its code (tail)
      output    mass * (2 ds + 16 e + 2 p + 2 e (keys / 8 + 64)) for numerator and denominator, then its rounding to fp16
    rounded: k and v go through fp16 (2^-11 of each) on their way into the products."""
    e, p, u = 2.0**-24, 2.0**-11, 2.0**-11 if rounded else 0.0
    ds = (dot * (2 * (hd + 8) * e + 4 * e + u))[..., None]
    return mass * (2 * ds + 16 * e + 2 * p + u + 2 * e * (keys[..., None] / 8 + 64)) + 2.0**-36 * tail * 1.01 + 2.0**-11 * np.abs(out) * 1.01 + 2.0**-25


def make_attn(rng, hq, hkv, hd, page, bits, group, prefix, lens, new, pad=2, scale_q=1.5, dirty=True):
    """A pool whose unused slots hold codes with scales and biases of NaN and infinities, tables in random order, q."""
    all_lens = list(lens) + [prefix]
    blocks = [-(-int(n) // page) for n in all_lens]
    n_pages = sum(blocks) + 3
    ids = rng.permutation(n_pages).astype(np.int32)
    table, at = np.full((len(all_lens), max(blocks) + 1), -1, np.int32), 0
    for b, n in enumerate(blocks):
        table[b, :n] = ids[at:at + n]
        at += n
    k = rng.standard_normal((n_pages, hkv, page, hd)) + rng.standard_normal((1, hkv, 1, hd))
    v = rng.standard_normal((n_pages, hkv, page, hd)) + 0.3
    data = oq.fill(k.astype(np.float32), v.astype(np.float32), bits, group)
    if dirty:
        used = np.zeros((n_pages, page), bool)
        for b, n in enumerate(all_lens):
            for i in range(n):
                used[table[b, i // page], i % page] = True
        odd = np.array([np.nan, np.inf, -np.inf, 6e4], np.float16).view(np.uint8).reshape(4, 2)
        blocks16 = data.reshape(n_pages, hkv, page // 16, -1)
        for side in (0, 1):
            for tok in range(16):
                for g in range(hd // group):
                    m = oq.meta_place(side, tok, g, hd, bits, group)
                    for pid, blk in np.argwhere(~used.reshape(n_pages, -1, 16)[:, :, tok]):
                        blocks16[pid, :, blk, m:m + 4] = odd[rng.integers(0, 4, 2)].reshape(4)
    rows = int(sum(new))
    q = torch.from_numpy(rng.standard_normal((rows + pad, hq * hd)) * scale_q).half()
    start = np.concatenate([[0], np.cumsum(new)])
    ptab = table[-1, : max(1, -(-prefix // page))] if prefix else np.zeros(1, np.int32)
    return dict(q=q, data=data, start=start, lens=np.array(lens), table=table[:-1].copy(), ptab=ptab.copy(), prefix=prefix, kind=(hd, page, bits, group))


def pool(d, cuda):
    return ops.QuantPages(torch.from_numpy(d["data"]).to(cuda), *d["kind"])


def run_attn(cuda, d, with_prefix=True, scale=None, workspace=None, out=None):
    if out is None:
        out = torch.full_like(d["q"], 5.0).to(cuda)
    pre = dict(prefix_table=i32(d["ptab"], cuda), prefix_len=i32([d["prefix"]], cuda)) if with_prefix else {}
    return ops.prefix_attn_q(d["q"].to(cuda), pool(d, cuda), i32(d["start"], cuda), i32(d["lens"], cuda), i32(d["table"], cuda), out=out, scale=scale,
                             workspace=workspace, **pre)


def check_attn(cuda, d, hq, with_prefix=True, scale=None, rounded=False):
    hd, page, bits, group = d["kind"]
    out = run_attn(cuda, d, with_prefix, scale)
    sc = 1 / math.sqrt(hd) if scale is None else scale
    want, mass, dot, keys, tail = oq.attention(d["q"].double().numpy(), d["data"], d["start"], d["lens"], d["table"], d["ptab"],
                                               d["prefix"] if with_prefix else 0, hq, hd, page, bits, group, sc)
    rows = int(d["start"][-1])
    got = out[:rows].double().cpu().numpy().reshape(want.shape)
    bound = attn_bound(want, mass, dot, keys, tail, hd, rounded)
    err = np.abs(got - want)
    assert np.isfinite(got).all()
    worst = np.unravel_index(np.argmax(err - bound), err.shape)
    assert (err <= bound).all(), (worst, got[worst], want[worst], bound[worst])
    assert (out[rows:] == 5.0).all()
    assert L.load().sc_prefix_attn_device_error(1) == 0
    return out


@pytest.mark.parametrize("hd,bits,group", KINDS)
@pytest.mark.parametrize("hq,hkv,page", [(8, 2, 16), (4, 4, 64), (6, 1, 32), (18, 2, 16)])
def test_attn_decode(cuda, rng, hd, bits, group, hq, hkv, page):
    d = make_attn(rng, hq, hkv, hd, page, bits, group, 77, [1, 16, 17, 5, 130, 64], [1] * 6)
    check_attn(cuda, d, hq)


@pytest.mark.parametrize("hd,bits,group", KINDS)
@pytest.mark.parametrize("hq,hkv,prefix", [(8, 2, 0), (3, 3, 1), (8, 1, 333)])
def test_attn_ragged_drafts(cuda, rng, hd, bits, group, hq, hkv, prefix):
    """Requests with no row, one row, drafts and short chunks, with and without tokens before them."""
    d = make_attn(rng, hq, hkv, hd, 16, bits, group, prefix, [20, 1, 5, 40, 0, 16, 40], [0, 1, 5, 13, 0, 16, 3])
    check_attn(cuda, d, hq)


@pytest.mark.parametrize("B,prefix,longest", [(1, 0, 1), (1, 2000, 700), (3, 5000, 40), (2, 0, 3001), (40, 129, 300)])
def test_attn_lengths(cuda, rng, B, prefix, longest):
    """From one token to many, few requests and many; queries far apart in size."""
    lens = [longest] + [int(x) for x in rng.integers(1, longest + 1, B - 1)]
    d = make_attn(rng, 4, 1, 64, 32, 4, 32, prefix, lens, [1] * B)
    d["q"] *= torch.from_numpy(10.0 ** rng.integers(-3, 2, (d["q"].shape[0], 1))).half()
    check_attn(cuda, d, 4)


@pytest.mark.parametrize("B,hq,hkv,hd", [(1, 8, 8, 128), (2, 6, 2, 64), (5, 8, 8, 128), (9, 16, 4, 64), (17, 8, 8, 128)])
@pytest.mark.parametrize("drafts", [False, True])
def test_attn_shares_joined(cuda, rng, B, hq, hkv, hd, drafts):
    """Few requests, whose keys several CTAs share, some without a key: the same bits every time."""
    new = [int(x) for x in rng.integers(0, 8, B)] if drafts else [1] * B
    lens = [n + int(rng.integers(0, 2)) * int(rng.integers(0, 900)) for n in new]
    lens[0] = new[0] + 900
    for prefix in (0, 130):
        d = make_attn(rng, hq, hkv, hd, 16, 4, 64, prefix, lens, new)
        out = check_attn(cuda, d, hq)
        for _ in range(4):
            assert torch.equal(out, run_attn(cuda, d))


@pytest.mark.parametrize("new", [[1, 1, 1], [9, 40, 30]])
def test_attn_no_prefix_and_scale(cuda, rng, new):
    d = make_attn(rng, 8, 2, 64, 16, 8, 64, 0, [30, 100, 41], new)
    check_attn(cuda, d, 8, with_prefix=False, scale=0.3)


def test_attn_scale_next_to_zero(cuda, rng):
    """Scores that vanish: every key that a row sees weighs the same, and what it does not see stays out."""
    d = make_attn(rng, 4, 2, 64, 16, 4, 64, 33, [5, 100, 40], [1, 4, 1])
    d["q"] = torch.full_like(d["q"], 2.0**-24)
    check_attn(cuda, d, 4, scale=1e-44)


@pytest.mark.parametrize("prefix", [0, 50])
def test_attn_rows_that_see_nothing(cuda, rng, prefix):
    """More rows than tokens: the first ones see the prefix only, or nothing at all, and are zero."""
    d = make_attn(rng, 4, 2, 64, 16, 4, 64, prefix, [3, 0, 20], [7, 2, 20])
    out = check_attn(cuda, d, 4)
    if not prefix:
        assert (out[:4] == 0).all() and (out[7:9] == 0).all()


def test_attn_absent_pages(cuda, rng):
    d = make_attn(rng, 8, 2, 128, 16, 4, 64, 100, [90, 70, 33], [1, 4, 1])
    d["ptab"][[0, len(d["ptab"]) - 1]] = [-1, len(d["data"]) + 5]
    d["table"][1, 0], d["table"][2, :] = -3, -1
    check_attn(cuda, d, 8)


@pytest.mark.parametrize("kv,qs", [(1e-6, 1.0), (1e-3, 300.0), (2e3, 1e-3), (2e3, 300.0)])
@pytest.mark.parametrize("bits", [4, 8])
def test_attn_values_of_any_size(cuda, rng, kv, qs, bits):
    """Scales down to fp16's subnormals, values up to its range, scores up to 10^9."""
    lens = [300, 40, 1, 77]
    d = make_attn(rng, 8, 2, 128, 16, bits, 64, 33, lens, [1, 1, 1, 5], dirty=False)
    k, v = (rng.standard_normal((len(d["data"]), 2, 16, 128)).astype(np.float32) * np.float32(kv) for _ in range(2))
    d["data"] = oq.fill(k, v, bits, 64)
    d["q"] = torch.from_numpy(rng.standard_normal(d["q"].shape) * qs).half()
    check_attn(cuda, d, 8)


def test_attn_scales_far_apart(cuda, rng):
    """Groups of one token, and tokens of one group, whose scales differ by 2^20: small weights of large scales and large weights
    of small ones both stay."""
    d = make_attn(rng, 4, 1, 128, 16, 4, 32, 0, [200, 190, 64], [1, 1, 3], dirty=False)
    n = len(d["data"])
    size = 2.0 ** rng.integers(-10, 11, (n, 1, 16, 4, 1))
    k = rng.standard_normal((n, 1, 16, 128)).astype(np.float32)
    v = (rng.standard_normal((n, 1, 16, 4, 32)) * size).reshape(n, 1, 16, 128).astype(np.float32)
    d["data"] = oq.fill(k, v, 4, 32)
    check_attn(cuda, d, 4)


def test_attn_small_weights_stay(cuda):
    """Thousands of keys 2^-25 below one that takes most of the weight and has a value of zero: what they add up to stays."""
    hd, page, n = 128, 64, 16384
    g = torch.Generator(device=cuda).manual_seed(3)
    k, v = np.zeros((n // page + 1, 1, page, hd), np.float32), np.zeros((n // page + 1, 1, page, hd), np.float32)
    k[0, 0, 0, :64] = 1.0
    v[:, 0, :, :] = np.random.default_rng(0).random((n // page + 1, page, hd)) + 0.5
    v[0, 0, 0] = 0.0
    data = oq.fill(k, v, 4, 64)
    q = torch.zeros(1, 2 * hd, dtype=torch.float16, device=cuda)
    q[:, :64] = 25 * math.log(2) / 64
    q[:, hd:] = torch.randn(1, hd, device=cuda, generator=g).half()
    table = torch.arange(n // page + 1, dtype=torch.int32, device=cuda)[None]
    pages = ops.QuantPages(torch.from_numpy(data).to(cuda), hd, page, 4, 64)
    out = ops.prefix_attn_q(q, pages, i32([0, 1], cuda), i32([n + 1], cuda), table, scale=1.0)
    want, mass, dot, keys, tail = oq.attention(q.double().cpu().numpy(), data, [0, 1], [n + 1], table.cpu().numpy(), [0], 0, 2, hd, page, 4, 64, 1.0)
    err = np.abs(out.double().cpu().numpy().reshape(want.shape) - want)
    assert (err <= attn_bound(want, mass, dot, keys, tail, hd)).all()
    assert np.linalg.norm(err[0, 0]) <= 2e-3 * np.linalg.norm(want[0, 0])  # 2 p of each weight, the output's rounding


def test_attn_hidden_scales_do_not_reach_other_rows(cuda, rng):
    """What is not finite in a chunk's later token shows in the rows that see it, and in no others."""
    d = make_attn(rng, 4, 2, 64, 16, 4, 32, 20, [30, 25], [6, 3], dirty=False)
    clean = run_attn(cuda, d)
    at = d["table"][0, 27 // 16]
    for side in (0, 1):
        for bad in (np.nan, np.inf, 6e4):
            e = dict(d, data=d["data"].copy())
            m = 27 % 32 // 16 * 0 + oq.meta_place(side, 27 % 16, 1, 64, 4, 32)
            e["data"][at, :, m:m + 4] = np.array([bad, bad], np.float16).view(np.uint8)
            out = run_attn(cuda, e)
            assert torch.equal(out[:3], clean[:3]) and torch.equal(out[6:9], clean[6:9])  # rows 24, 25, 26; the other request
            if not np.isfinite(bad):
                # (a K scale and bias of infinity, which the append does not write: s (q.c) + b (sum of q) is -inf where both
                # sums are negative, exp of it 0, and the token is out of the row, as one of an fp16 cache would be)
                sees = out[3:6].view(3, 4, 64)[..., 32:]
                assert not torch.isfinite(sees).any() or (side == 0 and bad == np.inf)


def test_a_run_of_all_against_the_cache_in_full(cuda, rng):
    """reserve, append, attention over drafts and single tokens for several steps, truncate: as the cache in fp16 does it on the
    values that the quantised one stands for."""
    hq, hkv, hd, page, B, n_pages, bits, group = 8, 2, 64, 16, 5, 40, 8, 32
    pages = ops.quant_pages(n_pages, hkv, page, hd, bits, group, cuda)
    kp, vp = (torch.zeros(n_pages, hkv, page, hd, device=cuda) for _ in range(2))
    lens, table = torch.zeros(B, dtype=torch.int32, device=cuda), torch.full((B, 8), -1, dtype=torch.int32, device=cuda)
    free, count = torch.arange(n_pages, dtype=torch.int32, device=cuda), torch.full((1,), n_pages, dtype=torch.int32, device=cuda)
    ang = torch.rand(200, hd // 2, device=cuda) * 6
    for new in ([5, 17, 1, 0, 40], [1, 1, 1, 1, 1], [3, 1, 5, 2, 1], [0, 0, 0, 1, 0], [6, 6, 6, 6, 6]):
        step = ops.paged_reserve(lens, i32(new, cuda), table, free, count, page, max_tokens=70, kv_lens=lens, free_count_out=count)
        assert int(step.status) == 0
        T, used = 70, sum(new)
        qkv = torch.randn(T, (hq + 2 * hkv) * hd, device=cuda)
        q, q32 = torch.zeros(T, hq * hd, dtype=torch.float16, device=cuda), torch.zeros(T, hq * hd, device=cuda)
        ops.paged_rope_append_q(qkv, step.q_start, step.slots, step.positions, ang.cos(), ang.sin(), q, pages)
        ops.paged_rope_append(qkv, step.q_start, step.slots, step.positions, ang.cos(), ang.sin(), q32, kp, vp)
        assert torch.equal(q[:used], q32[:used].half())
        every = torch.arange(n_pages * page, dtype=torch.int32, device=cuda)
        k, v = (x.view(n_pages, page, hkv, hd).transpose(1, 2).contiguous() for x in ops.paged_read_q(pages, every, dtype=torch.float32))
        held = torch.zeros(n_pages * page, dtype=torch.bool, device=cuda)
        held[step.slots[:used].long()] = True
        for a, b in ((k, kp), (v, vp)):  # half a step of 255 of a range of less than 12
            assert (a - b).transpose(1, 2).reshape(-1, hkv, hd)[held].abs().max() <= 12 / 255 / 2
        out = ops.prefix_attn_q(q, pages, step.q_start, step.kv_lens, table)
        want = ops.prefix_attn(q.float(), k, v, step.q_start, step.kv_lens, table)
        assert (out[:used].float() - want[:used]).abs().max() <= 2.0**-9 * 4 and (out[used:] == 0).all()
        ops.paged_truncate(lens, (lens - i32([1, 0, 2, 0, 1], cuda)).clamp_min(0), table, free, count, page, lens_out=lens, free_count_out=count)


# ------------------------------------------------------------------------------------------------ how it is called

def test_two_streams_and_graphs(cuda, rng):
    """Calls on two streams at once, and two captured calls replayed over new inputs, give what calls one by one do."""
    ds = [make_attn(rng, 8, 2, 128, 16, 4, 64, 500, [700 + i, 300], [1, 1]) for i in range(2)]
    want = [run_attn(cuda, d) for d in ds]
    streams = [torch.cuda.Stream() for _ in ds]
    args = []
    for d in ds:
        args.append((d["q"].to(cuda), pool(d, cuda), i32(d["start"], cuda), i32(d["lens"], cuda), i32(d["table"], cuda), i32(d["ptab"], cuda),
                     i32([d["prefix"]], cuda)))
    torch.cuda.synchronize()
    for _ in range(5):
        outs = []
        for s, a in zip(streams, args):
            with torch.cuda.stream(s):
                outs.append(ops.prefix_attn_q(*a))
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(o[:2], w[:2])
    graphs, outs = [], []
    for a in args:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.prefix_attn_q(*a))
        graphs.append(g)
    args[0][0].mul_(0.5)
    for g in graphs:
        g.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[1][:2], want[1][:2])
    assert torch.equal(outs[0][:2], ops.prefix_attn_q(*args[0])[:2])


def test_refusals_on_the_gpu(cuda, rng):
    d = make_attn(rng, 8, 2, 64, 16, 4, 64, 20, [30], [1])
    q, pages = d["q"].to(cuda), pool(d, cuda)
    start, lens, table = i32(d["start"], cuda), i32(d["lens"], cuda), i32(d["table"], cuda)
    ops.prefix_attn_q(q, pages, start, lens, table)
    with pytest.raises(ValueError, match="float16"):
        ops.prefix_attn_q(q.float(), pages, start, lens, table)
    with pytest.raises(ValueError, match="contiguous"):
        ops.prefix_attn_q(q, pages._replace(data=pages.data.transpose(0, 1).contiguous().transpose(0, 1)), start, lens, table)
    with pytest.raises(ValueError, match="int32"):
        ops.prefix_attn_q(q, pages, start, lens.long(), table)
    with pytest.raises(ValueError, match="together"):
        ops.prefix_attn_q(q, pages, start, lens, table, prefix_table=table[0])
    with pytest.raises(ValueError, match="multiple"):
        ops.prefix_attn_q(q[:, :-8].contiguous(), pages, start, lens, table)
    with pytest.raises(ValueError, match="block_table"):
        ops.prefix_attn_q(q, pages, start, lens, table[0])
    with pytest.raises(ValueError, match="q_start"):
        ops.prefix_attn_q(q, pages, start[:1], lens, table)
    with pytest.raises(ValueError, match="uint8"):
        ops.prefix_attn_q(q, pages, start, lens, table, workspace=torch.empty(1 << 20, device=cuda))
    with pytest.raises(ValueError, match="boundaries"):
        ops.prefix_attn_q(torch.empty(q.numel() + 1, dtype=torch.float16, device=cuda)[1:].view(q.shape), pages, start, lens, table)
    with pytest.raises(ValueError, match="scale"):
        ops.prefix_attn_q(q, pages, start, lens, table, scale=0.0)
    with pytest.raises(ValueError, match="k_out"):
        ops.paged_read_q(pages, lens, k_out=torch.empty(3, device=cuda), v_out=torch.empty(3, device=cuda))
    with pytest.raises(ValueError, match="slots"):
        ops.paged_rope_append_q(torch.zeros(2, 12 * 64, device=cuda), start, lens, lens, torch.zeros(4, 32, device=cuda), torch.zeros(4, 32, device=cuda),
                                torch.zeros(2, 512, dtype=torch.float16, device=cuda), pages)
    with pytest.raises(ValueError, match="q_out"):
        ops.paged_rope_append_q(torch.zeros(1, 12 * 64, device=cuda), start, lens, lens, torch.zeros(4, 32, device=cuda), torch.zeros(4, 32, device=cuda),
                                torch.zeros(1, 512, device=cuda), pages)
    none = torch.empty(0, 512, dtype=torch.float16, device=cuda)
    assert ops.prefix_attn_q(none, pages, i32([0, 0], cuda), lens, table).shape == (0, 512)
    assert [x.shape for x in ops.paged_read_q(pages, lens[:0])] == [(0, 2, 64)] * 2


# ------------------------------------------------------------------------------------------------ many rows of queries

@pytest.mark.parametrize("hd,bits,group", KINDS)
@pytest.mark.parametrize("hq,hkv,page,prefix", [(8, 1, 16, 0), (6, 2, 64, 333), (8, 2, 256, 1)])
def test_attn_chunks(cuda, rng, hd, bits, group, hq, hkv, page, prefix):
    """Prompt chunks, some over tokens that were there before, beside requests with one row and with none."""
    new = [0, 1, 5, 137, 0, 100, 3, 170]
    lens = [20, 1, 5, 160, 0, 100, 40, 500]
    d = make_attn(rng, hq, hkv, hd, page, bits, group, prefix, lens, new)
    out = check_attn(cuda, d, hq, rounded=True)
    for _ in range(4):
        assert torch.equal(out, run_attn(cuda, d))


@pytest.mark.parametrize("hd,bits,group", KINDS)
@pytest.mark.parametrize("prefix,longest", [(2900, 40), (1111, 300)])
def test_attn_shared_by_many_requests(cuda, rng, hd, bits, group, prefix, longest):
    """Batches large enough for the prefix to be taken once for all, with absent pages in it and in a request."""
    new = [int(x) for x in rng.integers(0, 6, 48)]
    lens = [n + int(rng.integers(0, longest)) for n in new]
    hq, hkv = (32, 4) if hd == 64 else (24, 8)
    d = make_attn(rng, hq, hkv, hd, 32 if hd == 64 else 16, bits, group, prefix, lens, new)
    check_attn(cuda, d, hq, rounded=True)
    d["ptab"][[0, len(d["ptab"]) - 1]] = [-1, len(d["data"]) + 5]
    d["table"][7, 0] = -3
    out = check_attn(cuda, d, hq, rounded=True)
    for _ in range(4):
        assert torch.equal(out, run_attn(cuda, d))


@pytest.mark.parametrize("bits,group", [(4, 64), (8, 32)])
def test_attn_chunk_of_many_tiles(cuda, rng, bits, group):
    """Several tiles of rows and of keys in one CTA, and several shares of the keys, over and over."""
    for lens, new, prefix in (([900, 700], [600, 300], 0), ([300], [300], 5000), ([2600, 10], [80, 2], 1500)):
        d = make_attn(rng, 8, 2, 128, 32, bits, group, prefix, lens, new)
        out = check_attn(cuda, d, 8, rounded=True)
        for _ in range(4):
            assert torch.equal(out, run_attn(cuda, d))


def test_chunk_hidden_scales_do_not_reach_other_rows(cuda, rng):
    """Many rows: what is not finite in a chunk's later token shows in the rows that see it, and in no others."""
    d = make_attn(rng, 8, 1, 64, 16, 4, 32, 20, [400, 250], [300, 200], dirty=False)
    clean = run_attn(cuda, d)
    first = 350 - 100  # the row that first sees token 350
    for side in (0, 1):
        e = dict(d, data=d["data"].copy())
        m = 350 % 16
        at = oq.meta_place(side, m, 1, 64, 4, 32)
        e["data"][d["table"][0, 350 // 16], :, at:at + 4] = np.array([np.nan, np.nan], np.float16).view(np.uint8)
        out = run_attn(cuda, e)
        assert torch.equal(out[:first], clean[:first]) and torch.equal(out[300:500], clean[300:500])
        sees = out[first:300].view(-1, 8, 64)
        assert sees[..., 32:].isnan().all() and (side == 0 or torch.equal(sees[..., :32], clean[first:300].view(-1, 8, 64)[..., :32]))


def test_attn_pages_of_any_size(cuda, rng):
    for page in (16, 128, 1024, 32768):
        for lens, new, prefix in (([200, 33], [1, 1], 100), ([200, 133], [150, 130], 100)):
            d = make_attn(rng, 8, 2, 64, page, 8, 64, prefix, lens, new, dirty=page < 1000)
            check_attn(cuda, d, 8, rounded=True)


# ------------------------------------------------------------------------------------------------ cut otherwise than usual

@pytest.mark.parametrize("hd,bits,group", [(64, 4, 64), (64, 8, 32), (128, 4, 64), (128, 8, 64), (128, 8, 32)])
@pytest.mark.parametrize("drafts", [False, True])
def test_attn_pieces_of_long_requests(cuda, rng, hd, bits, group, drafts):
    """Lengths from nothing to thousands: CTAs that take the end of one request, all of others, and the start of one more; the
    same bits every time."""
    B, hq, hkv = (24, 8, 2) if drafts else (26, 8, 8)
    new = [int(x) for x in rng.integers(0, 9, B)] if drafts else [int(x) for x in rng.integers(0, 2, B)]
    lens = [n + int(x) for n, x in zip(new, np.where(rng.random(B) < 0.5, rng.integers(0, 40, B), rng.integers(0, 1500, B)))]
    new[3], lens[3], new[5], lens[5] = 1, 0, 1, 1  # a row that sees nothing, a row that sees one token
    lens[0], new[0] = 9000, 1
    for prefix in (0, 60):
        d = make_attn(rng, hq, hkv, hd, 32, bits, group, prefix, lens, new, dirty=False)
        out = check_attn(cuda, d, hq)
        for _ in range(3):
            assert torch.equal(out, run_attn(cuda, d))


@pytest.mark.parametrize("prefix,new,rows", [(0, [3, 5, 2], 7), (77, [1, 1, 1], 2), (0, [9, 150, 70], 100), (300, [150, 150], 299),
                                             (9000, [1] * 40 + [4], 42), (40, [20, 0, 7], 20), (0, [4, 4], 1), (0, [1] * 30, 17)])
def test_q_ends_before_the_last_request(cuda, rng, prefix, new, rows):
    """Fewer rows of q than were reserved: the rows that are there see what they see in the whole call."""
    hq, hkv, hd = 8, 2, 64
    d = make_attn(rng, hq, hkv, hd, 16, 4, 32, prefix, [n + (5000 if len(new) == 30 else 30) for n in new], new, pad=0, dirty=len(new) < 30)
    want, mass, dot, keys, tail = (x[:rows] for x in oq.attention(d["q"].double().numpy(), d["data"], d["start"], d["lens"], d["table"], d["ptab"],
                                                                  prefix, hq, hd, 16, 4, 32, 1 / math.sqrt(hd)))
    d["q"] = d["q"][:rows].contiguous()
    got = run_attn(cuda, d).double().cpu().numpy().reshape(want.shape)
    assert (np.abs(got - want) <= attn_bound(want, mass, dot, keys, tail, hd, rounded=True)).all()
    assert L.load().sc_prefix_attn_device_error(1) == 0


def test_offsets_that_cannot_be(cuda, rng):
    """Rows and lengths on the device that no reservation writes: whatever comes out, nothing is read or written out of bounds
    (offsets that fall and pass the rows, lengths below zero and past the tables, pages that are none) and the next call is as
    before."""
    for lens, new, prefix in (([30, 25, 9, 40], [1, 1, 1, 1], 20), ([6000] * 4, [1, 1, 1, 1], 20), ([300, 200, 150, 90], [150, 100, 100, 64], 20),
                              ([30] * 4, [1, 1, 1, 1], 40000)):
        d = make_attn(rng, 8, 2, 64, 16, 4, 32, prefix, lens, new, dirty=False)
        clean = run_attn(cuda, d)
        guard = torch.full((clean.numel() + 4096,), 5.0, dtype=torch.float16, device=cuda)
        out = guard[:clean.numel()].view(clean.shape)
        odd = dict(d, start=np.array([0, 10**6, -5, 2**31 - 1, 3]), lens=np.array([-7, 2**31 - 1, 0, -(2**31)]), table=d["table"].copy())
        odd["table"][:, 0] = [-1, 2**31 - 1, -(2**31), 10**6]
        run_attn(cuda, odd, out=out)
        run_attn(cuda, dict(odd, prefix=2**31 - 1), out=out)
        run_attn(cuda, dict(odd, prefix=-4), out=out)
        torch.cuda.synchronize()
        assert (guard[clean.numel():] == 5.0).all()
        assert torch.equal(run_attn(cuda, d), clean)


def test_two_graphs_share_a_workspace(cuda, rng):
    """Captured calls of other shapes and plans with one workspace, replayed in turn on one stream."""
    ds = [make_attn(rng, 8, 2, 128, 16, 4, 64, 900, [40, 90, 33], [1, 1, 1]), make_attn(rng, 4, 1, 64, 32, 8, 32, 3000, [700], [2]),
          make_attn(rng, 8, 4, 64, 32, 4, 64, 0, [20000] + [50] * 20, [1] * 21, dirty=False),
          make_attn(rng, 32, 4, 64, 32, 4, 32, 2900, [20] * 48, [1] * 48, dirty=False)]
    ws, calls = torch.empty(64 << 20, dtype=torch.uint8, device=cuda), []
    for d in ds:
        t = [d["q"].to(cuda), pool(d, cuda), i32(d["start"], cuda), i32(d["lens"], cuda), i32(d["table"], cuda)]
        pre = dict(prefix_table=i32(d["ptab"], cuda), prefix_len=i32([d["prefix"]], cuda))
        want, out = ops.prefix_attn_q(*t, **pre), torch.zeros_like(t[0])
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            ops.prefix_attn_q(*t, out=out, workspace=ws, **pre)
        calls.append((graph, out, want, (t, pre)))
    for _ in range(3):
        for graph, out, _, _ in calls:
            out.zero_()
            graph.replay()
        for _, out, want, _ in calls:
            assert torch.equal(out, want)


def test_workspace_that_is_too_small(cuda, rng):
    d = make_attn(rng, 8, 4, 64, 32, 4, 64, 0, [20000] + [50] * 20, [1] * 21, dirty=False)
    need = ops.prefix_attn_q_workspace_bytes(23, 21, 8, 4, 64, d["table"].shape[1], 1, 32)
    assert need > 0
    with pytest.raises(ValueError, match="workspace"):
        run_attn(cuda, d, workspace=torch.empty(need - 16, dtype=torch.uint8, device=cuda))
    assert torch.equal(run_attn(cuda, d), run_attn(cuda, d, workspace=torch.empty(need, dtype=torch.uint8, device=cuda)))


def test_many_requests(cuda):
    """More requests than threads of a CTA, most without a row, a few long: against the same requests alone."""
    B, hd, page, hq, hkv = 1000, 64, 16, 4, 2
    g = torch.Generator(device=cuda).manual_seed(5)
    lens = torch.full((B,), 16, dtype=torch.int32, device=cuda)
    lens[::97] = 4000
    blocks = 250
    n_pages = B // 97 * blocks + 2 * blocks
    pages = ops.quant_pages(n_pages, hkv, page, hd, 4, 64, cuda)
    one = torch.ones(n_pages * page, hd // 2, device=cuda)
    at = torch.arange(n_pages * page, dtype=torch.int32, device=cuda)
    x = torch.randn(n_pages * page, (1 + 2 * hkv) * hd, device=cuda, generator=g)
    ops.paged_rope_append_q(x, i32([0, len(at)], cuda), at, at, one, one * 0, torch.empty(len(at), hd, dtype=torch.float16, device=cuda), pages)
    table = torch.randint(0, n_pages, (B, blocks), dtype=torch.int32, device=cuda, generator=g)
    new = torch.zeros(B, dtype=torch.int32, device=cuda)
    new[::97] = 1
    new[5::50] = 1
    start = torch.cat([new.new_zeros(1), new.cumsum(0).int()])
    rows = int(start[-1])
    q = torch.randn(rows, hq * hd, device=cuda, generator=g).half()
    out = ops.prefix_attn_q(q, pages, start, lens, table)
    for r, b in enumerate(new.nonzero().flatten().tolist()):
        alone = ops.prefix_attn_q(q[r:r + 1].contiguous(), pages, i32([0, 1], cuda), lens[b:b + 1].contiguous(), table[b:b + 1].contiguous())
        # two ways to cut the same sums: weights rounded by up to 2^-11 of each about another reference, outputs by 2^-11
        assert (out[r] - alone[0]).abs().max() <= 2.0**-9 * 4
