"""prefix_attn_q where the many-rows kernel takes part (shared prefixes, chunks): the plan is asserted, and the outputs are compared with
float64 attention over the very fp16 values that the kernel makes of k and v (k in two terms for rows that see few keys), in a bound that a
lost block of keys breaks."""

import math

import numpy as np
import pytest
import torch

from oracle import quant_pages as oq
from shardcompute_b200 import _lib as L
from shardcompute_b200 import ops
from tests.test_quant_pages_gpu import KINDS, make_attn, run_attn

pytestmark = pytest.mark.gpu
FP16 = {"few": "none", "shared": "prefix", "chunks": "all"}


def plan_of(d, hq):
    hd, page, bits, group = d["kind"]
    return ops.prefix_attn_q_plan(len(d["q"]), len(d["lens"]), hq, d["data"].shape[1], hd, d["table"].shape[1], len(d["ptab"]), page, bits, group)


def oracle(d, hq, kind, scale=None):
    hd, page, bits, group = d["kind"]
    return oq.attention(d["q"].double().numpy(), d["data"], d["start"], d["lens"], d["table"], d["ptab"], d["prefix"], hq, hd, page, bits, group,
                        1 / math.sqrt(hd) if scale is None else scale, fp16=FP16[kind])


def bounds(want, mass, dot, keys, tail, spread, split, hd):
    """How far an output, and the norm of a (row, head), may be off.  With e = 2^-24, p = 2^-11:
      score   S adds 16 dims at a time to an fp32 sum, each time off by at most 2 e of the largest sum; scales, biases and the difference
              to the maximum are a few roundings more: ds = dot (hd / 16 + 6) 2 e; and split, what two terms of fp16 are off k
      weight  w (1 + 2 ds + 8 e), rounded to fp16 (p; steps of 2^-36 of the largest weight: tail), codes' times s before
      output  mass (2 ds + 16 e + 2 p + 2 e (keys / 8 + 64)) for numerator and denominator, then its rounding to fp16
    In the norm the keys' roundings, up to p each whichever way, are independent of one another: six standard deviations of their sum,
    p / sqrt(3) spread, in place of p mass."""
    e, p = 2.0**-24, 2.0**-11
    ds = (dot * (hd / 16 + 6) * 2 * e + split)[..., None]
    sums = mass * (2 * ds + 16 * e + 2 * e * (keys[..., None] / 8 + 64)) + 2.0**-36 * 1.01 * tail + 2.0**-25
    last = p * 1.01 * np.abs(want)
    norm = lambda x: np.linalg.norm(x, axis=-1)  # noqa: E731
    return sums + 2 * p * mass + last, norm(sums) + 6 * p / math.sqrt(3) * norm(spread) + norm(last)


def check(cuda, d, hq, kind, scale=None, prepared=None):
    assert plan_of(d, hq).kind == kind
    out = run_attn(cuda, d, scale=scale)
    want, *parts = prepared or oracle(d, hq, kind, scale)
    rows = int(d["start"][-1])
    got = out[:rows].double().cpu().numpy().reshape(want.shape)
    each, whole = bounds(want, *parts, d["kind"][0])
    err = np.abs(got - want)
    worst = np.unravel_index(np.argmax(err / each), err.shape)
    assert np.isfinite(got).all() and (err <= each).all(), (worst, got[worst], want[worst], each[worst])
    off = np.linalg.norm(err, axis=-1)
    worst = np.unravel_index(np.argmax(off / whole), off.shape)
    assert (off <= whole).all(), (worst, off[worst], whole[worst])
    assert (out[rows:] == 5.0).all()
    assert L.load().sc_prefix_attn_device_error(1) == 0
    for _ in range(3):
        assert torch.equal(out, run_attn(cuda, d, scale=scale))
    return out


def chunks(rng, hq, hkv, hd, page, bits, group, prefix):
    """Prompt chunks, some over tokens that were there before, beside requests with one row and with none."""
    return make_attn(rng, hq, hkv, hd, page, bits, group, prefix, [20, 1, 5, 160, 0, 100, 40, 3300], [0, 1, 5, 137, 0, 100, 3, 170])


def shared(rng, hd, bits, group, prefix, longest):
    hq, hkv, page = (32, 4, 32) if hd == 64 else (24, 8, 16)
    new = [int(x) for x in rng.integers(0, 6, 48)]
    lens = [n + int(rng.integers(0, longest)) for n in new]
    lens[5], new[5], lens[6], new[6] = 0, 2, longest, 1  # rows that see the prefix alone
    return hq, make_attn(rng, hq, hkv, hd, page, bits, group, prefix, lens, new)


@pytest.mark.parametrize("hd,bits,group", KINDS)
@pytest.mark.parametrize("hq,hkv,page,prefix", [(8, 1, 16, 0), (6, 2, 64, 333), (8, 2, 256, 1)])
def test_chunks(cuda, rng, hd, bits, group, hq, hkv, page, prefix):
    check(cuda, chunks(rng, hq, hkv, hd, page, bits, group, prefix), hq, "chunks")


@pytest.mark.parametrize("hd,bits,group", KINDS)
@pytest.mark.parametrize("lens,new,prefix", [([900, 700], [600, 300], 0), ([300], [300], 5000), ([2600, 10], [80, 2], 1500)], ids=["own", "prefix", "both"])
def test_chunk_of_many_tiles(cuda, rng, hd, bits, group, lens, new, prefix):
    check(cuda, make_attn(rng, 8, 2, hd, 32, bits, group, prefix, lens, new), 8, "chunks")


@pytest.mark.parametrize("hd,bits,group", KINDS)
@pytest.mark.parametrize("prefix,longest", [(2900, 40), (4000, 300)])
def test_shared_by_many_requests(cuda, rng, hd, bits, group, prefix, longest):
    """The prefix once for all, then with absent pages in it and in a request."""
    hq, d = shared(rng, hd, bits, group, prefix, longest)
    check(cuda, d, hq, "shared")
    d["ptab"][[0, 3, len(d["ptab"]) - 1]] = [-1, -2, len(d["data"]) + 5]
    d["table"][6, 0] = -3
    check(cuda, d, hq, "shared")


def test_absent_pages_in_chunks(cuda, rng):
    d = chunks(rng, 8, 2, 128, 16, 4, 64, 333)
    d["ptab"][[0, 5, len(d["ptab"]) - 1]] = [-1, -7, len(d["data"]) + 5]
    d["table"][7, [0, 3, 100]], d["table"][5, :] = -1, -1
    check(cuda, d, 8, "chunks")


@pytest.mark.parametrize("hd,bits,group", [(128, 4, 64), (64, 8, 32)])
def test_values_of_any_size_in_chunks(cuda, rng, hd, bits, group):
    """Biases large beside their groups' ranges, subnormal values and large ones: what fp16 makes of s c + b."""
    for kv, shift in ((1.0, 30.0), (1e-6, 0.0), (2e3, -500.0)):
        d = make_attn(rng, 8, 2, hd, 32, bits, group, 100, [900, 700], [600, 300], dirty=False, scale_q=0.05 / kv if kv > 1 else 0.5)
        k, v = (rng.standard_normal((len(d["data"]), 2, 32, hd)) * kv + shift for _ in range(2))
        d["data"] = oq.fill(k.astype(np.float32), v.astype(np.float32), bits, group)
        check(cuda, d, 8, "chunks")


def test_hidden_groups_in_chunks(cuda, rng):
    """A chunk's later token that is not finite shows in the rows that see it: of k everywhere, of v in its group's dims, whatever the
    scale that stands beside the bias of NaN; the other rows and dims are what they were, bit for bit."""
    d = make_attn(rng, 8, 1, 64, 16, 4, 32, 20, [3400, 250], [300, 200], dirty=False)
    assert plan_of(d, 8).kind == "chunks"
    clean = run_attn(cuda, d)
    first = 3350 - 3100  # the row that first sees token 3350
    for side in (0, 1):
        for scale in (np.inf, 1.0):
            e = dict(d, data=d["data"].copy())
            at = oq.meta_place(side, 3350 % 16, 1, 64, 4, 32)
            e["data"][d["table"][0, 3350 // 16], :, at:at + 4] = np.array([scale, np.nan], np.float16).view(np.uint8)
            out = run_attn(cuda, e)
            assert torch.equal(out[:first], clean[:first]) and torch.equal(out[300:500], clean[300:500])
            sees, was = out[first:300].view(-1, 8, 64), clean[first:300].view(-1, 8, 64)
            assert sees[..., 32:].isnan().all() and (side == 0 or torch.equal(sees[..., :32], was[..., :32]))


@pytest.mark.parametrize("hd,bits,group", KINDS)
@pytest.mark.parametrize("middle", [0.0, 0.4, 30.0, -1000.0])
def test_scores_of_codes_beside_a_large_bias(cuda, rng, middle, hd, bits, group):
    """Keys whose codes the rounding of s c + b to fp16 would lose: two tokens of a prefix with equal scores, though their codes differ (q is
    the same over eight dims, over which both have one sum), of values 1 and 0.  The output is 1 / (1 + exp(-x)), x the difference of the
    scores, which two terms of fp16 leave off by no more than the oracle's bound of them and fp32's steps: the scale makes that 2."""
    hq, T, most = 8, 200, 2**bits - 1
    codes = rng.integers(0, most + 1, (2, hd // 8, 8))
    for a, c in ((codes[0, g], codes[1, g]) for g in range(hd // 8)):
        while a.sum() != c.sum():
            i = rng.integers(0, 8)
            c[i] = min(max(c[i] + np.sign(a.sum() - c.sum()), 0), most)
    n, s = hd // group, np.float16(1.37 / 2**bits)
    data = np.zeros((1, 1, oq.block_bytes(hd, bits, group)), np.uint8)
    half = float(s) * 2.0 ** (bits - 1)
    scales, biases = np.full((1, n), s, np.float16), np.full((1, n), middle - half, np.float16)
    for t in (0, 1):
        oq.put(data, t, 16, 0, codes[t].reshape(1, hd), scales, biases, bits, group)
        oq.put(data, t, 16, 1, np.full((1, hd), t), np.ones((1, n), np.float16), np.zeros((1, n), np.float16), bits, group)
    q = torch.from_numpy(np.repeat(rng.standard_normal((T, hq, hd // 8)), 8, -1).reshape(T, -1)).half()
    size = q.double().abs().view(T, hq, hd).sum(-1).max().item()
    # as in bounds(): split, and (hd / 16 + 6) 2^-23 of sum |q| |k|
    off = 2.0**-15 * half if abs(middle) < 0.9 * half else 2.0**-11 * half
    limit = 2 * size * (off + (hd / 16 + 6) * 2.0**-23 * (abs(middle) + half))
    pages = ops.QuantPages(torch.from_numpy(data).to(cuda), hd, 16, bits, group)
    i = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    table = torch.full((1, 2048), -1, dtype=torch.int32, device=cuda)  # room for many tokens, none there
    assert ops.prefix_attn_q_plan(T, 1, hq, 1, hd, 2048, 1, 16, bits, group).kind == "chunks"
    out = ops.prefix_attn_q(q.to(cuda), pages, i([0, T]), i([0]), table, prefix_table=i([0]), prefix_len=i([2]), scale=2.0 / limit)
    got = out.double().cpu().numpy()
    assert (np.abs(np.log(got / (1 - got))) <= 2.008).all(), (got.min(), got.max())


@pytest.mark.parametrize("hd,bits,group", [(128, 4, 64), (64, 8, 32)])
@pytest.mark.parametrize("prefix", [0, 1, 100, 1023, 1024, 2000])
def test_a_table_for_a_longer_prefix(cuda, rng, prefix, hd, bits, group):
    """A call planned for a prefix of 4096 that holds less: a short one is the few-rows kernel's, as codes; the same bits every time."""
    hq, d = shared(rng, hd, bits, group, prefix, 40)
    page = d["kind"][1]
    ptab = np.full(4096 // page, -1, np.int32)
    ptab[:len(d["ptab"])] = d["ptab"]
    check(cuda, dict(d, ptab=ptab), hq, "shared", prepared=oracle(d, hq, "shared"))


@pytest.mark.parametrize("hd,bits,group", [(128, 4, 64), (128, 8, 32), (64, 4, 32), (64, 8, 64)])
@pytest.mark.parametrize("lens,new,prefix", [([1500], [1500], 0), ([300, 1300, 90], [300, 700, 80], 700), ([3400, 20], [900, 20], 0)])
def test_rows_that_see_few_keys_beside_rows_that_see_many(cuda, rng, lens, new, prefix, hd, bits, group):
    """Tiles of rows on both sides of 1024 keys in one call."""
    d = make_attn(rng, 8, 2, hd, 16, bits, group, prefix, lens, new)
    page = d["kind"][1]
    table = np.full((len(lens), 8192 // page), -1, np.int32)
    table[:, :d["table"].shape[1]] = d["table"]
    check(cuda, dict(d, table=table), 8, "chunks", prepared=oracle(d, 8, "chunks"))


def wide(d, tokens=8192):
    """The same call with a block table that could hold `tokens` a request."""
    table = np.full((len(d["lens"]), tokens // d["kind"][1]), -1, np.int32)
    table[:, :d["table"].shape[1]] = d["table"]
    return dict(d, table=table)


def test_hidden_groups_in_chunks_of_few_keys(cuda, rng):
    """As test_hidden_groups_in_chunks, where k is taken as two terms."""
    d = wide(make_attn(rng, 8, 1, 64, 16, 4, 32, 20, [400, 250], [300, 200], dirty=False))
    assert plan_of(d, 8).kind == "chunks"
    clean = run_attn(cuda, d)
    first = 350 - 100  # the row that first sees token 350
    for side in (0, 1):
        for scale in (np.inf, 1.0):
            e = dict(d, data=d["data"].copy())
            at = oq.meta_place(side, 350 % 16, 1, 64, 4, 32)
            e["data"][d["table"][0, 350 // 16], :, at:at + 4] = np.array([scale, np.nan], np.float16).view(np.uint8)
            out = run_attn(cuda, e)
            assert torch.equal(out[:first], clean[:first]) and torch.equal(out[300:500], clean[300:500])
            sees, was = out[first:300].view(-1, 8, 64), clean[first:300].view(-1, 8, 64)
            assert sees[..., 32:].isnan().all() and (side == 0 or torch.equal(sees[..., :32], was[..., :32]))


@pytest.mark.parametrize("hd,bits,group", [(128, 4, 64), (128, 8, 64), (64, 8, 32)])
def test_keys_at_the_ends_of_fp16s_range_in_chunks(cuda, rng, hd, bits, group):
    """Groups of k that reach +-65504: neither term of theirs, nor the one, becomes an infinity."""
    for lens, new in (([300, 90], [200, 80]), ([1500], [300])):
        d = wide(make_attn(rng, 8, 2, hd, 16, bits, group, 0, lens, new, dirty=False))
        k = rng.uniform(-1, 1, (len(d["data"]), 2, 16, hd // group, group)) * 65504 * rng.choice([1.0, 0.6, 0.3], (len(d["data"]), 2, 16, hd // group, 1))
        k[..., 0], k[..., 1] = 65504 * rng.choice([1, 0.9, -0.5], k.shape[:-1]), -65504 * rng.choice([1, 0.8, -0.7], k.shape[:-1])
        v = rng.standard_normal((len(d["data"]), 2, 16, hd)) + 0.3
        d["data"] = oq.fill(k.reshape(v.shape).astype(np.float32), v.astype(np.float32), bits, group)
        d["q"] = (d["q"] * 2e-5).half()
        check(cuda, d, 8, "chunks")


def test_captured_chunks(cuda, rng):
    """Chunks on both sides of 1024 keys and a shared prefix, captured with one workspace and replayed in turn, and on two streams at once."""
    i = lambda a: torch.from_numpy(np.ascontiguousarray(np.asarray(a, np.int32))).to(cuda)  # noqa: E731
    ds = [(8, wide(make_attn(rng, 8, 2, 128, 16, 4, 64, 0, [1500, 90], [1200, 80]))), (8, wide(make_attn(rng, 8, 2, 64, 16, 8, 32, 1100, [500], [400]))),
          shared(rng, 64, 4, 32, 2900, 40), (32, wide(make_attn(rng, 32, 8, 128, 16, 4, 64, 40, [300] * 12, [290] * 12)))]
    ws, calls = torch.empty(256 << 20, dtype=torch.uint8, device=cuda), []
    for hq, d in ds:
        t = [d["q"].to(cuda), ops.QuantPages(torch.from_numpy(d["data"]).to(cuda), *d["kind"]), i(d["start"]), i(d["lens"]), i(d["table"])]
        pre = dict(prefix_table=i(d["ptab"]), prefix_len=i([d["prefix"]]))
        want, out = ops.prefix_attn_q(*t, **pre), torch.zeros_like(t[0])
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            ops.prefix_attn_q(*t, out=out, workspace=ws, **pre)
        calls.append((graph, out, want, t, pre))
    assert {plan_of(d, hq).kind for hq, d in ds} == {"chunks", "shared"}
    for _ in range(5):
        for graph, out, *_ in calls:
            out.zero_()
            graph.replay()
        for _, out, want, *_ in calls:
            assert torch.equal(out, want)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        outs = []
        for n, (_, _, want, t, pre) in enumerate(calls):
            with torch.cuda.stream(streams[n % 2]):
                outs.append(ops.prefix_attn_q(*t, **pre))
        torch.cuda.synchronize()
        for o, (_, _, want, *_) in zip(outs, calls):
            assert torch.equal(o, want)
