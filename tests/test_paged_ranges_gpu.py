"""The attention over a paged cache where number formats run out: weights far below the row's largest, values of any
size, scores past what fp32 steps finely, in every kernel that a call may be cut into.  Against float64 on the device."""

import math

import numpy as np
import pytest
import torch

from shardcompute_b200 import _lib as L
from shardcompute_b200 import ops
from tests.test_paged_gpu import DT, attn_bound, i32

pytestmark = pytest.mark.gpu

PAGE, HQ, HKV, HD = 16, 16, 4, 64
# requests, new tokens of each, whether the keys are a prefix: one token of one request (few rows), a token each of many
# behind a prefix (the prefix once for all), a prompt chunk
KINDS = {"few": (1, 1, False), "shared": (32, 1, True), "chunk": (1, 150, False)}


def batch(cuda, kind, dtype, keys, own=9):
    """Pools in order, tables and q of a kind of call whose rows see `keys` tokens, or almost: [n_pages, HKV, PAGE, HD] of
    zeros for k and v, and `at`, the flat token index of key j."""
    B, new, shared = KINDS[kind]
    lens = [own] * B if shared else [keys] * B
    per, pre = -(-lens[0] // PAGE), -(-keys // PAGE) if shared else 0
    n_pages = B * per + pre
    pool = lambda: torch.zeros(n_pages, HKV, PAGE, HD, dtype=torch.float64, device=cuda)  # noqa: E731
    table = torch.arange(B * per, dtype=torch.int32, device=cuda).view(B, per)
    ptab = torch.arange(B * per, n_pages, dtype=torch.int32, device=cuda)
    return dict(k=pool(), v=pool(), q=torch.zeros(B * new, HQ, HD, dtype=torch.float64, device=cuda), lens=lens, new=new, table=table, ptab=ptab,
                P=keys if shared else 0, first=B * per if shared else 0, kw=dict(prefix_table=ptab, prefix_len=i32([keys], cuda)) if shared else {})


def run(d, dtype, cuda, scale=None):
    """Rounds to the type, calls, and returns the outputs beside float64's and attn_bound's parts, all of the rounded values."""
    dt, B, new = DT[dtype], len(d["lens"]), d["new"]
    q, k, v = (d[n].to(dt) for n in "qkv")
    start = i32(np.arange(B + 1) * new, cuda)
    out = ops.prefix_attn(q.view(B * new, HQ * HD), k, v, start, i32(d["lens"], cuda), d["table"], scale=scale, **d["kw"]).view(B * new, HQ, HD)
    assert L.load().sc_prefix_attn_device_error(1) == 0
    scale = 1 / math.sqrt(HD) if scale is None else scale
    want, mass, tail = (torch.zeros(B * new, HQ, HD, dtype=torch.float64, device=cuda) for _ in range(3))
    dot, keys = (torch.zeros(B * new, HQ, dtype=torch.float64, device=cuda) for _ in range(2))
    G = HQ // HKV
    for b in range(B):
        n, rows = d["lens"][b], slice(b * new, (b + 1) * new)
        for h in range(HKV):
            flat = lambda x: torch.cat([x[d["ptab"].long(), h].reshape(-1, HD)[: d["P"]], x[d["table"][b].long(), h].reshape(-1, HD)[:n]]).double()  # noqa: E731
            kk, vv, qq = flat(k), flat(v), q[rows, h * G:(h + 1) * G].double()
            hidden = torch.arange(len(kk), device=cuda) > d["P"] + n - new + torch.arange(new, device=cuda)[:, None]
            s = ((qq @ kk.T) * scale).masked_fill(hidden[:, None], -math.inf)
            w = torch.exp(s - s.amax(-1, keepdim=True))
            l = w.sum(-1, keepdim=True)
            at = (rows, slice(h * G, (h + 1) * G))
            want[at], mass[at] = w @ vv / l, w @ vv.abs() / l
            tail[at] = (~hidden).double()[:, None] @ vv.abs() / l
            dot[at] = scale * (qq.abs() @ kk.abs().T).masked_fill(hidden[:, None], 0).amax(-1)
            keys[at] = (~hidden).sum(-1)[:, None].double()
    return [x.double().cpu().numpy() for x in (out, want, mass, dot, keys, tail)]


def check(dtype, out, want, mass, dot, keys, tail):
    """attn_bound, but that weights of fp16 keep 2^-11 of their size down to 2^-25 of the row's largest and a step of 2^-35
    below: a row's weights are taken 2^11 to 2^15 high into fp16, whose step below 2^-14 is 2^-24."""
    bound = attn_bound(dtype, want, mass, dot, keys, tail, HD)
    if dtype == "f16":
        bound = bound - 2.0**-25 * tail + 2.0**-36 * tail
    err = np.abs(out - want)
    worst = np.unravel_index(np.argmax(err - bound), err.shape)
    assert np.isfinite(out).all() and (err <= bound).all(), (worst, out[worst], want[worst], bound[worst])


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("keys,bits", [(4099, 20.6), (16384, 20.6), (16384, 25.3)])
@pytest.mark.parametrize("alike,sink", [(True, 0.0), (False, 0.0), (True, 1.0)])
def test_first_key_takes_most_of_the_weight(cuda, dtype, kind, keys, bits, alike, sink):
    """The first key's weight is 2^bits times any other's, its value `sink`; the thousands of others, alike or nearly, are
    what is left of the output, or a visible part of it."""
    g = torch.Generator(device=cuda).manual_seed(11)
    d = batch(cuda, kind, dtype, keys)
    u = torch.nn.functional.normalize(torch.randn(HKV, HD, generator=g, device=cuda, dtype=torch.float64), dim=-1)
    size = math.sqrt(bits * math.log(2) * math.sqrt(HD))
    if not alike:
        d["k"] += 0.02 * torch.randn(d["k"].shape, generator=g, device=cuda, dtype=torch.float64)
    d["k"][d["first"], :, 0] = u * size
    d["v"] += 0.5 + torch.rand(d["v"].shape, generator=g, device=cuda, dtype=torch.float64)
    d["v"][d["first"], :, 0] = sink
    d["q"] += (u * size).repeat_interleave(HQ // HKV, 0)
    check(dtype, *run(d, dtype, cuda))


def normal(d, cuda, seed=5):
    g = torch.Generator(device=cuda).manual_seed(seed)
    for n in "kvq":
        d[n] += torch.randn(d[n].shape, generator=g, device=cuda, dtype=torch.float64)
    return g


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("what,size", [("v", 1e-6), ("v", 1e-9), ("v", 1e-20), ("v", 1e5), ("v", 1e30), ("kq", 1e-6), ("kq", 1e6), ("kq", 1e-20),
                                       ("kq", 1e20)])
def test_fp32_values_of_any_size(cuda, kind, what, size):
    """v, or k against q, scaled far out of fp16's range: attn_bound is relative to the values, and holds as it is."""
    d = batch(cuda, kind, "f32", 4099)
    normal(d, cuda)
    if what == "v":
        d["v"] *= size
    else:
        d["k"] *= size
        d["q"] /= size
    check("f32", *run(d, "f32", cuda))


@pytest.mark.parametrize("kind", KINDS)
def test_fp32_values_of_all_sizes_at_once(cuda, kind):
    """Every value of v with a power of two of its own, every channel of k with one that q has the inverse of."""
    d = batch(cuda, kind, "f32", 4099)
    g = normal(d, cuda)
    two = lambda *shape: 2.0 ** torch.randint(-40, 41, shape, generator=g, device=cuda).double()  # noqa: E731
    d["v"] *= two(*d["v"].shape)
    e = two(HKV, HD)
    d["k"] *= e[:, None]
    d["q"] /= e.repeat_interleave(HQ // HKV, 0)
    check("f32", *run(d, "f32", cuda))


@pytest.mark.parametrize("keys", [200, 4099])
def test_fp32_large_hidden_values(cuda, keys):
    """Finite values of 1e30 among a chunk's last tokens: the rows before are the same bits as without, those that see them
    are within the bound."""
    outs = []
    for size in (1.0, 1e30):
        d = batch(cuda, "chunk", "f32", keys)
        normal(d, cuda)
        page, off = divmod(keys - 20, PAGE)
        d["v"][page, :, off] *= size
        r = run(d, "f32", cuda)
        check("f32", *r)
        outs.append(r[0])
    assert np.array_equal(outs[0][:130], outs[1][:130]) and (outs[0][130:] != outs[1][130:]).any()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype,size", [("f16", 200.0), ("f16", 1000.0), ("f16", 4000.0), ("f16", 15000.0), ("f32", 1e3), ("f32", 3e4), ("f32", 1e6),
                                        ("f32", 1e9), ("f32", 1e15)])
def test_large_scores(cuda, kind, dtype, size):
    """q and k so large that a row's largest score alone counts: its value comes out, by as much as its own weight (fp16:
    2^-11) and the output (as much again) are rounded; fp32: three roundings of 2^-24 and a quotient's, below 2^-20.  Rows
    whose two largest scores differ by less than the products' error, 2^-16 of sum |q| |k|, are only looked at for numbers."""
    d = batch(cuda, kind, dtype, 4099)
    normal(d, cuda)
    for n in "kq":
        d[n] = d[n].clamp(-4, 4) * size
    out, want, mass, dot, keys, tail = run(d, dtype, cuda)
    assert np.isfinite(out).all()
    q, k = d["q"].to(DT[dtype]).double(), d["k"].to(DT[dtype]).double()
    G, new, clear = HQ // HKV, d["new"], []
    for b, n in enumerate(d["lens"]):
        for h in range(HQ):
            flat = torch.cat([k[d["ptab"].long(), h // G].reshape(-1, HD)[: d["P"]], k[d["table"][b].long(), h // G].reshape(-1, HD)[:n]])
            s = q[b * new:(b + 1) * new, h] @ flat.T / math.sqrt(HD)
            s.masked_fill_(torch.arange(len(flat), device=cuda) > d["P"] + n - new + torch.arange(new, device=cuda)[:, None], -math.inf)
            two = s.topk(2).values
            clear.append((two[:, 0] - two[:, 1]).cpu().numpy())
    clear = np.concatenate([np.stack(clear[i:i + HQ], 1) for i in range(0, len(clear), HQ)])  # [rows, HQ]
    clear = clear > 20 + dot * 2.0**-16
    assert clear.mean() > 0.5
    assert np.abs(out - want)[clear].max() <= (2.0**-10 if dtype == "f16" else 2.0**-20) * 1.01 * np.abs(want).max()
