"""Without a GPU: how calls of prefix_attn_q are cut, and that the bound of tests/test_quant_many_rows_gpu.py sees what it should."""

import numpy as np
import pytest

from shardcompute_b200 import _lib as L
from shardcompute_b200 import ops
from tests.test_quant_many_rows_gpu import bounds, chunks, oracle, plan_of, shared
from tests.test_quant_pages_gpu import KINDS, make_attn


@pytest.mark.parametrize("kind", ["chunks", "shared"])
@pytest.mark.parametrize("hd,bits,group", [(128, 4, 64), (64, 8, 32)])
def test_the_bound_sees_a_lost_block(kind, hd, bits, group):
    """An output of zeros breaks the norm's bound in every row and head that sees a key, and one that lost 16 or 32 keys, of the prefix or of a
    request, in most of those that see them."""
    rng = np.random.default_rng(1234)
    if kind == "chunks":
        hq, d = 6, chunks(rng, 6, 2, hd, 16, bits, group, 333)
    else:
        hq, d = shared(rng, hd, bits, group, 2900, 40)
    assert plan_of(d, hq).kind == kind
    want, *parts = oracle(d, hq, kind)
    each, whole = bounds(want, *parts, hd)
    sees = parts[2] > 0
    assert (np.linalg.norm(want, axis=-1) > whole)[sees].all() and (np.abs(want) > each)[sees].mean() > 0.95
    for where in ("prefix", "request"):
        lost = dict(d, table=d["table"].copy(), ptab=d["ptab"].copy())
        if where == "prefix":
            lost["ptab"][7] = -1
        else:
            lost["table"][:, 1] = -1
        other, *less = oracle(lost, hq, kind)
        hit = less[2] < parts[2]
        assert hit.any() and (np.linalg.norm(want - other, axis=-1) > whole)[hit].mean() > 0.5, where


def test_plans():
    """(the sizes of the serving cases: 32 heads of 128 over 8, 4 bits)"""
    def kind(T, B, own, prefix, hq=32, hkv=8, hd=128, page=16, bits=4, group=64):
        return ops.prefix_attn_q_plan(T, B, hq, hkv, hd, -(-own // page), max(1, -(-prefix // page)), page, bits, group)

    one = kind(4, 4, 120, 700)
    assert one.kind == "few" and one.cluster >= 2 and one.line == 0 and one.many == 0
    long = kind(2, 2, 131000, 0, page=128)
    assert long.kind == "few" and long.cluster == 0 and long.line > 148 and long.many == 0
    many = kind(64, 64, 1500, 8197)
    assert many.kind == "shared" and 40 <= many.many <= 148 and many.line > 0
    chunk = kind(12 * 410, 12, 1200, 2050)
    assert chunk.kind == "chunks" and chunk.line == 0 and chunk.many >= 148
    # what the tables could hold decides, not what they do hold: a table far wider than the lengths moves the requests' share of the SMs
    wide = kind(64, 64, 32768, 8197)
    assert wide.kind == "shared" and wide.many < many.many


@pytest.mark.parametrize("hd,bits,group", KINDS)
def test_plans_of_the_tests(hd, bits, group):
    """tests/test_quant_pages_gpu.py: which kernels its ragged and shared cases meet."""
    rng = np.random.default_rng(1234)
    decode = make_attn(rng, 8, 2, hd, 16, bits, group, 77, [1, 16, 17, 5, 130, 64], [1] * 6)
    assert plan_of(decode, 8).kind == "few" and plan_of(decode, 8).cluster > 0
    hq, d = shared(rng, hd, bits, group, 2900, 40)
    assert plan_of(d, hq).kind == "shared"
    line = make_attn(rng, 8, 8, hd, 32, bits, group, 0, [9000] + [40] * 25, [1] * 26, dirty=False)
    assert plan_of(line, 8) == plan_of(line, 8)._replace(kind="few", cluster=0, many=0) and plan_of(line, 8).line > 0


def test_plan_refuses():
    good = (4, 4, 8, 2, 64, 4, 64, 8, 8, 16)
    out = (L.C.c_int32 * 4)()
    plan = L.load().sc_prefix_attn_q_plan
    assert plan(*good, out) == L.SC_OK
    for at, value, code in [(0, 0, L.SC_ERR_SHAPE), (1, 0, L.SC_ERR_SHAPE), (2, 7, L.SC_ERR_SHAPE), (3, 0, L.SC_ERR_SHAPE), (4, 96, L.SC_ERR_UNSUPPORTED),
                            (5, 5, L.SC_ERR_UNSUPPORTED), (6, 16, L.SC_ERR_UNSUPPORTED), (7, -1, L.SC_ERR_SHAPE), (8, -1, L.SC_ERR_SHAPE),
                            (9, 0, L.SC_ERR_SHAPE), (0, 1 << 28, L.SC_ERR_SHAPE)]:
        assert plan(*good[:at], value, *good[at + 1:], out) == code, (at, value)
    assert plan(*good, None) == L.SC_ERR_ARG
    with pytest.raises(ValueError):
        ops.prefix_attn_q_plan(0, 1, 8, 2, 64, 4, 4, 16)
    with pytest.raises(NotImplementedError):
        ops.prefix_attn_q_plan(1, 1, 8, 2, 96, 4, 4, 16)
