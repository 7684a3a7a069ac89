"""What the paged cache refuses and keeps, without a GPU."""

import pytest
import torch

from shardcompute_b200.parallel import PagedKVCache


def cache(**kw):
    a = dict(num_layers=1, kv_heads=2, head_dim=64, n_pages=4, max_batch=2, max_len=64, device=torch.device("cpu"))
    return PagedKVCache(**{**a, **kw})


@pytest.mark.parametrize("kw,match", [(dict(head_dim=40), "head_dim"), (dict(head_dim=256), "head_dim"), (dict(page_size=8), "page_size"),
                                      (dict(page_size=48), "page_size"), (dict(page_size=1 << 16), "page_size"),
                                      (dict(max_batch=16385), "requests"), (dict(max_tokens=0), "token"), (dict(max_tokens=-4), "token"),
                                      (dict(n_pages=1 << 26), "32 bits"), (dict(max_len=2**31 - 8), "32 bits"),
                                      (dict(max_prefix=2**31 - 1), "32 bits"), (dict(n_pages=0), "positive"), (dict(max_prefix=-1), "positive"),
                                      (dict(dtype=torch.bfloat16), "float16 or float32")])
def test_refuses_what_the_operators_do_not_take(kw, match):
    with pytest.raises(ValueError, match=match):
        cache(**kw)


@pytest.mark.parametrize("kw", [dict(), dict(head_dim=128, page_size=128, max_prefix=300), dict(dtype=torch.float16, max_tokens=1)])
def test_takes_the_rest(kw):
    c = cache(**kw)
    assert c.k.shape[2:] == (2, c.page_size, kw.get("head_dim", 64)) and int(c.free_count) == 4
    c.check()


def test_outgrown_rotary_tables_stay():
    """A captured step reads the tables that it was captured with: growing them must not free those."""
    import gc
    import weakref

    from shardcompute_b200.parallel import RoPE

    rope, cpu = RoPE(64), torch.device("cpu")
    first = weakref.ref(rope.tables(100, cpu)[0])
    small = rope.tables(100, cpu)[0].clone()
    big = rope.tables(5000, cpu)
    gc.collect()
    assert first() is not None and torch.equal(first(), small) and torch.equal(big[0][: len(small)], small)
    assert rope.tables(4000, cpu)[0] is big[0] and len(big[0]) == 5000
    assert sum(len(c) for c, _ in rope._outgrown) < len(big[0])


def test_attn_refuses_a_scale_that_overflows_with_log2_e():
    from shardcompute_b200 import _lib as L

    at = 1 << 20  # an address that no refused call reads
    call = lambda scale: L.load().sc_prefix_attn(at, at, at, L.SC_F16, 4, at, at, at, 4, 8, None, None, 0, 8, 2, 128, 100, 16, scale, at, at, 16,  # noqa: E731
                                                 None)
    assert call(3e38) == L.SC_ERR_ARG and "scale" in L.last_error()
