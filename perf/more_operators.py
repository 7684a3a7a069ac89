"""What the operators of a paged cache held in 8 or 4 bits are measured on.

Three operators, in the order in which a serving step meets them:

append    rotary embedding of q and k at each row's position; k and v quantised in groups and written to the rows' slots
          (read back here, so that what the cache stands for can be looked at)
read      tokens of a request read back from their slots
attn      each row attends to the shared prefix and to its own request's tokens, both held as codes

A group of `group` consecutive values x of one token and head is held as codes c of `bits` bits, a scale s and a bias b:
b is min(x) rounded down to fp16, s is (max(x) - b) / (2^bits - 1) rounded up to fp16, c = round((x - b) / s), and stands for
s c + b (c = 0 where s is zero).  Sixteen tokens of a head lie together as one block of bytes; ``_places`` has the order of the codes in it.

``run`` computes them in elementary torch operations in 32 bits, or, with ``own``, calls the framework.
"""

import functools
import math
import zlib

import torch

own = False

F16, F32 = "f16", "f32"
_DT = {F16: torch.float16, F32: torch.float32}


# ------------------------------------------------------------------------------------------------ cases

def listed():
    return [
        # the new tokens of 32 decoding requests, in the 32-layer 4096-wide model's head layout
        dict(name="append_step_32_q4", op="append", rows=32, pad=0, hq=32, hkv=8, hd=128, page=16, src=F32, bits=4, group=64),
        # chunks of prompts, padded to a bucket of rows, in the small model's head layout and the finer cache
        dict(name="append_chunk_8150_q8", op="append", rows=8150, pad=42, hq=32, hkv=4, hd=64, page=32, src=F32, bits=8, group=32),
        # one short request, moved to another server
        dict(name="read_700_q4", op="read", rows=700, pad=0, hkv=8, hd=128, page=16, out=F16, bits=4, group=64),
        # a long document's tokens, read back for a cache that holds them in full
        dict(name="read_40000_q8", op="read", rows=40000, pad=11, hkv=8, hd=128, page=64, out=F32, bits=8, group=32),
        # four requests behind a system prompt
        dict(name="attn_step_4_q4", op="attn", batch=4, min_new=1, max_new=1, prefix=700, max_own=120, hq=32, hkv=8, hd=128,
             page=16, pad=0, bits=4, group=64),
        # a full batch behind a long shared document whose last page is not full
        dict(name="attn_step_64_q4", op="attn", batch=64, min_new=1, max_new=1, prefix=8197, max_own=1500, hq=32, hkv=8, hd=128,
             page=16, pad=0, bits=4, group=64),
        # the largest batch, one rank of two of a 64-head model, larger pages
        dict(name="attn_step_256_q4", op="attn", batch=256, min_new=1, max_new=1, prefix=32768, max_own=2000, hq=32, hkv=4, hd=128,
             page=64, pad=0, bits=4, group=64),
        # two very long requests of their own, no prefix
        dict(name="attn_long_2_q4", op="attn", batch=2, min_new=1, max_new=1, prefix=0, max_own=131000, hq=32, hkv=8, hd=128,
             page=128, pad=0, bits=4, group=64),
        # as many kv heads as heads, the cache in 8 bits
        dict(name="attn_step_32_q8", op="attn", batch=32, min_new=1, max_new=1, prefix=0, max_own=3500, hq=16, hkv=16, hd=128,
             page=16, pad=3, bits=8, group=64),
        # speculative drafts of one to five tokens in the small model's layout, padded rows
        dict(name="attn_draft_16_q8", op="attn", batch=16, min_new=1, max_new=5, prefix=1000, max_own=400, hq=32, hkv=4, hd=64,
             page=32, pad=7, bits=8, group=32),
        # prompt chunks of a dozen requests behind the same instructions
        dict(name="attn_chunk_12_q4", op="attn", batch=12, min_new=120, max_new=700, prefix=2050, max_own=1200, hq=32, hkv=8, hd=128,
             page=16, pad=0, bits=4, group=64),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "read", "attn", "attn", "attn"])
    page = rng.choice([16, 32, 64, 128])
    hq, hkv, hd = rng.choice([(32, 8, 128), (16, 4, 128), (8, 1, 128), (32, 4, 64), (16, 16, 64), (6, 2, 64), (8, 8, 128)])
    kind = dict(hkv=hkv, hd=hd, page=page, bits=rng.choice([4, 4, 8]), group=rng.choice([32, 64]))
    if op == "append":
        return dict(op=op, rows=_log(rng, 1, 8150), pad=rng.choice([0, rng.randint(1, 63)]), hq=hq, src=rng.choice([F16, F32]), **kind)
    if op == "read":
        return dict(op=op, rows=_log(rng, 1, 40000), pad=rng.choice([0, rng.randint(1, 63)]), out=rng.choice([F16, F32]), **kind)
    if rng.random() < 0.3:  # chunks
        b, lo, hi = _log(rng, 1, 12), 1, _log(rng, 8, 700)
        prefix, most = rng.choice([0, _log(rng, 1, 2000)]), hi + _log(rng, 1, 1000)
    else:
        b, lo, hi = _log(rng, 1, 128), 1, rng.choice([1, 1, 1, 2, 6])
        prefix, most = rng.choice([0, _log(rng, 1, 16000), _log(rng, 1, 16000)]), hi + _log(rng, 1, min(60000, 200000 // b))
    return dict(op=op, batch=b, min_new=lo, max_new=hi, prefix=prefix, max_own=most, hq=hq, pad=rng.choice([0, rng.randint(1, 40)]), **kind)


# ------------------------------------------------------------------------------------------------ codes and their places

@functools.lru_cache(maxsize=None)
def _places(hd, bits, group, device):
    """Where a block of 16 tokens of one head has what: (bytes of the block, K's and V's code bytes, K's and V's scale bytes).

    The code bytes [16, hd * bits / 8]: the byte of the i-th 8 / bits consecutive dims of a token, the first of them in its low
    bits.  The scale bytes [16, hd / group]: a scale and the bias behind it, both fp16.  A token's K is split over four threads
    that each take a quarter of every group, one thread's share after another's (in 8 bits and heads of 128, where a share has
    two pieces of 16 bytes, first piece and second by halves of the row, changed over for odd tokens).  Its V is split over
    eight threads, each an eighth of every group, in units of two bytes that alternate between the two tokens of a pair; the
    threads' shares are exchanged by the pair's number.  So a warp's loads meet every bank of shared memory once."""
    row, per, n = hd * bits // 8, 8 // bits, hd // group
    tok = torch.arange(16)[:, None]
    d = torch.arange(0, hd, per)[None]
    g, r = d // group, d % group
    t, i = r // (group // 4), r % (group // 4)
    at = (t * (hd // 4) + g * (group // 4) + i) // per
    if row == 128:
        at = ((at % 32 // 16) ^ (tok % 2)) * 64 + t * 16 + at % 16
    k = tok * row + at
    lane, i = r // (group // 8), r % (group // 8)
    byte = (g * (group // 8) + i) // per
    byte = byte // 2 * 4 + tok % 2 * 2 + byte % 2  # in a share of two tokens
    pair, share = tok // 2, hd * bits // 32
    if share == 8:
        at = (lane ^ (pair // 2 % 2 * 4)) * 8 + byte
    else:
        at = byte // 16 * 128 + (lane ^ (pair % 4 * 2)) * 16 + byte % 16
    v = 16 * row + pair * 2 * row + at
    meta = 32 * row + (tok * n + torch.arange(n)[None]) * 4
    return (32 * row + 128 * n, *(x.expand(16, -1).contiguous().to(device) for x in (k, v, meta, meta + 64 * n)))


def _values(raw, meta, hd, bits, group):
    """Values [..., hd] in 32 bits of code bytes raw [..., hd * bits / 8] and scale bytes meta [..., hd / group, 4]."""
    codes = raw if bits == 8 else torch.stack([raw & 15, raw >> 4], -1).flatten(-2)
    sb = meta.contiguous().view(torch.float16).float()
    return (codes.float().unflatten(-1, (hd // group, group)) * sb[..., :1] + sb[..., 1:]).flatten(-2)


def _unpack(blocks, hd, bits, group):
    """Keys and values [..., 16, hd] in 32 bits of blocks [..., bytes]."""
    _, k, v, km, vm = _places(hd, bits, group, blocks.device)
    four = torch.arange(4, device=blocks.device)
    return [_values(blocks[..., at], blocks[..., meta[..., None] + four], hd, bits, group) for at, meta in ((k, km), (v, vm))]


def _down(x):
    """fp32 or fp64 to fp16, rounded down."""
    h = x.half()
    bits = h.view(torch.int16)
    less = torch.where(h == 0, torch.full_like(bits, -32767), torch.where(bits < 0, bits + 1, bits - 1)).view(torch.float16)
    return torch.where(h.to(x.dtype) > x, less, h)


def _quantise(x, bits, group):
    """x [..., hd] -> codes [..., hd] uint8, scales and biases [..., hd / group, 2] fp16."""
    x = x.float().unflatten(-1, (x.shape[-1] // group, group))
    most = 2 ** bits - 1
    b = _down(x.amin(-1))
    need = (x.amax(-1).double() - b.double()).clamp_min(0)
    s = -_down(-(need / most))  # to the side that 64 bits give, where the quotient is next to an fp16 value
    # in 64 bits: what lies next to the border of two codes goes to its own side
    c = ((x.double() - b.double()[..., None]) / s.double()[..., None]).round()
    c = torch.where(s[..., None] > 0, c, torch.zeros_like(c)).clamp(0, most).to(torch.uint8)
    return c.flatten(-2), torch.stack([s, b], -1)


def _base(data, slots, page, hd, bits, group):
    """The first byte [rows, hkv] of the block that holds each slot, in data [pages, hkv, bytes]."""
    size, hkv = _places(hd, bits, group, data.device)[0], data.shape[1]
    return ((slots // page * hkv)[:, None] + torch.arange(hkv, device=data.device)) * data.shape[-1] + (slots % page // 16 * size)[:, None]


def _store(data, slots, page, k, v, bits, group):
    """k and v [rows, hkv, hd], quantised, into the slots of data [pages, hkv, bytes]."""
    hd, slots, flat, four = k.shape[-1], slots.long(), data.view(-1), torch.arange(4, device=data.device)
    _, kat, vat, kmeta, vmeta = _places(hd, bits, group, data.device)
    base, tok = _base(data, slots, page, hd, bits, group), slots % 16
    for x, at, meta in ((k, kat, kmeta), (v, vat, vmeta)):
        codes, sb = _quantise(x, bits, group)
        flat[base[..., None] + at[tok][:, None]] = codes if bits == 8 else codes[..., ::2] | (codes[..., 1::2] << 4)
        flat[(base[..., None] + meta[tok][:, None])[..., None] + four] = sb.view(torch.uint8).view(*sb.shape[:-1], 4)


# ------------------------------------------------------------------------------------------------ inputs

def _dev():
    return torch.device("cuda", torch.cuda.current_device())


def _host(seed):
    g = torch.Generator().manual_seed(seed * 7919 + 29)
    return g, lambda lo, hi, n: torch.randint(lo, hi + 1, (n,), generator=g)


def _gpu(seed):
    return torch.Generator(device=_dev()).manual_seed(seed * 104729 + 11)


def _ceil(a, b):
    return -(-a // b)


def _page_bytes(case):
    return case["page"] // 16 * _places(case["hd"], case["bits"], case["group"], torch.device("cpu"))[0]


def _filled(case, pages, gg):
    """A cache full of tokens: keys with channels that stand out, as rotary keys have, and values off centre."""
    dev, hkv, hd, page = _dev(), case["hkv"], case["hd"], case["page"]
    data = torch.zeros(pages, hkv, _page_bytes(case), dtype=torch.uint8, device=dev)
    channel = torch.randn(hkv, hd, generator=gg, device=dev) * 1.5
    step = max(1, 200_000_000 // (hkv * hd * page * 8))
    for lo in range(0, pages, step):
        slots = torch.arange(lo * page, min(pages, lo + step) * page, device=dev)
        k = torch.randn(slots.numel(), hkv, hd, generator=gg, device=dev) + channel
        v = torch.randn(slots.numel(), hkv, hd, generator=gg, device=dev) * 0.7 + 0.2
        _store(data, slots, page, k, v, case["bits"], case["group"])
    return data


def _prepare_append(case, seed):
    g, ints = _host(seed)
    dev, gg = _dev(), _gpu(seed)
    rows, page, hd, hkv, hq = case["rows"], case["page"], case["hd"], case["hkv"], case["hq"]
    total = rows + case["pad"]
    pages = _ceil(rows, page) * 2 + 4
    # runs of tokens next to each other, as requests' chunks are, each in a place of its own
    run = min(total, 64 if rows > 200 else 1)
    starts = torch.randperm(pages * page // run, generator=g)[:_ceil(total, run)] * run
    slots = (starts[:, None] + torch.arange(run)).reshape(-1)[:total].int()
    most = 8192
    inv = 1.0 / (5e5 ** (torch.arange(0, hd, 2, dtype=torch.float64) / hd))
    ang = torch.outer(torch.arange(most, dtype=torch.float64), inv)
    back = torch.zeros(total, hkv, hd, dtype=torch.float16, device=dev)
    return dict(case, qkv=torch.randn(total, (hq + 2 * hkv) * hd, generator=gg, device=dev).to(_DT[case["src"]]), total=total,
                starts=torch.tensor([0, rows // 2, rows], dtype=torch.int32, device=dev), slots=slots.to(dev),
                positions=ints(0, most - 1, total).int().to(dev), cos=ang.cos().float().to(dev), sin=ang.sin().float().to(dev),
                data=torch.zeros(pages, hkv, _page_bytes(case), dtype=torch.uint8, device=dev),
                q=torch.zeros(total, hq * hd, dtype=torch.float16, device=dev), k=back, v=back.clone())


def _prepare_read(case, seed):
    g, _ = _host(seed)
    dev, gg = _dev(), _gpu(seed)
    rows, page = case["rows"], case["page"]
    total, blocks = rows + case["pad"], _ceil(rows + case["pad"], page)
    pages = blocks + 8
    table = torch.randperm(pages, generator=g)[:blocks]  # the request's pages lie scattered
    slots = (table[:, None] * page + torch.arange(page)).reshape(-1)[:total].int()
    out = torch.zeros(total, case["hkv"], case["hd"], dtype=_DT[case["out"]], device=dev)
    return dict(case, total=total, data=_filled(case, pages, gg), starts=torch.tensor([0, rows], dtype=torch.int32, device=dev),
                slots=slots.to(dev), k=out, v=out.clone())


def _prepare_attn(case, seed):
    # the case gives the lengths, so that outputs keep their shapes; the seed gives which request has which
    key = zlib.crc32(repr(sorted((k, v) for k, v in case.items() if k != "name")).encode())
    g, ints = _host(key)
    b, page, hd, hkv, hq, p = case["batch"], case["page"], case["hd"], case["hkv"], case["hq"], case["prefix"]
    new = ints(case["min_new"], case["max_new"], b)
    most = torch.maximum(torch.full((b,), case["max_own"]), new)
    lens = torch.minimum(new + (torch.rand(b, generator=g) * (most - new + 1)).long(), most)
    g, _ = _host(seed)
    dev, gg = _dev(), _gpu(seed)
    order = torch.randperm(b, generator=g)
    lens, new = lens[order], new[order]
    blocks, nb = (lens + page - 1) // page, _ceil(p, page)
    width, total = int(blocks.max()) + 1, int(blocks.sum())
    pages = total + nb + 8 + total // 10
    ids = torch.randperm(pages, generator=g).int()
    table = torch.full((b, width), -1, dtype=torch.int32)
    table[torch.arange(width)[None] < blocks[:, None]] = ids[:total]
    rows = int(new.sum())
    starts = torch.zeros(b + 1, dtype=torch.int32)
    starts[1:] = new.cumsum(0)
    q = (torch.randn(rows + case["pad"], hq * hd, generator=gg, device=dev) * 1.5).half()
    i32 = dict(dtype=torch.int32, device=dev)
    return dict(case, rows=rows, most_new=int(new.max()), most=int(lens.max()), q=q, data=_filled(case, pages, gg), starts=starts.to(dev),
                lens=lens.int().to(dev), table=table.to(dev), prefix_table=ids[total:total + nb].to(dev) if nb else torch.zeros(1, **i32),
                prefix_len=torch.tensor([p], **i32), out=torch.zeros_like(q))


def prepare(case, seed):
    return {"append": _prepare_append, "read": _prepare_read, "attn": _prepare_attn}[case["op"]](case, seed)


# ------------------------------------------------------------------------------------------------ plain forms

def _rows_of(s, slots):
    """Keys and values [rows, hkv, hd] in 32 bits that the slots hold."""
    slots, flat, four = slots.long(), s["data"].view(-1), torch.arange(4, device=s["data"].device)
    _, k, v, km, vm = _places(s["hd"], s["bits"], s["group"], flat.device)
    base, tok = _base(s["data"], slots, s["page"], s["hd"], s["bits"], s["group"]), slots % 16
    return [_values(flat[base[..., None] + at[tok][:, None]], flat[(base[..., None] + meta[tok][:, None])[..., None] + four], s["hd"], s["bits"],
                    s["group"]) for at, meta in ((k, km), (v, vm))]


def _plain_append(s):
    hq, hkv, hd, rows = s["hq"], s["hkv"], s["hd"], s["rows"]
    x = s["qkv"][:rows].float().view(rows, hq + 2 * hkv, hd)
    at = s["positions"][:rows].long()
    c, sn = s["cos"][at][:, None], s["sin"][at][:, None]
    x1, x2 = x[:, : hq + hkv, : hd // 2], x[:, : hq + hkv, hd // 2:]
    y = torch.cat([x1 * c - x2 * sn, x2 * c + x1 * sn], -1)
    s["q"][:rows] = y[:, :hq].reshape(rows, hq * hd).half()
    _store(s["data"], s["slots"][:rows], s["page"], y[:, hq:], x[:, hq + hkv:], s["bits"], s["group"])
    return dict(q=s["q"], **_plain_read(s))


def _plain_read(s):
    k, v = _rows_of(s, s["slots"][:s["rows"]])
    s["k"][:s["rows"]] = k.to(s["k"].dtype)
    s["v"][:s["rows"]] = v.to(s["v"].dtype)
    return dict(k=s["k"], v=s["v"])


def _pages_of(s, ids):
    """Keys and values [..., hkv, n * page, hd] in 32 bits of the pages ids [..., n]."""
    size = _places(s["hd"], s["bits"], s["group"], s["data"].device)[0]
    k, v = _unpack(s["data"][ids.long()].unflatten(-1, (-1, size)), s["hd"], s["bits"], s["group"])
    return [x.transpose(-5, -4).flatten(-4, -2) for x in (k, v)]


def _plain_attn(s):
    hq, hkv, hd, rows, page, p = s["hq"], s["hkv"], s["hd"], s["rows"], s["page"], s["prefix"]
    grp, b, dev = hq // hkv, s["lens"].numel(), s["q"].device
    q = s["q"][:rows].float().view(rows, hkv, grp, hd) * (1.0 / math.sqrt(hd))
    lens, starts = s["lens"].long(), s["starts"].long()
    t = torch.arange(rows, device=dev)
    seq = torch.searchsorted(starts[1:], t, right=True)
    i = t - starts[seq]
    # the requests' own tokens, padded to the longest
    nb = _ceil(s["most"], page)
    k2, v2 = _pages_of(s, s["table"][:, :nb].clamp_min(0))
    n = s["most_new"]
    qp = q.new_zeros(b, n, hkv, grp, hd)
    qp[seq, i] = q
    s2 = qp.permute(0, 2, 1, 3, 4).reshape(b, hkv, n * grp, hd) @ k2.transpose(-1, -2)
    last = lens - (starts[1:] - starts[:-1])
    seen = torch.arange(nb * page, device=dev)[None, None] <= (last[:, None] + torch.arange(n, device=dev)[None])[..., None]
    s2 = s2.view(b, hkv, n, grp, nb * page).masked_fill(~seen[:, None, :, None], -math.inf)
    m = s2.amax(-1)
    if p:
        k1, v1 = (x[:, :p] for x in _pages_of(s, s["prefix_table"]))
        s1 = (q.permute(1, 0, 2, 3).reshape(hkv, rows * grp, hd) @ k1.transpose(-1, -2)).view(hkv, rows, grp, p)
        m1 = s1.amax(-1)
        padded = m.new_full((b, n, hkv, grp), -math.inf)
        padded[seq, i] = m1.permute(1, 0, 2)
        m = torch.maximum(m, padded.permute(0, 2, 1, 3))
    s2 = (s2 - m.clamp_min(-1e30)[..., None]).exp()
    o2 = (s2.reshape(b, hkv, n * grp, nb * page) @ v2).view(b, hkv, n, grp, hd).permute(0, 2, 1, 3, 4)[seq, i]
    l = s2.sum(-1).permute(0, 2, 1, 3)[seq, i]
    if p:
        s1 = (s1 - m.permute(0, 2, 1, 3)[seq, i].permute(1, 0, 2)[..., None]).exp()
        o2 = o2 + (s1.view(hkv, rows * grp, p) @ v1).view(hkv, rows, grp, hd).permute(1, 0, 2, 3)
        l = l + s1.sum(-1).permute(1, 0, 2)
    o = torch.where(l[..., None] > 0, o2 / l[..., None], torch.zeros_like(o2))
    s["out"][:rows] = o.reshape(rows, hq * hd).half()
    return dict(out=s["out"])


def _own_pages(s):
    from shardcompute_b200 import ops
    return ops.QuantPages(s["data"], s["hd"], s["page"], s["bits"], s["group"])


def _own_append(s):
    from shardcompute_b200 import ops
    pages = _own_pages(s)
    ops.paged_rope_append_q(s["qkv"], s["starts"], s["slots"], s["positions"], s["cos"], s["sin"], s["q"], pages)
    ops.paged_read_q(pages, s["slots"], q_start=s["starts"], k_out=s["k"], v_out=s["v"])
    return dict(q=s["q"], k=s["k"], v=s["v"])


def _own_read(s):
    from shardcompute_b200 import ops
    ops.paged_read_q(_own_pages(s), s["slots"], q_start=s["starts"], k_out=s["k"], v_out=s["v"])
    return dict(k=s["k"], v=s["v"])


def _own_attn(s):
    from shardcompute_b200 import ops
    ops.prefix_attn_q(s["q"], _own_pages(s), s["starts"], s["lens"], s["table"], prefix_table=s["prefix_table"], prefix_len=s["prefix_len"],
                      out=s["out"])
    return dict(out=s["out"])


def run(state):
    if own:
        return {"append": _own_append, "read": _own_read, "attn": _own_attn}[state["op"]](state)
    return {"append": _plain_append, "read": _plain_read, "attn": _plain_attn}[state["op"]](state)


# ------------------------------------------------------------------------------------------------ work

def work(case):
    """Bytes and operations of the mean draw of lengths: a request's own length is even over its range."""
    op, hkv, hd = case["op"], case["hkv"], case["hd"]
    held = 2 * hkv * (hd * case["bits"] // 8 + 4 * hd // case["group"])  # a token's codes, scales and biases
    e = {F16: 2, F32: 4}
    if op == "append":
        rows, hq = case["rows"], case["hq"]
        return dict(bytes=rows * ((hq + 2 * hkv) * hd * e[case["src"]] + hq * hd * 2 + held + 4 * hkv * hd + 4 * hd + 8), flops=rows * hd * (6 * (hq + hkv) + 12 * hkv))
    if op == "read":
        return dict(bytes=case["rows"] * (held + 2 * hkv * hd * e[case["out"]] + 4), flops=4 * case["rows"] * hkv * hd)
    b, n, p, hq = case["batch"], (case["min_new"] + case["max_new"]) / 2, case["prefix"], case["hq"]
    own_len = (n + max(case["max_own"], n)) / 2
    pairs = b * n * p + b * n * (own_len - (n - 1) / 2)
    return dict(bytes=(p + b * own_len) * held + 4 * b * n * hq * hd, flops=4 * pairs * hq * hd)


# ------------------------------------------------------------------------------------------------ 64 bits

def _exact_tokens(raw, hd, bits, group):
    """Keys and values [n, 16, hd] in 64 bits of blocks raw [n, bytes], by cutting the bytes up as they lie."""
    n, row, per, dev = raw.shape[0], hd * bits // 8, 8 // bits, raw.device
    groups, share, out = hd // group, hd * bits // 32, []
    values = lambda x: x.double() if bits == 8 else torch.stack([x % 16, torch.div(x, 16, rounding_mode="floor")], -1).flatten(-2).double()  # noqa: E731
    k = raw[:, :16 * row].reshape(n, 16, row)
    if row == 128:  # [half, thread, 16 bytes]
        k = k.reshape(n, 8, 2, 2, 4, 16)
        k = torch.stack([k[:, :, 0], k[:, :, 1].flip(-3)], 2).reshape(n, 16, 2, 4, 16).permute(0, 1, 3, 2, 4).reshape(n, 16, row)
    k = k.reshape(n, 16, 4, groups, group // 4 // per).permute(0, 1, 3, 2, 4).reshape(n, 16, row)
    v = raw[:, 16 * row:32 * row].reshape(n, 8, 2 * row)
    place = torch.arange(8, device=dev)
    if share == 8:
        v = v.reshape(n, 8, 8, 8)
        v = torch.stack([v[:, pair][:, place ^ (4 if pair & 2 else 0)] for pair in range(8)], 1)
    else:
        v = v.reshape(n, 8, share // 16, 8, 16)
        v = torch.stack([v[:, pair][:, :, place ^ (2 * (pair & 3))] for pair in range(8)], 1).permute(0, 1, 3, 2, 4)
    v = v.reshape(n, 8, 8, share // 4, 2, 2).permute(0, 1, 4, 2, 3, 5).reshape(n, 16, 8, groups, group // 8 // per)
    v = v.permute(0, 1, 3, 2, 4).reshape(n, 16, row)
    meta = raw[:, 32 * row:].contiguous().view(torch.float16).double().reshape(n, 2, 16, groups, 2)
    for side, codes in enumerate((k, v)):
        c = values(codes).reshape(n, 16, groups, group)
        out.append((c * meta[:, side, ..., 0:1] + meta[:, side, ..., 1:2]).reshape(n, 16, hd))
    return out


def _exact_pages(s, ids, head, count):
    """The first count tokens of head in the pages ids: keys and values [count, hd]."""
    size = 4 * s["hd"] * s["bits"] + 128 * (s["hd"] // s["group"])
    raw = s["data"][ids.long(), head].reshape(-1, size)
    return [x.reshape(-1, s["hd"])[:count] for x in _exact_tokens(raw, s["hd"], s["bits"], s["group"])]


def _exact_quantised(x, bits, group):
    x = x.reshape(*x.shape[:-1], -1, group)
    low, high, most = x.min(-1, keepdim=True).values, x.max(-1, keepdim=True).values, 2.0 ** bits - 1

    def floor16(y):  # the largest fp16 value that is not above y
        e = torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -14)))
        step = torch.exp2(torch.where(torch.exp2(e) > y.abs().clamp_min(2.0 ** -14), e - 1, e) - 10)
        return torch.floor(y / step) * step

    bias = floor16(low)
    scale = -floor16(-(high - bias) / most)
    code = torch.round((x - bias) / scale.clamp_min(1e-300)).clamp(0, most)
    return torch.where(scale > 0, code * scale + bias, bias).flatten(-2)


def _exact_append(s):
    rows, hq, hkv, hd = s["rows"], s["hq"], s["hkv"], s["hd"]
    x = s["qkv"][:rows].double().reshape(rows, hq + 2 * hkv, 2, hd // 2)
    at = s["positions"][:rows].long()
    turn = torch.complex(s["cos"].double()[at], s["sin"].double()[at])[:, None]
    z = torch.complex(x[:, : hq + hkv, 0], x[:, : hq + hkv, 1]) * turn
    y = torch.stack([z.real, z.imag], 2).reshape(rows, hq + hkv, hd)
    q, k, v = s["q"].double(), s["k"].double(), s["v"].double()
    q[:rows] = y[:, :hq].reshape(rows, -1)
    k[:rows] = _exact_quantised(y[:, hq:], s["bits"], s["group"])
    v[:rows] = _exact_quantised(x[:, hq + hkv:].reshape(rows, hkv, hd), s["bits"], s["group"])
    return dict(q=q, k=k, v=v)


def _exact_read(s):
    k, v = s["k"].double(), s["v"].double()
    slots, page = s["slots"][:s["rows"]].long(), s["page"]
    ids, which = torch.unique(torch.div(slots, page, rounding_mode="floor"), return_inverse=True)
    for h in range(s["hkv"]):
        keys, vals = _exact_pages(s, ids, h, None)
        k[:s["rows"], h], v[:s["rows"], h] = keys[which * page + slots % page], vals[which * page + slots % page]
    return dict(k=k, v=v)


def _exact_attn(s):
    hq, hkv, hd, page, p = s["hq"], s["hkv"], s["hd"], s["page"], s["prefix"]
    out = s["out"].double()
    starts, lens = s["starts"].tolist(), s["lens"].tolist()
    for h in range(hkv):
        kp, vp = _exact_pages(s, s["prefix_table"], h, p)
        for b, n_own in enumerate(lens):
            lo, hi = starts[b], starts[b + 1]
            if lo == hi:
                continue
            ks, vs = _exact_pages(s, s["table"][b, : _ceil(n_own, page)], h, n_own)
            keys, vals = torch.cat([kp, ks]), torch.cat([vp, vs])
            q = s["q"][lo:hi].double().view(hi - lo, hkv, hq // hkv, hd)[:, h]
            score = torch.einsum("tgd,kd->tgk", q, keys) / math.sqrt(hd)
            last = p + n_own - (hi - lo) + torch.arange(hi - lo, device=q.device)
            hidden = torch.arange(p + n_own, device=q.device)[None] > last[:, None]
            w = torch.softmax(score.masked_fill(hidden[:, None], -math.inf), -1)
            out.view(out.shape[0], hkv, hq // hkv, hd)[lo:hi, h] = torch.einsum("tgk,kd->tgd", w, vals)
    return dict(out=out)


def exact(case, seed):
    return {"append": _exact_append, "read": _exact_read, "attn": _exact_attn}[case["op"]](prepare(case, seed))
