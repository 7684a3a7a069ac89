"""What the paged serving operators are measured on: a cache of pages shared by ragged requests, and the attention of
a batch that shares a long prefix.

Four operators, in the order in which a serving step calls them:

reserve   from the requests' lengths: the pages of their new tokens taken from a stack of free pages and written into
          the block table, the row offsets, each new token's slot in the cache and its position
truncate  a request's length cut to `keep` tokens (0: it is finished): its pages go back on the stack
append    rotary embedding of q and k at each row's position; k and v written to the rows' slots
attn      each row attends to the shared prefix (its keys and values held once) and to its own request's tokens

``run`` computes them in elementary torch operations in 32 bits, or, with ``own``, calls the framework.
"""

import math
import zlib

import torch

own = False

F16, F32 = "f16", "f32"
_DT = {F16: torch.float16, F32: torch.float32}


# ------------------------------------------------------------------------------------------------ cases

def listed():
    return [
        # one decoding step of a small batch: every request gets one token, every 16th of them a new page
        dict(name="reserve_step_8", op="reserve", batch=8, page=16, max_new=1, max_len=700, pad=0),
        # a step of a large server that mixes decoding requests with chunks of new prompts, rows padded to a bucket
        dict(name="reserve_mixed_1500", op="reserve", batch=1500, page=16, max_new=129, max_len=4000, pad=1000),
        # two of eight requests have ended
        dict(name="truncate_end_8", op="truncate", batch=8, page=16, max_len=700, share=0.25),
        # a large batch after speculation: most requests drop a few rejected tokens, some end
        dict(name="truncate_spec_1024", op="truncate", batch=1024, page=16, max_len=4000, share=0.1),
        # the new tokens of 32 decoding requests, in the 32-layer 4096-wide model's head layout
        dict(name="append_step_32", op="append", rows=32, pad=0, hq=32, hkv=8, hd=128, page=16, src=F32, cache=F16),
        # chunks of prompts, padded to a bucket of rows, in the small model's head layout and the exact cache
        dict(name="append_chunk_8150", op="append", rows=8150, pad=42, hq=32, hkv=4, hd=64, page=32, src=F32, cache=F32),
        # four requests behind a system prompt
        dict(name="attn_step_4_f16", op="attn", batch=4, min_new=1, max_new=1, prefix=700, max_own=120, hq=32, hkv=8,
             hd=128, page=16, pad=0, dtype=F16),
        # a full batch behind a long shared document whose last page is not full
        dict(name="attn_step_64_f16", op="attn", batch=64, min_new=1, max_new=1, prefix=8197, max_own=1500, hq=32,
             hkv=8, hd=128, page=16, pad=0, dtype=F16),
        # the largest batch and prefix, one rank of two of a 64-head model, larger pages
        dict(name="attn_step_256_f16", op="attn", batch=256, min_new=1, max_new=1, prefix=32768, max_own=2000, hq=32,
             hkv=4, hd=128, page=64, pad=0, dtype=F16),
        # the exact cache, as the 4096-wide model serves it
        dict(name="attn_step_32_f32", op="attn", batch=32, min_new=1, max_new=1, prefix=4099, max_own=600, hq=32, hkv=8,
             hd=128, page=16, pad=0, dtype=F32),
        # speculative drafts of one to five tokens in the small model's layout, exact cache, padded rows
        dict(name="attn_draft_16_f32", op="attn", batch=16, min_new=1, max_new=5, prefix=1000, max_own=400, hq=32, hkv=4,
             hd=64, page=32, pad=7, dtype=F32),
        # prompt chunks of a dozen requests behind the same instructions
        dict(name="attn_chunk_12_f16", op="attn", batch=12, min_new=120, max_new=700, prefix=2050, max_own=1200, hq=32,
             hkv=8, hd=128, page=16, pad=0, dtype=F16),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["reserve", "truncate", "append", "attn", "attn", "attn"])
    page = rng.choice([16, 32, 64, 128])
    if op == "reserve":
        b = _log(rng, 1, 1500)
        return dict(op=op, batch=b, page=page, max_new=_log(rng, 1, 129), max_len=_log(rng, 1, 4000), pad=rng.choice([0, rng.randint(1, 999)]))
    if op == "truncate":
        return dict(op=op, batch=_log(rng, 1, 1024), page=page, max_len=_log(rng, 1, 4000), share=round(rng.uniform(0.02, 0.9), 3))
    hq, hkv, hd = rng.choice([(32, 8, 128), (16, 4, 128), (8, 1, 128), (32, 4, 64), (16, 16, 64), (6, 2, 64), (8, 8, 128)])
    if op == "append":
        return dict(op=op, rows=_log(rng, 1, 8150), pad=rng.choice([0, rng.randint(1, 63)]), hq=hq, hkv=hkv, hd=hd, page=page,
                    src=rng.choice([F16, F32]), cache=rng.choice([F16, F32]))
    dtype = rng.choice([F16, F16, F32])
    if rng.random() < 0.3:  # chunks
        b, lo, hi = _log(rng, 1, 12), 1, _log(rng, 8, 700)
        prefix, most = rng.choice([0, _log(rng, 1, 4000)]), hi + _log(rng, 1, 1000)
    else:
        b, lo, hi = _log(rng, 1, 128), 1, rng.choice([1, 1, 1, 2, 6])
        prefix, most = rng.choice([0, _log(rng, 1, 16000), _log(rng, 1, 16000)]), hi + _log(rng, 1, 1500)
    return dict(op=op, batch=b, min_new=lo, max_new=hi, prefix=prefix, max_own=most, hq=hq, hkv=hkv, hd=hd, page=page,
                pad=rng.choice([0, rng.randint(1, 40)]), dtype=dtype)


# ------------------------------------------------------------------------------------------------ inputs

def _dev():
    return torch.device("cuda", torch.cuda.current_device())


def _host(case, seed):
    g = torch.Generator().manual_seed(seed * 7919 + 17)
    return g, lambda lo, hi, n: torch.randint(lo, hi + 1, (n,), generator=g)


def _gpu(seed):
    return torch.Generator(device=_dev()).manual_seed(seed * 104729 + 5)


def _ceil(a, b):
    return -(-a // b)


def _lengths(case, seed):
    """The requests' lengths, on the host: what a program has that made the batch. The case gives them, so that outputs
    keep their shapes; the seed gives which request has which."""
    key = zlib.crc32(repr(sorted((k, v) for k, v in case.items() if k != "name")).encode())
    g, ints = _host(case, key)
    b = case["batch"]
    new = None
    if case["op"] == "truncate":
        lens = ints(1, case["max_len"], b)
    elif case["op"] == "reserve":
        new = ints(0 if case["max_new"] > 1 else 1, case["max_new"], b)
        if case["max_new"] > 1:  # most requests decode, some bring a chunk
            new = torch.where(torch.rand(b, generator=g) < 0.6, torch.ones_like(new), new)
        lens = ints(0, case["max_len"], b)
    else:
        new = ints(case["min_new"], case["max_new"], b)
        most = torch.maximum(torch.full((b,), case["max_own"]), new)
        lens = torch.minimum(new + (torch.rand(b, generator=g) * (most - new + 1)).long(), most)
    ends = torch.rand(b, generator=g) < case["share"] if case["op"] == "truncate" else None
    g = _host(case, seed)[0]
    order = torch.randperm(b, generator=g)
    return g, lens[order], (ends if new is None else new)[order]


def _table(lens, page, extra, g):
    """A block table whose pages lie scattered in the cache, and the ids of the pages that no request holds."""
    blocks = (lens + page - 1) // page
    width = int(blocks.max()) + extra
    total = int(blocks.sum())
    spare = 8 + int(0.1 * total) + extra * lens.numel()
    ids = torch.randperm(total + spare, generator=g).to(torch.int32)
    table = torch.full((lens.numel(), width), -1, dtype=torch.int32)
    inside = torch.arange(width)[None] < blocks[:, None]
    table[inside] = ids[:total]
    return table, ids[total:], total + spare


def _prepare_reserve(case, seed):
    g, lens, new = _lengths(case, seed)
    page, dev = case["page"], _dev()
    extra = _ceil(case["max_new"], page) + 1
    table, free, pages = _table(lens, page, extra, g)
    rows = int(new.sum()) + case["pad"]
    stack = torch.full((pages,), -1, dtype=torch.int32)
    stack[: free.numel()] = free
    i32 = dict(dtype=torch.int32, device=dev)
    return dict(op="reserve", page=page, rows=max(rows, 1), lens=lens.int().to(dev), new=new.int().to(dev), table=table.to(dev), free=stack.to(dev),
                count=torch.tensor([free.numel()], **i32), prefix=torch.tensor([int(torch.randint(0, 5000, (1,), generator=g))], **i32),
                kv=torch.zeros(case["batch"], **i32), starts=torch.zeros(case["batch"] + 1, **i32), slots=torch.full((max(rows, 1),), -7, **i32),
                positions=torch.full((max(rows, 1),), -7, **i32), left=torch.zeros(1, **i32), status=torch.zeros(1, **i32))


def _prepare_truncate(case, seed):
    g, lens, ends = _lengths(case, seed)
    page, dev = case["page"], _dev()
    table, free, pages = _table(lens, page, 1, g)
    keep = torch.where(ends, torch.zeros_like(lens), (lens - torch.randint(0, 9, (case["batch"],), generator=g)).clamp_min(0))
    stack = torch.full((pages,), -1, dtype=torch.int32)
    stack[: free.numel()] = free
    i32 = dict(dtype=torch.int32, device=dev)
    return dict(op="truncate", page=page, lens=lens.int().to(dev), keep=keep.int().to(dev), table=table.to(dev), free=stack.to(dev),
                count=torch.tensor([free.numel()], **i32), out=torch.zeros(case["batch"], **i32), left=torch.zeros(1, **i32), status=torch.zeros(1, **i32))


def _prepare_append(case, seed):
    g, ints = _host(case, seed)
    dev, gg = _dev(), _gpu(seed)
    rows, page, hd, hkv, hq = case["rows"], case["page"], case["hd"], case["hkv"], case["hq"]
    total = rows + case["pad"]
    pages = _ceil(rows, page) * 2 + 4
    slots = torch.randperm(pages * page, generator=g)[:total].int()
    most = 8192
    inv = 1.0 / (5e5 ** (torch.arange(0, hd, 2, dtype=torch.float64) / hd))
    ang = torch.outer(torch.arange(most, dtype=torch.float64), inv)
    src, cache = _DT[case["src"]], _DT[case["cache"]]
    shape = (pages, hkv, page, hd)
    return dict(op="append", rows=rows, hq=hq, hkv=hkv, hd=hd, page=page, qkv=torch.randn(total, (hq + 2 * hkv) * hd, generator=gg, device=dev).to(src),
                starts=torch.tensor([0, rows // 2, rows], dtype=torch.int32, device=dev), slots=slots.to(dev),
                positions=ints(0, most - 1, total).int().to(dev), cos=ang.cos().float().to(dev), sin=ang.sin().float().to(dev),
                q=torch.zeros(total, hq * hd, dtype=cache, device=dev), k=torch.zeros(shape, dtype=cache, device=dev), v=torch.zeros(shape, dtype=cache, device=dev))


def _prepare_attn(case, seed):
    g, lens, new = _lengths(case, seed)
    dev, gg = _dev(), _gpu(seed)
    page, hd, hkv, hq, p, dt = case["page"], case["hd"], case["hkv"], case["hq"], case["prefix"], _DT[case["dtype"]]
    table, free, pages = _table(lens, page, 1, g)
    nb = _ceil(p, page)
    # the prefix's pages lie scattered among the others
    move = torch.randperm(pages + nb, generator=g).int()
    table = torch.where(table >= 0, move[table.clamp_min(0).long()], table)
    prefix_table = move[pages:pages + nb]
    pages += nb
    rows = int(new.sum())
    # keys with channels that stand out, as rotary keys have, and values off centre; slots that no token holds keep what was there
    channel = torch.randn(hkv, 1, hd, generator=gg, device=dev)
    k = (torch.randn(pages, hkv, page, hd, generator=gg, device=dev) + channel).to(dt)
    v = (torch.randn(pages, hkv, page, hd, generator=gg, device=dev) * 0.7 + 0.2).to(dt)
    q = (torch.randn(rows + case["pad"], hq * hd, generator=gg, device=dev) * 1.5).to(dt)
    starts = torch.zeros(case["batch"] + 1, dtype=torch.int32)
    starts[1:] = new.cumsum(0)
    i32 = dict(dtype=torch.int32, device=dev)
    return dict(op="attn", rows=rows, hq=hq, hkv=hkv, hd=hd, page=page, p=p, most_new=int(new.max()), most=int(lens.max()), q=q, k=k, v=v, starts=starts.to(dev),
                lens=lens.int().to(dev), table=table.to(dev), prefix_table=prefix_table.to(dev) if nb else torch.zeros(1, **i32), prefix=torch.tensor([p], **i32),
                out=torch.zeros(rows + case["pad"], hq * hd, dtype=dt, device=dev))


def prepare(case, seed):
    return {"reserve": _prepare_reserve, "truncate": _prepare_truncate, "append": _prepare_append, "attn": _prepare_attn}[case["op"]](case, seed)


# ------------------------------------------------------------------------------------------------ plain forms

def _plain_reserve(s):
    page, lens, new, table = s["page"], s["lens"].long(), s["new"].long(), s["table"]
    b, width = table.shape
    kv = lens + new
    have, need = (lens + page - 1) // page, (kv + page - 1) // page
    need = need - have
    ends, taken = new.cumsum(0), need.cumsum(0)
    count = s["count"].long()
    bad = (lens < 0).any() | (new < 0).any()
    status = (taken[-1] > count[0]).int() + 2 * (kv > width * page).any().int() + 4 * (ends[-1] > s["rows"]).int() + 8 * bad.int()
    ok = status == 0
    # the page of block j of request r: the stack's top, taken in the order of requests and blocks
    j = torch.arange(width, device=lens.device)[None]
    nth = (taken - need)[:, None] + j - have[:, None]
    fresh = (j >= have[:, None]) & (j < (have + need)[:, None]) & ok
    table = torch.where(fresh, s["free"][(count - 1 - nth).clamp(0, s["free"].numel() - 1)], table)
    starts = torch.cat([ends.new_zeros(1), ends]) * ok
    t = torch.arange(s["rows"], device=lens.device)
    seq = torch.searchsorted(ends, t, right=True).clamp_max(b - 1)
    at = lens[seq] + t - (ends - new)[seq]
    page_of = table[seq, (at // page).clamp(0, width - 1)].long()
    used = (t < ends[-1]) & ok
    slots = torch.where(used, (page_of * page + at % page).int(), s["slots"])
    positions = torch.where(used, (s["prefix"] + at).int(), s["positions"])
    return dict(table=table, kv=torch.where(ok, kv, lens).int(), starts=starts.int(), slots=slots, positions=positions,
                left=(count - taken[-1] * ok).int(), status=status.reshape(1).int())


def _plain_truncate(s):
    page, lens, table = s["page"], s["lens"].long(), s["table"]
    keep = torch.minimum(s["keep"].long().clamp_min(0), lens)
    have, left = (lens + page - 1) // page, (keep + page - 1) // page
    give = have - left
    given = give.cumsum(0)
    n = s["free"].numel()
    j = torch.arange(table.shape[1], device=lens.device)[None]
    back = (j >= left[:, None]) & (j < have[:, None])
    at = s["count"].long() + (given - give)[:, None] + j - left[:, None]
    free = torch.cat([s["free"], s["free"].new_zeros(1)])
    free[torch.where(back, at, torch.full_like(at, n)).reshape(-1)] = table.reshape(-1)
    return dict(free=free[:n], out=keep.int(), left=(s["count"] + given[-1]).int(), status=torch.zeros_like(s["status"]))


def _plain_append(s):
    hq, hkv, hd, rows, page = s["hq"], s["hkv"], s["hd"], s["rows"], s["page"]
    x = s["qkv"][:rows].float().view(rows, hq + 2 * hkv, hd)
    at = s["positions"][:rows].long()
    c, sn = s["cos"][at][:, None], s["sin"][at][:, None]
    x1, x2 = x[:, : hq + hkv, : hd // 2], x[:, : hq + hkv, hd // 2:]
    y = torch.cat([x1 * c - x2 * sn, x2 * c + x1 * sn], -1)
    dt = s["k"].dtype
    s["q"][:rows] = y[:, :hq].reshape(rows, hq * hd).to(dt)
    slot = s["slots"][:rows].long()
    s["k"][slot // page, :, slot % page] = y[:, hq:].to(dt)
    s["v"][slot // page, :, slot % page] = x[:, hq + hkv:].to(dt)
    return dict(q=s["q"], k=s["k"], v=s["v"])


def _plain_attn(s):
    hq, hkv, hd, rows, page, p = s["hq"], s["hkv"], s["hd"], s["rows"], s["page"], s["p"]
    grp, b, dev = hq // hkv, s["lens"].numel(), s["q"].device
    q = s["q"][:rows].float().view(rows, hkv, grp, hd) * (1.0 / math.sqrt(hd))
    lens, starts = s["lens"].long(), s["starts"].long()
    t = torch.arange(rows, device=dev)
    seq = torch.searchsorted(starts[1:], t, right=True)
    i = t - starts[seq]
    # the requests' own tokens, padded to the longest
    nb = _ceil(s["most"], page)
    own_pages = s["table"][:, :nb].long().clamp_min(0)
    k2 = s["k"][own_pages].permute(0, 2, 1, 3, 4).reshape(b, hkv, nb * page, hd).float()
    v2 = s["v"][own_pages].permute(0, 2, 1, 3, 4).reshape(b, hkv, nb * page, hd).float()
    n = s["most_new"]
    qp = q.new_zeros(b, n, hkv, grp, hd)
    qp[seq, i] = q
    s2 = qp.permute(0, 2, 1, 3, 4).reshape(b, hkv, n * grp, hd) @ k2.transpose(-1, -2)
    last = lens - (starts[1:] - starts[:-1])
    seen = torch.arange(nb * page, device=dev)[None, None] <= (last[:, None] + torch.arange(n, device=dev)[None])[..., None]
    s2 = s2.view(b, hkv, n, grp, nb * page).masked_fill(~seen[:, None, :, None], -math.inf)
    m = s2.amax(-1)
    if p:
        k1 = s["k"][s["prefix_table"].long()].permute(1, 0, 2, 3).reshape(hkv, -1, hd)[:, :p].float()
        v1 = s["v"][s["prefix_table"].long()].permute(1, 0, 2, 3).reshape(hkv, -1, hd)[:, :p].float()
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
    s["out"][:rows] = o.reshape(rows, hq * hd).to(s["out"].dtype)
    return dict(out=s["out"])


def _own_reserve(s):
    from shardcompute_b200 import ops
    ops.paged_reserve(s["lens"], s["new"], s["table"], s["free"], s["count"], s["page"], kv_lens=s["kv"], q_start=s["starts"], slots=s["slots"],
                      positions=s["positions"], free_count_out=s["left"], status=s["status"], prefix_len=s["prefix"])
    return {k: s[k] for k in ("table", "kv", "starts", "slots", "positions", "left", "status")}


def _own_truncate(s):
    from shardcompute_b200 import ops
    ops.paged_truncate(s["lens"], s["keep"], s["table"], s["free"], s["count"], s["page"], lens_out=s["out"], free_count_out=s["left"], status=s["status"])
    return {k: s[k] for k in ("free", "out", "left", "status")}


def _own_append(s):
    from shardcompute_b200 import ops
    ops.paged_rope_append(s["qkv"], s["starts"], s["slots"], s["positions"], s["cos"], s["sin"], s["q"], s["k"], s["v"])
    return dict(q=s["q"], k=s["k"], v=s["v"])


def _own_attn(s):
    from shardcompute_b200 import ops
    ops.prefix_attn(s["q"], s["k"], s["v"], s["starts"], s["lens"], s["table"], prefix_table=s["prefix_table"], prefix_len=s["prefix"], out=s["out"])
    return dict(out=s["out"])


def run(state):
    if own:
        return {"reserve": _own_reserve, "truncate": _own_truncate, "append": _own_append, "attn": _own_attn}[state["op"]](state)
    return {"reserve": _plain_reserve, "truncate": _plain_truncate, "append": _plain_append, "attn": _plain_attn}[state["op"]](state)


# ------------------------------------------------------------------------------------------------ work

def work(case):
    """Bytes and operations of the mean draw of lengths: a request's own length is even over its range."""
    op = case["op"]
    if op == "reserve":
        b, rows = case["batch"], case["batch"] * (1 if case["max_new"] == 1 else 0.6 + 0.4 * case["max_new"] / 2)
        return dict(bytes=16 * b + 8 * rows + 8 * rows / case["page"], flops=0)
    if op == "truncate":
        b, blocks = case["batch"], case["batch"] * case["share"] * case["max_len"] / 2 / case["page"]
        return dict(bytes=12 * b + 8 * blocks, flops=0)
    e = {F16: 2, F32: 4}
    hq, hkv, hd = case["hq"], case["hkv"], case["hd"]
    if op == "append":
        rows, w = case["rows"], (hq + 2 * hkv) * hd
        return dict(bytes=rows * (w * (e[case["src"]] + e[case["cache"]]) + 4 * hd + 8), flops=6 * rows * (hq + hkv) * hd)
    b, n, p = case["batch"], (case["min_new"] + case["max_new"]) / 2, case["prefix"]
    own_len = (n + max(case["max_own"], n)) / 2
    size = e[case["dtype"]]
    keys = p + b * own_len
    pairs = b * n * p + b * n * (own_len - (n - 1) / 2)
    return dict(bytes=keys * hkv * hd * 2 * size + 2 * b * n * hq * hd * size, flops=4 * pairs * hq * hd)


# ------------------------------------------------------------------------------------------------ 64 bits

def _exact_append(s):
    rows, hq, hkv, hd, page = s["rows"], s["hq"], s["hkv"], s["hd"], s["page"]
    x = s["qkv"][:rows].double().reshape(rows, hq + 2 * hkv, 2, hd // 2)
    at = s["positions"][:rows].long()
    turn = torch.complex(s["cos"].double()[at], s["sin"].double()[at])[:, None]
    z = torch.complex(x[:, : hq + hkv, 0], x[:, : hq + hkv, 1]) * turn
    y = torch.stack([z.real, z.imag], 2).reshape(rows, hq + hkv, hd)
    q, k, v = s["q"].double(), s["k"].double(), s["v"].double()
    q[:rows] = y[:, :hq].reshape(rows, -1)
    flat = s["slots"][:rows].long()
    pages, off = torch.div(flat, page, rounding_mode="floor"), torch.remainder(flat, page)
    for h in range(hkv):
        k[pages, h, off] = y[:, hq + h]
        v[pages, h, off] = x[:, hq + hkv + h].reshape(rows, hd)
    return dict(q=q, k=k, v=v)


def _exact_attn(s):
    hq, hkv, hd, page, p = s["hq"], s["hkv"], s["hd"], s["page"], s["p"]
    out = s["out"].double()
    starts, lens = s["starts"].tolist(), s["lens"].tolist()
    for h in range(hkv):
        kp = s["k"][s["prefix_table"].long(), h].reshape(-1, hd)[:p].double()
        vp = s["v"][s["prefix_table"].long(), h].reshape(-1, hd)[:p].double()
        for b, n_own in enumerate(lens):
            lo, hi = starts[b], starts[b + 1]
            if lo == hi:
                continue
            ids = s["table"][b, : _ceil(n_own, page)].long()
            keys = torch.cat([kp, s["k"][ids, h].reshape(-1, hd)[:n_own].double()])
            vals = torch.cat([vp, s["v"][ids, h].reshape(-1, hd)[:n_own].double()])
            q = s["q"][lo:hi].double().view(hi - lo, hkv, hq // hkv, hd)[:, h]
            score = torch.einsum("tgd,kd->tgk", q, keys) / math.sqrt(hd)
            last = p + n_own - (hi - lo) + torch.arange(hi - lo, device=q.device)
            hidden = torch.arange(p + n_own, device=q.device)[None] > last[:, None]
            w = torch.softmax(score.masked_fill(hidden[:, None], -math.inf), -1)
            out.view(out.shape[0], hkv, hq // hkv, hd)[lo:hi, h] = torch.einsum("tgk,kd->tgd", w, vals)
    return dict(out=out)


def exact(case, seed):
    if case["op"] in ("reserve", "truncate"):
        return None  # whole numbers: the plain form is the definition
    s = prepare(case, seed)
    return _exact_append(s) if case["op"] == "append" else _exact_attn(s)
