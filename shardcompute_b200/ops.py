"""Tensor-level wrappers over the C ABI (torch tensors are only handles).

Every function checks devices, dtypes and shapes on the host, passes raw
pointers plus the current CUDA stream to ``libsc_b200.so`` and raises the
reference's exception types on failure.  All tensors must live on a CUDA
device; there is no CPU path.
"""

from __future__ import annotations

import ctypes as C
import functools
import math
from typing import NamedTuple, Optional, Sequence

import torch

from . import _lib as L

_F16, _F32 = torch.float16, torch.float32


def _dt(t: torch.Tensor) -> int:
    if t.dtype == _F16:
        return L.SC_F16
    if t.dtype == _F32:
        return L.SC_F32
    if t.dtype == torch.int32:
        return L.SC_I32
    raise ValueError(f"unsupported dtype {t.dtype}")


def _cuda(*ts: Optional[torch.Tensor]) -> None:
    for t in ts:
        if t is not None and not t.is_cuda:
            raise RuntimeError("libsc_b200 ops take CUDA tensors only (no CPU path)")


def _f32_cache(*ts: torch.Tensor) -> None:
    for t in ts:
        if t.dtype != torch.float32:
            raise ValueError(f"KV cache must be float32 (the reference caches fp32 keys/values), got {t.dtype}")


def _p(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def stream_handle(device: Optional[torch.device] = None) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def as_u32(t: torch.Tensor) -> torch.Tensor:
    """Packed words are handled as 4-byte storage; int32/uint32 both accepted."""
    if t.dtype in (torch.int32, getattr(torch, "uint32", torch.int32)):
        return t
    raise ValueError(f"packed weights must be uint32/int32, got {t.dtype}")


class Workspace:
    """Grow-only device scratch buffer, one per device.

    Sized before a CUDA graph capture so the captured pointer stays valid.
    """

    _bufs: dict = {}

    @classmethod
    def get(cls, nbytes: int, device: torch.device) -> Optional[torch.Tensor]:
        if nbytes <= 0:
            return None
        key = (device.type, device.index if device.index is not None else torch.cuda.current_device())
        buf = cls._bufs.get(key)
        if buf is None or buf.numel() < nbytes:
            buf = torch.empty(max(nbytes, 1 << 20), dtype=torch.uint8, device=device)
            cls._bufs[key] = buf
        return buf


# ---------------------------------------------------------------- K1

def qlinear_workspace_bytes(M: int, K: int, N: int, bits: int) -> int:
    return int(L.load().sc_qlinear_workspace_bytes(M, K, N, bits))


def qlinear(x: torch.Tensor, wq: torch.Tensor, scales: torch.Tensor, biases: torch.Tensor, group_size: int,
            bits: int, bias: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None,
            out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x @ dequant(wq, scales, biases).T (+ bias)`` — mx.quantized_matmul(transpose=True)."""
    _cuda(x, wq, scales, biases, bias, out)
    wq = as_u32(wq)
    K = x.shape[-1]
    N = wq.shape[0]
    if wq.shape[1] * (32 // bits) != K:
        raise ValueError(f"weight packs {wq.shape[1] * (32 // bits)} inputs, x has {K}")
    if scales.shape != (N, K // group_size) or biases.shape != scales.shape:
        raise ValueError(f"scales {tuple(scales.shape)} / biases {tuple(biases.shape)} do not match "
                         f"[{N}, {K // group_size}]")
    x2 = x.reshape(-1, K)
    if not x2.is_contiguous():
        x2 = x2.contiguous()
    M = x2.shape[0]
    y = out if out is not None else torch.empty(M, N, dtype=out_dtype or x.dtype, device=x.device)
    ws_bytes = qlinear_workspace_bytes(M, K, N, bits)
    ws = Workspace.get(ws_bytes, x.device)
    L.call("sc_qlinear", _p(x2), _dt(x2), M, K, K, _p(wq), _p(scales), _p(biases), N, group_size, bits,
           _p(bias), _p(y), _dt(y), N, _p(ws), ws_bytes, stream_handle(x.device))
    return y.reshape(*x.shape[:-1], N)


def qlinear_fused(x: torch.Tensor, segments: Sequence, group_size: int, bits: int, epilogue: int = L.SC_EPI_STORE,
                  norm_weight: Optional[torch.Tensor] = None, eps: float = 1e-5,
                  bias: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None,
                  out: Optional[torch.Tensor] = None, out_dtype: torch.dtype = _F32) -> torch.Tensor:
    """Fused RMSNorm -> segments of quantized linears -> epilogue.

    ``segments`` is a list of ``(wq, scales, biases)`` sharing ``x``.
    """
    _cuda(x, norm_weight, bias, residual, out)
    n = len(segments)
    K = x.shape[-1]
    x2 = x.reshape(-1, K)
    if not x2.is_contiguous():
        x2 = x2.contiguous()
    M = x2.shape[0]
    rows = [int(s[0].shape[0]) for s in segments]
    N = rows[0] if epilogue == L.SC_EPI_SWIGLU else sum(rows)
    for wq, sc, bi in segments:
        _cuda(wq, sc, bi)
        if wq.shape[1] * (32 // bits) != K:
            raise ValueError("segment K mismatch")
    y = out if out is not None else torch.empty(M, N, dtype=out_dtype, device=x.device)
    W = (C.c_void_p * n)(*[s[0].data_ptr() for s in segments])
    S = (C.c_void_p * n)(*[s[1].data_ptr() for s in segments])
    B = (C.c_void_p * n)(*[s[2].data_ptr() for s in segments])
    R = (C.c_int * n)(*rows)
    ws_bytes = qlinear_workspace_bytes(M, K, N, bits)
    ws = Workspace.get(ws_bytes, x.device)
    res = residual.reshape(-1, N) if residual is not None else None
    L.call("sc_qlinear_fused", _p(x2), _dt(x2), M, K, K, _p(norm_weight), float(eps), n,
           C.cast(W, L._pp), C.cast(S, L._pp), C.cast(B, L._pp), R, group_size, bits, _p(bias), epilogue,
           _p(y), _dt(y), N, _p(res), N if res is not None else 0, _p(ws), ws_bytes, stream_handle(x.device))
    return y


# ---------------------------------------------------------------- K3

def embed_gather_q(ids: torch.Tensor, wq, scales, biases, vocab_start: int, vocab_end: int, hidden: int,
                   group_size: int, bits: int, out_dtype=_F16, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    _cuda(ids, wq, scales, biases, out)
    if wq.shape[0] < vocab_end - vocab_start or scales.shape[0] < vocab_end - vocab_start:
        raise ValueError(f"table has {wq.shape[0]} rows, vocab range needs {vocab_end - vocab_start}")
    if wq.shape[1] * (32 // bits) != hidden:
        raise ValueError(f"table packs {wq.shape[1] * (32 // bits)} values per row, hidden is {hidden}")
    ids32 = ids.reshape(-1).to(torch.int32).contiguous()
    n = ids32.numel()
    y = out if out is not None else torch.empty(n, hidden, dtype=out_dtype, device=ids.device)
    L.call("sc_embed_gather_q", _p(ids32), n, _p(as_u32(wq)), _p(scales), _p(biases), vocab_start, vocab_end,
           hidden, group_size, bits, _p(y), _dt(y), stream_handle(ids.device))
    return y.reshape(*ids.shape, hidden)


def embed_gather_f16(ids: torch.Tensor, table: torch.Tensor, vocab_start: int, vocab_end: int,
                     out_dtype=_F16) -> torch.Tensor:
    _cuda(ids, table)
    if table.shape[0] < vocab_end - vocab_start:
        raise ValueError(f"table has {table.shape[0]} rows, vocab range needs {vocab_end - vocab_start}")
    ids32 = ids.reshape(-1).to(torch.int32).contiguous()
    H = table.shape[1]
    y = torch.empty(ids32.numel(), H, dtype=out_dtype, device=ids.device)
    L.call("sc_embed_gather_f16", _p(ids32), ids32.numel(), _p(table), vocab_start, vocab_end, H, _p(y), _dt(y),
           stream_handle(ids.device))
    return y.reshape(*ids.shape, H)


def dequantize(wq, scales, biases, group_size: int, bits: int) -> torch.Tensor:
    _cuda(wq, scales, biases)
    rows = wq.shape[0]
    K = wq.shape[1] * (32 // bits)
    out = torch.empty(rows, K, dtype=_F16, device=wq.device)
    L.call("sc_dequantize", _p(as_u32(wq)), _p(scales), _p(biases), rows, K, group_size, bits, _p(out),
           stream_handle(wq.device))
    return out


def quantize(w: torch.Tensor, group_size: int = 64, bits: int = 4):
    """fp16 [rows, K] -> (wq int32 [rows, K*bits/32], scales fp16, biases fp16)."""
    _cuda(w)
    w = w.to(_F16).contiguous()
    rows, K = w.shape
    wq = torch.empty(rows, K * bits // 32, dtype=torch.int32, device=w.device)
    s = torch.empty(rows, K // group_size, dtype=_F16, device=w.device)
    b = torch.empty_like(s)
    L.call("sc_quantize", _p(w), rows, K, group_size, bits, _p(wq), _p(s), _p(b), stream_handle(w.device))
    return wq, s, b


# ---------------------------------------------------------------- K4

def rope_append(qkv: torch.Tensor, B: int, S: int, Hq: int, Hkv: int, hd: int, pos: torch.Tensor,
                cos_tab: torch.Tensor, sin_tab: torch.Tensor, q_out: torch.Tensor, k_cache: torch.Tensor,
                v_cache: torch.Tensor) -> None:
    _cuda(qkv, pos, cos_tab, sin_tab, q_out, k_cache, v_cache)
    _f32_cache(k_cache, v_cache)
    Lmax = k_cache.shape[2]
    L.call("sc_rope_append", _p(qkv), B, S, Hq, Hkv, hd, _p(pos), _p(cos_tab), _p(sin_tab), cos_tab.shape[0],
           _p(q_out), _p(k_cache), _p(v_cache), Lmax, stream_handle(qkv.device))


def flash_decode_workspace_bytes(B: int, S: int, Hq: int, hd: int, splits: int) -> int:
    return int(L.load().sc_flash_decode_workspace_bytes(B, S, Hq, hd, splits))


def flash_decode(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, pos: torch.Tensor, B: int, S: int,
                 Hq: int, Hkv: int, hd: int, splits: int, out: torch.Tensor,
                 workspace: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> torch.Tensor:
    _cuda(q, k_cache, v_cache, pos, out)
    _f32_cache(k_cache, v_cache)
    nbytes = flash_decode_workspace_bytes(B, S, Hq, hd, splits)
    if workspace is None:
        workspace = Workspace.get(nbytes, q.device)
    sc = (1.0 / math.sqrt(hd)) if scale is None else scale
    L.call("sc_flash_decode", _p(q), _p(k_cache), _p(v_cache), _p(pos), B, S, Hq, Hkv, hd, k_cache.shape[2],
           float(sc), splits, _p(out), _dt(out), _p(workspace), nbytes if workspace is not None else 0,
           stream_handle(q.device))
    return out


def attn_decode_workspace_bytes(B: int, Hq: int, hd: int, splits: int) -> int:
    return int(L.load().sc_attn_decode_workspace_bytes(B, Hq, hd, splits))


def attn_decode(qkv: torch.Tensor, B: int, Hq: int, Hkv: int, hd: int, pos: torch.Tensor, cos_tab: torch.Tensor,
                sin_tab: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, splits: int, out: torch.Tensor,
                tickets: torch.Tensor, workspace: Optional[torch.Tensor] = None,
                scale: Optional[float] = None) -> torch.Tensor:
    """One decode token per sequence: RoPE + KV append + split-KV attention
    (+ merge) in one launch.  ``tickets`` is int32 [B*Hkv], zero on entry
    and left zero."""
    _cuda(qkv, pos, cos_tab, sin_tab, k_cache, v_cache, out, tickets, workspace)
    _f32_cache(k_cache, v_cache)
    nbytes = attn_decode_workspace_bytes(B, Hq, hd, splits)
    if workspace is None:
        workspace = Workspace.get(nbytes, qkv.device)
    sc = (1.0 / math.sqrt(hd)) if scale is None else scale
    L.call("sc_attn_decode", _p(qkv), B, Hq, Hkv, hd, _p(pos), _p(cos_tab), _p(sin_tab), cos_tab.shape[0],
           _p(k_cache), _p(v_cache), k_cache.shape[2], float(sc), splits, _p(out), _dt(out), _p(workspace),
           nbytes if workspace is not None else 0, _p(tickets), stream_handle(qkv.device))
    return out


# ---------------------------------------------------------------- paged cache

class PagedStep(NamedTuple):
    """What ``paged_reserve`` wrote (all int32 on the device)."""

    kv_lens: torch.Tensor      # [B] tokens of each request, the new ones among them
    q_start: torch.Tensor      # [B + 1] rows of each request
    slots: torch.Tensor        # [max_tokens] each row's slot in the cache
    positions: torch.Tensor    # [max_tokens] each row's position
    free_count: torch.Tensor   # [1] pages left
    status: torch.Tensor       # [1] 0, or why nothing was reserved


_I32 = torch.int32


def _refuse(what: str, dev: int, ts: Sequence[torch.Tensor], dtype: Optional[torch.dtype]) -> None:
    """Raises for the first of the tensors that is not a contiguous CUDA tensor of device ``dev`` and type ``dtype``."""
    for t in ts:
        if not t.is_cuda:
            raise RuntimeError("libsc_b200 ops take CUDA tensors only (no CPU path)")
        if t.get_device() != dev:
            raise ValueError(f"{what}: tensors on cuda:{dev} and {t.device}")
        if dtype is not None and t.dtype is not dtype:
            raise ValueError(f"{what}: lengths, tables, slots and counts must be int32, got {t.dtype}")
        if not t.is_contiguous():
            raise ValueError(f"{what}: tensors must be contiguous")
    raise ValueError(f"{what}: unsupported tensors")


def _check(what: str, dev: int, ts: Sequence[torch.Tensor], dtype: Optional[torch.dtype] = None) -> None:
    """One pass over the tensors of a call, which a serving loop makes for every layer and token."""
    if dev < 0:
        _refuse(what, dev, ts, dtype)
    if dtype is None:
        for t in ts:
            if t.get_device() != dev or not t.is_contiguous():
                _refuse(what, dev, ts, dtype)
    else:
        for t in ts:
            if t.dtype is not dtype or t.get_device() != dev or not t.is_contiguous():
                _refuse(what, dev, ts, dtype)


def _sized(what: str, n: int, **named: Optional[torch.Tensor]) -> None:
    for name, t in named.items():
        if t is not None and t.numel() != n:
            raise ValueError(f"{what}: {name} holds {t.numel()} values, {n} are needed")


_bound = None


def _native():
    """The binding of the paged operators (csrc/sc_binding.cpp): each of its functions checks the tensors and makes the call in
    one go, and returns the status, or -1 where the checks below have to say what is wrong or the device has to be changed."""
    global _bound
    if _bound is None:
        L.load()
        try:
            from . import _native as m
        except ImportError as e:
            raise RuntimeError(f"_native.so is missing or does not load ({e}); build it with `python -m shardcompute_b200.build`") from e
        _bound = m
    return _bound


def _call_on(dev: int, name: str, *args) -> None:
    """The call with device ``dev`` as the current one, on its current stream."""
    if dev == torch._C._cuda_getDevice():
        st = getattr(L.load(), name)(*args, torch._C._cuda_getCurrentRawStream(dev))
        if st:
            L.check(st, name)
    else:
        with torch.cuda.device(dev):
            L.call(name, *args, torch._C._cuda_getCurrentRawStream(dev))


def paged_reserve(lens: torch.Tensor, new_lens: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor,
                  free_count: torch.Tensor, page_size: int, max_tokens: Optional[int] = None,
                  prefix_len: Optional[torch.Tensor] = None, kv_lens: Optional[torch.Tensor] = None,
                  q_start: Optional[torch.Tensor] = None, slots: Optional[torch.Tensor] = None,
                  positions: Optional[torch.Tensor] = None, free_count_out: Optional[torch.Tensor] = None,
                  status: Optional[torch.Tensor] = None) -> PagedStep:
    """Pages, slots and row offsets for ``new_lens[b]`` more tokens of every request.

    ``block_table`` [B, max_blocks] gets the new pages, taken from the top of the stack ``free_pages`` [:free_count].
    Outputs not passed are allocated (``slots`` and ``positions`` of ``max_tokens`` rows, -1 behind the last one);
    ``kv_lens`` may be ``lens`` and ``free_count_out`` may be ``free_count``.  If ``status`` is not 0 nothing was
    reserved and ``q_start`` is all zeros: 1 not enough pages, 2 a request exceeds ``max_blocks`` pages, 4 more than
    ``max_tokens`` new tokens, 8 a negative length, 16 ``free_count`` outside the stack (the sum of those that hold)."""
    if slots is None:
        if max_tokens is None:
            raise ValueError("paged_reserve: max_tokens or slots is needed")
        slots = torch.full((max_tokens,), -1, dtype=_I32, device=lens.device)
    rows = slots.numel() if max_tokens is None else max_tokens
    if positions is None:
        positions = torch.full((rows,), -1, dtype=_I32, device=lens.device)
    new = lambda n: torch.empty(n, dtype=_I32, device=lens.device)  # noqa: E731
    kv_lens = new(lens.numel()) if kv_lens is None else kv_lens
    q_start = new(lens.numel() + 1) if q_start is None else q_start
    free_count_out = new(1) if free_count_out is None else free_count_out
    status = new(1) if status is None else status
    st = _native().paged_reserve(lens, new_lens, block_table, free_pages, free_count, page_size, rows, prefix_len, kv_lens, q_start, slots,
                                 positions, free_count_out, status)
    if st == 0:
        return PagedStep(kv_lens, q_start, slots, positions, free_count_out, status)
    B, dev = lens.numel(), lens.get_device()
    ts = (lens, new_lens, block_table, free_pages, free_count, kv_lens, q_start, slots, positions, free_count_out, status)
    _check("paged_reserve", dev, ts if prefix_len is None else (*ts, prefix_len), _I32)
    tab = block_table.shape
    if len(tab) != 2 or tab[0] != B:
        raise ValueError(f"paged_reserve: block_table {tuple(tab)} is not [{B}, max_blocks]")
    if (new_lens.numel() != B or kv_lens.numel() != B or q_start.numel() != B + 1 or free_count.numel() != 1
            or free_count_out.numel() != 1 or status.numel() != 1 or (prefix_len is not None and prefix_len.numel() != 1)):
        _sized("paged_reserve", B, new_lens=new_lens, kv_lens=kv_lens)
        _sized("paged_reserve", B + 1, q_start=q_start)
        _sized("paged_reserve", 1, free_count=free_count, prefix_len=prefix_len, free_count_out=free_count_out, status=status)
    if slots.numel() < rows or positions.numel() < rows:
        raise ValueError(f"paged_reserve: slots and positions hold {slots.numel()} and {positions.numel()} rows, {rows} are needed")
    _call_on(dev, "sc_paged_reserve", lens.data_ptr(), new_lens.data_ptr(), B, _p(prefix_len), block_table.data_ptr(),
             tab[1], free_pages.data_ptr(), free_pages.numel(), free_count.data_ptr(), page_size, rows,
             kv_lens.data_ptr(), q_start.data_ptr(), slots.data_ptr(), positions.data_ptr(), free_count_out.data_ptr(),
             status.data_ptr())
    return PagedStep(kv_lens, q_start, slots, positions, free_count_out, status)


def paged_truncate(lens: torch.Tensor, keep: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor,
                   free_count: torch.Tensor, page_size: int, lens_out: Optional[torch.Tensor] = None,
                   free_count_out: Optional[torch.Tensor] = None, status: Optional[torch.Tensor] = None):
    """Cut every request to its first ``keep[b]`` tokens (0: it has ended) and put the pages that it no longer needs
    back on the stack.  ``lens_out`` may be ``lens``, ``free_count_out`` may be ``free_count``.  Returns ``(lens_out,
    free_count_out, status)``; unless ``status`` is 0 nothing changed (1: the stack has no room, as when a page is given
    back twice; 2, 8, 16 as for ``paged_reserve``)."""
    lens_out = torch.empty_like(lens) if lens_out is None else lens_out
    free_count_out = torch.empty_like(free_count) if free_count_out is None else free_count_out
    status = torch.empty(1, dtype=_I32, device=lens.device) if status is None else status
    st = _native().paged_truncate(lens, keep, block_table, free_pages, free_count, page_size, lens_out, free_count_out, status)
    if st == 0:
        return lens_out, free_count_out, status
    B, dev = lens.numel(), lens.get_device()
    _check("paged_truncate", dev, (lens, keep, block_table, free_pages, free_count, lens_out, free_count_out, status), _I32)
    tab = block_table.shape
    if len(tab) != 2 or tab[0] != B:
        raise ValueError(f"paged_truncate: block_table {tuple(tab)} is not [{B}, max_blocks]")
    if keep.numel() != B or lens_out.numel() != B or free_count.numel() != 1 or free_count_out.numel() != 1 or status.numel() != 1:
        _sized("paged_truncate", B, keep=keep, lens_out=lens_out)
        _sized("paged_truncate", 1, free_count=free_count, free_count_out=free_count_out, status=status)
    _call_on(dev, "sc_paged_truncate", lens.data_ptr(), keep.data_ptr(), B, block_table.data_ptr(), tab[1],
             free_pages.data_ptr(), free_pages.numel(), free_count.data_ptr(), page_size, lens_out.data_ptr(),
             free_count_out.data_ptr(), status.data_ptr())
    return lens_out, free_count_out, status


def _pools(what: str, k_pages: torch.Tensor, v_pages: torch.Tensor):
    shape, dt = k_pages.shape, k_pages.dtype
    if len(shape) != 4 or shape != v_pages.shape:
        raise ValueError(f"{what}: k_pages {tuple(shape)} and v_pages {tuple(v_pages.shape)} must be one [n_pages, Hkv, page, hd]")
    if dt is not v_pages.dtype or (dt is not _F16 and dt is not _F32):
        raise ValueError(f"{what}: pages must both be float16 or float32, got {dt} and {v_pages.dtype}")
    return shape


def paged_rope_append(qkv: torch.Tensor, q_start: torch.Tensor, slots: torch.Tensor, positions: torch.Tensor,
                      cos_tab: torch.Tensor, sin_tab: torch.Tensor, q_out: torch.Tensor, k_pages: torch.Tensor,
                      v_pages: torch.Tensor) -> torch.Tensor:
    """``rope_append`` for a paged cache: q and k of each row (``qkv`` [T, (Hq + 2 Hkv) hd], float16 or float32) rotated
    at ``positions``, k and v written to ``slots`` of the pools, q to ``q_out`` [T, Hq hd] in the pools' type.  Rows from
    ``q_start[-1]`` on are left as they were; a slot outside the pool or a position past the tables is not written."""
    st = _native().paged_rope_append(qkv, q_start, slots, positions, cos_tab, sin_tab, q_out, k_pages, v_pages)
    if st == 0:
        return q_out
    dev = qkv.get_device()
    _check("paged_rope_append", dev, (qkv, cos_tab, sin_tab, q_out, k_pages, v_pages))
    _check("paged_rope_append", dev, (q_start, slots, positions), _I32)
    n_pages, Hkv, page, hd = _pools("paged_rope_append", k_pages, v_pages)
    if qkv.dim() != 2 or qkv.dtype not in (_F16, _F32):
        raise ValueError(f"paged_rope_append: qkv must be a float16 or float32 [T, (Hq + 2 Hkv) hd], got {qkv.dtype} {tuple(qkv.shape)}")
    T, width = qkv.shape
    Hq = width // hd - 2 * Hkv
    if width % hd or Hq < 1:
        raise ValueError(f"paged_rope_append: qkv rows of {width} do not hold q beside {Hkv} heads of {hd}")
    if q_out.dtype != k_pages.dtype or q_out.numel() != T * Hq * hd:
        raise ValueError(f"paged_rope_append: q_out must be a {k_pages.dtype} [{T}, {Hq * hd}], got {q_out.dtype} {tuple(q_out.shape)}")
    if slots.numel() < T or positions.numel() < T:
        raise ValueError(f"paged_rope_append: {slots.numel()} slots and {positions.numel()} positions for {T} rows")
    if cos_tab.dtype != _F32 or sin_tab.dtype != _F32 or cos_tab.dim() != 2 or cos_tab.shape[1] * 2 != hd or cos_tab.shape != sin_tab.shape:
        raise ValueError(f"paged_rope_append: cos_tab and sin_tab must be float32 [max_pos, {hd // 2}]")
    if q_start.numel() < 1:
        raise ValueError("paged_rope_append: q_start is empty")
    if T:
        _call_on(dev, "sc_paged_rope_append", qkv.data_ptr(), _dt(qkv), T, q_start.data_ptr() + 4 * (q_start.numel() - 1),
                 slots.data_ptr(), positions.data_ptr(), cos_tab.data_ptr(), sin_tab.data_ptr(), cos_tab.shape[0], Hq, Hkv, hd,
                 q_out.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), _dt(k_pages), n_pages, page)
    return q_out


@functools.lru_cache(maxsize=1024)
def _prefix_attn_bytes(*args: int) -> int:
    return int(L.load().sc_prefix_attn_workspace_bytes(*args))


def prefix_attn_workspace_bytes(T: int, B: int, Hq: int, Hkv: int, hd: int, max_blocks: int, max_prefix_blocks: int,
                                page_size: int, dtype: torch.dtype) -> int:
    return _prefix_attn_bytes(T, B, Hq, Hkv, hd, max_blocks, max_prefix_blocks, page_size, L.SC_F16 if dtype == _F16 else L.SC_F32)


def prefix_attn(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, q_start: torch.Tensor, kv_lens: torch.Tensor,
                block_table: torch.Tensor, prefix_table: Optional[torch.Tensor] = None,
                prefix_len: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                scale: Optional[float] = None, workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of a ragged batch behind a prefix that all its requests share.

    Row ``q_start[b] + i`` of request b (n rows) sees the ``prefix_len`` tokens in the pages ``prefix_table`` and its own
    tokens ``0 .. kv_lens[b] - n + i`` in the pages ``block_table[b]``; GQA by heads.  ``q`` and ``out`` [T, Hq hd] have
    the pools' type.  Rows from ``q_start[-1]`` on are left as they were (an ``out`` that is allocated here is zero
    there); a row that sees no token is zero; pages outside the pool count as absent.  ``workspace``: uint8, at least
    ``prefix_attn_workspace_bytes``; without it scratch is allocated per call, so calls on two streams do not meet."""
    if out is None:
        out = torch.zeros_like(q)
    st = _native().prefix_attn(q, k_pages, v_pages, q_start, kv_lens, block_table, prefix_table, prefix_len, out, scale, workspace)
    if st == 0:
        return out
    n_pages, Hkv, page, hd = _pools("prefix_attn", k_pages, v_pages)
    dev, dt = q.get_device(), k_pages.dtype
    _check("prefix_attn", dev, (q, k_pages, v_pages, out))
    nbp, pt, pl = 0, None, None
    if prefix_len is not None and prefix_table is not None:
        _check("prefix_attn", dev, (q_start, kv_lens, block_table, prefix_table, prefix_len), _I32)
        if prefix_len.numel() != 1:
            _sized("prefix_attn", 1, prefix_len=prefix_len)
        nbp, pt, pl = prefix_table.numel(), prefix_table.data_ptr(), prefix_len.data_ptr()
    elif prefix_len is None and prefix_table is None:
        _check("prefix_attn", dev, (q_start, kv_lens, block_table), _I32)
    else:
        raise ValueError("prefix_attn: prefix_table and prefix_len go together")
    B, nq = kv_lens.numel(), q.numel()
    T = q.shape[0] if q.dim() else 0
    if q.dtype is not dt or out.dtype is not dt or out.numel() != nq:
        raise ValueError(f"prefix_attn: q and out must have the pages' type {dt} and one size, got {q.dtype} "
                         f"{tuple(q.shape)} and {out.dtype} {tuple(out.shape)}")
    Hq = nq // (T * hd) if T else Hkv
    if T and Hq * T * hd != nq:
        raise ValueError(f"prefix_attn: q rows of {nq // T} are no multiple of head_dim {hd}")
    tab = block_table.shape
    if len(tab) != 2 or tab[0] != B:
        raise ValueError(f"prefix_attn: block_table {tuple(tab)} is not [{B}, max_blocks]")
    if q_start.numel() != B + 1:
        _sized("prefix_attn", B + 1, q_start=q_start)
    if not T or not B:
        return out
    code = L.SC_F16 if dt is _F16 else L.SC_F32
    mb = tab[1]
    nbytes = _prefix_attn_bytes(T, B, Hq, Hkv, hd, mb, nbp, page, code)
    wp, wb = None, 0
    if workspace is not None:
        _check("prefix_attn", dev, (workspace,))
        if workspace.dtype != torch.uint8:
            raise ValueError(f"prefix_attn: workspace must be uint8, got {workspace.dtype}")
        wp, wb = workspace.data_ptr(), workspace.numel()
    elif nbytes:
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        wp, wb = workspace.data_ptr(), nbytes
    _call_on(dev, "sc_prefix_attn", q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), code, T, q_start.data_ptr(),
             kv_lens.data_ptr(), block_table.data_ptr(), B, mb, pt, pl, nbp, Hq, Hkv, hd, n_pages, page,
             1.0 / math.sqrt(hd) if scale is None else float(scale), out.data_ptr(), wp, wb)
    return out


def prefix_attn_device_error(device: Optional[torch.device] = None, reset: bool = True) -> int:
    """Nonzero after a CTA of ``prefix_attn`` on this device gave up a bounded wait: outputs since the last reset are undefined.
    Waits for the device's current stream."""
    with torch.cuda.device(device):
        torch.cuda.current_stream().synchronize()
        return int(L.load().sc_prefix_attn_device_error(int(reset)))


# ---------------------------------------------------------------- K5 / K7

def rmsnorm(x: torch.Tensor, w: torch.Tensor, eps: float, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    _cuda(x, w)
    H = x.shape[-1]
    x2 = x.reshape(-1, H).contiguous()
    y = torch.empty(x2.shape, dtype=out_dtype or x.dtype, device=x.device)
    L.call("sc_rmsnorm", _p(x2), _dt(x2), x2.shape[0], H, _p(w.to(_F16).contiguous()), float(eps), _p(y), _dt(y),
           stream_handle(x.device))
    return y.reshape(x.shape)


def silu_mul(gate: torch.Tensor, up: torch.Tensor, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    _cuda(gate, up)
    if gate.shape != up.shape or gate.dtype != up.dtype:
        raise ValueError("gate/up shape or dtype mismatch")
    g, u = gate.contiguous(), up.contiguous()
    y = torch.empty(g.shape, dtype=out_dtype or g.dtype, device=g.device)
    L.call("sc_silu_mul", _p(g), _p(u), _dt(g), g.numel(), _p(y), _dt(y), stream_handle(g.device))
    return y


def add(a: torch.Tensor, b: torch.Tensor, out: Optional[torch.Tensor] = None,
        out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    _cuda(a, b, out)
    if a.shape != b.shape:
        raise ValueError(f"add: shapes {tuple(a.shape)} vs {tuple(b.shape)}")
    a, b = a.contiguous(), b.contiguous()
    y = out if out is not None else torch.empty(a.shape, dtype=out_dtype or torch.promote_types(a.dtype, b.dtype),
                                                device=a.device)
    L.call("sc_add", _p(a), _dt(a), _p(b), _dt(b), a.numel(), _p(y), _dt(y), stream_handle(a.device))
    return y


def argmax_workspace_bytes(M: int, N: int) -> int:
    return int(L.load().sc_argmax_workspace_bytes(M, N))


def argmax(logits: torch.Tensor, index_offset: int = 0, val: Optional[torch.Tensor] = None,
           idx: Optional[torch.Tensor] = None):
    """Per-row (max value, lowest index of it + offset) of fp32 logits [M, N]."""
    _cuda(logits)
    if logits.dtype != _F32:
        logits = logits.float()
    N = logits.shape[-1]
    lg = logits.reshape(-1, N).contiguous()
    M = lg.shape[0]
    val = val if val is not None else torch.empty(M, dtype=_F32, device=lg.device)
    idx = idx if idx is not None else torch.empty(M, dtype=torch.int32, device=lg.device)
    nb = argmax_workspace_bytes(M, N)
    ws = Workspace.get(nb, lg.device)
    L.call("sc_argmax", _p(lg), M, N, N, index_offset, _p(val), _p(idx), _p(ws), nb, stream_handle(lg.device))
    return val, idx


def argmax_merge(vals: torch.Tensor, idxs: torch.Tensor, world: int, token_out: torch.Tensor,
                 pos: Optional[torch.Tensor] = None, pos_advance: int = 0) -> torch.Tensor:
    _cuda(vals, idxs, token_out, pos)
    M = token_out.numel()
    L.call("sc_argmax_merge", _p(vals), _p(idxs), M, world, _p(token_out), _p(pos), pos_advance,
           stream_handle(vals.device))
    return token_out


# ---------------------------------------------------------------- K7b: temperature + top-p sampling

_ST_N, _ST_MAX, _ST_Z, _ST_KEPT, _ST_TOKEN = 8, 0, 1, 4, 7


def sample_workspace_bytes(B: int) -> int:
    return int(L.load().sc_sample_workspace_bytes(B))


def sample_uniforms(seed: int, counter: torch.Tensor, u: torch.Tensor) -> torch.Tensor:
    """Fill ``u`` (float32 [B]) with uniforms from (seed, the int64 device
    ``counter``), advancing the counter on the device (capturable)."""
    _cuda(counter, u)
    if counter.dtype != torch.int64 or u.dtype != torch.float32:
        raise ValueError("counter must be int64 and u float32")
    L.call("sc_sample_uniforms", C.c_uint64(seed & 0xFFFFFFFFFFFFFFFF), _p(counter), u.numel(), _p(u),
           stream_handle(u.device))
    return u


def sample_topp(logits: torch.Tensor, temperature: float, top_p: float, u: torch.Tensor, tok: torch.Tensor,
                comm=None, vocab_start: int = 0, workspace: Optional[torch.Tensor] = None,
                gather: Optional[torch.Tensor] = None):
    """Temperature + top-p draw from ``logits`` (float32 [B, V_local]) into
    ``tok`` (int32 [B]) -- the sampled branch of the reference's generate
    (worker/executor.py:270-306).  ``comm`` (tensor parallel): each rank
    passes its vocab slice and the ranks exchange only per-row scalars and
    256-bin histograms (all-gather / all-reduce on the current stream), never
    the logits; every rank ends with the same token in ``tok`` (global ids).
    ``tok`` keeps its value for a row whose draw found no token."""
    _cuda(logits, u, tok, workspace, gather)
    if logits.dtype != torch.float32 or logits.dim() != 2 or not logits.is_contiguous():
        raise ValueError("logits must be a contiguous float32 [B, V] tensor")
    if temperature <= 0.0 or top_p <= 0.0:
        raise ValueError("temperature and top_p must be positive (temperature 0 is the greedy argmax)")
    B, V = logits.shape
    nbytes = sample_workspace_bytes(B)
    if workspace is None:
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=logits.device)
    stream = stream_handle(logits.device)
    ws = workspace.data_ptr()
    world = 1 if comm is None else comm.world_size
    if world == 1:
        L.call("sc_sample_topp", _p(logits), B, V, V, float(temperature), float(top_p), _p(u), int(vocab_start),
               _p(tok), ws, nbytes, stream)
        return tok
    rank = comm.rank
    st = workspace[: _ST_N * B * 4].view(torch.float32).view(_ST_N, B)
    hist = workspace[_ST_N * B * 4: nbytes].view(torch.float32)
    if gather is None:
        gather = torch.empty(world, B, dtype=torch.float32, device=logits.device)

    def phase(ph, level=0):
        L.call("sc_sample_phase", _p(logits), B, V, V, float(temperature), float(top_p), _p(u), int(vocab_start), ph,
               level, ws, nbytes, stream)

    phase(0)
    comm.allgather_into(st[_ST_MAX], gather)
    L.call("sc_sample_combine", ws, _p(gather), B, world, rank, 0, None, stream)
    phase(1)
    comm.allreduce_into(st[_ST_Z], st[_ST_Z], "sum")
    for level in range(4):
        phase(2, level)
        comm.allreduce_into(hist, hist, "sum")
        phase(3, level)
    phase(4)
    comm.allgather_into(st[_ST_KEPT], gather)
    L.call("sc_sample_combine", ws, _p(gather), B, world, rank, 1, None, stream)
    phase(5)
    comm.allreduce_into(st[_ST_TOKEN], st[_ST_TOKEN], "sum")
    L.call("sc_sample_combine", ws, None, B, world, rank, 2, _p(tok), stream)
    return tok
