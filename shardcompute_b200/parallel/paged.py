"""A KV cache of pages for a ragged batch, next to the contiguous ``KVCache``.

``PagedKVCache`` holds every layer's pool of pages ``[n_pages, Hkv/TP, page, hd]`` and, shared by all layers, the block
table, the requests' lengths and the stack of free pages -- all on the device, so that a step can be captured (with counts
that are device tensors; the first step runs outside of the capture, for it makes the model's rotary tables).  A step
is: ``reserve`` room for each request's new tokens, run the model on the new tokens of all requests in a row
(``input_ids`` ``[1, T]``) with ``past_key_values=cache.layers()``, then ``truncate`` what did not stay (rejected
drafts, ended requests).  A request can be made the prefix that all others share (``share_prefix``): its keys and values
are held once and attended to once for the whole batch.

With ``bits`` 8 or 4 the pages hold codes (``ops.QuantPages``): a quarter to a half of float16's room, 72 bytes in place of
256 for a token's key or value of a head of 128.  Keys and values are quantised as they are written and attended to as they
lie; ``read`` gives back what the cache stands for.

The attention is cut by what the tables have room for, since the lengths live on the device: ``max_len`` and ``max_prefix`` far
past what is held cost time (64 requests behind 8197 tokens with room for 32768: the prefix's kernel runs as 8 CTAs, not 48), not
correctness.  ``ops.prefix_attn_q_plan`` says how a call is cut.
"""

from __future__ import annotations

from typing import List, NamedTuple, Optional, Sequence, Union

import torch

from .. import ops

_WHY = {1: "not enough free pages", 2: "a request exceeds its block table", 4: "more new tokens than rows",
        8: "a negative length", 16: "the count of free pages is outside the stack"}
_WHY_BACK = {**_WHY, 1: "no room for the pages given back (a page held twice)"}


class PagedLayer(NamedTuple):
    """One layer of a ``PagedKVCache``: what ``ParallelAttention`` takes as ``past_key_value``.  ``pages`` in place of ``k``
    and ``v`` where they are held in 8 or 4 bits."""

    cache: "PagedKVCache"
    k: Optional[torch.Tensor]
    v: Optional[torch.Tensor]
    pages: Optional["ops.QuantPages"] = None


class PagedKVCache:
    def __init__(self, num_layers: int, kv_heads: int, head_dim: int, n_pages: int, max_batch: int, max_len: int,
                 page_size: int = 16, max_prefix: int = 0, max_tokens: Optional[int] = None,
                 dtype: torch.dtype = torch.float32, device: Optional[torch.device] = None, bits: Optional[int] = None,
                 group_size: int = 64):
        """``max_len`` / ``max_prefix``: tokens of a request and of the shared prefix at most (0: none).
        ``max_tokens``: new tokens of a step at most (default ``max_batch``, one each).  ``bits``: 8 or 4, by groups of
        ``group_size`` (32 or 64) dims, and queries and outputs of the attention are float16; ``dtype`` is that of pages
        which are not.  What the operators do not take is
        refused here, not after pages were reserved and keys written: heads of 64 or 128, pages of a power of two from 16 to
        32768 tokens, 16384 requests at most, and a pool whose rows (pages x heads x page size) count in 32 bits."""
        if dtype not in (torch.float16, torch.float32):
            raise ValueError(f"pages must be float16 or float32, got {dtype}")
        if min(num_layers, kv_heads, head_dim, n_pages, max_batch, max_len, page_size) < 1 or max_prefix < 0:
            raise ValueError("PagedKVCache: sizes must be positive")
        if head_dim not in (64, 128):
            raise ValueError(f"PagedKVCache: head_dim {head_dim} unsupported (64, 128)")
        if not 16 <= page_size <= 32768 or page_size & (page_size - 1):
            raise ValueError(f"PagedKVCache: page_size {page_size} unsupported (a power of two from 16 to 32768)")
        if max_batch > 16384 or (max_tokens is not None and max_tokens < 1):
            raise ValueError(f"PagedKVCache: 1..16384 requests and at least one new token, got {max_batch} and {max_tokens}")
        if max(n_pages * kv_heads * page_size, max_len + page_size, max_prefix + page_size) >= 2**31:
            raise ValueError("PagedKVCache: rows of the pool, or tokens of a request, past 32 bits")
        dev = device or torch.device("cuda", torch.cuda.current_device())
        i32 = dict(dtype=torch.int32, device=dev)
        blocks = -(-max_len // page_size)
        if max_prefix:  # a request of this batch becomes the prefix
            blocks = max(blocks, -(-max_prefix // page_size))
        self.page_size, self.max_batch = page_size, max_batch
        self.max_tokens = max_batch if max_tokens is None else max_tokens
        self.max_positions = blocks * page_size * (2 if max_prefix else 1)
        self.k = self.v = self.pages = None
        if bits is None:
            self.k = torch.zeros(num_layers, n_pages, kv_heads, page_size, head_dim, dtype=dtype, device=dev)
            self.v = torch.zeros_like(self.k)
        else:
            nbytes = ops.quant_page_bytes(page_size, head_dim, bits, group_size)
            data = torch.zeros(num_layers, n_pages, kv_heads, nbytes, dtype=torch.uint8, device=dev)
            self.pages = [ops.QuantPages(d, head_dim, page_size, bits, group_size) for d in data]
        self.free_pages = torch.arange(n_pages - 1, -1, -1, **i32)  # page 0 on top
        self.free_count = torch.full((1,), n_pages, **i32)
        self.block_table = torch.full((max_batch, blocks), -1, **i32)
        self.lens = torch.zeros(max_batch, **i32)
        self.prefix_table = torch.full((blocks,), -1, **i32) if max_prefix else None
        self.prefix_len = torch.zeros(1, **i32) if max_prefix else None
        # of the last reservation, and of the last truncation or release: a step's truncation must not cover its reservation's
        self._status = torch.zeros(2, **i32)
        self.status, self.truncate_status = self._status[:1], self._status[1:]
        self._q_start = torch.zeros(max_batch + 1, **i32)
        self._slots = torch.full((self.max_tokens,), -1, **i32)
        self._positions = torch.zeros(self.max_tokens, **i32)
        self.step = ops.PagedStep(self.lens, self._q_start, self._slots, self._positions, self.free_count, self.status)

    def _per_request(self, what: str, values: Union[torch.Tensor, Sequence[int]]) -> torch.Tensor:
        t = values if isinstance(values, torch.Tensor) else torch.tensor(list(values), dtype=torch.int32)
        if t.numel() != self.max_batch:
            raise ValueError(f"{what}: {t.numel()} values for {self.max_batch} requests")
        return t.to(device=self.lens.device, dtype=torch.int32)

    def reserve(self, new_lens: Union[torch.Tensor, Sequence[int]]) -> "ops.PagedStep":
        """Room for ``new_lens[b]`` more tokens of every request (0: it takes no part in this step)."""
        self.step = ops.paged_reserve(self.lens, self._per_request("reserve", new_lens), self.block_table, self.free_pages,
                                      self.free_count, self.page_size, prefix_len=self.prefix_len, kv_lens=self.lens,
                                      q_start=self._q_start, slots=self._slots, positions=self._positions,
                                      free_count_out=self.free_count, status=self.status)
        return self.step

    def truncate(self, keep: Union[torch.Tensor, Sequence[int]]) -> None:
        """Cut every request to its first ``keep[b]`` tokens; 0 ends it and gives its pages back."""
        ops.paged_truncate(self.lens, self._per_request("truncate", keep), self.block_table, self.free_pages, self.free_count,
                           self.page_size, lens_out=self.lens, free_count_out=self.free_count, status=self.truncate_status)

    def share_prefix(self, request: int) -> None:
        """Make this request's tokens the prefix of the whole batch; the request is empty after it."""
        if self.prefix_table is None:
            raise ValueError("this cache was made without room for a prefix (max_prefix)")
        if not 0 <= request < self.max_batch:
            raise IndexError(f"request {request} out of range [0, {self.max_batch})")
        if int(self.prefix_len):
            raise ValueError("the batch has a prefix already: release_prefix first")
        if int(self.lens.sum()) != int(self.lens[request]):
            raise ValueError("the other requests' tokens would move behind the prefix: share it before they start")
        self.prefix_table.copy_(self.block_table[request])
        self.prefix_len.copy_(self.lens[request:request + 1])
        self.lens[request] = 0

    def release_prefix(self) -> None:
        """Give the prefix's pages back; no request may have tokens behind it."""
        if self.prefix_table is None:
            raise ValueError("this cache was made without room for a prefix (max_prefix)")
        if int(self.lens.sum()):
            raise ValueError("requests still hold tokens behind the prefix")
        ops.paged_truncate(self.prefix_len, torch.zeros_like(self.prefix_len), self.prefix_table.view(1, -1), self.free_pages,
                           self.free_count, self.page_size, lens_out=self.prefix_len, free_count_out=self.free_count,
                           status=self.truncate_status)

    def check(self) -> None:
        """Raise ``ValueError`` if the last ``reserve`` was refused, or the last ``truncate`` or ``release_prefix`` (reads both
        status words from the device), and ``RuntimeError`` if the attention gave up a wait since the last check."""
        why = [f"{what}: " + ", ".join(w for bit, w in names.items() if st & bit)
               for what, names, st in zip(("reserve", "truncate"), (_WHY, _WHY_BACK), self._status.tolist()) if st]
        if why:
            raise ValueError("paged cache, " + "; ".join(why))
        if self.lens.is_cuda and ops.prefix_attn_device_error(self.lens.device):
            raise RuntimeError("prefix_attn gave up a bounded wait: the attention's outputs since the last check are undefined")

    def layers(self) -> List[PagedLayer]:
        """``past_key_values`` of ``ParallelTransformer.forward``."""
        if self.pages is not None:
            return [PagedLayer(self, None, None, p) for p in self.pages]
        return [PagedLayer(self, k, v) for k, v in zip(self.k, self.v)]

    def read(self, layer: int, request: int, dtype: Optional[torch.dtype] = None):
        """The request's tokens in one layer, as ``(k, v)`` ``[len, Hkv/TP, hd]`` of ``dtype`` (default: that of the pages; of pages
        in 8 or 4 bits float16): what the cache holds, keys as they were rotated, to look at or to compare.  Zeros where the
        block table has no page.  Waits for the device (a request's length lives there).  The shared prefix is not among
        them, and no call writes them back: an append takes keys before their rotation."""
        if not 0 <= request < self.max_batch:
            raise IndexError(f"request {request} out of range [0, {self.max_batch})")
        n = int(self.lens[request])
        at = torch.arange(n, device=self.lens.device)
        slots = self.block_table[request, at // self.page_size] * self.page_size + at.int() % self.page_size
        if self.pages is not None:
            return ops.paged_read_q(self.pages[layer], slots, dtype=dtype or torch.float16)
        page, off = slots.long() // self.page_size, slots.long() % self.page_size
        there = (page >= 0) & (page < self.k.shape[1])
        page = page.where(there, 0)
        return tuple(x[layer][page, :, off].masked_fill(~there[:, None, None], 0).to(dtype or x.dtype) for x in (self.k, self.v))
