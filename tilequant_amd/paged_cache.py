"""A paged INT8 KV cache for serving ragged requests (HIP, gfx950).

Next to the fixed-length 16-bit ``StaticCache`` of ``graph_decode`` (the reference's only cache,
src/runtime/graph_decode.py:96-479), three pieces that a serving loop puts around its model:

* ``BlockTables``: which pages hold which request, kept on the device.  ``step`` releases the pages of
  finished requests, takes pages for the new tokens and returns their slots and positions; nothing comes
  back to the host, so a captured graph follows the requests' lengths by itself.
* ``PagedKVCache``: the pages themselves, INT8 codes with one fp32 scale per 16 tokens and kv head.
  ``append`` quantizes new keys and values into their slots, ``read`` gives them back in 16 bits, and
  ``attend`` is attention over the cache, for one new token per sequence or whole prompts.

One step of a serving loop, per layer after the first line::

    step = tables.step(new_tokens, max_tokens=T, finished=done)
    cache.append(layer, k, v, step.slots)
    out = cache.attend(layer, q, tables.block_table, tables.lengths, scale=scale,
                       query_start=step.query_start, max_query=longest)

Kernels: ``csrc/tq_paged.hip``, ``csrc/tq_paged_attention.hip``; formats and rules: ``include/tilequant.h``.
Every call only enqueues work on the current stream of the tensors' device.
"""
from __future__ import annotations

import ctypes
from functools import lru_cache
from typing import NamedTuple, Optional, Tuple

import torch

from . import _native as nat

UNIT = 16   # tokens that share a scale


def _check_block(block_size: int) -> None:
    if block_size < UNIT or block_size > 1024 or block_size & (block_size - 1):
        raise ValueError(f"block size must be a power of two in [16, 1024], got {block_size}")


def _int32(name: str, t: torch.Tensor, shape, device) -> None:
    if t.dtype != torch.int32 or t.shape != shape or not t.is_contiguous() or t.device != device:
        raise ValueError(f"{name} must be a contiguous int32 tensor of shape {tuple(shape)} on {device}")


class StepSlots(NamedTuple):
    """The new tokens of one ``BlockTables.step``, in request order."""

    slots: torch.Tensor         # [max_tokens] int32, -1 behind the last token
    positions: torch.Tensor     # [max_tokens] int32, 0 behind the last token
    query_start: torch.Tensor   # [requests + 1] int32: each request's first new token
    granted: torch.Tensor       # [requests] bool: its tokens found room


class BlockTables:
    """Pages of up to ``requests`` concurrent requests, on the device.

    ``block_table`` [requests, blocks_per_request], ``lengths`` [requests], ``free_blocks`` [pages] (a stack) and
    ``free_count`` [1], all int32; ``step`` updates them in place.  ``allocate`` makes empty tables over pages
    0 .. pages - 1."""

    def __init__(self, block_table: torch.Tensor, lengths: torch.Tensor, free_blocks: torch.Tensor,
                 free_count: torch.Tensor, block_size: int) -> None:
        nat.require_device(block_table, lengths, free_blocks, free_count)
        if block_size < 1:
            raise ValueError("block size must be positive")
        if block_table.dim() != 2 or block_table.dtype != torch.int32 or block_table.stride(1) != 1:
            raise ValueError("block_table must be an int32 matrix with unit column stride")
        rows, width = block_table.shape
        if rows > 1 and block_table.stride(0) < width:
            raise ValueError("block_table rows overlap")
        if free_blocks.dim() != 1:
            raise ValueError("free_blocks must be a vector")
        _int32("lengths", lengths, (rows,), block_table.device)
        _int32("free_blocks", free_blocks, free_blocks.shape, block_table.device)
        _int32("free_count", free_count, (1,), block_table.device)
        if max(width, free_blocks.numel()) * block_size >= 1 << 31:
            raise ValueError("slots are 32-bit: pages * block size must stay below 2^31")
        self._tensors = block_table, lengths, free_blocks, free_count   # held, as their addresses are below
        self.block_size = int(block_size)
        self._state = (block_table.data_ptr(), max(block_table.stride(0), width), lengths.data_ptr(),
                       free_blocks.data_ptr(), free_blocks.numel(), free_count.data_ptr())

    block_table = property(lambda self: self._tensors[0])
    lengths = property(lambda self: self._tensors[1])
    free_blocks = property(lambda self: self._tensors[2])
    free_count = property(lambda self: self._tensors[3])

    @classmethod
    def allocate(cls, *, requests: int, blocks_per_request: int, blocks: int, block_size: int = 64,
                 device="cuda") -> "BlockTables":
        new = lambda *s, fill: torch.full(s, fill, dtype=torch.int32, device=device)   # noqa: E731
        # the stack's top is its end: pages come out in ascending order at first
        free = torch.arange(blocks - 1, -1, -1, dtype=torch.int32, device=device)
        return cls(new(requests, blocks_per_request, fill=-1), new(requests, fill=0), free, new(1, fill=blocks),
                   block_size)

    def step(self, new_tokens: torch.Tensor, *, max_tokens: int, finished: Optional[torch.Tensor] = None) -> StepSlots:
        """Release the rows of ``finished`` [requests] (bool), then give every row room for ``new_tokens`` [requests]
        (int32; none where <= 0) more tokens, in row order.  A finished row starts a new request with its new tokens.

        A row whose tokens do not fit (its table's width, the free pages, ``max_tokens`` of one step) is refused:
        ``granted`` is False and its length stays.  Rows that come after a refused one do not take pages or places
        that it was waiting for (a row that needs no new page goes on)."""
        rows, width = self.block_table.shape
        dev = self.block_table.device
        nat.require_device(new_tokens, finished)
        _int32("new_tokens", new_tokens, (rows,), dev)
        if finished is not None:
            if finished.dtype not in (torch.bool, torch.uint8) or tuple(finished.shape) != (rows,) \
                    or not finished.is_contiguous() or finished.device != dev:
                raise ValueError("finished must be a contiguous bool vector with one entry per request")
        if not 0 <= max_tokens < 1 << 30:
            raise ValueError("max_tokens must be in [0, 2^30)")
        # one allocation for the three int32 results
        out = torch.empty((2 * max_tokens + rows + 1,), dtype=torch.int32, device=dev)
        granted = torch.empty((rows,), dtype=torch.bool, device=dev)
        at = out.data_ptr()
        nat.launch(dev, "tq_block_tables_step", nat.lib().tq_block_tables_step,
                   new_tokens.data_ptr(), nat.ptr(finished), *self._state, at, at + 4 * max_tokens, at + 8 * max_tokens,
                   granted.data_ptr(), rows, width, self.block_size, max_tokens)
        return StepSlots(*out.split((max_tokens, max_tokens, rows + 1)), granted)


@lru_cache(maxsize=1024)
def _attention_elems(*sizes: int) -> int:
    return int(nat.lib().tq_kv8_attention_workspace_elems(*sizes))


def paged_attention_workspace(tokens: int, batch: int, q_heads: int, kv_heads: int, head_dim: int, max_query: int,
                              max_length: int, device) -> Optional[torch.Tensor]:
    """fp32 scratch for the split partials of ``PagedKVCache.attend`` (``max_length``: the bound it is called with, at
    most the table's width in tokens); None when the call needs none."""
    elems = _attention_elems(tokens, batch, q_heads, kv_heads, head_dim, min(max_query, tokens), max_length)
    return torch.empty((elems,), device=device, dtype=torch.float32) if elems else None


class PagedKVCache:
    """INT8 keys and values of all layers, in pages of ``block_size`` tokens.

    ``k_codes`` [layers, pages, kv_heads, block_size / 16, 16, head_dim] and ``v_codes`` [..., head_dim, 16] int8,
    ``k_scales`` and ``v_scales`` [layers, pages, kv_heads, block_size / 16] fp32; head_dim 64 or 128.  ``allocate``
    makes them."""

    def __init__(self, k_codes: torch.Tensor, v_codes: torch.Tensor, k_scales: torch.Tensor,
                 v_scales: torch.Tensor) -> None:
        nat.require_device(k_codes, v_codes, k_scales, v_scales)
        if k_codes.dim() != 6 or k_codes.shape[4] != UNIT:
            raise ValueError("k_codes must be [layers, pages, kv_heads, block / 16, 16, head_dim]")
        layers, pages, kv_heads, units, _, dim = k_codes.shape
        if tuple(v_codes.shape) != (layers, pages, kv_heads, units, dim, UNIT):
            raise ValueError("v_codes must be [layers, pages, kv_heads, block / 16, head_dim, 16]")
        if dim not in (64, 128):
            raise ValueError(f"head_dim must be 64 or 128, got {dim}")
        _check_block(units * UNIT)
        if pages * units * UNIT >= 1 << 31:
            raise ValueError("slots are 32-bit: pages * block size must stay below 2^31")
        for name, t, dt in (("k_codes", k_codes, torch.int8), ("v_codes", v_codes, torch.int8),
                            ("k_scales", k_scales, torch.float32), ("v_scales", v_scales, torch.float32)):
            if t.dtype != dt or not t.is_contiguous() or t.device != k_codes.device:
                raise ValueError(f"{name} must be contiguous {dt} on one device")
        for name, t in (("k_scales", k_scales), ("v_scales", v_scales)):
            if tuple(t.shape) != (layers, pages, kv_heads, units):
                raise ValueError(f"{name} must be [layers, pages, kv_heads, block / 16]")
        self._tensors = k_codes, v_codes, k_scales, v_scales   # held, as their addresses are below
        self.layers, self.pages, self.kv_heads, self.head_dim = layers, pages, kv_heads, dim
        self.block_size = units * UNIT
        self.device = k_codes.device
        self._layers = [ctypes.byref(nat.Kv8Cache(nat.ptr(k_codes[i]), nat.ptr(v_codes[i]), nat.ptr(k_scales[i]),
                                                  nat.ptr(v_scales[i]), pages, kv_heads, dim, self.block_size))
                        for i in range(layers)]

    k_codes = property(lambda self: self._tensors[0])
    v_codes = property(lambda self: self._tensors[1])
    k_scales = property(lambda self: self._tensors[2])
    v_scales = property(lambda self: self._tensors[3])

    @classmethod
    def allocate(cls, *, layers: int, blocks: int, kv_heads: int, head_dim: int = 128, block_size: int = 64,
                 device="cuda") -> "PagedKVCache":
        _check_block(block_size)
        units = block_size // UNIT
        new = lambda *s, dt: torch.zeros((layers, blocks, kv_heads, units) + s, dtype=dt, device=device)   # noqa: E731
        return cls(new(UNIT, head_dim, dt=torch.int8), new(head_dim, UNIT, dt=torch.int8), new(dt=torch.float32),
                   new(dt=torch.float32))

    def _layer(self, layer: int):
        if not 0 <= layer < self.layers:
            raise IndexError(f"layer {layer} of {self.layers}")
        return self._layers[layer]

    def _rows(self, name: str, t: torch.Tensor, heads: int, dtype=None) -> None:
        if t.dim() != 3 or t.shape[1] != heads or t.shape[2] != self.head_dim or t.stride(2) != 1:
            raise ValueError(f"{name} must be [tokens, {heads}, {self.head_dim}] with unit stride in the head")
        if t.device != self.device or (dtype is not None and t.dtype != dtype):
            raise ValueError(f"{name} must be {dtype} on {self.device}")

    def _slots(self, slots: torch.Tensor) -> None:
        if slots.dtype != torch.int32 or slots.dim() != 1 or not slots.is_contiguous() or slots.device != self.device:
            raise ValueError(f"slots must be a contiguous int32 vector on {self.device}")

    def append(self, layer: int, key: torch.Tensor, value: torch.Tensor, slots: torch.Tensor) -> None:
        """Quantize ``key`` and ``value`` [tokens, kv_heads, head_dim] (bf16 or fp16) into ``slots`` [tokens].

        Slots outside the cache (-1) are skipped.  The new tokens of a unit (16 aligned slots) stand next to each
        other in the list, as ``BlockTables.step`` lists them; a slot named twice there keeps the later token.  A unit
        holds the tokens below the first offset written: writing its offset 0 starts it afresh.  Its scale grows
        with its largest value, and the codes it held are rounded to the grown scale."""
        nat.require_device(key, value, slots)
        self._rows("key", key, self.kv_heads)
        self._rows("value", value, self.kv_heads, key.dtype)
        self._slots(slots)
        if key.shape[0] != slots.shape[0] or value.shape[0] != slots.shape[0]:
            raise ValueError("key, value and slots must have as many tokens")
        nat.launch(self.device, "tq_kv8_append", nat.lib().tq_kv8_append, self._layer(layer), key.data_ptr(),
                   key.stride(0), key.stride(1), value.data_ptr(), value.stride(0), value.stride(1),
                   nat.dtype_code(key.dtype), slots.data_ptr(), slots.shape[0])

    def read(self, layer: int, slots: torch.Tensor, dtype: torch.dtype) -> Tuple[torch.Tensor, torch.Tensor]:
        """Keys and values [n, kv_heads, head_dim] of ``slots`` [n] in ``dtype``; zeros for slots outside the cache."""
        nat.require_device(slots)
        self._slots(slots)
        code = nat.dtype_code(dtype)
        out = torch.empty((2, slots.shape[0], self.kv_heads, self.head_dim), dtype=dtype, device=self.device)
        k, v = out.unbind(0)
        row, head = self.kv_heads * self.head_dim, self.head_dim
        nat.launch(self.device, "tq_kv8_read", nat.lib().tq_kv8_read, self._layer(layer), slots.data_ptr(),
                   slots.shape[0], code, k.data_ptr(), row, head, v.data_ptr(), row, head)
        return k, v

    def attend(self, layer: int, query: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor, *, scale: float,
               query_start: Optional[torch.Tensor] = None, max_query: int = 1, max_length: Optional[int] = None,
               out: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
        """softmax(scale * q k^T) v over each sequence's cached tokens.

        ``query`` [tokens, q_heads, head_dim] (bf16 or fp16); ``block_table`` [batch, width] and ``lengths`` [batch]
        (int32) say where each sequence's tokens are, the queried ones among them (appended before).  Without
        ``query_start`` there is one query per sequence; with it, queries query_start[b] .. query_start[b + 1] - 1
        are the last tokens of sequence b, causal among themselves, at most ``max_query`` of them.  A query that
        sees no key gives zeros; rows of ``out`` behind the last sequence are left as they were (a new ``out`` is
        zeroed when ``query_start`` is given).  batch * kv_heads is at most 65535.  ``max_length``: an upper bound of the lengths (default: the
        table's width), longer ones count as that; a tight one gives the best schedule."""
        nat.require_device(query, block_table, lengths, query_start, out, workspace)
        if query.dim() != 3 or query.shape[1] % self.kv_heads:
            raise ValueError(f"query must be [tokens, q_heads, {self.head_dim}] with q_heads a multiple of {self.kv_heads}")
        tokens, hq, dim = query.shape
        self._rows("query", query, hq)
        if block_table.dim() != 2 or block_table.dtype != torch.int32 or block_table.device != self.device \
                or (block_table.shape[1] > 1 and block_table.stride(1) != 1):
            raise ValueError(f"block_table must be an int32 matrix with unit column stride on {self.device}")
        batch, width = block_table.shape
        if batch > 1 and block_table.stride(0) < width:
            raise ValueError("block_table rows overlap")
        _int32("lengths", lengths, (batch,), self.device)
        if query_start is not None:
            _int32("query_start", query_start, (batch + 1,), self.device)
            if max_query < 1:
                raise ValueError("max_query must be positive")
            max_query = min(max_query, tokens)
        elif tokens != batch or max_query != 1:
            raise ValueError("without query_start there is one query per sequence")
        bound = width * self.block_size
        if max_length is not None:
            if max_length < 0:
                raise ValueError("max_length must not be negative")
            bound = min(bound, int(max_length))
        zero_rest = out is None and query_start is not None
        if out is None:
            if batch == 0:
                out = torch.zeros((tokens, hq, dim), device=self.device, dtype=query.dtype)
            elif query.is_contiguous():
                out = torch.empty_like(query)   # half a microsecond less than spelling it out
            else:
                out = torch.empty((tokens, hq, dim), device=self.device, dtype=query.dtype)
        else:
            self._rows("out", out, hq, query.dtype)
            if out.shape[0] != tokens:
                raise ValueError("out must have the query's shape")
        if workspace is None:
            workspace = paged_attention_workspace(tokens, batch, hq, self.kv_heads, dim, max_query, bound, self.device)
        elif workspace.dtype != torch.float32 or not workspace.is_contiguous() or workspace.device != self.device:
            raise ValueError(f"workspace must be contiguous fp32 on {self.device}")
        nat.launch(self.device, "tq_kv8_attention", nat.lib().tq_kv8_attention,
                   self._layer(layer), query.data_ptr(), query.stride(0), query.stride(1), nat.dtype_code(query.dtype),
                   block_table.data_ptr(), max(block_table.stride(0), width), width, lengths.data_ptr(),
                   nat.ptr(query_start), tokens, batch, hq, max_query, bound, float(scale), out.data_ptr(), out.stride(0),
                   out.stride(1), zero_rest, nat.ptr(workspace), workspace.numel() if workspace is not None else 0)
        return out
