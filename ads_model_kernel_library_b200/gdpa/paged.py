"""Serving from a paged key / value cache in 8 bits: block tables, the quantiser that fills the cache, and the GDPA forward over it.

The reference has no cache: its callers pack every request's keys and values anew for each call.  Here they stay on the GPU
between calls, as e4m3 values in blocks of 16, 32, 64 or 128 tokens with one fp32 scale per (block, head):

    k_cache, v_cache    [num_blocks, block_size, H_kv, D]  float8_e4m3fn   (value = e4m3 * scale)
    k_scales, v_scales  [num_blocks, H_kv]                 float32
    block_tables        [B, width]                         int32: the blocks of a request's tokens, in order

One step of a batch is :func:`build_block_tables` (blocks and slots of the new tokens), :func:`append_kv_cache_fp8` (their keys
and values) and :func:`generalized_dot_product_attention_paged_fp8` (their queries).  :class:`PagedKVCache` holds the tensors
and makes the three calls.  Nothing here synchronises with the host, and there are no gradients.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Sequence, Tuple

import torch

from . import _cabi
from .math import activation_string_to_int
from .ops import (
    _SUPPORTED_HEAD_DIMS,
    _define_op,
    _on_device,
    _raise_if_wait_ran_out,
    _set_timing,
    _status_word,
    _stream_ptr,
)
from . import ops as _ops

__all__ = ["build_block_tables", "append_kv_cache_fp8", "generalized_dot_product_attention_paged_fp8", "PagedKVCache"]

_BLOCK_SIZES = (16, 32, 64, 128)
_INTS = (torch.int32, torch.int64)


def _check_vector(name: str, t: torch.Tensor, device: torch.device, dtypes, length: Optional[int] = None) -> None:
    if t.device != device:
        raise RuntimeError(f"{name} must be on {device}, got {t.device}")
    if t.dtype not in dtypes:
        raise TypeError(f"{name} must be {' or '.join(str(d) for d in dtypes)}, got {t.dtype}")
    if t.dim() != 1 or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous 1-D tensor")
    if length is not None and t.numel() != length:
        raise ValueError(f"{name} must have {length} entries, got {t.numel()}")


def _check_table(block_tables: torch.Tensor, batch: int, block_size: int) -> None:
    if block_tables.dtype != torch.int32:
        raise TypeError(f"block_tables must be torch.int32, got {block_tables.dtype}")
    if block_tables.dim() != 2 or block_tables.shape[0] != batch:
        raise ValueError(f"block_tables must be [{batch}, width], got {tuple(block_tables.shape)}")
    if block_tables.shape[1] > 1 and block_tables.stride(1) != 1:
        raise ValueError("block_tables must have contiguous rows")
    if block_tables.shape[1] * block_size > 1 << 30:
        raise ValueError("block_tables: a request can hold 2^30 tokens at most")


def _check_cache(k_cache, v_cache, k_scales, v_scales, device: torch.device) -> Tuple[int, int, int, int]:
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache)):
        if t.device != device:
            raise RuntimeError(f"{name} must be on {device}, got {t.device}")
        if t.dtype != torch.float8_e4m3fn:
            raise TypeError(f"{name} must be torch.float8_e4m3fn, got {t.dtype}")
        if t.dim() != 4:
            raise ValueError(f"{name} must be [num_blocks, block_size, H_kv, D], got {tuple(t.shape)}")
        if t.stride(3) != 1 or t.data_ptr() % 16 or any(s % 16 or s <= 0 for s, n in zip(t.stride()[:3], t.shape) if n > 1):
            raise ValueError(f"{name} must have a contiguous head dimension and 16-byte aligned strides")
    if k_cache.shape != v_cache.shape:
        raise ValueError("k_cache and v_cache must have the same shape")
    blocks, size, heads, dim = k_cache.shape
    if size not in _BLOCK_SIZES:
        raise NotImplementedError(f"a block size of {size} is not supported (supported: {_BLOCK_SIZES})")
    if dim not in _SUPPORTED_HEAD_DIMS:
        raise NotImplementedError(f"head_dim {dim} is not supported (supported: {_SUPPORTED_HEAD_DIMS})")
    if heads < 1:
        raise ValueError("a cache must have at least one head")
    for name, t in (("k_scales", k_scales), ("v_scales", v_scales)):
        if t.device != device:
            raise RuntimeError(f"{name} must be on {device}, got {t.device}")
        if t.dtype != torch.float32:
            raise TypeError(f"{name} must be torch.float32, got {t.dtype}")
        if t.shape != (blocks, heads) or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous [{blocks}, {heads}] tensor")
    return blocks, size, heads, dim


def _cache_strides(field, t: torch.Tensor) -> None:
    # a dimension of one entry has no stride that matters: the contiguous one is taken (0)
    for i in range(3):
        field[i] = t.stride(i) if t.shape[i] > 1 else 0


def _check_rows(name: str, t: torch.Tensor, dtypes) -> None:
    if t.dim() != 3:
        raise ValueError(f"{name} must be [total_tokens, H, D], got {tuple(t.shape)}")
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor: this operator has no CPU path")
    if t.dtype not in dtypes:
        raise TypeError(f"{name} must be {' or '.join(str(d) for d in dtypes)}, got {t.dtype}")
    size = t.element_size()
    if t.shape[2] > 0 and t.numel() > 0 and (
            t.stride(2) != 1 or t.data_ptr() % 16 or any((s * size) % 16 or s < 0 for s, n in zip(t.stride()[:2], t.shape) if n > 1)):
        raise ValueError(f"{name} must have a contiguous head dimension and 16-byte aligned row / head strides "
                         "(a contiguous tensor, or a slice of a packed QKV / KV tensor along the last dimension)")


def _row_strides(field, t: torch.Tensor) -> None:
    for i in range(2):
        field[i] = t.stride(i) if t.shape[i] > 1 else 0


# ------------------------------------------------------------------------------------------ block tables, slot maps


def _tables_outputs(cached_lens, total_new):
    def empty(n, dtype):
        return torch.empty(n, dtype=dtype, device=cached_lens.device)

    batch = cached_lens.shape[0]
    return empty(total_new, torch.int64), empty(batch + 1, torch.int32), empty(batch, torch.int32), empty(1, torch.int32)


def _build_block_tables(block_tables, cached_lens, new_lens, free_blocks, num_free, block_size: int, total_new: int):
    if not cached_lens.is_cuda:
        raise RuntimeError("cached_lens must be a CUDA tensor: this operator has no CPU path")
    device, batch = cached_lens.device, cached_lens.numel()
    _check_vector("cached_lens", cached_lens, device, _INTS)
    _check_vector("new_lens", new_lens, device, (cached_lens.dtype,), batch)
    _check_vector("free_blocks", free_blocks, device, (torch.int32,))
    _check_vector("num_free", num_free, device, (torch.int32,), 1)
    if block_size not in _BLOCK_SIZES:
        raise NotImplementedError(f"a block size of {block_size} is not supported (supported: {_BLOCK_SIZES})")
    if block_tables.device != device:
        raise RuntimeError(f"block_tables must be on {device}, got {block_tables.device}")
    _check_table(block_tables, batch, block_size)
    if not 0 <= total_new < 1 << 31:
        raise ValueError(f"total_new must be in [0, 2^31), got {total_new}")
    with _on_device(cached_lens):
        slots, query_offset, seq_lens, num_free_after = _tables_outputs(cached_lens, total_new)
        p = _cabi.GdpaBlockTableParams()
        p.struct_size = C.sizeof(_cabi.GdpaBlockTableParams)
        p.lens_are_int64 = int(cached_lens.dtype == torch.int64)
        p.cached_lens, p.new_lens = cached_lens.data_ptr(), new_lens.data_ptr()
        p.batch, p.block_size = batch, block_size
        p.block_tables, p.table_stride, p.table_width = block_tables.data_ptr(), block_tables.stride(0), block_tables.shape[1]
        p.free_blocks, p.free_capacity, p.num_free = free_blocks.data_ptr(), free_blocks.numel(), num_free.data_ptr()
        p.total_new, p.slots = total_new, slots.data_ptr()
        p.query_offset, p.seq_lens, p.num_free_after = query_offset.data_ptr(), seq_lens.data_ptr(), num_free_after.data_ptr()
        _cabi.check(_cabi.lib.gdpa_build_block_tables(C.byref(p), _stream_ptr()), "gdpa_build_block_tables")
    return slots, query_offset, seq_lens, num_free_after


_define_op("build_block_tables(Tensor(a!) block_tables, Tensor cached_lens, Tensor new_lens, Tensor free_blocks, Tensor num_free, "
           "SymInt block_size, SymInt total_new) -> (Tensor, Tensor, Tensor, Tensor)",
           _build_block_tables,
           lambda block_tables, cached_lens, new_lens, free_blocks, num_free, block_size, total_new: _tables_outputs(cached_lens, total_new))


def build_block_tables(
    block_tables: torch.Tensor,
    cached_lens: torch.Tensor,
    new_lens: torch.Tensor,
    free_blocks: torch.Tensor,
    num_free: torch.Tensor,
    block_size: int,
    total_new: int,
) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """Blocks for the new tokens of a batch, and the slots of these tokens, in one kernel.

    Request ``b`` holds ``cached_lens[b]`` tokens in ``ceil(cached / block_size)`` blocks and gets ``new_lens[b]`` more (int32 or
    int64).  The further blocks it needs are taken from the top of the stack ``free_blocks[:num_free]`` (int32; ``num_free`` a
    tensor of one entry), in the order of the requests, and written into its row of ``block_tables`` (int32 ``[B, width]``, changed
    in place).  ``total_new`` is the number of new tokens, known to the caller who has their rows.

    Returns ``(slot_mapping, query_offset, seq_lens, num_free_after)``: int64 ``[total_new]``, the slot ``block * block_size + row``
    of each new token, -1 for one without a block; int32 ``[B + 1]`` prefix sums of ``new_lens``; int32 ``[B]`` ``cached + new``; int32
    ``[1]``, the entries of the stack that are left.  Where the stack runs out the table gets -1 and ``num_free_after`` is negative by
    the number of missing blocks; tokens beyond the width of the table get slot -1 and no block.  The stack itself is not changed.
    """
    return torch.ops.gdpa.build_block_tables(block_tables, cached_lens, new_lens, free_blocks, num_free, int(block_size), int(total_new))


# ------------------------------------------------------------------------------------------ new keys and values


def _append(key, value, k_cache, v_cache, k_scales, v_scales, slot_mapping) -> None:
    _check_rows("key", key, (torch.bfloat16, torch.float32))
    _check_rows("value", value, (key.dtype,))
    blocks, size, heads, dim = _check_cache(k_cache, v_cache, k_scales, v_scales, key.device)
    if key.shape != value.shape or value.device != key.device:
        raise ValueError("key and value must have the same shape and device")
    if key.shape[1:] != (heads, dim):
        raise ValueError(f"key and value must be [tokens, {heads}, {dim}] for this cache, got {tuple(key.shape)}")
    _check_vector("slot_mapping", slot_mapping, key.device, (torch.int64,), key.shape[0])
    if _ops._validate_offsets:
        _check_slots(slot_mapping, blocks, size)
    with _on_device(key):
        p = _cabi.GdpaCacheAppendParams()
        p.struct_size = C.sizeof(_cabi.GdpaCacheAppendParams)
        p.x_is_fp32 = int(key.dtype == torch.float32)
        p.key, p.value = key.data_ptr(), value.data_ptr()
        _row_strides(p.key_strides, key)
        _row_strides(p.value_strides, value)
        p.k_cache, p.v_cache = k_cache.data_ptr(), v_cache.data_ptr()
        _cache_strides(p.k_cache_strides, k_cache)
        _cache_strides(p.v_cache_strides, v_cache)
        p.k_scales, p.v_scales, p.slot_mapping = k_scales.data_ptr(), v_scales.data_ptr(), slot_mapping.data_ptr()
        p.tokens, p.num_blocks, p.block_size, p.kv_heads, p.head_dim = key.shape[0], blocks, size, heads, dim
        _cabi.check(_cabi.lib.gdpa_append_kv_cache_fp8(C.byref(p), _stream_ptr()), "gdpa_append_kv_cache_fp8")


def _check_slots(slot_mapping: torch.Tensor, blocks: int, size: int) -> None:
    """The host's look at a slot map (offset validation): every block's tokens are one run."""
    s = slot_mapping.detach().to("cpu")
    s = s[(s >= 0) & (s < blocks * size)]
    if s.numel() == 0:
        return
    begins = torch.ones_like(s, dtype=torch.bool)
    begins[1:] = (s[1:] != s[:-1] + 1) | (s[1:] % size == 0)
    runs = s[begins] // size
    if runs.unique().numel() != runs.numel():
        raise ValueError("slot_mapping must hold the tokens of a block one after the other, with consecutive slots")


_define_op("append_kv_cache_fp8(Tensor key, Tensor value, Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor(c!) k_scales, "
           "Tensor(d!) v_scales, Tensor slot_mapping) -> ()",
           _append, lambda *args: None)


def append_kv_cache_fp8(
    key: torch.Tensor,
    value: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    k_scales: torch.Tensor,
    v_scales: torch.Tensor,
    slot_mapping: torch.Tensor,
) -> None:
    """Quantise new keys and values (``[tokens, H_kv, D]``, bf16 or fp32, strided as for the attention) into their slots of a cache.

    The new tokens of a block are a run: they follow one another and have consecutive slots (as :func:`build_block_tables` gives them).
    Its scale is a power of two, the smallest with ``amax / scale <= 448`` over the run's finite values (at least 2^-100), or, if
    the block has rows before the run, the larger of that and the block's scale: these rows are rescaled when the scale grows (which
    loses nothing but bits below e4m3's smallest normal value).  Values round to nearest even; infinities become ``448 * scale``, NaN stays
    NaN.  Tokens whose slot is not in the cache (-1) are skipped.  Two runs of one block in a call are not allowed (and raise
    ``ValueError`` with offset validation on); rows after a run count as unused.
    """
    torch.ops.gdpa.append_kv_cache_fp8(key, value, k_cache, v_cache, k_scales, v_scales, slot_mapping)


# ------------------------------------------------------------------------------------------ attention over the cache


def _paged_forward(query, k_cache, v_cache, k_scales, v_scales, block_tables, query_offset, seq_lens, max_seq_len_q: int,
                   qk_scale: float, activation: int, is_causal: bool, window_size: int) -> torch.Tensor:
    _check_rows("query", query, (torch.bfloat16,))
    device = query.device
    _raise_if_wait_ran_out(device)
    blocks, size, kv_heads, dim = _check_cache(k_cache, v_cache, k_scales, v_scales, device)
    total_q, heads = query.shape[:2]
    if query.shape[2] != dim:
        raise ValueError(f"query must have the cache's head_dim {dim}, got {query.shape[2]}")
    if heads < 1 or heads % kv_heads != 0:
        raise ValueError("the number of query heads must be a multiple of the number of key/value heads")
    _check_vector("seq_lens", seq_lens, device, _INTS)
    batch = seq_lens.numel()
    _check_vector("query_offset", query_offset, device, _INTS, batch + 1)
    if block_tables.device != device:
        raise RuntimeError(f"block_tables must be on {device}, got {block_tables.device}")
    _check_table(block_tables, batch, size)
    if max_seq_len_q < 0:
        raise ValueError("max_seq_len_q must not be negative")
    if _ops._validate_offsets:
        _ops._check_offsets("query_offset", query_offset, total_q, False)
        n = seq_lens.detach().to("cpu", torch.int64)
        if n.numel() and (int(n.min()) < 0 or int(n.max()) > block_tables.shape[1] * size):
            raise ValueError("seq_lens has entries outside [0, width of block_tables * block size]")
    with _on_device(query):
        o = torch.empty((total_q, heads, dim), dtype=torch.bfloat16, device=device)
        if total_q == 0 or batch == 0:
            return o
        p = _cabi.GdpaPagedParams()
        p.struct_size = C.sizeof(_cabi.GdpaPagedParams)
        p.activation, p.qk_scale = activation, qk_scale
        p.q, p.o = query.data_ptr(), o.data_ptr()
        _row_strides(p.q_strides, query)
        p.k_cache, p.v_cache = k_cache.data_ptr(), v_cache.data_ptr()
        _cache_strides(p.k_cache_strides, k_cache)
        _cache_strides(p.v_cache_strides, v_cache)
        p.k_scales, p.v_scales = k_scales.data_ptr(), v_scales.data_ptr()
        p.block_tables, p.table_stride, p.table_width = block_tables.data_ptr(), block_tables.stride(0), block_tables.shape[1]
        p.block_size, p.num_blocks = size, blocks
        p.q_offsets, p.offsets_are_int64 = query_offset.data_ptr(), int(query_offset.dtype == torch.int64)
        p.seq_lens, p.lens_are_int64 = seq_lens.data_ptr(), int(seq_lens.dtype == torch.int64)
        p.batch, p.heads, p.kv_heads, p.head_dim = batch, heads, kv_heads, dim
        p.total_q, p.max_seq_len_q = total_q, max_seq_len_q
        p.causal = int(is_causal)
        p.window_plus_one = window_size + 1 if window_size >= 0 else 0
        nbytes = _cabi.lib.gdpa_paged_workspace_bytes(heads, kv_heads, dim, max_seq_len_q)
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=device)
        p.workspace, p.workspace_bytes = workspace.data_ptr(), nbytes
        p.status = _status_word(device).data_ptr()
        _set_timing(p, "fwd")
        _cabi.check(_cabi.lib.gdpa_fwd_paged_fp8(C.byref(p), _stream_ptr()), "gdpa_fwd_paged_fp8")
    return o


_define_op("generalized_dot_product_attention_paged_fp8(Tensor query, Tensor k_cache, Tensor v_cache, Tensor k_scales, Tensor v_scales, "
           "Tensor block_tables, Tensor query_offset, Tensor seq_lens, SymInt max_seq_len_q, float qk_scale, int activation, bool is_causal, "
           "SymInt window_size) -> Tensor",
           _paged_forward,
           lambda query, *args: torch.empty(query.shape, dtype=torch.bfloat16, device=query.device))


def generalized_dot_product_attention_paged_fp8(
    query: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    k_scales: torch.Tensor,
    v_scales: torch.Tensor,
    block_tables: torch.Tensor,
    query_offset: torch.Tensor,
    seq_lens: torch.Tensor,
    max_seq_len_q: int,
    qk_scale: Optional[float] = None,
    activation: str = "softmax",
    is_causal: bool = False,
    window_size: Optional[int] = None,
) -> torch.Tensor:
    """``O = act(Q K^T) qk_scale V`` (or the softmax form, as :func:`generalized_dot_product_attention`) of each request's queries over its
    cached keys and values; bf16 ``[total_q, H, D]``, ``H`` a multiple of ``H_kv``.

    The queries of request ``b`` are the rows ``query_offset[b]:query_offset[b + 1]`` of ``query`` (at most ``max_seq_len_q``), its keys the
    first ``seq_lens[b]`` tokens of its row of ``block_tables``.  Query ``i`` of ``n`` has position ``seq_lens[b] - n + i``: with ``is_causal`` it
    takes part with keys up to its position, with ``window_size`` with those at most that far from it.  Without either every query sees all
    keys (candidates of a request that attend to its history).  A row without keys gives zeros.  Tokens past ``seq_lens[b]``, and blocks
    that the table has not (-1), take no part, whatever their memory holds.  Scales must be positive.  ``seq_lens`` and ``query_offset`` are
    trusted like the offsets of the other operators (clamped in the kernel, checked on the host with offset validation on).
    """
    return torch.ops.gdpa.generalized_dot_product_attention_paged_fp8(
        query, k_cache, v_cache, k_scales, v_scales, block_tables, query_offset, seq_lens, int(max_seq_len_q),
        1.0 if qk_scale is None else float(qk_scale), activation_string_to_int(activation), bool(is_causal),
        -1 if window_size is None else int(window_size))


class PagedKVCache:
    """The cache of a batch of requests, with its free blocks, and the three calls of a step.

    ``step`` appends the new tokens' keys and values of every request and attends with their queries; ``release`` gives back the blocks
    of requests that are done.  Everything stays on the GPU; ``num_free`` (a tensor of one entry) is for the host to read when it wants to
    know how much room is left: negative, a step wanted more blocks than there were.
    """

    def __init__(self, num_blocks: int, block_size: int, kv_heads: int, head_dim: int, batch: int, max_tokens: int, device="cuda"):
        shape = (num_blocks, block_size, kv_heads, head_dim)
        self.block_size = block_size
        self.k_cache, self.v_cache = (torch.zeros(shape, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn) for _ in range(2))
        self.k_scales, self.v_scales = (torch.ones(num_blocks, kv_heads, device=device) for _ in range(2))
        width = (max_tokens + block_size - 1) // block_size
        self.block_tables = torch.full((batch, width), -1, dtype=torch.int32, device=device)
        self.seq_lens = torch.zeros(batch, dtype=torch.int32, device=device)
        self.free_blocks = torch.arange(num_blocks - 1, -1, -1, dtype=torch.int32, device=device)
        self.num_free = torch.full((1,), num_blocks, dtype=torch.int32, device=device)

    def append(self, key: torch.Tensor, value: torch.Tensor, new_lens: torch.Tensor) -> torch.Tensor:
        """Store the keys and values of ``new_lens[b]`` (int32) new tokens of each request; returns their offsets ``[B + 1]``."""
        slots, query_offset, self.seq_lens, self.num_free = build_block_tables(
            self.block_tables, self.seq_lens, new_lens, self.free_blocks, self.num_free, self.block_size, key.shape[0])
        append_kv_cache_fp8(key, value, self.k_cache, self.v_cache, self.k_scales, self.v_scales, slots)
        return query_offset

    def attend(self, query: torch.Tensor, query_offset: torch.Tensor, max_seq_len_q: int, **options) -> torch.Tensor:
        """:func:`generalized_dot_product_attention_paged_fp8` over what the cache holds."""
        return generalized_dot_product_attention_paged_fp8(
            query, self.k_cache, self.v_cache, self.k_scales, self.v_scales, self.block_tables, query_offset, self.seq_lens, max_seq_len_q,
            **options)

    def step(self, query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, new_lens: torch.Tensor, max_seq_len_q: int,
             **options) -> torch.Tensor:
        """Append, then attend with the new tokens' queries (causal unless ``is_causal=False`` is given)."""
        return self.attend(query, self.append(key, value, new_lens), max_seq_len_q, **{"is_causal": True, **options})

    def release(self, requests: Sequence[int]) -> None:
        """Give back the blocks of these requests (rows of the tables), which are empty afterwards."""
        rows = torch.as_tensor(requests, dtype=torch.int64, device=self.block_tables.device)
        table = self.block_tables[rows]
        held = torch.arange(table.shape[1], device=table.device) < ((self.seq_lens[rows] + self.block_size - 1) // self.block_size)[:, None]
        held &= table >= 0
        place = self.num_free.clamp_min(0) + torch.cumsum(held.flatten(), 0) - 1
        # entries that are not held go to a place behind the stack
        stack = torch.cat([self.free_blocks, self.free_blocks.new_zeros(1)])
        stack[torch.where(held.flatten(), place, self.free_blocks.numel())] = table.flatten()
        self.free_blocks = stack[:-1]
        self.num_free = self.num_free.clamp_min(0) + held.sum().to(torch.int32)
        self.block_tables[rows] = -1
        self.seq_lens[rows] = 0
