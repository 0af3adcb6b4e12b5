"""Serving from a paged key / value cache in 8 bits: block tables, the quantiser that fills the cache, and the GDPA forward over it.

The reference has no cache: its callers pack every request's keys and values anew for each call.  Here they stay on the GPU
between calls, as e4m3 values in blocks of 16, 32, 64 or 128 tokens with one fp32 scale per (block, head):

    k_cache, v_cache    [num_blocks, block_size, H_kv, D]  float8_e4m3fn   (value = e4m3 * scale)
    k_scales, v_scales  [num_blocks, H_kv]                 float32
    block_tables        [B, width]                         int32: the blocks of a request's tokens, in order

One step of a batch is :func:`build_block_tables` (blocks and slots of the new tokens), :func:`append_kv_cache_fp8` (their keys
and values) and :func:`generalized_dot_product_attention_paged_fp8` (their queries).  :func:`append_rotated_kv_cache_fp8` norms and rotates queries
and keys on the way, :func:`read_kv_cache_fp8` gives packed keys and values back, :func:`drop_cached_tokens` takes tokens out again (drafts
that were refused).  :class:`PagedKVCache` holds the tensors and makes the calls.  Nothing here synchronises with the host, and there are no
gradients.
"""
from __future__ import annotations

import ctypes as C
import operator
import os
import threading
from typing import Optional, Sequence, Tuple

import torch

from . import _cabi, ops
from .math import activation_string_to_int

__all__ = ["build_block_tables", "append_kv_cache_fp8", "append_rotated_kv_cache_fp8", "generalized_dot_product_attention_paged_fp8", "read_kv_cache_fp8",
           "drop_cached_tokens", "PagedKVCache"]

LIB_PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "libgdpa_b200_torch.so")


@C.CFUNCTYPE(C.c_void_p, C.c_int, C.POINTER(C.c_char), C.c_int)
def _look_at_status(device: int, message, size: int):
    """The address of a device's status word, for the operators' C++ side: called for a device's first call, and when the word is set."""
    where = torch.device("cuda", device)
    word = ops._status_word(where).data_ptr()
    try:
        ops._raise_if_wait_ran_out(where)
    except RuntimeError as e:
        text = str(e).encode()[:size - 1] + b"\0"
        C.memmove(message, text, len(text))
    return word


class _Operators:
    """The torch operators that libgdpa_b200_torch.so registers (checks, outputs and launch in C++: a step of generation is host
    time), with their fake kernels."""

    def __init__(self):
        if not os.path.exists(LIB_PATH):
            raise ImportError(f"{LIB_PATH} is missing: build it with `python -m ads_model_kernel_library_b200.build` (needs g++ and torch's "
                              "headers); these operators have no other path")
        lib = _cabi.lib if "lib" in vars(_cabi) else _cabi.__getattr__("lib")
        first = not hasattr(torch.ops.gdpa, "append_kv_cache_fp8")  # a second load of this module finds them registered
        torch.ops.load_library(LIB_PATH)
        self.native = C.CDLL(LIB_PATH)
        entries = (lib.gdpa_build_block_tables, lib.gdpa_append_kv_cache_fp8, lib.gdpa_paged_workspace_bytes, lib.gdpa_fwd_paged_fp8, lib.gdpa_strerror)
        self.native.gdpa_torch_init(*(C.cast(f, C.c_void_p) for f in entries))
        entries = (lib.gdpa_qk_norm_rotary, lib.gdpa_qk_norm_rotary_bwd, lib.gdpa_rotary_workspace_bytes, lib.gdpa_append_rotated_kv_cache_fp8,
                   lib.gdpa_read_kv_cache_fp8, lib.gdpa_verify_workspace_bytes, lib.gdpa_verify_draft_tokens, lib.gdpa_drop_workspace_bytes, lib.gdpa_drop_cached_tokens)
        self.native.gdpa_torch_init_heads((C.c_void_p * len(entries))(*(C.cast(f, C.c_void_p) for f in entries)))
        self.native.gdpa_torch_set_timing.argtypes = [C.c_void_p, C.c_void_p]
        self.native.gdpa_torch_set_status_look(_look_at_status)
        if first:
            torch.library.register_fake("gdpa::build_block_tables", _fake_tables)
            torch.library.register_fake("gdpa::append_kv_cache_fp8", lambda *args: None)
            torch.library.register_fake("gdpa::generalized_dot_product_attention_paged_fp8",
                                        lambda query, *args: torch.empty(query.shape, dtype=torch.bfloat16, device=query.device))
            torch.library.register_fake("gdpa::qk_norm_rotary", lambda query, key, *args: (_packed(query), _packed(key)))
            torch.library.register_fake("gdpa::qk_norm_rotary_backward", _fake_rotary_backward)
            torch.library.register_fake("gdpa::append_rotated_kv_cache_fp8", lambda query, *args: _packed(query))
            torch.library.register_fake("gdpa::read_kv_cache_fp8", _fake_read)
            torch.library.register_fake("gdpa::verify_draft_tokens", _fake_verify)
            torch.library.register_fake("gdpa::drop_cached_tokens",
                                        lambda table, lens, *args: (torch.empty_like(lens, dtype=torch.int32), lens.new_empty(1, dtype=torch.int32)))
        self.tables = torch.ops.gdpa.build_block_tables.default
        self.append = torch.ops.gdpa.append_kv_cache_fp8.default
        self.attend = torch.ops.gdpa.generalized_dot_product_attention_paged_fp8.default
        self.rotary = torch.ops.gdpa.qk_norm_rotary.default
        self.append_rotated = torch.ops.gdpa.append_rotated_kv_cache_fp8.default
        self.read = torch.ops.gdpa.read_kv_cache_fp8.default
        self.verify = torch.ops.gdpa.verify_draft_tokens.default
        self.drop = torch.ops.gdpa.drop_cached_tokens.default


_operators: Optional[_Operators] = None
_loading = threading.Lock()


def _load() -> _Operators:
    global _operators
    with _loading:  # first calls of two threads: the operators are registered once
        if _operators is None:
            _operators = _Operators()
    return _operators


def _fake_tables(block_tables, cached_lens, new_lens, free_blocks, num_free, block_size, total_new):
    def empty(n, dtype):
        return torch.empty(n, dtype=dtype, device=cached_lens.device)

    batch = cached_lens.shape[0]
    return empty(total_new, torch.int64), empty(batch + 1, torch.int32), empty(batch, torch.int32), empty(1, torch.int32)


def _packed(x):
    return x.new_empty(x.shape)


def _fake_rotary_backward(query_grad, key_grad, query, key, inv_freq, query_positions, key_positions, query_weight, key_weight, eps, norm, interleaved, sections,
                          weight_grads):
    def of(weight):
        return query.new_empty(0, dtype=torch.float32) if weight is None or not (weight_grads and norm) else weight.new_empty(weight.shape)

    return _packed(query), _packed(key), of(query_weight), of(key_weight)


def _fake_read(k_cache, v_cache, k_scales, v_scales, block_tables, key_offset, total_tokens, first_tokens, dtype):
    return tuple(torch.empty((total_tokens, *k_cache.shape[2:]), dtype=dtype, device=k_cache.device) for _ in range(2))


def _fake_verify(target_probs, draft_probs, draft_tokens, query_offset, draft_offset, accept_uniform, sample_uniform, max_drafts):
    batch = sample_uniform.shape[0]
    return draft_tokens.new_empty((batch, max_drafts + 1)), *(draft_tokens.new_empty(batch, dtype=torch.int32) for _ in range(2))


# ------------------------------------------------------------------------------------------ block tables, slot maps


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
    return (_operators or _load()).tables(block_tables, cached_lens, new_lens, free_blocks, num_free, block_size, total_new)


# ------------------------------------------------------------------------------------------ new keys and values


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
    if ops._validate_offsets:
        _check_slots(slot_mapping, k_cache)
    (_operators or _load()).append(key, value, k_cache, v_cache, k_scales, v_scales, slot_mapping)


def _check_slots(slot_mapping: torch.Tensor, cache: torch.Tensor) -> None:
    """The host's look at a slot map (offset validation): every block's tokens are one run."""
    blocks, size = cache.shape[:2]
    s = slot_mapping.detach().to("cpu")
    held = (s >= 0) & (s < blocks * size)
    begins = held.clone()  # a token that is skipped ends a run, as any other slot than the next does
    begins[1:] &= ~held[:-1] | (s[1:] != s[:-1] + 1) | (s[1:] % size == 0)
    runs = s[begins] // size
    if runs.unique().numel() != runs.numel():
        raise ValueError("slot_mapping must hold the tokens of a block one after the other, with consecutive slots")


# ------------------------------------------------------------------------------------------ attention over the cache


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
    keys (candidates of a request that attend to its history).  A row without keys gives zeros.  Tokens past ``seq_lens[b]``, those past
    the table's width and those of blocks that the table has not (-1) take no part, whatever their memory holds.  Scales are finite, V's not negative (a block whose scale is 0
    holds zeros, and its tokens take part).  ``seq_lens`` and ``query_offset`` are
    trusted like the offsets of the other operators (clamped in the kernel, checked on the host with offset validation on).
    """
    call = _operators or _load()
    if ops._validate_offsets and not torch.compiler.is_compiling():
        _check_lengths(query, k_cache, block_tables, query_offset, seq_lens)
    args = (query, k_cache, v_cache, k_scales, v_scales, block_tables, query_offset, seq_lens, max_seq_len_q,
            1.0 if qk_scale is None else qk_scale, activation_string_to_int(activation), is_causal, -1 if window_size is None else window_size)
    events = ops._timing_events["fwd"]
    if events is None:
        return call.attend(*args)
    call.native.gdpa_torch_set_timing(events[0].cuda_event, events[1].cuda_event)
    try:
        return call.attend(*args)
    finally:
        call.native.gdpa_torch_set_timing(None, None)


def _check_lengths(query, k_cache, block_tables, query_offset, seq_lens) -> None:
    ops._check_offsets("query_offset", query_offset, query.shape[0], False)
    n = seq_lens.detach().to("cpu", torch.int64)
    if n.numel() and (int(n.min()) < 0 or int(n.max()) > block_tables.shape[1] * k_cache.shape[1]):
        raise ValueError("seq_lens has entries outside [0, width of block_tables * block size]")


# ------------------------------------------------------------------------------------------ queries and keys on their way in


def append_rotated_kv_cache_fp8(
    query: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    k_scales: torch.Tensor,
    v_scales: torch.Tensor,
    slot_mapping: torch.Tensor,
    query_offset: torch.Tensor,
    seq_lens: torch.Tensor,
    inv_freq: torch.Tensor,
    positions: Optional[torch.Tensor] = None,
    query_weight: Optional[torch.Tensor] = None,
    key_weight: Optional[torch.Tensor] = None,
    eps: float = 1e-6,
    norm: bool = True,
    interleaved: bool = False,
    sections: Optional[Sequence[int]] = None,
) -> torch.Tensor:
    """:func:`~.rotary.qk_norm_rotary` of a step's queries and keys and :func:`append_kv_cache_fp8` of the rotated keys and the values, in one
    kernel; returns the rotated queries for the attention.

    ``query`` ``[tokens, H, D]``, ``key`` and ``value`` ``[tokens, H_kv, D]`` (bf16 or fp32, strided as slices of one packed projection are).
    ``positions`` (``[tokens]``, or ``[axes, tokens]`` with ``sections``) may be left out: token ``i`` of the ``n`` that request ``b`` has, rows
    ``query_offset[b]:query_offset[b + 1]``, is at ``seq_lens[b] - n + i`` (``seq_lens`` with the new tokens, as :func:`build_block_tables` returns
    it), on every axis.  Rotated keys go from fp32 to e4m3: they are rounded once, where the two operators one after the other round to bf16
    in between.  A query whose token has no slot (-1) is rotated all the same; what holds for the slots holds as in the append.
    """
    if ops._validate_offsets and not torch.compiler.is_compiling():
        _check_slots(slot_mapping, k_cache)
        ops._check_offsets("query_offset", query_offset, query.shape[0], False)
    return (_operators or _load()).append_rotated(
        query, key, value, k_cache, v_cache, k_scales, v_scales, slot_mapping, query_offset, seq_lens, inv_freq, positions, query_weight, key_weight, eps, norm,
        interleaved, () if sections is None else sections)


# ------------------------------------------------------------------------------------------ what the cache holds


def read_kv_cache_fp8(
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    k_scales: torch.Tensor,
    v_scales: torch.Tensor,
    block_tables: torch.Tensor,
    key_offset: torch.Tensor,
    total_tokens: int,
    first_tokens: Optional[torch.Tensor] = None,
    dtype: torch.dtype = torch.bfloat16,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """The cached keys and values of a batch as packed ``[total_tokens, H_kv, D]`` tensors (bf16 or fp32), as the operators that have no paged form
    take them.

    Rows ``key_offset[b]:key_offset[b + 1]`` are request ``b``'s tokens ``first_tokens[b]``, ``first_tokens[b] + 1``, ... (from 0 without
    ``first_tokens``; both int32 or int64).  A value is e4m3 times scale in fp32, rounded once: with scales that the append made (powers of two)
    bf16 holds it exactly.  Tokens past the table's width, those of blocks that the table has not (-1) and rows that no request has are zeros.
    ``key_offset`` is trusted like the offsets of the other operators.
    """
    if ops._validate_offsets and not torch.compiler.is_compiling():
        ops._check_offsets("key_offset", key_offset, total_tokens, False)
    return (_operators or _load()).read(k_cache, v_cache, k_scales, v_scales, block_tables, key_offset, total_tokens, first_tokens, dtype)


def drop_cached_tokens(
    block_tables: torch.Tensor,
    seq_lens: torch.Tensor,
    dropped: torch.Tensor,
    free_blocks: torch.Tensor,
    num_free: torch.Tensor,
    block_size: int,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """The last ``dropped[b]`` tokens of each request leave the cache (drafts that were refused; all of them: the request is done), in one kernel.

    Blocks that none of a request's remaining tokens needs go onto the stack ``free_blocks[:num_free]`` (int32, changed in place), in the order of the
    requests and of their tables; entries that are no block (-1) do not.  ``dropped`` is clamped to what a request has, a negative ``num_free``
    counts as 0.  Returns ``(seq_lens_after, num_free_after)``, int32 ``[B]`` and ``[1]``.  The tables are left as they are: what lies behind
    a request's length is not looked at, and :func:`build_block_tables` writes over it.

    Tokens that stay in a block with dropped ones keep the block's scale.  Where the append of a draft made it grow, they were rescaled then, and the bits of
    theirs that fell below e4m3's smallest normal value do not come back (:func:`append_kv_cache_fp8`).
    """
    return (_operators or _load()).drop(block_tables, seq_lens, dropped, free_blocks, num_free, block_size)


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

    def _append(self, query, key, value, new_lens, rotary):
        """Store new tokens without counting them: the queries (rotated, if they are to be), their offsets, and the lengths and free blocks from then on."""
        slots, query_offset, seq_lens, num_free = build_block_tables(
            self.block_tables, self.seq_lens, new_lens, self.free_blocks, self.num_free, self.block_size, key.shape[0])
        if rotary is None:
            append_kv_cache_fp8(key, value, self.k_cache, self.v_cache, self.k_scales, self.v_scales, slots)
        else:
            query = append_rotated_kv_cache_fp8(query, key, value, self.k_cache, self.v_cache, self.k_scales, self.v_scales, slots, query_offset, seq_lens,
                                                **rotary)
        return query, query_offset, seq_lens, num_free

    def append(self, key: torch.Tensor, value: torch.Tensor, new_lens: torch.Tensor) -> torch.Tensor:
        """Store the keys and values of ``new_lens[b]`` (int32) new tokens of each request; returns their offsets ``[B + 1]``."""
        _, query_offset, seq_lens, num_free = self._append(None, key, value, new_lens, None)
        # not before: keys or values that were refused are not in the cache (the blocks that the tables have for them count as free)
        self.seq_lens, self.num_free = seq_lens, num_free
        return query_offset

    def append_rotated(self, query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, new_lens: torch.Tensor, rotary: dict):
        """As :meth:`append`, with queries and keys normed and rotated on the way (``rotary``: :func:`append_rotated_kv_cache_fp8`'s arguments from
        ``inv_freq`` on); returns ``(queries, offsets)``."""
        query, query_offset, seq_lens, num_free = self._append(query, key, value, new_lens, rotary)
        self.seq_lens, self.num_free = seq_lens, num_free  # not before, as in append
        return query, query_offset

    def read(self, key_offset: torch.Tensor, total_tokens: int, first_tokens: Optional[torch.Tensor] = None, dtype: torch.dtype = torch.bfloat16):
        """:func:`read_kv_cache_fp8` of what the cache holds."""
        return read_kv_cache_fp8(self.k_cache, self.v_cache, self.k_scales, self.v_scales, self.block_tables, key_offset, total_tokens, first_tokens, dtype)

    def drop(self, dropped: torch.Tensor) -> None:
        """Take the last ``dropped[b]`` tokens of each request out of the cache, and their blocks back (:func:`drop_cached_tokens`)."""
        self.seq_lens, self.num_free = drop_cached_tokens(self.block_tables, self.seq_lens, dropped, self.free_blocks, self.num_free, self.block_size)

    def attend(self, query: torch.Tensor, query_offset: torch.Tensor, max_seq_len_q: int, **options) -> torch.Tensor:
        """:func:`generalized_dot_product_attention_paged_fp8` over what the cache holds."""
        return generalized_dot_product_attention_paged_fp8(
            query, self.k_cache, self.v_cache, self.k_scales, self.v_scales, self.block_tables, query_offset, self.seq_lens, max_seq_len_q,
            **options)

    def step(self, query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, new_lens: torch.Tensor, max_seq_len_q: int,
             rotary: Optional[dict] = None, **options) -> torch.Tensor:
        """Append, then attend with the new tokens' queries (causal unless ``is_causal=False`` is given); with ``rotary``, queries and keys are
        normed and rotated first (:meth:`append_rotated`).  A step that is refused, by its append or by its attention, counts no tokens: it can be made again."""
        if query.dtype != torch.bfloat16:  # of all that the attention refuses what an append of fp32 lets through: before anything is stored
            raise TypeError(f"query must be bf16 for a step (the attention's type), got {query.dtype}")
        query, query_offset, seq_lens, num_free = self._append(query, key, value, new_lens, rotary)
        out = generalized_dot_product_attention_paged_fp8(
            query, self.k_cache, self.v_cache, self.k_scales, self.v_scales, self.block_tables, query_offset, seq_lens, max_seq_len_q,
            **{"is_causal": True, **options})
        self.seq_lens, self.num_free = seq_lens, num_free  # not before
        return out

    def release(self, requests: Sequence[int]) -> None:
        """Give back the blocks of these requests (rows of the tables, negative ones from the end), which are empty afterwards."""
        batch = self.block_tables.shape[0]
        asked = [operator.index(r) for r in requests]
        for r in asked:  # on the host: an index out of range would be an assertion on the GPU, whose context is lost with it
            if not -batch <= r < batch:
                raise IndexError(f"request {r} is not one of this cache's {batch}")
        rows = torch.tensor(sorted({r % batch for r in asked}), dtype=torch.int64)
        if self.block_tables.is_cuda:  # from pinned memory: a copy from pageable memory waits for the stream
            rows = rows.pin_memory().to(self.block_tables.device, non_blocking=True)
        table = self.block_tables[rows]
        held = torch.arange(table.shape[1], device=table.device) < ((self.seq_lens[rows] + self.block_size - 1) // self.block_size)[:, None]
        held &= table >= 0
        place = self.num_free.clamp_min(0) + torch.cumsum(held.flatten(), 0) - 1
        # entries that are not held go to a place behind the stack
        stack = torch.cat([self.free_blocks, self.free_blocks.new_zeros(1)])
        stack[torch.where(held.flatten(), place, self.free_blocks.numel())] = table.flatten()
        self.free_blocks = stack[:-1]
        self.num_free = self.num_free.clamp_min(0) + held.sum().to(torch.int32)
        self.block_tables.index_fill_(0, rows, -1)
        self.seq_lens.index_fill_(0, rows, 0)


# The libraries are loaded here if they are built, so that a compiler that traces a first call finds the operators; if that fails, the first call says why.
if os.path.exists(LIB_PATH) and os.path.exists(_cabi.LIB_PATH):
    try:
        _load()
    except OSError:
        pass
