"""Block tables, positions and cache slots of a batch, built on the GPU (sm_100a, libkvbm_cuda.so).

A slot is ``block * page + offset``, the address the cache-writing kernels take; -1 is a token that
has no block and is not written.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib

MAX_BATCH = 8192  # requests a call of batch_tables takes (kMaxBatch of batch_tables.cu)


class BatchTables(NamedTuple):
    block_table: torch.Tensor  # int32 [B, max_blocks], or the caller's table
    seq_lens: torch.Tensor     # int32 [B]: context + query
    cu_query: torch.Tensor     # int32 [B + 1]: where each request's tokens begin
    positions: torch.Tensor    # int32 [num_tokens]
    slots: torch.Tensor        # int64 [num_tokens]


def _check(t: torch.Tensor, name: str, dtype: torch.dtype, n: int | None = None, device=None) -> None:
    if t.dtype != dtype or t.dim() != 1 or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous 1-D {dtype} tensor")
    if n is not None and t.numel() != n:
        raise ValueError(f"{name} has {t.numel()} entries, expected {n}")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")


def _check_table(t: torch.Tensor, device) -> None:
    if t.device != device or t.dtype != torch.int32 or t.dim() != 2 or (t.shape[1] > 1 and t.stride(1) != 1):
        raise ValueError("a block table must be int32 [rows, max_blocks] with unit inner stride, on the same device")


def batch_tables(query_lens: torch.Tensor, context_lens: torch.Tensor, block_ids: torch.Tensor, *, page: int,
                 max_blocks: int | None = None, num_tokens: int = 0, block_counts: torch.Tensor | None = None,
                 table: torch.Tensor | None = None, rows: torch.Tensor | None = None, pad_block: int = 0,
                 stream=None) -> BatchTables:
    """Tables of requests that bring ``query_lens`` new tokens behind ``context_lens`` cached ones, in one launch.

    All lengths are int32 [B] on the GPU (negative ones count as 0; B up to 8,192). ``block_ids`` (int32, flat)
    lists the requests' blocks one request after another: ``block_counts[b]`` of them each, or as many as its
    tokens need. ``num_tokens`` is the token capacity of ``positions`` and ``slots``: tokens behind the last
    request's get position 0 and slot -1 (a padded batch), tokens beyond the capacity are left out. A token
    whose block is missing, negative or beyond ``max_blocks`` gets slot -1.

    The table is new ([B, max_blocks], ``pad_block`` behind each request's blocks) or ``table``, a persistent one
    (``max_blocks`` is its width): request b's blocks then go to row ``rows[b]`` (int32 [B], distinct; b itself
    without ``rows``), rows outside the table are skipped and rows not named are left as they were.
    """
    dev, B = query_lens.device, query_lens.numel()
    _check(query_lens, "query_lens", torch.int32)
    _check(context_lens, "context_lens", torch.int32, B, dev)
    _check(block_ids, "block_ids", torch.int32, None, dev)
    if block_counts is not None:
        _check(block_counts, "block_counts", torch.int32, B, dev)
    if page <= 0 or num_tokens < 0:
        raise ValueError("page must be positive and num_tokens not negative")
    if B > MAX_BATCH:
        raise ValueError(f"batch_tables takes at most {MAX_BATCH} requests, got {B}")
    if table is None:
        if max_blocks is None or max_blocks < 0 or rows is not None:
            raise ValueError("without a table, max_blocks is required and rows has no meaning")
    else:
        _check_table(table, dev)
        if max_blocks is not None and max_blocks != table.shape[1]:
            raise ValueError(f"max_blocks {max_blocks} differs from the table's {table.shape[1]}")
        max_blocks = table.shape[1]
        if rows is not None:
            _check(rows, "rows", torch.int32, B, dev)
        elif table.shape[0] < B:
            raise ValueError(f"the table has {table.shape[0]} rows for {B} requests")
    with _lib.on_device(dev, stream) as st:
        if table is None:
            table = query_lens.new_empty((B, max_blocks))
        seq_lens, cu_query, positions = query_lens.new_empty(2 * B + 1 + num_tokens).split_with_sizes(
            (B, B + 1, num_tokens))
        slots = query_lens.new_empty(num_tokens, dtype=torch.int64)
        _lib.call("kvbm_batch_tables", query_lens.data_ptr(), context_lens.data_ptr(),
                  block_counts.data_ptr() if block_counts is not None else None, block_ids.data_ptr(),
                  block_ids.numel(), B, page, max_blocks, pad_block, table.data_ptr() or None, table.stride(0),
                  rows.data_ptr() if rows is not None else None, table.shape[0], seq_lens.data_ptr(),
                  cu_query.data_ptr(), positions.data_ptr(), slots.data_ptr(), num_tokens, st)
    return BatchTables(table, seq_lens, cu_query, positions, slots)


def slot_map(block_table: torch.Tensor, positions: torch.Tensor, *, page: int, out: torch.Tensor | None = None,
             stream=None) -> torch.Tensor:
    """Slots (int64 [T]) of tokens at ``positions`` (int32 [T]) from an existing table (int32).

    ``block_table`` [T, max_blocks]: token t looks in row t (a decode step); 1-D [max_blocks]: one row for all
    tokens (one request's prefill). A negative position, one beyond the table and a negative block give -1.
    """
    _check(positions, "positions", torch.int32)
    dev, T = positions.device, positions.numel()
    one = block_table.dim() == 1
    if one:
        block_table = block_table.unsqueeze(0)
    _check_table(block_table, dev)
    if not one and block_table.shape[0] != T:
        raise ValueError(f"block_table has {block_table.shape[0]} rows for {T} tokens")
    if page <= 0:
        raise ValueError("page must be positive")
    if out is not None:
        _check(out, "out", torch.int64, T, dev)
    with _lib.on_device(dev, stream) as st:
        if out is None:
            out = positions.new_empty(T, dtype=torch.int64)
        _lib.call("kvbm_slot_map", block_table.data_ptr() or None, 0 if one else block_table.stride(0),
                  block_table.shape[1], positions.data_ptr(), T, page, out.data_ptr(), st)
    return out
