"""Block tables and slot maps built on the GPU from request lengths: what the cache write (slot_mapping) and the
attention (block_tables, seq_lens) of a step take, without a host round trip.

A serving loop keeps `block_tables` [R, width], `seq_lens` [R], a list `free_blocks` [N] of block ids and a one-element
int64 `free_cursor`: entries from the cursor on are free, those below it have been handed out.

    build_block_tables     blocks for the tokens that a step adds, and the slots of those tokens
    build_slot_mapping     the slots alone, through tables that somebody else keeps
    release_block_tables   blocks of finished requests back to the list

Argument violations raise AssertionError, as in the other operators; nothing synchronises, and every call can be
captured in a CUDA graph.  The reference builds both on the host (tests/test_int8_paged_attention.py:16-43).
"""

from __future__ import annotations

import contextlib
from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib
from .ops import _require_lib, _stream_ptr

_INDEX = (torch.int32, torch.int64)


class BlockTableStep(NamedTuple):
    """What build_block_tables returns."""

    slot_mapping: torch.Tensor  # [num_tokens] int64, -1 = no slot
    query_start: torch.Tensor  # [R + 1] int32, exclusive prefix sums of new_lens
    seq_lens: torch.Tensor  # [R], lengths after the step
    free_cursor: torch.Tensor  # [1] int64


def _on_device(device: torch.device):
    """The launch context of `device`: a no-op when it is the current one already."""
    if device.index is None or device.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(device)


def _check_lists(device, block_tables, seq_lens, block_size, written):
    assert block_tables.is_cuda and block_tables.ndim == 2 and block_tables.dtype in _INDEX
    assert seq_lens.ndim == 1 and seq_lens.dtype in _INDEX and seq_lens.device == device
    assert seq_lens.numel() == block_tables.shape[0]
    assert int(block_size) > 0
    if written:  # an expanded table has one memory cell for several entries
        assert all(st != 0 or n <= 1 for st, n in zip(block_tables.stride(), block_tables.shape))


def _check_free_list(device, free_blocks, free_cursor):
    assert free_blocks.ndim == 1 and free_blocks.dtype in _INDEX and free_blocks.device == device
    assert free_cursor.numel() == 1 and free_cursor.dtype == torch.int64 and free_cursor.device == device


def _check_out(out, like, shape, dtype):
    assert out.shape == shape and out.dtype == dtype and out.device == like.device and out.is_contiguous()


def _workspace(lib, requests: int, items: int, device) -> Tuple[Optional[torch.Tensor], int, int]:
    """(tensor, address, bytes) of a call's workspace.  It belongs to the call: a captured call gets memory of its
    graph's own pool, so two graphs never share it."""
    nbytes = lib.int8kv_block_tables_workspace_bytes(requests, items)
    if nbytes <= 0:
        return None, 0, 0
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
    return ws, ws.data_ptr(), nbytes


def build_block_tables(
    block_tables: torch.Tensor,
    seq_lens: torch.Tensor,
    new_lens: torch.Tensor,
    free_blocks: torch.Tensor,
    free_cursor: torch.Tensor,
    block_size: int,
    *,
    num_tokens: int,
    out: Optional[BlockTableStep] = None,
) -> BlockTableStep:
    """Make room for new_lens[b] more tokens behind the seq_lens[b] tokens that request b holds: extend the rows of
    `block_tables` (in place) with blocks from `free_blocks`, in request order, and return the new tokens' slots.

    num_tokens: length of the slot mapping, at least the sum of new_lens (a captured step passes its padded size);
    tokens are packed in request order, the rest is -1.  A request that does not fit its table row, or that needs
    blocks when the list has not enough left, is refused: no blocks, the old length, slots -1.
    out: preallocated outputs; its seq_lens and free_cursor may be the inputs themselves, which then advance in place.
    """
    device = block_tables.device
    _check_lists(device, block_tables, seq_lens, block_size, True)
    _check_free_list(device, free_blocks, free_cursor)
    R, width = block_tables.shape
    num_tokens = int(num_tokens)
    assert new_lens.ndim == 1 and new_lens.numel() == R and new_lens.dtype in _INDEX and new_lens.device == device
    assert 0 <= num_tokens < 2**31 - 1
    if out is None:
        out = BlockTableStep(torch.empty(num_tokens, dtype=torch.int64, device=device),
                             torch.empty(R + 1, dtype=torch.int32, device=device),
                             torch.empty(R, dtype=seq_lens.dtype, device=device),
                             torch.empty(1, dtype=torch.int64, device=device))
    else:
        _check_out(out.slot_mapping, block_tables, (num_tokens,), torch.int64)
        _check_out(out.query_start, block_tables, (R + 1,), torch.int32)
        _check_out(out.seq_lens, block_tables, (R,), seq_lens.dtype)
        _check_out(out.free_cursor, block_tables, (1,), torch.int64)
    lib = _require_lib()
    seq_lens, new_lens, free_blocks = seq_lens.contiguous(), new_lens.contiguous(), free_blocks.contiguous()
    ws, ws_ptr, ws_bytes = _workspace(lib, R, num_tokens + num_tokens // int(block_size) + R, device)
    with _on_device(device):
        rc = lib.int8kv_build_block_tables(
            seq_lens.data_ptr(), int(seq_lens.dtype == torch.int64),
            new_lens.data_ptr(), int(new_lens.dtype == torch.int64), R, int(block_size),
            block_tables.data_ptr(), int(block_tables.dtype == torch.int64), _lib.i64(block_tables.stride()), width,
            free_blocks.data_ptr(), int(free_blocks.dtype == torch.int64), free_blocks.numel(),
            free_cursor.data_ptr(), out.free_cursor.data_ptr(), out.seq_lens.data_ptr(),
            out.slot_mapping.data_ptr(), num_tokens, out.query_start.data_ptr(),
            ws_ptr, ws_bytes, _stream_ptr(device),
        )
    _lib.check("int8kv_build_block_tables", rc)
    return out


def build_slot_mapping(
    block_tables: torch.Tensor,
    seq_lens: torch.Tensor,
    new_lens: torch.Tensor,
    block_size: int,
    *,
    num_tokens: int,
    out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """(slot_mapping [num_tokens] int64, query_start [R + 1] int32) of new_lens[b] tokens that follow the seq_lens[b]
    cached ones of request b, through tables that hold their blocks already.  Packing and padding as in
    build_block_tables; a token beyond its table row, or on a negative block id, gets slot -1."""
    device = block_tables.device
    _check_lists(device, block_tables, seq_lens, block_size, False)
    R, width = block_tables.shape
    num_tokens = int(num_tokens)
    assert new_lens.ndim == 1 and new_lens.numel() == R and new_lens.dtype in _INDEX and new_lens.device == device
    assert 0 <= num_tokens < 2**31 - 1
    if out is None:
        out = (torch.empty(num_tokens, dtype=torch.int64, device=device),
               torch.empty(R + 1, dtype=torch.int32, device=device))
    else:
        _check_out(out[0], block_tables, (num_tokens,), torch.int64)
        _check_out(out[1], block_tables, (R + 1,), torch.int32)
    lib = _require_lib()
    seq_lens, new_lens = seq_lens.contiguous(), new_lens.contiguous()
    ws, ws_ptr, ws_bytes = _workspace(lib, R, num_tokens, device)
    with _on_device(device):
        rc = lib.int8kv_build_slot_mapping(
            seq_lens.data_ptr(), int(seq_lens.dtype == torch.int64),
            new_lens.data_ptr(), int(new_lens.dtype == torch.int64), R, int(block_size),
            block_tables.data_ptr(), int(block_tables.dtype == torch.int64), _lib.i64(block_tables.stride()), width,
            out[0].data_ptr(), num_tokens, out[1].data_ptr(), ws_ptr, ws_bytes, _stream_ptr(device),
        )
    _lib.check("int8kv_build_slot_mapping", rc)
    return out


def release_block_tables(
    block_tables: torch.Tensor,
    seq_lens: torch.Tensor,
    finished: torch.Tensor,
    free_blocks: torch.Tensor,
    free_cursor: torch.Tensor,
    block_size: int,
    *,
    out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """Give the blocks of the requests with finished[b] (bool [R]) back: they are written to `free_blocks` (in place)
    just below the cursor, in request order.  Returns (seq_lens with 0 for the finished ones, free_cursor); out:
    preallocated outputs, which may be the inputs themselves.  The table is not written.  Every block of a list is
    handed out once, so requests that share blocks must not both be released."""
    device = block_tables.device
    _check_lists(device, block_tables, seq_lens, block_size, False)
    _check_free_list(device, free_blocks, free_cursor)
    R, width = block_tables.shape
    assert finished.ndim == 1 and finished.numel() == R and finished.dtype == torch.bool and finished.device == device
    assert free_blocks.is_contiguous()
    if out is None:
        out = (torch.empty(R, dtype=seq_lens.dtype, device=device), torch.empty(1, dtype=torch.int64, device=device))
    else:
        _check_out(out[0], block_tables, (R,), seq_lens.dtype)
        _check_out(out[1], block_tables, (1,), torch.int64)
    lib = _require_lib()
    seq_lens, finished = seq_lens.contiguous(), finished.contiguous()
    ws, ws_ptr, ws_bytes = _workspace(lib, R, min(R * width, free_blocks.numel()), device)
    with _on_device(device):
        rc = lib.int8kv_release_block_tables(
            seq_lens.data_ptr(), int(seq_lens.dtype == torch.int64), finished.data_ptr(), R, int(block_size),
            block_tables.data_ptr(), int(block_tables.dtype == torch.int64), _lib.i64(block_tables.stride()), width,
            free_blocks.data_ptr(), int(free_blocks.dtype == torch.int64), free_blocks.numel(),
            free_cursor.data_ptr(), out[1].data_ptr(), out[0].data_ptr(), ws_ptr, ws_bytes, _stream_ptr(device),
        )
    _lib.check("int8kv_release_block_tables", rc)
    return out
