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

from functools import lru_cache
from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib
from .ops import _call, _require_lib, _stream_ptr

_INDEX_CODES = {torch.int32: 0, torch.int64: 1}
_MAX_TOKENS = 2**31 - 1


class BlockTableStep(NamedTuple):
    """What build_block_tables returns."""

    slot_mapping: torch.Tensor  # [num_tokens] int64, -1 = no slot
    query_start: torch.Tensor  # [R + 1] int32, exclusive prefix sums of new_lens
    seq_lens: torch.Tensor  # [R], lengths after the step
    free_cursor: torch.Tensor  # [1] int64


def _check_lists(block_tables, seq_lens, block_size):
    """(device, requests, width, index code of the table, of the lengths)"""
    device = block_tables.device
    assert device.type == "cuda" and block_tables.ndim == 2 and seq_lens.ndim == 1 and seq_lens.device == device
    requests, width = block_tables.shape
    bt_code, sl_code = _INDEX_CODES.get(block_tables.dtype), _INDEX_CODES.get(seq_lens.dtype)
    assert bt_code is not None and sl_code is not None and seq_lens.shape[0] == requests
    assert 0 < block_size < 2**31  # the library takes it as a C int
    return device, requests, width, bt_code, sl_code


def _check_free_list(device, free_blocks, free_cursor):
    code = _INDEX_CODES.get(free_blocks.dtype)
    assert free_blocks.ndim == 1 and code is not None and free_blocks.device == device
    assert free_cursor.numel() == 1 and free_cursor.dtype == torch.int64 and free_cursor.device == device
    return code


def _check_out(out, device, shape, dtype):
    assert out.shape == shape and out.dtype == dtype and out.device == device and out.is_contiguous()


@lru_cache(maxsize=1024)
def _workspace_bytes(requests: int, items: int, in_place: bool) -> int:
    return _require_lib().int8kv_block_tables_workspace_bytes(requests, items, in_place)


def _workspace(requests: int, items: int, in_place: bool, device) -> Tuple[Optional[torch.Tensor], int, int]:
    """(tensor, address, bytes) of a call's workspace.  It belongs to the call: a captured call gets memory of its
    graph's own pool, so two graphs never share it."""
    nbytes = _workspace_bytes(requests, items, in_place)
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
    device, R, width, bt_code, sl_code = _check_lists(block_tables, seq_lens, block_size)
    bt_st = block_tables.stride()  # an expanded table has one memory cell for several entries
    assert (bt_st[0] != 0 or R <= 1) and (bt_st[1] != 0 or width <= 1)
    fb_code, nl_code = _check_free_list(device, free_blocks, free_cursor), _INDEX_CODES.get(new_lens.dtype)
    assert new_lens.shape == seq_lens.shape and nl_code is not None and new_lens.device == device
    assert 0 <= num_tokens < _MAX_TOKENS
    if out is None:
        out = BlockTableStep(torch.empty(num_tokens, dtype=torch.int64, device=device),
                             torch.empty(R + 1, dtype=torch.int32, device=device),
                             seq_lens.new_empty(R), free_cursor.new_empty(1))
    else:
        _check_out(out.slot_mapping, device, (num_tokens,), torch.int64)
        _check_out(out.query_start, device, (R + 1,), torch.int32)
        _check_out(out.seq_lens, device, (R,), seq_lens.dtype)
        _check_out(out.free_cursor, device, (1,), torch.int64)
    lib = _require_lib()
    seq_lens, new_lens, free_blocks = seq_lens.contiguous(), new_lens.contiguous(), free_blocks.contiguous()
    lens_ptr, new_ptr, lens_out = seq_lens.data_ptr(), new_lens.data_ptr(), out.seq_lens.data_ptr()
    cursor_ptr, cursor_out = free_cursor.data_ptr(), out.free_cursor.data_ptr()
    in_place = lens_out == lens_ptr or lens_out == new_ptr or cursor_ptr == cursor_out
    ws, ws_ptr, ws_bytes = _workspace(R, num_tokens + num_tokens // block_size + R, in_place, device)
    rc = _call(device, lib.int8kv_build_block_tables, _lib.TABLE_ARGS.pack(
        lens_ptr, new_ptr, 0, block_tables.data_ptr(), free_blocks.data_ptr(), cursor_ptr, cursor_out, lens_out,
        out.slot_mapping.data_ptr(), out.query_start.data_ptr(), ws_ptr, _stream_ptr(device),
        sl_code, nl_code, bt_code, fb_code, R, block_size, *bt_st, width, free_blocks.shape[0], num_tokens, ws_bytes))
    if rc != _lib.OK:
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
    device, R, width, bt_code, sl_code = _check_lists(block_tables, seq_lens, block_size)
    nl_code = _INDEX_CODES.get(new_lens.dtype)
    assert new_lens.shape == seq_lens.shape and nl_code is not None and new_lens.device == device
    assert 0 <= num_tokens < _MAX_TOKENS
    if out is None:
        out = (torch.empty(num_tokens, dtype=torch.int64, device=device),
               torch.empty(R + 1, dtype=torch.int32, device=device))
    else:
        _check_out(out[0], device, (num_tokens,), torch.int64)
        _check_out(out[1], device, (R + 1,), torch.int32)
    lib = _require_lib()
    seq_lens, new_lens = seq_lens.contiguous(), new_lens.contiguous()
    ws, ws_ptr, ws_bytes = _workspace(R, num_tokens, False, device)
    rc = _call(device, lib.int8kv_build_slot_mapping, _lib.TABLE_ARGS.pack(
        seq_lens.data_ptr(), new_lens.data_ptr(), 0, block_tables.data_ptr(), 0, 0, 0, 0,
        out[0].data_ptr(), out[1].data_ptr(), ws_ptr, _stream_ptr(device),
        sl_code, nl_code, bt_code, 0, R, block_size, *block_tables.stride(), width, 0, num_tokens, ws_bytes))
    if rc != _lib.OK:
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
    device, R, width, bt_code, sl_code = _check_lists(block_tables, seq_lens, block_size)
    fb_code = _check_free_list(device, free_blocks, free_cursor)
    assert finished.shape == seq_lens.shape and finished.dtype == torch.bool and finished.device == device
    assert free_blocks.is_contiguous()
    if out is None:
        out = (seq_lens.new_empty(R), free_cursor.new_empty(1))
    else:
        _check_out(out[0], device, (R,), seq_lens.dtype)
        _check_out(out[1], device, (1,), torch.int64)
    lib = _require_lib()
    seq_lens, finished = seq_lens.contiguous(), finished.contiguous()
    N = free_blocks.shape[0]
    lens_ptr, lens_out, cursor_ptr, cursor_out = (
        seq_lens.data_ptr(), out[0].data_ptr(), free_cursor.data_ptr(), out[1].data_ptr())
    ws, ws_ptr, ws_bytes = _workspace(R, min(R * width, N), lens_ptr == lens_out or cursor_ptr == cursor_out, device)
    rc = _call(device, lib.int8kv_release_block_tables, _lib.TABLE_ARGS.pack(
        lens_ptr, 0, finished.data_ptr(), block_tables.data_ptr(), free_blocks.data_ptr(), cursor_ptr, cursor_out, lens_out,
        0, 0, ws_ptr, _stream_ptr(device),
        sl_code, 0, bt_code, fb_code, R, block_size, *block_tables.stride(), width, N, 0, ws_bytes))
    if rc != _lib.OK:
        _lib.check("int8kv_release_block_tables", rc)
    return out
