"""Block tables and slot maps, request by request in Python integers: the oracle of the device operators."""

from __future__ import annotations

from typing import List, Sequence, Tuple

import torch


def _ceil(a: int, b: int) -> int:
    return -(-a // b)


def _slots(row: List[int], cached: int, new: int, block_size: int) -> List[int]:
    """Slots of tokens cached .. cached + new - 1 through one row; -1 beyond the row and on negative ids."""
    out = []
    for pos in range(cached, cached + new):
        j = pos // block_size
        blk = row[j] if j < len(row) else -1
        out.append(blk * block_size + pos % block_size if blk >= 0 else -1)
    return out


def _packed(per_request: Sequence[List[int]], num_tokens: int) -> Tuple[torch.Tensor, torch.Tensor]:
    starts = [0]
    for s in per_request:
        starts.append(starts[-1] + len(s))
    flat = [x for s in per_request for x in s][:num_tokens]
    flat += [-1] * (num_tokens - len(flat))
    return torch.tensor(flat, dtype=torch.int64), torch.tensor(starts, dtype=torch.int32)


def build_block_tables(block_tables, seq_lens, new_lens, free_blocks, free_cursor, block_size, num_tokens):
    """(block_tables, slot_mapping, query_start, seq_lens, free_cursor) after the step; the inputs are not changed."""
    rows = [list(map(int, r)) for r in block_tables.tolist()]
    free = list(map(int, free_blocks.tolist()))
    cursor = max(0, int(free_cursor))
    width = block_tables.shape[1]
    lens_out, slots, exhausted = [], [], False
    for b, (c, n) in enumerate(zip(seq_lens.tolist(), new_lens.tolist())):
        c, n = max(0, int(c)), max(0, int(n))
        have = _ceil(c, block_size)
        granted = c + n <= width * block_size
        if granted:
            need = _ceil(c + n, block_size) - have
            if need and (exhausted or cursor + need > len(free)):
                granted, exhausted = False, True
            else:
                for j in range(need):
                    rows[b][have + j] = free[cursor + j]
                cursor += need
        lens_out.append(c + n if granted else c)
        slots.append(_slots(rows[b], c, n, block_size) if granted else [-1] * n)
    table = torch.tensor(rows, dtype=block_tables.dtype).reshape(block_tables.shape)
    slot_mapping, query_start = _packed(slots, num_tokens)
    return table, slot_mapping, query_start, torch.tensor(lens_out, dtype=seq_lens.dtype), cursor


def build_slot_mapping(block_tables, seq_lens, new_lens, block_size, num_tokens):
    rows = [list(map(int, r)) for r in block_tables.tolist()]
    return _packed([_slots(row, max(0, int(c)), max(0, int(n)), block_size)
                    for row, c, n in zip(rows, seq_lens.tolist(), new_lens.tolist())], num_tokens)


def release_block_tables(block_tables, seq_lens, finished, free_blocks, free_cursor, block_size):
    """(free_blocks, seq_lens, free_cursor) after the release."""
    free = free_blocks.clone()
    width = block_tables.shape[1]
    back = []
    for b, (n, done) in enumerate(zip(seq_lens.tolist(), finished.tolist())):
        if done:
            n = min(max(0, int(n)), width * block_size)
            back += block_tables[b, : _ceil(n, block_size)].tolist()
    base = min(int(free_cursor), free.numel()) - len(back)
    for k, blk in enumerate(back):
        if base + k >= 0:
            free[base + k] = blk
    lens = torch.where(finished, torch.zeros_like(seq_lens), seq_lens)
    return free, lens, max(base, 0)
