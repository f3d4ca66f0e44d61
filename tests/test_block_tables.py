"""Block tables and slot maps without a GPU: the checker against the package's host-side builders, the refusals of
the Python entry points, and the argument checks of the C ABI."""

import ctypes as C

import pytest
import torch

from conftest import package
from oracle import block_tables as oracle_tables


def test_checker_agrees_with_the_host_side_builders(workloads):
    """Tables grown from nothing out of a permuted pool are the tables and slots that the workloads build on the host."""
    lens = [17, 1, 0, 64, 33]
    need = workloads.blocks_needed(lens, 16)
    pool = torch.randperm(20, generator=torch.Generator().manual_seed(3 * 31337 + 3)).to(torch.int32)
    table, slots, start, seq, cursor = oracle_tables.build_block_tables(
        torch.zeros(5, 4, dtype=torch.int32), torch.zeros(5, dtype=torch.int32), torch.tensor(lens), pool, 0, 16, 115)
    want = workloads.permuted_block_tables(lens, 16, 20, seed=3)
    assert torch.equal(table, want) and cursor == int(need.sum()) and seq.tolist() == lens
    assert torch.equal(slots, workloads.slot_mapping_for(want, lens, 16))
    assert start.tolist() == [0, 17, 18, 18, 82, 115]
    free, seq, cursor = oracle_tables.release_block_tables(table, seq, torch.tensor([True] * 5), torch.zeros_like(pool),
                                                           cursor, 16)
    assert cursor == 0 and seq.tolist() == [0] * 5 and torch.equal(free[: int(need.sum())], pool[: int(need.sum())])


def test_entry_points_refuse_host_tensors_and_bad_shapes(kv):
    bt = torch.zeros(2, 4, dtype=torch.int32)
    lens, one = torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int64)
    with pytest.raises(AssertionError):
        kv.build_block_tables(bt, lens, lens, torch.zeros(4, dtype=torch.int32), one, 16, num_tokens=4)
    with pytest.raises(AssertionError):
        kv.build_slot_mapping(bt, lens, lens, 16, num_tokens=4)
    with pytest.raises(AssertionError):
        kv.release_block_tables(bt, lens, torch.zeros(2, dtype=torch.bool), torch.zeros(4, dtype=torch.int32), one, 16)


def test_c_abi_argument_checks():
    """Null pointers, sizes out of range and a missing workspace are refused before anything is launched."""
    lm = package("_lib")
    lib = lm.load()
    st = lm.i64((4, 1))
    p = C.c_void_p(256)  # never dereferenced: every call below is refused

    def build(R=2, bs=16, width=4, free=8, tokens=4, lens=p, lens_out=p, bt=p, cursor=p, start=p, slots=p, ws=None, ws_bytes=0):
        return lib.int8kv_build_block_tables(lens, 0, p, 0, R, bs, bt, 0, st, width, p, 0, free, cursor, cursor, lens_out,
                                             slots, tokens, start, ws, ws_bytes, None)

    assert build(R=-1) == lm.E_BAD_SHAPE and build(bs=0) == lm.E_BAD_SHAPE and build(width=-1) == lm.E_BAD_SHAPE
    assert build(tokens=-1) == lm.E_BAD_SHAPE and build(tokens=2**31) == lm.E_BAD_SHAPE
    assert build(free=-1) == lm.E_BAD_SHAPE and build(width=2**31) == lm.E_BAD_SHAPE
    assert build(lens=None) == lm.E_NULLPTR and build(bt=None) == lm.E_NULLPTR and build(cursor=None) == lm.E_NULLPTR
    assert build(start=None) == lm.E_NULLPTR and build(slots=None) == lm.E_NULLPTR
    big = 1 << 20
    need = lib.int8kv_block_tables_workspace_bytes(2, big + big // 16 + 2, 1)
    assert need > 0 and build(tokens=big) == lm.E_WORKSPACE
    assert build(tokens=big, ws=p, ws_bytes=need - 1) == lm.E_WORKSPACE
    assert build(tokens=big, ws=C.c_void_p(264), ws_bytes=need) == lm.E_WORKSPACE
    assert lib.int8kv_block_tables_workspace_bytes(64, 128, 1) == 0  # small: one kernel
    assert lib.int8kv_block_tables_workspace_bytes(64, 1 << 20, 0) == 0  # outputs of its own: one kernel of many CTAs
    assert lib.int8kv_block_tables_workspace_bytes(5000, 128, 0) > 0
    assert lib.int8kv_block_tables_workspace_bytes(-1, 128, 0) == -1
    assert lib.int8kv_build_slot_mapping(p, 0, None, 0, 2, 16, p, 0, st, 4, p, 4, p, None, 0, None) == lm.E_NULLPTR
    assert lib.int8kv_build_slot_mapping(p, 0, p, 0, 2, 0, p, 0, st, 4, p, 4, p, None, 0, None) == lm.E_BAD_SHAPE
    assert lib.int8kv_release_block_tables(p, 0, None, 2, 16, p, 0, st, 4, p, 0, 8, p, p, p, None, 0, None) == lm.E_NULLPTR
    assert lib.int8kv_release_block_tables(p, 0, p, 2, 16, p, 0, st, 4, None, 0, 8, p, p, p, None, 0, None) == lm.E_NULLPTR
