"""Block tables and slot maps without a GPU: the oracle against the package's host-side builders, the refusals of
the Python entry points, and the argument checks of the C ABI."""

import pytest
import torch

from conftest import package
from oracle import block_tables as oracle_tables


def test_oracle_agrees_with_the_host_side_builders(workloads):
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
    p = 256  # never dereferenced: every call below is refused

    def call(fn, R=2, bs=16, width=4, free=8, tokens=4, lens=p, new=p, done=p, bt=p, cursor=p, start=p, slots=p, fb=p, lens_out=p,
             ws=0, ws_bytes=0):
        return fn(lm.TABLE_ARGS.pack(lens, new, done, bt, fb, cursor, cursor, lens_out, slots, start, ws, 0,
                                     0, 0, 0, 0, R, bs, 4, 1, width, free, tokens, ws_bytes))

    build, slot, release = lib.int8kv_build_block_tables, lib.int8kv_build_slot_mapping, lib.int8kv_release_block_tables
    for fn in (build, slot, release):
        assert fn(None) == lm.E_NULLPTR
        assert call(fn, R=-1) == lm.E_BAD_SHAPE and call(fn, R=2**31) == lm.E_BAD_SHAPE
        assert call(fn, bs=0) == lm.E_BAD_SHAPE and call(fn, bs=2**32 + 16) == lm.E_BAD_SHAPE
        assert call(fn, width=-1) == lm.E_BAD_SHAPE and call(fn, width=2**31) == lm.E_BAD_SHAPE
        assert call(fn, lens=0) == lm.E_NULLPTR and call(fn, bt=0) == lm.E_NULLPTR
    for fn in (build, slot):
        assert call(fn, tokens=-1) == lm.E_BAD_SHAPE and call(fn, tokens=2**31) == lm.E_BAD_SHAPE
        assert call(fn, start=0) == lm.E_NULLPTR and call(fn, slots=0) == lm.E_NULLPTR and call(fn, new=0) == lm.E_NULLPTR
    for fn in (build, release):
        assert call(fn, free=-1) == lm.E_BAD_SHAPE and call(fn, cursor=0) == lm.E_NULLPTR
        assert call(fn, fb=0) == lm.E_NULLPTR and call(fn, lens_out=0) == lm.E_NULLPTR
    assert call(release, done=0) == lm.E_NULLPTR
    big = 1 << 20
    need = lib.int8kv_block_tables_workspace_bytes(2, big + big // 16 + 2, 1)
    assert need > 0 and call(build, tokens=big) == lm.E_WORKSPACE  # in place: lens_out is lens
    assert call(build, tokens=big, ws=p, ws_bytes=need - 1) == lm.E_WORKSPACE
    assert call(build, tokens=big, ws=264, ws_bytes=need) == lm.E_WORKSPACE
    assert lib.int8kv_block_tables_workspace_bytes(64, 128, 1) == 0  # small: one kernel
    assert lib.int8kv_block_tables_workspace_bytes(64, 1 << 20, 0) == 0  # outputs of its own: one kernel of many CTAs
    assert lib.int8kv_block_tables_workspace_bytes(5000, 128, 0) > 0
    assert lib.int8kv_block_tables_workspace_bytes(-1, 128, 0) == -1


def test_argument_records_have_the_size_of_the_structs(tmp_path):
    """The flat records that the binding packs are the structs of the header."""
    import shutil
    import subprocess

    from conftest import REPO

    lm = package("_lib")
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("no C compiler")
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "int8kv_b200.h"\nint main(void) {\n'
                   'printf("%zu %zu %zu %zu %zu\\n", sizeof(int8kv_diff_args), sizeof(int8kv_table_args),'
                   ' offsetof(int8kv_diff_args, lam_stride), offsetof(int8kv_diff_args, norm_eps),'
                   ' offsetof(int8kv_table_args, num_requests)); return 0; }\n')
    subprocess.run([gcc, "-I", str(REPO / "include"), str(src), "-o", str(tmp_path / "sizes")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "sizes")], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [lm.DIFF_ARGS.size, lm.TABLE_ARGS.size, 8 * 29, 8 * 47, 8 * 16]
