"""Block tables and slot maps on the GPU against the request-by-request oracle: every value is an integer and has
to be equal."""

import random

import pytest
import torch

from oracle import block_tables as oracle_tables

pytestmark = pytest.mark.gpu
DEV = "cuda"


def make_state(seed, requests, width, block_size, lo, hi, new_hi, spare, index=torch.int32, lens_type=torch.int32):
    """Rows holding `lo`..`hi` tokens each out of a permuted pool, and what a step asks for."""
    r = random.Random(seed)
    cached = [r.randint(lo, hi) for _ in range(requests)]
    new = [r.choice([0, 1, 1, r.randint(0, new_hi)]) for _ in range(requests)]
    need = [-(-c // block_size) for c in cached]
    used = sum(need)
    grow = sum(-(-(c + n) // block_size) - -(-c // block_size) for c, n in zip(cached, new)
               if c + n <= width * block_size)
    pool = torch.randperm(max(0, used + grow + spare), generator=torch.Generator().manual_seed(seed)).to(index)
    table = torch.full((requests, width), -7, dtype=index)
    at = 0
    for b, k in enumerate(need):
        table[b, :k] = pool[at:at + k]
        at += k
    return (table, torch.tensor(cached, dtype=lens_type), torch.tensor(new, dtype=lens_type), pool,
            torch.tensor([used], dtype=torch.int64))


CASES = [  # requests, width, block size, lo, hi, new_hi, spare
    (1, 4, 16, 0, 0, 1, 0),
    (1, 1, 1, 0, 0, 1, 5),
    (3, 9, 16, 0, 140, 3, 0),
    (64, 40, 16, 1, 600, 30, 0),
    (255, 17, 7, 0, 100, 15, 2),
    (256, 33, 16, 0, 500, 1, -3),      # the list runs out
    (300, 25, 1, 0, 20, 4, -20),       # a block per token, a few tokens each, the list runs out
    (1000, 9, 16, 0, 143, 4, 0),       # a few tokens each, some beyond their row
    (1, 600, 16, 0, 0, 9000, 3),       # one prompt
    (3, 300, 64, 100, 9000, 9000, 0),
    (257, 12, 32, 0, 384, 200, 0),     # rows that some requests do not fit
    (1025, 20, 24, 0, 400, 80, -40),   # more requests than threads, the list runs out, the two-kernel form
    (2049, 6, 16, 0, 80, 2, 1),        # more requests than the one-kernel form takes
]


@pytest.mark.parametrize("case", CASES, ids=str)
@pytest.mark.parametrize("types", [(torch.int32, torch.int32), (torch.int64, torch.int64), (torch.int32, torch.int64)],
                         ids=["i32", "i64", "mixed"])
def test_build_and_release_match_the_oracle(kv, case, types):
    requests, width, bs, lo, hi, new_hi, spare = case
    table, lens, new, pool, cursor = make_state(hash(case) & 0xffff, requests, width, bs, lo, hi, new_hi, spare, *types)
    total = int(new.sum())
    for num_tokens in (total, total + 131, max(0, total - 1)):
        bt = table.to(DEV)
        got = kv.build_block_tables(bt, lens.to(DEV), new.to(DEV), pool.to(DEV), cursor.to(DEV), bs, num_tokens=num_tokens)
        want = oracle_tables.build_block_tables(table, lens, new, pool, int(cursor), bs, num_tokens)
        assert torch.equal(bt.cpu(), want[0])
        assert torch.equal(got.slot_mapping.cpu(), want[1])
        assert torch.equal(got.query_start.cpu(), want[2])
        assert torch.equal(got.seq_lens.cpu(), want[3]) and got.seq_lens.dtype == lens.dtype
        assert got.free_cursor.tolist() == [want[4]]
        # the slots alone, through the grown table, are the same wherever the request was granted
        slots, start = kv.build_slot_mapping(bt, lens.to(DEV), new.to(DEV), bs, num_tokens=num_tokens)
        want_slots, want_start = oracle_tables.build_slot_mapping(want[0], lens, new, bs, num_tokens)
        assert torch.equal(slots.cpu(), want_slots) and torch.equal(start.cpu(), want_start)
    r = random.Random(requests)
    done = torch.tensor([r.random() < 0.4 for _ in range(requests)])
    free = pool.to(DEV)
    lens_out, cur = kv.release_block_tables(bt, got.seq_lens, done.to(DEV), free, got.free_cursor, bs)
    want_free, want_lens, want_cur = oracle_tables.release_block_tables(want[0], want[3], done, pool, want[4], bs)
    assert torch.equal(free.cpu(), want_free) and torch.equal(lens_out.cpu(), want_lens) and cur.tolist() == [want_cur]


def test_lengths_that_do_not_make_sense(kv):
    """Negative lengths count as nothing, absurd ones are refused, and nothing outside the buffers is touched."""
    big = 2**31 - 1
    table = torch.arange(24, dtype=torch.int32).reshape(6, 4)
    lens = torch.tensor([-5, 3, big, 16, 0, 63], dtype=torch.int32)
    new = torch.tensor([2, -4, 1, big, big, 1], dtype=torch.int32)
    pool = torch.arange(100, 108, dtype=torch.int32)
    bt = table.to(DEV)
    got = kv.build_block_tables(bt, lens.to(DEV), new.to(DEV), pool.to(DEV), torch.tensor([6], device=DEV), 16, num_tokens=5)
    assert bt.cpu()[0].tolist() == [106, 1, 2, 3]
    assert torch.equal(bt.cpu()[1:], table[1:])
    # packed behind request 3 nothing is reached any more: its 2^31 - 1 tokens fill the mapping
    assert got.slot_mapping.tolist() == [106 * 16, 106 * 16 + 1, -1, -1, -1]
    assert got.seq_lens.tolist() == [2, 3, big, 16, 0, 64]
    assert got.free_cursor.tolist() == [7]
    assert got.query_start.tolist() == [0, 2, 2, 3, big, big, big]
    first = torch.tensor([big, 1], dtype=torch.int32)
    slots, start = kv.build_slot_mapping(bt[:2], torch.zeros(2, dtype=torch.int64, device=DEV), first.to(DEV), 1, num_tokens=6)
    assert slots.tolist() == [106, 1, 2, 3, -1, -1] and start.tolist() == [0, big, big]


def test_lengths_and_slots_beyond_32_bits(kv):
    """Positions past 2^32 in a wide table of large blocks, and block ids whose slots need 64 bits."""
    bs = 1 << 28
    table = torch.full((2, 20), -1, dtype=torch.int64)
    table[0, 16], table[0, 17], table[1, 0] = 2**33, 5, 3
    lens = torch.tensor([17 * bs - 2, 0], dtype=torch.int64)
    new = torch.tensor([4, 2], dtype=torch.int64)
    slots, _ = kv.build_slot_mapping(table.to(DEV), lens.to(DEV), new.to(DEV), bs, num_tokens=6)
    assert slots.tolist() == [(2**33 + 1) * bs - 2, (2**33 + 1) * bs - 1, 5 * bs, 5 * bs + 1, 3 * bs, 3 * bs + 1]
    bt = table.to(DEV)
    got = kv.build_block_tables(bt, lens.to(DEV), new.to(DEV), torch.tensor([9, 8, 7], device=DEV),
                                torch.zeros(1, dtype=torch.int64, device=DEV), bs, num_tokens=6)
    assert bt[0, 17].item() == 9 and bt[1, 0].item() == 8 and got.free_cursor.tolist() == [2]
    assert got.slot_mapping.tolist()[2:] == [9 * bs, 9 * bs + 1, 8 * bs, 8 * bs + 1]
    assert got.seq_lens.tolist() == [17 * bs + 2, 2]


def test_no_requests_no_tokens_no_blocks(kv):
    empty32 = torch.zeros(0, dtype=torch.int32, device=DEV)
    cur = torch.tensor([0], device=DEV)
    got = kv.build_block_tables(torch.zeros(0, 4, dtype=torch.int32, device=DEV), empty32, empty32, empty32, cur, 16, num_tokens=3)
    assert got.slot_mapping.tolist() == [-1] * 3 and got.query_start.tolist() == [0] and got.free_cursor.tolist() == [0]
    bt = torch.zeros(2, 0, dtype=torch.int32, device=DEV)
    two = torch.tensor([0, 0], dtype=torch.int32, device=DEV)
    got = kv.build_block_tables(bt, two, two + 1, empty32, cur, 16, num_tokens=2)
    assert got.slot_mapping.tolist() == [-1, -1] and got.seq_lens.tolist() == [0, 0]
    lens, c = kv.release_block_tables(bt, two, torch.tensor([True, True], device=DEV), empty32, cur, 16)
    assert lens.tolist() == [0, 0] and c.tolist() == [0]


def test_strided_tables_and_lists(kv):
    """A column-major table, a table that is a window of a larger one, and lists with a stride."""
    table, lens, new, pool, cursor = make_state(5, 33, 21, 16, 0, 300, 20, 4)
    total = int(new.sum())
    want = oracle_tables.build_block_tables(table, lens, new, pool, int(cursor), 16, total)
    wide = torch.full((33, 64), 77, dtype=torch.int32, device=DEV)
    wide[:, 5:26] = table.to(DEV)
    views = {"window": wide[:, 5:26], "columns": table.to(DEV).t().contiguous().t()}
    pick = lambda t: torch.stack([t, t], 1).to(DEV)[:, 0]
    for bt in views.values():
        got = kv.build_block_tables(bt, pick(lens), pick(new), pick(pool), cursor.to(DEV), 16, num_tokens=total)
        assert torch.equal(bt.cpu(), want[0]) and torch.equal(got.slot_mapping.cpu(), want[1])
    assert (wide[:, :5] == 77).all() and (wide[:, 26:] == 77).all()


def test_release_more_than_was_handed_out(kv):
    """Entries that would fall below the list are dropped, whatever the cursor says."""
    table = torch.arange(12, dtype=torch.int32).reshape(2, 6)
    lens = torch.tensor([96, 1000], dtype=torch.int32)
    done = torch.tensor([True, True])
    for cursor in (5, 12, 40, 0):
        free = torch.full((14,), -1, dtype=torch.int32)
        want = oracle_tables.release_block_tables(table, lens, done, free, cursor, 16)
        f = free.to(DEV)
        out_lens, out_cur = kv.release_block_tables(table.to(DEV), lens.to(DEV), done.to(DEV), f, torch.tensor([cursor], device=DEV), 16)
        assert torch.equal(f.cpu(), want[0]) and out_cur.tolist() == [want[2]] and out_lens.tolist() == [0, 0]


def test_refusals(kv):
    bt = torch.zeros(2, 4, dtype=torch.int32, device=DEV)
    lens, one = torch.zeros(2, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int64, device=DEV)
    free = torch.zeros(4, dtype=torch.int32, device=DEV)
    build = lambda t=bt, s=lens, n=lens, f=free, c=one, bs=16, tok=4, **kw: kv.build_block_tables(t, s, n, f, c, bs, num_tokens=tok, **kw)
    build()
    for bad in (dict(t=bt.float()), dict(t=bt[0]), dict(s=lens[:1]), dict(s=lens.float()), dict(n=lens.cpu()), dict(bs=0), dict(bs=2**32 + 16),
                dict(f=free.float()), dict(c=one.int()), dict(c=torch.zeros(2, dtype=torch.int64, device=DEV)), dict(tok=-1),
                dict(tok=2**31), dict(t=torch.zeros(1, 4, dtype=torch.int32, device=DEV).expand(2, 4)), dict(f=free.cpu())):
        with pytest.raises(AssertionError):
            build(**bad)
    good = build()
    with pytest.raises(AssertionError):
        build(out=good._replace(slot_mapping=good.slot_mapping[:3]))
    with pytest.raises(AssertionError):
        build(out=good._replace(seq_lens=good.seq_lens.long()))
    with pytest.raises(AssertionError):
        kv.release_block_tables(bt, lens, lens, free, one, 16)
    with pytest.raises(AssertionError):
        kv.release_block_tables(bt, lens, lens.bool(), free[::2], one, 16)


@pytest.mark.parametrize("requests,prompt", [(37, 0), (9, 12000)], ids=["one_kernel", "two_kernels"])
def test_captured_step_advances_its_own_state(kv, requests, prompt):
    """Lengths and cursor in place, captured once: every replay is one more step of the oracle."""
    table, lens, new, pool, cursor = make_state(11, requests, 900, 16, 0, 90, 1, 64 * 16 + 8 * prompt)
    new[:] = 1
    new[requests // 2] = max(1, prompt)
    total = int(new.sum())
    bt, l, n, f, c = (t.to(DEV) for t in (table, lens, new, pool, cursor))
    out = kv.BlockTableStep(torch.empty(total, dtype=torch.int64, device=DEV),
                            torch.empty(requests + 1, dtype=torch.int32, device=DEV), l, c)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            kv.build_block_tables(bt, l, n, f, c, 16, num_tokens=total, out=out)
    torch.cuda.synchronize()
    state = (table, None, None, lens, int(cursor))
    for _ in range(4):
        with torch.cuda.stream(stream):
            graph.replay()
        torch.cuda.synchronize()
        state = oracle_tables.build_block_tables(state[0], state[3], new, pool, state[4], 16, total)
        assert torch.equal(bt.cpu(), state[0]) and torch.equal(out.slot_mapping.cpu(), state[1])
        assert torch.equal(l.cpu(), state[3]) and c.tolist() == [state[4]]


def test_two_graphs_on_two_streams(kv):
    """Two captured two-kernel calls replayed at the same time: each has a workspace of its own."""
    runs = []
    for seed in (1, 2):
        table, lens, new, pool, cursor = make_state(seed, 300, 200, 16, 0, 900, 400, 0)
        total = int(new.sum())
        dev = [t.to(DEV) for t in (table, lens, new, pool, cursor)]
        stream = torch.cuda.Stream()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            got = kv.build_block_tables(*dev, 16, num_tokens=total)
        runs.append((graph, stream, got, dev[0], oracle_tables.build_block_tables(table, lens, new, pool, int(cursor), 16, total)))
    for _ in range(20):
        for graph, stream, *_ in runs:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for _, _, got, bt, want in runs:
        assert torch.equal(bt.cpu(), want[0]) and torch.equal(got.slot_mapping.cpu(), want[1])


def test_serving_loop_writes_and_attends(kv, workloads):
    """The operators together: rows grow from prompts through decode steps, every step's K/V goes through the slots
    into the cache, attention reads it back through the tables; finished requests' blocks are reused."""
    import oracle

    shape = workloads.QWEN25_7B
    gen = torch.Generator(device=DEV).manual_seed(0)
    gain = workloads.channel_gain(shape, 0, DEV)
    ks, vs = (t.to(DEV) for t in workloads.calibrate_scales(shape, 0))
    R, width, blocks = 5, 6, 20
    kc = torch.zeros(blocks, 16, shape.num_kv_heads, shape.head_dim, dtype=torch.int8, device=DEV)
    vc = torch.zeros_like(kc)
    bt = torch.zeros(R, width, dtype=torch.int32, device=DEV)
    lens = torch.zeros(R, dtype=torch.int32, device=DEV)
    free = torch.randperm(blocks, generator=torch.Generator().manual_seed(1)).to(torch.int32).to(DEV)
    cursor = torch.zeros(1, dtype=torch.int64, device=DEV)
    history = [[] for _ in range(R)]
    prompts = torch.tensor([3, 40, 17, 1, 30], dtype=torch.int32, device=DEV)
    for step in range(12):
        if step == 8:  # two requests end and start again with new prompts, out of the blocks they gave back
            done = torch.tensor([False, True, False, False, True], device=DEV)
            lens, cursor = kv.release_block_tables(bt, lens, done, free, cursor, 16)
            history[1], history[4] = [], []
            new = torch.where(done, torch.tensor([0, 50, 0, 0, 20], dtype=torch.int32, device=DEV), torch.ones_like(lens))
        else:
            new = prompts if step == 0 else torch.ones_like(lens)
        total = int(new.sum())
        plan = kv.build_block_tables(bt, lens, new, free, cursor, 16, num_tokens=total + 3)
        lens, cursor = plan.seq_lens, plan.free_cursor
        k, v = workloads.draw_kv(total + 3, shape, gen, gain)
        kv.int8_kv_cache_write(k, v, kc, vc, plan.slot_mapping, ks, vs)
        for b in range(R):
            lo, hi = plan.query_start[b].item(), plan.query_start[b + 1].item()
            history[b].append((k[lo:hi], v[lo:hi]))
        q = workloads.draw_query(R, shape, gen)
        out = kv.int8_paged_attention(q, kc, vc, bt, lens, ks, vs, max_seq_len=width * 16)
        for b in range(R):
            kb, vb = (torch.cat([h[i] for h in history[b]]).cpu() for i in (0, 1))
            n = kb.shape[0]
            assert n == lens[b].item()
            flat = -(-n // 16)
            okc = torch.zeros(flat, 16, shape.num_kv_heads, shape.head_dim, dtype=torch.int8)
            ovc = torch.zeros_like(okc)
            oracle.cache_write(kb, vb, okc, ovc, torch.arange(n), ks.cpu(), vs.cpu())
            want = oracle.int8_paged_attention_oracle(q[b:b + 1].cpu(), okc, ovc, torch.arange(flat)[None], [n], ks.cpu(), vs.cpu())
            assert (out[b:b + 1].float().cpu() - want).abs().max() <= 2e-2
