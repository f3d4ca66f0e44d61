"""Measured cases of the block-table operators and of differential paged decode attention.

Five operators of the serving step, each in a plain form (elementary torch operations, `own` false) and as the calls
that a user makes of this package (`own` true):

  tables   build_block_tables        blocks for the tokens that a step adds, and the slots of those tokens
  slots    build_slot_mapping        the slots alone, from tables that the host keeps
  release  release_block_tables      blocks of finished requests back to the free list
  diff8    int8_paged_diff_attention differential decode attention over the INT8 paged cache
  diff16   bf16_paged_diff_attention the same over a bf16 or fp16 paged cache

Every size of a case is a plain value; the lengths follow from the case's own `len_seed`, the contents (queries,
caches, block placement) from the seed that `prepare` is given.
"""

import importlib
import math
import random

import numpy as np
import torch

own = False

_DEVICE = "cuda"
_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_EPS = 1e-5


def _package():
    return importlib.import_module("int8-kvcache_b200")


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one decode step of a batch of 256: every request adds a token, about one in sixteen needs a block; latency
        dict(name="tables_decode_256", op="tables", requests=256, lo=1024, hi=8192, new_lo=1, new_hi=1, prompts=0,
             block_size=16, width=513, spare=64, pad=0, len_seed=1),
        # a prompt phase: 384 new requests of 1 to 8192 tokens, tables from nothing, block size 32, pool just enough
        dict(name="tables_prompts_384", op="tables", requests=384, lo=0, hi=0, new_lo=1, new_hi=8192, prompts=384,
             block_size=32, width=260, spare=0, pad=517, len_seed=2),
        # the slot map of a decode step whose tables the engine keeps, with padding rows of a captured batch; latency
        dict(name="slots_decode_64", op="slots", requests=64, lo=1, hi=4096, new_lo=1, new_hi=1, prompts=0,
             block_size=16, width=257, spare=0, pad=7, len_seed=3),
        # chunks of prompts behind cached tokens next to decoding requests: 1024 requests, 128 of them with a chunk
        dict(name="slots_chunks_1024", op="slots", requests=1024, lo=1, hi=8192, new_lo=1, new_hi=4096, prompts=128,
             block_size=16, width=769, spare=0, pad=0, len_seed=4),
        # eight of 64 running requests end; latency
        dict(name="release_8_of_64", op="release", requests=64, lo=1, hi=4096, finished=8, block_size=16, width=257,
             len_seed=5),
        # a whole batch of 512 long requests is dropped (an aborted job)
        dict(name="release_512", op="release", requests=512, lo=4096, hi=32768, finished=512, block_size=16,
             width=2048, len_seed=6),
        # a lone request of 512 tokens on a layer of 14 differential heads over 2 pairs of KV heads (28 / 4 heads of
        # 128 in the cache's terms): latency
        dict(name="diff8_1x512", op="diff8", batch=1, lo=512, hi=512, heads=14, kv_pairs=2, head_dim=128,
             block_size=16, empty=0, dtype="bf16", norm=True, len_seed=7),
        # the everyday decode call of the same layer: 8 sequences of 4096 tokens
        dict(name="diff8_8x4096", op="diff8", batch=8, lo=4096, hi=4096, heads=14, kv_pairs=2, head_dim=128,
             block_size=16, empty=0, dtype="bf16", norm=True, len_seed=8),
        # a ragged batch with padding rows: head size 64, 8 heads without grouping, fp16, pages of 32 tokens
        dict(name="diff8_ragged_d64", op="diff8", batch=61, lo=1, hi=8191, heads=8, kv_pairs=8, head_dim=64,
             block_size=32, empty=3, dtype="fp16", norm=False, len_seed=9),
        # long contexts, the largest call: 32 sequences of up to 32768 tokens, 32 heads over 4 pairs of KV heads
        dict(name="diff8_long", op="diff8", batch=32, lo=24576, hi=32768, heads=32, kv_pairs=4, head_dim=128,
             block_size=16, empty=0, dtype="bf16", norm=True, len_seed=10),
        # the float-cache baseline of the everyday call
        dict(name="diff16_8x4096", op="diff16", batch=8, lo=4096, hi=4096, heads=14, kv_pairs=2, head_dim=128,
             block_size=16, empty=0, dtype="bf16", norm=True, len_seed=11),
        # a ragged fp16 batch, groups of four, no norm
        dict(name="diff16_ragged", op="diff16", batch=45, lo=1, hi=8191, heads=16, kv_pairs=4, head_dim=128,
             block_size=16, empty=2, dtype="fp16", norm=False, len_seed=12),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["tables", "slots", "release", "diff8", "diff8", "diff16"])
    len_seed = rng.randrange(1 << 30)
    block_size = rng.choice([16, 16, 32, 64])
    if op in ("tables", "slots", "release"):
        requests = _log_int(rng, 1, 1024)
        if op != "release":
            block_size = rng.choice([1, 8, 16, 24, 32, 64])
        hi = _log_int(rng, 1, 8192)
        case = dict(op=op, requests=requests, lo=rng.choice([0, 1, hi // 2]), hi=hi, block_size=block_size,
                    len_seed=len_seed)
        if op == "release":
            case["finished"] = rng.randint(0, requests)
            case["width"] = -(-hi // block_size) + rng.randint(0, 33)
        else:
            case["prompts"] = rng.randint(0, min(requests, 128))
            case["new_lo"] = rng.choice([0, 1])
            case["new_hi"] = _log_int(rng, 1, 4096)
            # now and then a table too narrow or a pool too small for all that is asked for
            case["width"] = max(1, -(-(hi + case["new_hi"]) // block_size) - rng.choice([0, 0, 1]))
            case["spare"] = rng.choice([0, 17, 1000, -3]) if op == "tables" else 0
            case["pad"] = rng.choice([0, 0, 1, 130])
        return case
    head_dim = rng.choice([64, 128, 128])
    kv_pairs = rng.randint(1, 8)
    heads = kv_pairs * rng.randint(1, 8)
    hi = _log_int(rng, 1, 32768)
    # at most half the bytes of the largest listed case
    room = 500_000_000 // (4 * head_dim * kv_pairs * (2 if op == "diff16" else 1) * hi)
    batch = _log_int(rng, 1, max(1, min(128, room)))
    return dict(op=op, batch=batch, lo=rng.choice([1, max(1, hi // 2), hi]), hi=hi, heads=heads, kv_pairs=kv_pairs,
                head_dim=head_dim, block_size=block_size, empty=rng.choice([0, 0, 1]) if batch > 1 else 0,
                dtype=rng.choice(["bf16", "fp16"]), norm=rng.random() < 0.5, len_seed=len_seed)


def _lengths(case):
    """The case's lengths: (cached, new) per request for the table operators, sequence lengths for attention."""
    r = random.Random(case["len_seed"])
    if case["op"] in ("diff8", "diff16"):
        lens = [r.randint(case["lo"], case["hi"]) for _ in range(case["batch"])]
        for b in r.sample(range(case["batch"]), case["empty"]):
            lens[b] = 0
        return lens
    cached = [r.randint(case["lo"], case["hi"]) for _ in range(case["requests"])]
    if case["op"] == "release":
        return cached, set(r.sample(range(case["requests"]), case["finished"]))
    prompts = set(r.sample(range(case["requests"]), case["prompts"]))
    new = [r.randint(case["new_lo"], case["new_hi"]) if b in prompts else 1 for b in range(case["requests"])]
    return cached, new


def _ceil(a, b):
    return -(-a // b)


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device=_DEVICE).manual_seed(int(seed))


def _placed_tables(lens, block_size, width, num_blocks, gen):
    """int32 [B, width]: the blocks of every sequence from a random permutation of the pool, 0 behind its last one;
    and that permutation with the number of its entries that are in use."""
    need = torch.tensor([_ceil(n, block_size) for n in lens], dtype=torch.int64, device=_DEVICE)
    perm = torch.randperm(num_blocks, generator=gen, device=_DEVICE).to(torch.int32)
    first = torch.cumsum(need, 0) - need
    col = torch.arange(width, device=_DEVICE)
    idx = (first[:, None] + col[None, :]).clamp_max(max(num_blocks - 1, 0))
    table = torch.where(col[None, :] < need[:, None], perm[idx], torch.zeros((), dtype=torch.int32, device=_DEVICE))
    return table.contiguous(), perm


def prepare(case, seed):
    gen = _generator(seed)
    if case["op"] in ("diff8", "diff16"):
        return _prepare_attention(case, gen)
    i32 = dict(dtype=torch.int32, device=_DEVICE)
    bs, width = case["block_size"], case["width"]
    state = dict(case=case, block_size=bs)
    if case["op"] == "release":
        cached, finished = _lengths(case)
    else:
        cached, new = _lengths(case)
    cached = [min(n, width * bs) for n in cached]
    used = sum(_ceil(n, bs) for n in cached)
    wanted = 0
    if case["op"] == "tables":
        wanted = sum(_ceil(c + n, bs) - _ceil(c, bs) for c, n in zip(cached, new) if c + n <= width * bs)
        wanted = max(0, wanted + case["spare"])
    table, pool = _placed_tables(cached, bs, width, max(1, used + wanted), gen)
    state["seq_lens"] = torch.tensor(cached, **i32)
    state["block_tables"] = table
    if case["op"] == "release":
        state["finished"] = torch.tensor([b in finished for b in range(len(cached))], device=_DEVICE)
        # the free list as the requests' own growth left it: its first `used` entries have been handed out
        state["free_blocks"] = pool
        state["free_cursor"] = torch.tensor([used], dtype=torch.int64, device=_DEVICE)
        return state
    state["new_lens"] = torch.tensor(new, **i32)
    state["num_tokens"] = sum(new) + case["pad"]
    if case["op"] == "tables":
        state["free_blocks"] = pool
        state["free_cursor"] = torch.tensor([used], dtype=torch.int64, device=_DEVICE)
    return state


def _prepare_attention(case, gen):
    lens = _lengths(case)
    B, heads, pairs, D, bs = case["batch"], case["heads"], case["kv_pairs"], case["head_dim"], case["block_size"]
    dtype = _DTYPES[case["dtype"]]
    used = sum(_ceil(n, bs) for n in lens)
    num_blocks = used + used // 8 + 4
    width = max(1, max(_ceil(n, bs) for n in lens))
    table, _ = _placed_tables(lens, bs, width, num_blocks, gen)
    # keys with four strong channels per head and calmer values, as real layers have them; a few values lie outside
    # what the scales can hold and saturate
    gain = torch.ones(2 * pairs, D, device=_DEVICE)
    for h in range(2 * pairs):
        gain[h, torch.randperm(D, generator=gen, device=_DEVICE)[:4]] = 8.0
    k_scale = 30.0 / 127.0 * (0.9 + 0.2 * torch.rand(2 * pairs, generator=gen, device=_DEVICE))
    v_scale = 2.0 / 127.0 * (0.9 + 0.2 * torch.rand(2 * pairs, generator=gen, device=_DEVICE))
    cache_dtype = torch.int8 if case["op"] == "diff8" else dtype
    keys = torch.empty(num_blocks, bs, 2 * pairs, D, dtype=cache_dtype, device=_DEVICE)
    values = torch.empty_like(keys)
    step = max(1, (1 << 26) // (bs * 2 * pairs * D))
    for lo in range(0, num_blocks, step):
        shape = keys[lo:lo + step].shape
        k = torch.randn(shape, generator=gen, device=_DEVICE) * gain
        v = torch.randn(shape, generator=gen, device=_DEVICE) * 0.5
        if cache_dtype == torch.int8:
            k = (k / k_scale[:, None]).round_().clamp_(-127, 127)
            v = (v / v_scale[:, None]).round_().clamp_(-127, 127)
        keys[lo:lo + step] = k.to(cache_dtype)
        values[lo:lo + step] = v.to(cache_dtype)
    state = dict(
        case=case, lens=lens, block_tables=table, key_cache=keys, value_cache=values,
        query=torch.randn(B, 2 * heads, D, generator=gen, device=_DEVICE).to(dtype),
        seq_lens=torch.tensor(lens, dtype=torch.int32, device=_DEVICE), max_seq_len=max(lens),
        lam=0.2 + 0.6 * torch.rand(heads, generator=gen, device=_DEVICE),
        norm_weight=1.0 + 0.1 * torch.randn(2 * D, generator=gen, device=_DEVICE) if case["norm"] else None,
        out_scale=0.2 if case["norm"] else 1.0,
    )
    if case["op"] == "diff8":
        state["k_scale"], state["v_scale"] = k_scale, v_scale
    return state


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    if own:
        return _RUN_OWN[op](state)
    return _RUN_PLAIN[op](state)


def _own_tables(s):
    return (s["block_tables"],) + tuple(_package().build_block_tables(
        s["block_tables"], s["seq_lens"], s["new_lens"], s["free_blocks"], s["free_cursor"], s["block_size"],
        num_tokens=s["num_tokens"]))


def _own_slots(s):
    return _package().build_slot_mapping(s["block_tables"], s["seq_lens"], s["new_lens"], s["block_size"],
                                         num_tokens=s["num_tokens"])


def _own_release(s):
    return (s["free_blocks"],) + tuple(_package().release_block_tables(
        s["block_tables"], s["seq_lens"], s["finished"], s["free_blocks"], s["free_cursor"], s["block_size"]))


def _own_diff8(s):
    return _package().int8_paged_diff_attention(
        s["query"], s["key_cache"], s["value_cache"], s["block_tables"], s["seq_lens"], s["k_scale"], s["v_scale"],
        s["lam"], norm_weight=s["norm_weight"], norm_eps=_EPS, out_scale=s["out_scale"], max_seq_len=s["max_seq_len"])


def _own_diff16(s):
    return _package().bf16_paged_diff_attention(
        s["query"], s["key_cache"], s["value_cache"], s["block_tables"], s["seq_lens"], s["lam"],
        norm_weight=s["norm_weight"], norm_eps=_EPS, out_scale=s["out_scale"], max_seq_len=s["max_seq_len"])


def _slots_of(table_block, seq_lens, new_lens, alive, block_size, num_tokens):
    """slot_mapping [num_tokens] and query_start [R + 1]; `table_block(request, logical block)` gives block ids."""
    start = torch.zeros(new_lens.numel() + 1, dtype=torch.int64, device=new_lens.device)
    start[1:] = torch.cumsum(new_lens, 0)
    token = torch.arange(num_tokens, device=new_lens.device)
    owner = torch.searchsorted(start[1:], token, right=True).clamp_max(new_lens.numel() - 1)
    pos = seq_lens[owner] + token - start[owner]
    block = table_block(owner, pos // block_size)
    live = (token < start[-1]) & alive[owner] & (block >= 0)
    slots = torch.where(live, block * block_size + pos % block_size, torch.full_like(token, -1))
    return slots, start.to(torch.int32)


def _plain_tables(s):
    bs, table, free = s["block_size"], s["block_tables"], s["free_blocks"]
    cached = s["seq_lens"].long().clamp_min(0)
    new = s["new_lens"].long().clamp_min(0)
    cursor = s["free_cursor"].clamp_min(0)
    width = table.shape[1]
    old = (cached + bs - 1) // bs
    fits = cached + new <= width * bs
    want = torch.where(fits, (cached + new + bs - 1) // bs - old, torch.zeros_like(old))
    end = torch.cumsum(want, 0)
    first = end - want
    granted = fits & ((want == 0) | (end <= free.numel() - cursor))
    taken = torch.where(granted & (want > 0), end, torch.zeros_like(end)).amax().reshape(1)

    def new_block(owner, j):
        return free[(cursor + first[owner] + j - old[owner]).clamp(0, free.numel() - 1)].long()

    def block_of(owner, j):
        known = table[owner, j.clamp(0, width - 1)].long()
        return torch.where(j < old[owner], known, new_block(owner, j))

    slots, start = _slots_of(block_of, cached, new, granted, bs, s["num_tokens"])
    col = torch.arange(width, device=table.device)[None, :]
    row = torch.arange(table.shape[0], device=table.device)[:, None]
    grown = granted[:, None] & (col >= old[:, None]) & (col < (old + want)[:, None])
    table = torch.where(grown, new_block(row, col).to(table.dtype), table)
    seq_lens = torch.where(granted, cached + new, cached).to(s["seq_lens"].dtype)
    return table, slots, start, seq_lens, cursor + taken


def _plain_slots(s):
    bs, table = s["block_size"], s["block_tables"]
    cached = s["seq_lens"].long().clamp_min(0)
    new = s["new_lens"].long().clamp_min(0)
    width = table.shape[1]

    def block_of(owner, j):
        known = table[owner, j.clamp(0, width - 1)].long()
        return torch.where(j < width, known, torch.full_like(known, -1))

    return _slots_of(block_of, cached, new, torch.ones_like(cached, dtype=torch.bool), bs, s["num_tokens"])


def _plain_release(s):
    bs, table, free, cursor = s["block_size"], s["block_tables"], s["free_blocks"], s["free_cursor"]
    done = s["finished"]
    lens = s["seq_lens"].long().clamp(0, table.shape[1] * bs)
    count = torch.where(done, (lens + bs - 1) // bs, torch.zeros_like(lens))
    end = torch.cumsum(count, 0)
    base = cursor - end[-1]
    place = torch.arange(free.numel(), device=free.device) - base
    owner = torch.searchsorted(end, place.clamp_min(0), right=True).clamp_max(lens.numel() - 1)
    j = (place - (end - count)[owner]).clamp(0, table.shape[1] - 1)
    free = torch.where((place >= 0) & (place < end[-1]), table[owner, j].to(free.dtype), free)
    seq_lens = torch.where(done, torch.zeros_like(s["seq_lens"]), s["seq_lens"])
    return free, seq_lens, base.clamp_min(0)


def _plain_attention(s):
    case = s["case"]
    heads, pairs, D, bs = case["heads"], case["kv_pairs"], case["head_dim"], case["block_size"]
    group = heads // pairs
    q = s["query"].float().view(-1, pairs, group, 2, D) / math.sqrt(D)
    out = torch.zeros(q.shape[0], heads, 2 * D, device=q.device)
    for b, n in enumerate(s["lens"]):
        if n == 0:
            continue
        blocks = s["block_tables"][b, :_ceil(n, bs)].long()
        k = s["key_cache"][blocks].reshape(-1, 2 * pairs, D)[:n].float()
        v = s["value_cache"][blocks].reshape(-1, 2 * pairs, D)[:n].float()
        if "k_scale" in s:
            k = k * s["k_scale"][:, None]
            v = v * s["v_scale"][:, None]
        k = k.view(n, pairs, 2, D).permute(1, 2, 3, 0)        # [pairs, 2, D, n]
        v = v.view(n, pairs, 2 * D).permute(1, 0, 2)          # [pairs, n, 2D]
        scores = q[b].permute(0, 2, 1, 3) @ k                 # [pairs, 2, group, n]
        p = torch.exp(scores - scores.amax(-1, keepdim=True))
        maps = (p @ v[:, None]) / p.sum(-1, keepdim=True)     # [pairs, 2, group, 2D]
        out[b] = (maps[:, 0] - s["lam"].view(pairs, group, 1) * maps[:, 1]).reshape(heads, 2 * D)
    if s["norm_weight"] is not None:
        out = out * torch.rsqrt(out.square().mean(-1, keepdim=True) + _EPS) * s["norm_weight"]
    return (out * s["out_scale"]).to(s["query"].dtype)


_RUN_OWN = dict(tables=_own_tables, slots=_own_slots, release=_own_release, diff8=_own_diff8, diff16=_own_diff16)
_RUN_PLAIN = dict(tables=_plain_tables, slots=_plain_slots, release=_plain_release, diff8=_plain_attention,
                  diff16=_plain_attention)


# ---------------------------------------------------------------------------------------------------------------------
# what one pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------
def work(case):
    bs = case["block_size"]
    if case["op"] in ("diff8", "diff16"):
        lens = _lengths(case)
        D, pairs, heads = case["head_dim"], case["kv_pairs"], case["heads"]
        elem = 1 if case["op"] == "diff8" else 2
        # K and V rows of both halves of a pair, the block ids, queries in and outputs out
        nbytes = sum(lens) * pairs * 4 * D * elem + sum(_ceil(n, bs) for n in lens) * 4
        nbytes += case["batch"] * (4 + heads * 2 * D * 2 * 2) + heads * 4
        # two score maps, and one product of their difference with V
        return dict(bytes=nbytes, flops=sum(lens) * heads * 8 * D)
    width = case["width"]
    R = case["requests"]
    if case["op"] == "release":
        cached, finished = _lengths(case)
        moved = sum(_ceil(min(n, width * bs), bs) for b, n in enumerate(cached) if b in finished)
        return dict(bytes=moved * 8 + R * (4 + 1 + 4) + 16, flops=moved)
    cached, new = _lengths(case)
    cached = [min(n, width * bs) for n in cached]
    tokens = sum(new)
    read = written = 0
    for c, n in zip(cached, new):
        if case["op"] == "tables":
            read += 1 if n and c % bs else 0
            written += _ceil(c + n, bs) - _ceil(c, bs) if c + n <= width * bs else 0
        elif n:
            read += min(_ceil(c + n, bs), width) - c // bs
    # lengths in, prefix sums and lengths out, a slot per token, old block ids in, new ones in and out
    out_lens = 4 if case["op"] == "tables" else 0
    return dict(bytes=R * (4 + 4 + 4 + out_lens) + (tokens + case["pad"]) * 8 + read * 4 + written * 8,
                flops=tokens)


# ---------------------------------------------------------------------------------------------------------------------
# the definitions, in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    return {"tables": _exact_tables, "slots": _exact_slots, "release": _exact_release,
            "diff8": _exact_attention, "diff16": _exact_attention}[case["op"]](state)


def _host(t):
    return t.cpu().numpy().astype(np.int64)


def _request_slots(row, cached, n, bs):
    """Slots of tokens cached .. cached + n - 1 through one request's list of blocks; -1 where it has none."""
    pos = np.arange(cached, cached + n)
    block = pos // bs
    ids = np.full(n, -1, dtype=np.int64)
    inside = block < len(row)
    ids[inside] = row[block[inside]]
    return np.where(ids >= 0, ids * bs + pos % bs, -1)


def _exact_tables(s):
    bs = s["block_size"]
    table, free = _host(s["block_tables"]), _host(s["free_blocks"])
    cached, new, cursor = _host(s["seq_lens"]), _host(s["new_lens"]), int(s["free_cursor"].item())
    slots = np.full(s["num_tokens"], -1, dtype=np.int64)
    start, lens = [0], []
    next_free, stuck = cursor, False
    for b in range(len(cached)):
        c, n = int(cached[b]), int(new[b])
        have = _ceil(c, bs)
        ok = c + n <= table.shape[1] * bs
        need = _ceil(c + n, bs) - have if ok else 0
        if need and (stuck or next_free + need > len(free)):
            ok, stuck = False, True
        if ok:
            table[b, have:have + need] = free[next_free:next_free + need]
            next_free += need
            slots[start[-1]:start[-1] + n] = _request_slots(table[b], c, n, bs)
        lens.append(c + n if ok else c)
        start.append(start[-1] + n)
    as_tensor = lambda a, dt: torch.as_tensor(np.asarray(a), dtype=dt, device=_DEVICE)
    return (as_tensor(table, torch.int32), as_tensor(slots, torch.int64), as_tensor(start, torch.int32),
            as_tensor(lens, torch.int32), as_tensor([next_free], torch.int64))


def _exact_slots(s):
    bs, table = s["block_size"], _host(s["block_tables"])
    slots = np.full(s["num_tokens"], -1, dtype=np.int64)
    start = [0]
    for b, (c, n) in enumerate(zip(_host(s["seq_lens"]), _host(s["new_lens"]))):
        slots[start[-1]:start[-1] + n] = _request_slots(table[b], int(c), int(n), bs)
        start.append(start[-1] + int(n))
    return (torch.as_tensor(slots, device=_DEVICE),
            torch.as_tensor(np.asarray(start), dtype=torch.int32, device=_DEVICE))


def _exact_release(s):
    bs, table, free = s["block_size"], _host(s["block_tables"]), _host(s["free_blocks"])
    done, lens, cursor = s["finished"].cpu().numpy(), _host(s["seq_lens"]), int(s["free_cursor"].item())
    back = [table[b, :_ceil(int(lens[b]), bs)] for b in range(len(lens)) if done[b]]
    back = np.concatenate(back) if back else np.zeros(0, dtype=np.int64)
    free[cursor - len(back):cursor] = back
    as_tensor = lambda a, dt: torch.as_tensor(np.asarray(a), dtype=dt, device=_DEVICE)
    return (as_tensor(free, torch.int32), as_tensor(np.where(done, 0, lens), torch.int32),
            as_tensor([cursor - len(back)], torch.int64))


def _exact_attention(s):
    case = s["case"]
    heads, pairs, D, bs = case["heads"], case["kv_pairs"], case["head_dim"], case["block_size"]
    group = heads // pairs
    out = torch.zeros(len(s["lens"]), heads, 2 * D, dtype=torch.float64, device=_DEVICE)
    for b, n in enumerate(s["lens"]):
        if n == 0:
            continue
        token = torch.arange(n, device=_DEVICE)
        block, offset = s["block_tables"][b, token // bs].long(), token % bs
        for g in range(pairs):
            weights = []
            for m in range(2):
                k = s["key_cache"][block, offset, 2 * g + m].double()
                if "k_scale" in s:
                    k = k * s["k_scale"][2 * g + m].double()
                q = s["query"][b, 2 * group * g + m:2 * group * (g + 1):2].double()
                weights.append(torch.softmax(torch.einsum("hd,nd->hn", q, k) * D ** -0.5, dim=-1))
            lam = s["lam"][group * g:group * (g + 1)].double()
            mixed = weights[0] - lam[:, None] * weights[1]
            for half in range(2):
                v = s["value_cache"][block, offset, 2 * g + half].double()
                if "v_scale" in s:
                    v = v * s["v_scale"][2 * g + half].double()
                out[b, group * g:group * (g + 1), half * D:(half + 1) * D] = torch.einsum("hn,nd->hd", mixed, v)
    if s["norm_weight"] is not None:
        rms = (out.pow(2).sum(-1, keepdim=True) / (2 * D) + _EPS).sqrt()
        out = out / rms * s["norm_weight"].double()
    return out * s["out_scale"]
