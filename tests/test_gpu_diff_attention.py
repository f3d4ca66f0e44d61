"""Differential paged decode attention on the GPU against its definition in 64 bits; every tolerance is the bound that
oracle/diff_attention.py derives from the operator's documented roundings."""

import pytest
import torch

from oracle.diff_attention import check, diff_paged_attention

pytestmark = pytest.mark.gpu
DEV = "cuda"


def make_case(seed, lens, heads, pairs, D, bs, cache=torch.int8, qtype=torch.bfloat16, sharp=1.0, extra_blocks=3, index=torch.int32):
    """Tensors on the GPU: caches filled everywhere (what lies behind a sequence's last token is never to be read into
    the result), blocks in random order, queries scaled by `sharp` (large: few tokens carry the softmax)."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // bs) for n in lens]
    blocks = sum(need) + extra_blocks
    perm = torch.randperm(blocks, generator=g)
    width = max(1, max(need, default=1))
    bt = torch.zeros(len(lens), width, dtype=index)
    at = 0
    for b, k in enumerate(need):
        bt[b, :k] = perm[at:at + k].to(index)
        at += k
    shape = (blocks, bs, 2 * pairs, D)
    kc = torch.randn(shape, generator=g)
    kc[..., 0] *= 4
    vc = torch.randn(shape, generator=g) * 0.5
    scales = (None, None)
    if cache == torch.int8:
        scales = (0.02 + 0.01 * torch.rand(2 * pairs, generator=g), 0.01 + 0.01 * torch.rand(2 * pairs, generator=g))
        kc = (kc / scales[0][:, None]).round().clamp(-127, 127)
        vc = (vc / scales[1][:, None]).round().clamp(-127, 127)
    q = (torch.randn(len(lens), 2 * heads, D, generator=g) * sharp).to(qtype)
    lam = 0.1 + torch.rand(heads, generator=g)
    dev = lambda t: None if t is None else t.to(DEV)
    return dict(q=dev(q), kc=dev(kc.to(cache)), vc=dev(vc.to(cache)), bt=dev(bt), lens=torch.tensor(lens, dtype=index, device=DEV),
                ks=dev(scales[0]), vs=dev(scales[1]), lam=dev(lam))


def call(kv, c, **kw):
    kw.setdefault("max_seq_len", c["bt"].shape[1] * c["kc"].shape[1])
    if c["kc"].dtype == torch.int8:
        return kv.int8_paged_diff_attention(c["q"], c["kc"], c["vc"], c["bt"], c["lens"], c["ks"], c["vs"], c["lam"], **kw)
    return kv.bf16_paged_diff_attention(c["q"], c["kc"], c["vc"], c["bt"], c["lens"], c["lam"], **kw)


def verify(kv, c, **kw):
    norm = {k: kw[k] for k in ("norm_weight", "norm_eps", "out_scale") if k in kw}
    want, bound = diff_paged_attention(c["q"], c["kc"], c["vc"], c["bt"], c["lens"].tolist(), c["lam"], c["ks"], c["vs"], **norm)
    got = call(kv, c, **kw)
    check(got, want, bound)
    return got


LENS = [0, 1, 15, 16, 17, 100, 257]
SHAPES = [  # heads, pairs, head_dim, block size
    (1, 1, 128, 16), (4, 1, 128, 16), (14, 2, 128, 16), (8, 1, 128, 32), (6, 2, 64, 16), (8, 8, 64, 32), (16, 2, 64, 64),
    (5, 1, 64, 16), (5, 1, 128, 48),
    # shapes outside the tiled kernels: odd head dims and block sizes, large groups
    (9, 1, 128, 16), (2, 1, 32, 16), (3, 3, 80, 16), (2, 2, 50, 7), (2, 1, 37, 5), (4, 2, 128, 24), (2, 1, 256, 16), (4, 2, 1, 16),
]


@pytest.mark.parametrize("cache", [torch.int8, torch.bfloat16, torch.float16], ids=["int8", "bf16", "fp16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("sharp", [1.0, 4.0])
def test_shapes(kv, cache, shape, sharp):
    heads, pairs, D, bs = shape
    c = make_case(hash(shape) & 0xfff, LENS, heads, pairs, D, bs, cache, sharp=sharp)
    out = verify(kv, c)
    assert out.shape == (len(LENS), heads, 2 * D) and (out[0] == 0).all()
    w = 1 + 0.2 * torch.randn(2 * D, generator=torch.Generator().manual_seed(1))
    out = verify(kv, c, norm_weight=w.to(DEV), norm_eps=1e-3, out_scale=0.3)
    assert (out[0] == 0).all()


@pytest.mark.parametrize("cache", [torch.int8, torch.bfloat16], ids=["int8", "bf16"])
@pytest.mark.parametrize("shape", [(14, 2, 128, 16), (4, 2, 64, 16), (3, 3, 80, 16)], ids=str)
@pytest.mark.parametrize("splits", [1, 2, 3, 7, 64, 1000])
def test_split_counts(kv, cache, shape, splits):
    heads, pairs, D, bs = shape
    c = make_case(3, [500, 1, 0, 333, 64], heads, pairs, D, bs, cache, sharp=2.0)
    verify(kv, c, num_splits=splits)


@pytest.mark.parametrize("qtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("cache", [torch.int8, torch.bfloat16, torch.float16], ids=["int8", "bf16", "fp16"])
def test_types_of_query_output_weights_and_indices(kv, qtype, cache):
    for D in (128, 64, 40):
        c = make_case(4, [70, 33], 6, 2, D, 16, cache, qtype=qtype, index=torch.int64)
        assert verify(kv, c).dtype == qtype
        out = torch.empty(2, 6, 2 * D, dtype=torch.float32, device=DEV)
        w = torch.rand(2 * D, device=DEV).to(torch.bfloat16)
        c["lam"] = c["lam"].to(torch.float16)
        assert verify(kv, c, norm_weight=w, out=out) is out
        c["lam"] = torch.tensor([0.7], device=DEV)
        verify(kv, c)


def test_strides(kv):
    """Queries, caches, tables and outputs that are views of larger tensors; a query and an output that start on an
    odd element."""
    for cache in (torch.int8, torch.bfloat16):
        for D in (128, 64):
            c = make_case(5, [130, 40, 0, 16], 6, 2, D, 16, cache)
            want = call(kv, c)
            B, H2 = c["q"].shape[:2]
            for shift in (0, 1, 3):
                big = torch.zeros(B, H2 + 4, D + 8, dtype=c["q"].dtype, device=DEV)
                q = big[:, 2:2 + H2, shift:shift + D]
                q.copy_(c["q"])
                out = torch.full((B, H2 // 2, 2 * D + 8), 9.0, dtype=c["q"].dtype, device=DEV)
                d = dict(c, q=q)
                call(kv, d, out=out[..., shift:shift + 2 * D])
                assert torch.equal(out[..., shift:shift + 2 * D], want)
                assert (out[..., :shift] == 9).all() and (out[..., shift + 2 * D:] == 9).all()
            # head-major pages (another order of the same rows), a fused K/V pool, padding between tokens
            kc = c["kc"].permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
            vc = c["vc"].permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
            verify(kv, dict(c, kc=kc, vc=vc))
            pool = torch.stack([c["kc"], c["vc"]], 1)
            verify(kv, dict(c, kc=pool[:, 0], vc=pool[:, 1]))
            wide = torch.zeros(*c["kc"].shape[:3], D + 24, dtype=cache, device=DEV)
            wide[..., :D] = c["kc"]
            verify(kv, dict(c, kc=wide[..., :D]))
            odd = torch.zeros(c["kc"].numel() + 1, dtype=cache, device=DEV)[1:].view(c["kc"].shape)
            odd.copy_(c["kc"])
            verify(kv, dict(c, kc=odd))
            bt = torch.stack([c["bt"], c["bt"]], 2)[..., 0]
            lens = torch.stack([c["lens"], c["lens"]], 1)[:, 0]
            verify(kv, dict(c, bt=bt, lens=lens))


@pytest.mark.parametrize("cache", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("D", [128, 64, 48])
def test_nothing_behind_the_last_token_is_used(kv, cache, D):
    """NaN and infinities behind every sequence's end, in unused blocks and behind the last table entry."""
    c = make_case(6, [1, 17, 30, 48, 0], 4, 2, D, 16, cache)
    want = call(kv, c)
    for bad in (float("nan"), float("inf")):
        kc, vc = c["kc"].clone(), c["vc"].clone()
        used = torch.zeros(kc.shape[:2], dtype=torch.bool, device=DEV)
        for b, n in enumerate(c["lens"].tolist()):
            for t in range(n):
                used[c["bt"][b, t // 16], t % 16] = True
        kc[~used] = bad
        vc[~used] = bad
        assert torch.equal(call(kv, dict(c, kc=kc, vc=vc)), want)


def test_large_magnitudes(kv):
    """Scores of several hundred, one token that takes everything, all keys equal, and lam of 0 and below."""
    for D in (128, 64, 72):
        c = make_case(7, [200, 65], 4, 2, D, 16, torch.int8, sharp=100.0)
        verify(kv, c)
        c["kc"][:] = 3
        verify(kv, c)
        c["lam"] = torch.tensor([0.0, -0.5, 1.0, 3.0], device=DEV)
        c["q"] = c["q"] / 100
        verify(kv, c)
        c["q"].zero_()
        verify(kv, c)


def test_maps_of_different_size(kv):
    """Queries of the two maps, and of the heads of a group, four orders of magnitude apart: each head has its own scale."""
    for D, heads in ((128, 4), (128, 7), (64, 4), (64, 7)):
        for small in (0, 1):
            c = make_case(21, [150, 31], heads, 1, D, 16, torch.int8, sharp=2.0)
            c["q"][:, small::2] *= 1e-4
            c["q"][:, 2] *= 30
            c["ks"][small::2] *= 1e4  # the scores of the small queries matter all the same
            verify(kv, c)


def test_bad_values_stay_in_their_head(kv):
    """A NaN or an infinity in one query head reaches that differential head only."""
    for cache in (torch.int8, torch.bfloat16):
        for D, heads in ((128, 4), (128, 7), (64, 4), (64, 7), (40, 3)):
            c = make_case(22, [150, 31], heads, 1, D, 16, cache)
            want = call(kv, c)
            c["q"][0, 3, 5] = float("nan")
            got = call(kv, c)
            assert torch.isnan(got[0, 1]).all()
            got[0, 1] = want[0, 1]
            assert torch.equal(got, want)


@pytest.mark.parametrize("cache", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("D", [128, 64, 48])
@pytest.mark.parametrize("heads", [4, 14])
def test_tokens_masked_by_an_infinite_key(kv, cache, D, heads):
    """A first block whose scores are -inf is as if it were not there; a sequence of nothing else attends to
    nothing."""
    c = make_case(23, [96, 33], heads, 2, D, 16, cache)
    c["q"][..., 0] = c["q"][..., 0].abs() + 0.5
    out = lambda: torch.empty(2, heads, 2 * D, dtype=torch.float32, device=DEV)
    rest = dict(c, bt=c["bt"][:, 1:].contiguous(), lens=c["lens"] - 16)
    kc = c["kc"].clone()
    kc[c["bt"][:, 0].long(), :, :, 0] = float("-inf")
    # one part: the masked block leaves sums of 0, and what follows is the same arithmetic
    assert torch.equal(call(kv, dict(c, kc=kc), num_splits=1, out=out()), call(kv, rest, num_splits=1, out=out()))
    # a block per part: the join adds the same six values in another order, each addition off by 2^-24 of sum p |v|
    a, b = call(kv, dict(c, kc=kc), num_splits=6, out=out()), call(kv, rest, num_splits=5, out=out())
    room = 16 * 2.0 ** -24 * c["vc"].float().abs().max().item() * (1 + c["lam"].abs().max().item())
    assert (a - b).abs().max().item() <= room
    kc[..., 0] = float("-inf")
    assert (call(kv, dict(c, kc=kc)) == 0).all()


@pytest.mark.parametrize("cache", [torch.int8, torch.float16], ids=["int8", "fp16"])
@pytest.mark.parametrize("D", [128, 64])
def test_a_crowd_far_below_one_token(kv, cache, D):
    """20000 tokens, each 2^-27 of a token that dominates but has no value: together they are the whole output, and each
    of them is below what fp16 holds next to 1."""
    n, bs = 20000, 16
    c = make_case(30, [n], 2, 1, D, bs, cache)
    first = c["bt"][0, 0].item()
    c["kc"].zero_()
    c["kc"][first, 0] = 100 if cache == torch.int8 else 2.0
    c["vc"].fill_(100 if cache == torch.int8 else 1.0)
    c["vc"][first, 0] = 0
    if cache == torch.int8:
        c["ks"].fill_(0.02)
        c["vs"].fill_(0.01)
    c["q"].fill_(27 / 2.0 / D ** 0.5 / 1.4426950408889634)
    c["lam"].fill_(0.25)
    out = torch.empty(1, 2, 2 * D, dtype=torch.float32, device=DEV)
    got = verify(kv, c, out=out)
    assert (got > 0.75 * 0.9 * n * 2.0 ** -27).all()


def test_equal_maps_cancel(kv):
    """The same queries and keys in both maps and lam = 1: what is left is rounding, whatever the length."""
    for D in (128, 64):
        c = make_case(8, [1000, 5], 2, 1, D, 16, torch.int8)
        c["q"][:, 1::2] = c["q"][:, 0::2]
        c["kc"][:, :, 1::2] = c["kc"][:, :, 0::2]
        c["ks"][1::2] = c["ks"][0::2]
        c["lam"].fill_(1.0)
        out = call(kv, c)
        # equal inputs go through equal steps: the maps agree to the last few bits of fp32
        assert out.abs().max() <= 2.0 ** -18


def test_agrees_with_two_ordinary_calls(kv):
    """lam = 0 is ordinary attention of the first map, half of V by half.  Both results are rounded to bf16 (2^-8 each),
    and both operators round queries and probabilities: 2 (2 ds + 2^-11) sum p |v| < 2^-9 with ds < 2^-11 and |v| < 0.8
    on average over any of these maps."""
    c = make_case(9, [300, 77, 1], 14, 2, 128, 16, torch.int8)
    c["lam"].zero_()
    got = call(kv, c).float()
    for half in range(2):
        pick = lambda t, i: t[:, :, i::2].contiguous()
        ref = kv.int8_paged_attention(c["q"][:, 0::2].contiguous(), pick(c["kc"], 0), pick(c["vc"], half), c["bt"], c["lens"],
                                      c["ks"][0::2].contiguous(), c["vs"][half::2].contiguous(), max_seq_len=512).float()
        torch.testing.assert_close(got[..., 128 * half:128 * (half + 1)], ref, rtol=2 ** -7, atol=2 ** -9)


def test_cache_written_by_the_cache_write(kv):
    """int8_kv_cache_write with the 2P heads and the same scale tensors, then the operator: K and V rows of 2D values
    seen as two heads are the same memory."""
    H, P, D, n = 6, 2, 128, 50
    g = torch.Generator(device=DEV).manual_seed(10)
    k = torch.randn(n, P, 2, D, generator=g, device=DEV).bfloat16()
    v = torch.randn(n, P, 2 * D, generator=g, device=DEV).bfloat16()
    ks, vs = torch.full((2 * P,), 0.03, device=DEV), torch.full((2 * P,), 0.03, device=DEV)
    kc = torch.zeros(8, 16, 2 * P, D, dtype=torch.int8, device=DEV)
    vc = torch.zeros(8, 16, P, 2 * D, dtype=torch.int8, device=DEV)
    bt = torch.tensor([[5, 2, 7, 0]], dtype=torch.int32, device=DEV)
    lens, none = torch.tensor([n], dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    slots, _ = kv.build_slot_mapping(bt, none, lens, 16, num_tokens=n)
    kv.int8_kv_cache_write(k.view(n, 2 * P, D), v.view(n, 2 * P, D), kc, vc.view(8, 16, 2 * P, D), slots, ks, vs)
    q = torch.randn(1, 2 * H, D, generator=g, device=DEV).bfloat16()
    c = dict(q=q, kc=kc, vc=vc.view(8, 16, 2 * P, D), bt=bt, lens=lens, ks=ks, vs=vs, lam=torch.full((H,), 0.4, device=DEV))
    verify(kv, c, norm_weight=torch.ones(2 * D, device=DEV), out_scale=0.2)


def test_lengths_beyond_the_table_and_bad_blocks(kv):
    """A length past what the table row can address is cut there; block ids outside the cache are never read."""
    for D in (128, 64, 40):
        for cache in (torch.int8, torch.float16):
            c = make_case(11, [48, 32], 4, 2, D, 16, cache)
            c["lens"] = torch.tensor([4800, 32], dtype=torch.int32, device=DEV)
            verify(kv, c)
            c["lens"] = torch.tensor([-3, 32], dtype=torch.int32, device=DEV)
            out = verify(kv, c)
            assert (out[0] == 0).all()
            c["bt"][0] = torch.tensor([10**6, -1, 2**31 - 1], dtype=torch.int32, device=DEV)
            c["lens"] = torch.tensor([48, 32], dtype=torch.int32, device=DEV)
            assert torch.isfinite(call(kv, c)[1]).all()


def test_long_cache_past_32_bit_offsets(kv):
    """A cache of more than 2^32 bytes whose used blocks lie at its end."""
    P, D, bs, blocks = 4, 128, 16, 280000  # 16 * 8 * 128 = 16 KB per block and tensor: 4.6 GB
    kc = torch.zeros(blocks, bs, 2 * P, D, dtype=torch.int8, device=DEV)
    vc = torch.zeros_like(kc)
    small = make_case(12, [40, 16], 8, P, D, bs, torch.int8)
    n = small["kc"].shape[0]
    kc[-n:], vc[-n:] = small["kc"], small["vc"]
    want = call(kv, small)
    got = call(kv, dict(small, kc=kc, vc=vc, bt=small["bt"] + (blocks - n)))
    assert torch.equal(got, want)


def test_several_tokens_of_one_sequence(kv):
    """Rows that repeat a sequence's table row with lengths of their own: a causal chunk of new tokens."""
    c = make_case(13, [70], 6, 2, 128, 16)
    lens = torch.tensor([66, 67, 68, 69, 70], dtype=torch.int32, device=DEV)
    q = torch.randn(5, 12, 128, device=DEV).bfloat16()
    verify(kv, dict(c, q=q, lens=lens, bt=c["bt"].expand(5, -1)))


def test_refusals(kv):
    c = make_case(14, [20, 30], 4, 2, 64, 16)
    call(kv, c)
    bf = dict(c, kc=c["kc"].bfloat16(), vc=c["vc"].bfloat16())
    bad = [
        (c, dict(kc=c["kc"][:, :, :3], vc=c["vc"][:, :, :3])), (c, dict(lam=c["lam"][:3])), (c, dict(lam=c["lam"].int())),
        (c, dict(lam=c["lam"].cpu())), (c, dict(q=c["q"][:, :6])), (c, dict(ks=c["ks"][:2])), (c, dict(vs=c["vs"].cpu())),
        (c, dict(bt=c["bt"].cpu())), (c, dict(bt=c["bt"].float())), (c, dict(lens=c["lens"][:1])), (c, dict(vc=c["vc"].bfloat16())),
        (bf, dict(vc=c["vc"].half())), (c, dict(kc=c["kc"].transpose(2, 3).contiguous().transpose(2, 3))),
    ]
    for base, change in bad:
        with pytest.raises(AssertionError):
            call(kv, dict(base, **change))
    for kw in (dict(norm_weight=torch.ones(64, device=DEV)), dict(norm_weight=torch.ones(128, device=DEV), norm_eps=0.0),
               dict(norm_weight=torch.ones(128)), dict(num_splits=0), dict(out=torch.empty(2, 4, 64, device=DEV)),
               dict(out=torch.empty(2, 4, 128, dtype=torch.int32, device=DEV))):
        with pytest.raises(AssertionError):
            call(kv, c, **kw)
    with pytest.raises(AssertionError):  # without an upper bound the lengths are read, and have to be positive
        call(kv, dict(c, lens=torch.tensor([0, 30], dtype=torch.int32, device=DEV)), max_seq_len=None)
    big = make_case(15, [20], 2, 1, 257, 16)
    with pytest.raises(AssertionError):
        call(kv, big)
    none = make_case(16, [20], 2, 1, 64, 16)
    assert call(kv, dict(none, q=none["q"][:0], bt=none["bt"][:0], lens=none["lens"][:0])).shape == (0, 2, 128)


def test_without_an_upper_bound(kv):
    c = make_case(17, [20, 75], 4, 2, 128, 16)
    assert torch.equal(call(kv, c, max_seq_len=None), call(kv, c, max_seq_len=75))
    assert kv.device_status() == 0


def test_captured_calls_and_two_streams(kv):
    """Two graphs captured on one stream, replayed on two: each has its own partial rows."""
    cases = [make_case(18 + i, [900, 300, 1], 14, 2, 128, 16) for i in range(2)]
    want = [call(kv, c) for c in cases]
    side = torch.cuda.Stream()
    graphs = []
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        call(kv, cases[0])  # the stream's status word exists before a capture
        for c in cases:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                out = call(kv, c)
            graphs.append((g, out))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(30):
        for (g, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for (_, out), w in zip(graphs, want):
        assert torch.equal(out, w)
    # new lengths, queries and blocks reach a replay
    cases[0]["lens"].copy_(torch.tensor([64, 0, 1], device=DEV))
    cases[0]["q"].mul_(-1)
    graphs[0][0].replay()
    torch.cuda.synchronize()
    assert torch.equal(graphs[0][1], call(kv, cases[0]))
    assert kv.device_status() == 0


def test_whole_step(kv):
    """A differential layer's serving steps: tables grown on the GPU, the write through the slots, the attention
    through the tables, against the definition over the written cache."""
    H, P, D, bs, R, width, blocks = 4, 2, 64, 16, 3, 5, 14
    g = torch.Generator(device=DEV).manual_seed(20)
    kc = torch.zeros(blocks, bs, 2 * P, D, dtype=torch.int8, device=DEV)
    vc = torch.zeros_like(kc)
    ks, vs = torch.full((2 * P,), 0.03, device=DEV), torch.full((2 * P,), 0.02, device=DEV)
    bt = torch.zeros(R, width, dtype=torch.int32, device=DEV)
    lens = torch.zeros(R, dtype=torch.int32, device=DEV)
    free = torch.arange(blocks, dtype=torch.int32, device=DEV).flip(0).contiguous()
    cursor = torch.zeros(1, dtype=torch.int64, device=DEV)
    new = torch.tensor([30, 1, 16], dtype=torch.int32, device=DEV)
    for step in range(5):
        total = int(new.sum())
        plan = kv.build_block_tables(bt, lens, new, free, cursor, bs, num_tokens=total)
        lens, cursor = plan.seq_lens, plan.free_cursor
        k, v = (torch.randn(total, 2 * P, D, generator=g, device=DEV).bfloat16() for _ in range(2))
        kv.int8_kv_cache_write(k, v, kc, vc, plan.slot_mapping, ks, vs)
        q = torch.randn(R, 2 * H, D, generator=g, device=DEV).bfloat16()
        c = dict(q=q, kc=kc, vc=vc, bt=bt, lens=lens, ks=ks, vs=vs, lam=torch.full((1,), 0.6, device=DEV))
        verify(kv, c, norm_weight=torch.ones(2 * D, device=DEV), out_scale=0.4)
        new = torch.ones_like(new)
