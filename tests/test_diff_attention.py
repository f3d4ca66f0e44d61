"""Differential attention without a GPU: the oracle against the elementary formula, refusals of host tensors, and the
argument checks of the C ABI."""

import pytest
import torch

from conftest import package
from oracle.diff_attention import diff_paged_attention


def test_oracle_is_the_difference_of_two_ordinary_attentions():
    """Against the fp32 oracle of ordinary decode attention, run once per map and half of V."""
    import oracle

    torch.manual_seed(0)
    B, H, P, D, bs = 2, 6, 2, 16, 16
    q = torch.randn(B, 2 * H, D)
    kc, vc = torch.randn(5, bs, 2 * P, D, dtype=torch.float64).to(torch.bfloat16), torch.randn(5, bs, 2 * P, D).to(torch.bfloat16)
    bt = torch.tensor([[3, 1, 0], [4, 2, 0]])
    lens, lam = [40, 7], torch.rand(H)
    want, _ = diff_paged_attention(q, kc, vc, bt, lens, lam)
    pick = lambda c, m: c[:, :, m::2].contiguous()
    for half in range(2):
        maps = [oracle.float_paged_attention_oracle(q[:, m::2].contiguous(), pick(kc, m), pick(vc, half), bt, lens) for m in range(2)]
        got = maps[0] - lam[None, :, None] * maps[1]
        assert (got - want[..., half * D:(half + 1) * D]).abs().max() < 1e-5


def test_entry_points_refuse_host_tensors(kv):
    q, c = torch.zeros(1, 4, 64), torch.zeros(1, 16, 2, 64, dtype=torch.int8)
    args = (torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32))
    with pytest.raises(AssertionError):
        kv.int8_paged_diff_attention(q, c, c, *args, torch.ones(2), torch.ones(2), torch.ones(2))
    with pytest.raises(AssertionError):
        kv.bf16_paged_diff_attention(q, c.bfloat16(), c.bfloat16(), *args, torch.ones(2))


def test_c_abi_argument_checks():
    lm = package("_lib")
    lib = lm.load()
    p = 256  # never dereferenced: every call below is refused or empty

    def call(B=2, H=4, P=2, D=128, bs=16, width=4, q=p, lam=p, ks=p, out=p, qd=lm.BF16, cd=lm.INT8, ld=lm.FP32, norm=0, eps=1e-5,
             splits=1, ws=p, ws_bytes=1 << 20, last=1):
        return lib.int8kv_paged_diff_attn(lm.DIFF_ARGS.pack(
            q, p, p, p, p, ks, p, lam, norm, out, ws, 0, 0, 512, 128, 1, 8192, 512, 128, last, 8192, 512, 128, last, width, 1, 1024,
            256, 1, 1, B, H, P, D, 4, bs, width, 64, splits, ws_bytes, qd, cd, ld, lm.FP32, lm.BF16, 0, 0, eps, 1.0))

    assert lib.int8kv_paged_diff_attn(None) == lm.E_NULLPTR
    assert call(B=0) == lm.OK
    assert call(B=-1) == lm.E_BAD_SHAPE and call(H=3) == lm.E_BAD_SHAPE and call(P=0) == lm.E_BAD_SHAPE
    assert call(bs=0) == lm.E_BAD_SHAPE and call(bs=2**32 + 16) == lm.E_BAD_SHAPE and call(B=2**31) == lm.E_BAD_SHAPE
    assert call(splits=-1) == lm.E_BAD_SHAPE and call(splits=1000) == lm.E_BAD_SHAPE and call(width=-1) == lm.E_BAD_SHAPE
    assert call(qd=lm.INT8) == lm.E_BAD_DTYPE and call(ld=-1) == lm.E_BAD_DTYPE and call(cd=lm.FP32) == lm.E_BAD_DTYPE
    assert call(norm=p, eps=0.0) == lm.E_BAD_SHAPE and call(norm=p, eps=float("nan")) == lm.E_BAD_SHAPE
    assert call(D=257) == lm.E_UNSUPPORTED and call(last=2) == lm.E_UNSUPPORTED and call(H=65536, P=1) == lm.E_UNSUPPORTED
    for missing in ("q", "lam", "ks", "out"):
        assert call(**{missing: 0}) == lm.E_NULLPTR
    need = lib.int8kv_diff_workspace_bytes(2, 4, 2, 128, 64, 16, 1, 148)
    assert need == 2 * 8 * 260 * 4
    assert call(ws=0) == lm.E_WORKSPACE and call(ws_bytes=need - 1) == lm.E_WORKSPACE and call(ws=264) == lm.E_WORKSPACE
    assert lib.int8kv_diff_workspace_bytes(2, 3, 2, 128, 64, 16, 1, 148) == -1
