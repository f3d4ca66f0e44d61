"""Differential paged decode attention in 64 bits, from its definition, with a bound of what the operator's own roundings
may move each output."""

from __future__ import annotations

import math

import torch


def diff_paged_attention(query, key_cache, value_cache, block_tables, seq_lens, lam, k_scale=None, v_scale=None,
                         norm_weight=None, norm_eps=1e-5, out_scale=1.0):
    """(out [B, H, 2D] float64, bound [B, H, 2D] float64).

    The bound, without the rounding of the output itself: the operator may hold each query head as 16-bit fixed point
    over its largest element (step amax / 32000, off by at most half of it), or round it to the cache's 16-bit type
    (2^-8 relative for bf16, of which fp16's 2^-11 is a part), and each probability as a 16-bit float (dp = 2^-11
    relative for fp16, 2^-8 for a bf16 cache), in the product and in the sum it is divided by alike.  A score moves by at
    most ds = max_n sum_d |dq_d k_nd| / sqrt(D); with it every weight by a factor within exp(+-ds), numerator and
    denominator both, and a map's output by 2 ds sum_n p_n |v_n|.  Rounded weights p (1 + e), |e| <= dp, move
    o = sum p v / sum p by at most dp sum p |v - o| <= 2 dp sum p |v| (normalised p).  Where fp16 runs out of
    exponents, 2^-32 below the largest probability, a weight is off by at most that much, which moves o by at most
    2^-32 sum (|v| + |o|).  fp32 sums, exponentials and
    divisions add less than 2^-14 of the same.  The norm divides by the row's root mean square r and moves with it, which at most doubles
    a relative error.
    """
    B, H2, D = query.shape
    H, P, bs = H2 // 2, key_cache.shape[2] // 2, key_cache.shape[1]
    group = H // P
    int8 = key_cache.dtype == torch.int8
    dp = 2.0 ** -8 if key_cache.dtype == torch.bfloat16 else 2.0 ** -11
    out = torch.zeros(B, H, 2 * D, dtype=torch.float64)
    bound = torch.zeros_like(out)
    query, bt = query.cpu().double(), block_tables.cpu().long()
    kc, vc, lam = key_cache.cpu(), value_cache.cpu(), lam.cpu().double().expand(H)
    for b, n in enumerate(int(x) for x in seq_lens):
        n = min(n, bt.shape[1] * bs)
        if n <= 0:
            continue
        token = torch.arange(n)
        block, offset = bt[b, token // bs], token % bs
        k, v = kc[block, offset].double(), vc[block, offset].double()  # [n, 2P, D]
        if int8:
            k = k * k_scale.cpu().double().clamp_min(1e-6)[:, None]
            v = v * v_scale.cpu().double().clamp_min(1e-6)[:, None]
        v = v.reshape(n, P, 2 * D)
        for h in range(H):
            g = h // group
            for m in range(2):
                q = query[b, 2 * h + m]
                p = torch.softmax(k[:, 2 * g + m] @ q / math.sqrt(D), 0)
                dq = q.abs().amax().expand(D) / 64000.0 if int8 else q.abs() * (2.0 ** -8)
                ds = float((k[:, 2 * g + m].abs() @ dq).amax()) / math.sqrt(D)
                f = 1.0 if m == 0 else float(lam[h])
                out[b, h] += (1.0 if m == 0 else -1.0) * f * (p @ v[:, g])
                bound[b, h] += abs(f) * 2.0 ** -32 * (v[:, g].abs().sum(0) + n * (p @ v[:, g]).abs())
                bound[b, h] += abs(f) * math.exp(2 * ds) * (2 * ds + 2 * dp + 2.0 ** -14) * (p @ v[:, g].abs())
    bound *= abs(out_scale)
    scaled = out * out_scale
    if norm_weight is not None:
        w = norm_weight.cpu().double()
        r = (out.square().mean(-1, keepdim=True) + norm_eps).sqrt()
        # y = o w / r: |dy| <= |w| (|do| + |o| |dr| / r) / r, and |dr| <= root mean square of do
        spread = bound.square().mean(-1, keepdim=True).sqrt()
        bound = w.abs() / r * (bound + out.abs() * spread / r) * 1.5  # 1.5: second-order terms
        scaled = scaled / r * w
    return scaled, bound


def check(got, want, bound):
    """Every output within the bound plus half a step of its own type."""
    eps = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).smallest_normal if got.dtype == torch.float16 else 1e-30
    err = (got.cpu().double() - want).abs()
    allowed = bound + eps * (want.abs() + bound) + 2.0 ** -20 * want.abs() + tiny
    assert torch.isfinite(got).all()
    worst = float((err / allowed).amax()) if err.numel() else 0.0
    assert worst <= 1.0, f"error is {worst:.3g} times what the roundings allow (largest {float(err.amax()):.3g})"
    return worst
