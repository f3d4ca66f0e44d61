"""Differential decode attention over the paged caches: the difference of two softmax maps, per head, with a learned
weight.

A layer has H differential heads over P pairs of KV heads.  Everything around the operator keeps its ordinary shape, with
2 H query heads and 2 P KV heads of head_dim D: the caches are those that int8_kv_cache_write fills (K heads 2g and
2g + 1 are the keys of pair g's two maps, V heads 2g and 2g + 1 the two halves of its value rows of 2 D), the scales
are the [2 P] tensors they were written with, block_tables and seq_lens are the same.

    o[b, h] = (softmax(q[b, 2h] K[2g]^T / sqrt(D)) - lam[h] softmax(q[b, 2h+1] K[2g+1]^T / sqrt(D))) [V[2g] | V[2g+1]]

with g = h // (H // P), optionally followed by a root-mean-square norm over the 2 D values.  One query token per row;
several new tokens of one sequence are several rows that repeat its block-table row, each with its own seq_len.

Argument violations raise AssertionError, as in the other operators.  The reference has no counterpart.
"""

from __future__ import annotations

from typing import Optional

import torch

from . import _lib
from .block_tables import _on_device
from .ops import (_FLOAT_CODES, _as_f32_scale, _check_decode_args, _max_seq_len, _require_lib, _sm_count, _stream_ptr,
                  _workspace)


def _run(int8, query, key_cache, value_cache, block_tables, seq_lens, k_scale, v_scale, lam, norm_weight, norm_eps,
         out_scale, num_splits, max_seq_len, out):
    B, Hq, Hkv, D, block_size = _check_decode_args(query, key_cache, value_cache, block_tables, seq_lens)
    device = query.device
    assert Hq % 2 == 0 and Hkv % 2 == 0 and D <= 256
    H, P = Hq // 2, Hkv // 2
    for t in (key_cache, value_cache, block_tables, seq_lens, lam):
        assert t.device == device
    assert lam.dtype in _FLOAT_CODES and lam.ndim <= 1 and lam.numel() in (1, H)
    if norm_weight is not None:
        assert norm_weight.dtype in _FLOAT_CODES and norm_weight.shape == (2 * D,) and norm_weight.device == device
        assert norm_eps > 0
        norm_weight = norm_weight.contiguous()
    assert num_splits is None or int(num_splits) >= 1
    max_seq = _max_seq_len(seq_lens, block_tables, block_size, max_seq_len)
    if out is None:
        out = torch.empty((B, H, 2 * D), device=device, dtype=query.dtype)
    else:
        assert out.shape == (B, H, 2 * D) and out.dtype in _FLOAT_CODES and out.device == device
    if B == 0:
        return out
    if seq_lens.stride(0) != 1:
        seq_lens = seq_lens.contiguous()
    lib = _require_lib()
    splits = 0 if num_splits is None else min(int(num_splits), lib.int8kv_max_splits())
    limit = block_tables.shape[1] * block_size
    nbytes = lib.int8kv_diff_workspace_bytes(B, H, P, D, min(max_seq, limit) if max_seq > 0 else limit, block_size,
                                             splits, _sm_count(device))
    with _on_device(device):
        # The partial rows belong to the call: memory of the current stream, or of the pool of the graph that captures
        # the call.  The status word is the stream's, the one that device_status() reads.
        ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
        shared = _workspace(device, 16)
        status = shared.data_ptr() + lib.int8kv_workspace_status_offset(shared.numel())
        head = (query.data_ptr(), _FLOAT_CODES[query.dtype], _lib.i64(query.stride()), B, H, P, D,
                key_cache.data_ptr(), value_cache.data_ptr())
        mid = (_lib.i64(key_cache.stride()), _lib.i64(value_cache.stride()), key_cache.shape[0], block_size,
               block_tables.data_ptr(), int(block_tables.dtype == torch.int64), _lib.i64(block_tables.stride()),
               block_tables.shape[1], seq_lens.data_ptr(), int(seq_lens.dtype == torch.int64), max_seq)
        tail = (lam.data_ptr(), _FLOAT_CODES[lam.dtype], 0 if lam.numel() == 1 else lam.stride(0),
                0 if norm_weight is None else norm_weight.data_ptr(),
                0 if norm_weight is None else _FLOAT_CODES[norm_weight.dtype], float(norm_eps), float(out_scale),
                out.data_ptr(), _FLOAT_CODES[out.dtype], _lib.i64(out.stride()),
                splits, ws.data_ptr(), nbytes, status, _stream_ptr(device))
        if int8:
            rc = lib.int8kv_paged_diff_attn_int8(*head, *mid, k_scale.data_ptr(), v_scale.data_ptr(), *tail)
        else:
            rc = lib.int8kv_paged_diff_attn_bf16(*head, _FLOAT_CODES[key_cache.dtype], *mid, *tail)
    _lib.check("int8kv_paged_diff_attn_int8" if int8 else "int8kv_paged_diff_attn_bf16", rc)
    return out


def int8_paged_diff_attention(
    query: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    block_tables: torch.Tensor,
    seq_lens: torch.Tensor,
    k_scale: torch.Tensor,
    v_scale: torch.Tensor,
    lam: torch.Tensor,
    *,
    norm_weight: Optional[torch.Tensor] = None,
    norm_eps: float = 1e-5,
    out_scale: float = 1.0,
    num_splits: Optional[int] = None,
    max_seq_len: Optional[int] = None,
    out: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Differential decode attention of query [B, 2H, D] over an INT8 paged cache [num_blocks, BS, 2P, D]; returns
    [B, H, 2D] in query.dtype.

    k_scale / v_scale: [2P], the scales of int8_kv_cache_write.  lam: [H], or one value for all heads, any float type.
    norm_weight [2D]: out = out_scale * norm_weight * o / sqrt(mean(o^2) + norm_eps); without it out = out_scale * o.
    num_splits / max_seq_len / out as in int8_paged_attention: with max_seq_len the call does not synchronise, and
    sequences of length 0 (padding rows) yield zeros.
    """
    assert key_cache.dtype == torch.int8 and value_cache.dtype == torch.int8
    assert k_scale.device == query.device and v_scale.device == query.device
    assert k_scale.ndim == 1 and v_scale.ndim == 1
    assert k_scale.numel() == key_cache.shape[2] and v_scale.numel() == key_cache.shape[2]
    return _run(True, query, key_cache, value_cache, block_tables, seq_lens, _as_f32_scale(k_scale),
                _as_f32_scale(v_scale), lam, norm_weight, norm_eps, out_scale, num_splits, max_seq_len, out)


def bf16_paged_diff_attention(
    query: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    block_tables: torch.Tensor,
    seq_lens: torch.Tensor,
    lam: torch.Tensor,
    *,
    norm_weight: Optional[torch.Tensor] = None,
    norm_eps: float = 1e-5,
    out_scale: float = 1.0,
    num_splits: Optional[int] = None,
    max_seq_len: Optional[int] = None,
    out: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """The same over a bf16 or fp16 paged cache, the same-run baseline of the INT8 form."""
    assert key_cache.dtype in (torch.bfloat16, torch.float16) and value_cache.dtype == key_cache.dtype
    return _run(False, query, key_cache, value_cache, block_tables, seq_lens, None, None, lam, norm_weight, norm_eps,
                out_scale, num_splits, max_seq_len, out)
