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

from functools import lru_cache
from typing import Optional

import torch

from . import _lib
from .ops import (_FLOAT_CODES, _as_f32_scale, _call, _max_seq_len, _require_lib, _sm_count, _status_ptr,
                  _stream_ptr)

_INDEX_CODES = {torch.int32: 0, torch.int64: 1}
_CACHE_CODES = {torch.int8: _lib.INT8, torch.bfloat16: _lib.BF16, torch.float16: _lib.FP16}


@lru_cache(maxsize=1024)
def _workspace_bytes(B, H, P, D, max_seq, block_size, splits, sm_count) -> int:
    return _require_lib().int8kv_diff_workspace_bytes(B, H, P, D, max_seq, block_size, splits, sm_count)


def _run(int8, query, key_cache, value_cache, block_tables, seq_lens, k_scale, v_scale, lam, norm_weight, norm_eps,
         out_scale, num_splits, max_seq_len, out):
    device = query.device
    assert device.type == "cuda" and query.ndim == 3 and key_cache.ndim == 4
    for t in (key_cache, value_cache, block_tables, seq_lens, lam):
        assert t.device == device
    B, Hq, D = query.shape
    num_blocks, block_size, Hkv, cache_D = key_cache.shape
    kc_st, vc_st, bt_st = key_cache.stride(), value_cache.stride(), block_tables.stride()
    assert value_cache.shape == key_cache.shape and cache_D == D and kc_st[3] == 1 and vc_st[3] == 1
    assert Hq % 2 == 0 and Hkv % 2 == 0 and Hkv > 0 and Hq % Hkv == 0 and 0 < D <= 256
    assert block_tables.ndim == 2 and block_tables.shape[0] == B and seq_lens.ndim == 1 and seq_lens.shape[0] == B
    q_code, lam_code = _FLOAT_CODES.get(query.dtype), _FLOAT_CODES.get(lam.dtype)
    bt_code, sl_code = _INDEX_CODES.get(block_tables.dtype), _INDEX_CODES.get(seq_lens.dtype)
    assert None not in (q_code, lam_code, bt_code, sl_code)
    H, P = Hq // 2, Hkv // 2
    lams = lam.numel()
    assert lam.ndim <= 1 and (lams == 1 or lams == H)
    norm_ptr = norm_code = 0
    if norm_weight is not None:
        norm_code = _FLOAT_CODES.get(norm_weight.dtype)
        assert norm_code is not None and norm_weight.shape == (2 * D,) and norm_weight.device == device and norm_eps > 0
        norm_weight = norm_weight.contiguous()
        norm_ptr = norm_weight.data_ptr()
    if out is None:
        out, out_code = query.new_empty((B, H, 2 * D)), q_code
    else:
        out_code = _FLOAT_CODES.get(out.dtype)
        assert out.shape == (B, H, 2 * D) and out_code is not None and out.device == device
    splits = 0
    lib = _require_lib()
    if num_splits is not None:
        assert int(num_splits) >= 1
        splits = min(int(num_splits), lib.int8kv_max_splits())
    max_seq = _max_seq_len(seq_lens, block_tables, block_size, max_seq_len)
    if B == 0:
        return out
    if seq_lens.stride(0) != 1:
        seq_lens = seq_lens.contiguous()
    width = block_tables.shape[1]
    limit = width * block_size
    nbytes = _workspace_bytes(B, H, P, D, min(max_seq, limit) if max_seq > 0 else limit, block_size, splits, _sm_count(device))
    # The partial rows belong to the call: memory of the current stream, or of the pool of the graph that captures the
    # call.  The status word is the stream's, the one that device_status() reads.
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
    packed = _lib.DIFF_ARGS.pack(
        query.data_ptr(), key_cache.data_ptr(), value_cache.data_ptr(), block_tables.data_ptr(), seq_lens.data_ptr(),
        k_scale.data_ptr() if int8 else 0, v_scale.data_ptr() if int8 else 0, lam.data_ptr(), norm_ptr, out.data_ptr(),
        ws.data_ptr(), _status_ptr(device), _stream_ptr(device),
        *query.stride(), *kc_st, *vc_st, *bt_st, *out.stride(),
        0 if lams == 1 else lam.stride(0), B, H, P, D, num_blocks, block_size, width, max_seq, splits, nbytes,
        q_code, _CACHE_CODES[key_cache.dtype], lam_code, norm_code, out_code, bt_code, sl_code,
        norm_eps, out_scale,
    )
    rc = _call(device, lib.int8kv_paged_diff_attn, packed)
    if rc != _lib.OK:
        _lib.check("int8kv_paged_diff_attn", rc)
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
    assert key_cache.ndim == 4 and k_scale.shape == v_scale.shape == key_cache.shape[2:3]
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
    """The same over a bf16 or fp16 paged cache, the same-run baseline of the INT8 form.  The query is rounded to the
    caches' type, so with fp16 caches it has to lie in fp16's range.  A key that makes a token's scores -inf masks it."""
    assert key_cache.dtype in (torch.bfloat16, torch.float16) and value_cache.dtype == key_cache.dtype
    return _run(False, query, key_cache, value_cache, block_tables, seq_lens, None, None, lam, norm_weight, norm_eps,
                out_scale, num_splits, max_seq_len, out)
