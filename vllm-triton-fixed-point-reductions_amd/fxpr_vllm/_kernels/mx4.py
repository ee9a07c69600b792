"""The paged KV cache in 4 bits: its write, its read back and the attention over it
(csrc/cache_mx4.hip, csrc/attn_mx4*.hip).

Codes [num_blocks, 2, block_size, num_kv_heads, head_size / 2] and scales
[num_blocks, 2, block_size, num_kv_heads, head_size / 32], both uint8: 32 consecutive
elements share a power-of-two scale byte, an element is a 4-bit E2M1 code (the format
in bytes: include/fxpr.h). empty_cache() allocates the pair. No counterpart in the
reference, whose backend refuses a quantised cache
(fxpr_vllm/attention_backend.py:40-277).
"""

from __future__ import annotations

import math

import torch

from .. import _hip
from .fxp import fxp_constants

HEAD_SIZES = (64, 128, 256)
BLOCK = 32  # elements that share a scale
_FLOATS = (torch.float16, torch.bfloat16, torch.float32)
_RCP_LN2 = 1.4426950408889634


def empty_cache(num_blocks: int, block_size: int, num_kv_heads: int, head_size: int,
                device: torch.device | str) -> tuple[torch.Tensor, torch.Tensor]:
    """An uninitialised (kv_codes, kv_scales) pair in the order that attention reads
    fastest: per block, K or V and head, the block's code rows and then its scales,
    in one allocation of num_blocks * 2 * num_kv_heads * block_size * head_size * 17 / 32
    bytes."""
    if head_size not in HEAD_SIZES:
        raise ValueError(f"empty_cache: head_size must be one of {HEAD_SIZES}, got {head_size}")
    if num_blocks < 0 or num_kv_heads <= 0 or block_size <= 0 or block_size % 16:
        raise ValueError("empty_cache: num_blocks >= 0, num_kv_heads > 0 and a block_size of whole 16s")
    code, scale = head_size // 2, head_size // BLOCK
    raw = torch.empty(num_blocks, 2, num_kv_heads, block_size * (code + scale), dtype=torch.uint8, device=device)
    codes, scales = raw.split([block_size * code, block_size * scale], -1)
    shape = (num_blocks, 2, num_kv_heads, block_size)
    return (codes.unflatten(-1, (block_size, code)).view(*shape, code).transpose(2, 3),
            scales.unflatten(-1, (block_size, scale)).view(*shape, scale).transpose(2, 3))


def _check_cache(what: str, codes: torch.Tensor, scales: torch.Tensor) -> None:
    if not (codes.is_cuda and scales.is_cuda):
        raise RuntimeError(f"{what}: tensors must be CUDA")
    if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
        raise TypeError(f"{what}: kv_codes and kv_scales must be uint8")
    if codes.dim() != 5 or codes.shape[1] != 2:
        raise ValueError(f"{what}: kv_codes must be (num_blocks, 2, block_size, num_kv_heads, head_size / 2)")
    if 2 * codes.shape[4] not in HEAD_SIZES:
        raise ValueError(f"{what}: head_size must be one of {HEAD_SIZES}, got {2 * codes.shape[4]}")
    if scales.dim() != 5 or scales.shape[:4] != codes.shape[:4] or scales.shape[4] * 16 != codes.shape[4]:
        raise ValueError(f"{what}: kv_scales must be (num_blocks, 2, block_size, num_kv_heads, head_size / 32)")
    if codes.stride(4) != 1 or scales.stride(4) != 1:
        raise ValueError(f"{what}: kv_codes and kv_scales must be contiguous along a row")
    if max(codes.shape[2:4]) > 1 << 30:
        raise ValueError(f"{what}: block_size and num_kv_heads must be at most 2^30")


def _same_device(what: str, first: torch.Tensor, *others: torch.Tensor) -> None:
    if any(t.device != first.device for t in others):
        raise RuntimeError(f"{what}: tensors must be on one device")


def _rows(t: torch.Tensor) -> torch.Tensor:
    """`t` [tokens, heads, head_size] with 16-byte aligned rows (a copy where they are not)."""
    n = t.element_size()
    if t.stride(2) == 1 and (t.stride(0) * n) % 16 == 0 and (t.stride(1) * n) % 16 == 0 and t.data_ptr() % 16 == 0:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _slots(what: str, slot_mapping: torch.Tensor, least: int) -> torch.Tensor:
    if slot_mapping.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{what}: slot_mapping must be int32 or int64")
    if slot_mapping.dim() != 1 or slot_mapping.shape[0] < least:
        raise ValueError(f"{what}: slot_mapping must be 1-D with one slot per token")
    return slot_mapping.to(torch.int64).contiguous()


def reshape_and_cache_run(key: torch.Tensor, value: torch.Tensor, kv_codes: torch.Tensor, kv_scales: torch.Tensor,
                          slot_mapping: torch.Tensor) -> None:
    what = "reshape_and_cache_mx4"
    if not (key.is_cuda and value.is_cuda and slot_mapping.is_cuda):
        raise RuntimeError(f"{what}: tensors must be CUDA")
    _check_cache(what, kv_codes, kv_scales)
    if key.dtype not in _FLOATS:
        raise TypeError(f"{what}: unsupported dtype {key.dtype}; expected one of {_FLOATS}")
    if value.dtype != key.dtype:
        raise TypeError(f"{what}: key and value must share a dtype")
    _same_device(what, kv_codes, kv_scales, key, value, slot_mapping)
    num_blocks, _, block_size, num_kv_heads, code = kv_codes.shape
    if key.dim() == 2 and key.shape[1] == num_kv_heads * 2 * code:
        key = key.unflatten(1, (num_kv_heads, 2 * code))
    if value.dim() == 2 and value.shape[1] == num_kv_heads * 2 * code:
        value = value.unflatten(1, (num_kv_heads, 2 * code))
    if key.dim() != 3 or key.shape != value.shape or tuple(key.shape[1:]) != (num_kv_heads, 2 * code):
        raise ValueError(f"{what}: key / value must be [num_tokens, num_kv_heads, head_size] matching the cache")
    num_tokens = key.shape[0]
    slots = _slots(what, slot_mapping, num_tokens)
    if num_tokens == 0:
        return
    key, value = _rows(key), _rows(value)
    with torch.cuda.device(kv_codes.device):
        _hip.call(
            "fxpr_reshape_and_cache_mx4", key.data_ptr(), value.data_ptr(), kv_codes.data_ptr(), kv_scales.data_ptr(),
            _hip.DTYPE_CODE[key.dtype], slots.data_ptr(), num_tokens, num_kv_heads, 2 * code, block_size, num_blocks,
            key.stride(0), key.stride(1), value.stride(0), value.stride(1), *kv_codes.stride()[:4],
            *kv_scales.stride()[:4], _hip.stream_ptr(kv_codes.device),
        )


def gather_cache_run(kv_codes: torch.Tensor, kv_scales: torch.Tensor, slot_mapping: torch.Tensor,
                     out_dtype: torch.dtype) -> tuple[torch.Tensor, torch.Tensor]:
    what = "gather_cache_mx4"
    if not slot_mapping.is_cuda:
        raise RuntimeError(f"{what}: tensors must be CUDA")
    _check_cache(what, kv_codes, kv_scales)
    if out_dtype not in _FLOATS:
        raise TypeError(f"{what}: unsupported output dtype {out_dtype}; expected one of {_FLOATS}")
    _same_device(what, kv_codes, kv_scales, slot_mapping)
    slots = _slots(what, slot_mapping, 0)
    num_blocks, _, block_size, num_kv_heads, code = kv_codes.shape
    key = torch.empty(slots.shape[0], num_kv_heads, 2 * code, dtype=out_dtype, device=kv_codes.device)
    value = torch.empty_like(key)
    if key.numel():
        with torch.cuda.device(kv_codes.device):
            _hip.call(
                "fxpr_gather_cache_mx4", kv_codes.data_ptr(), kv_scales.data_ptr(), key.data_ptr(), value.data_ptr(),
                _hip.DTYPE_CODE[out_dtype], slots.data_ptr(), slots.shape[0], num_kv_heads, 2 * code, block_size,
                num_blocks, *kv_codes.stride()[:4], *kv_scales.stride()[:4], _hip.stream_ptr(kv_codes.device),
            )
    return key, value


def unified_attention_run(
    q: torch.Tensor,
    kv_codes: torch.Tensor,
    kv_scales: torch.Tensor,
    o: torch.Tensor,
    query_start_loc: torch.Tensor,
    seq_lens: torch.Tensor,
    block_table: torch.Tensor,
    max_query_len: int,
    alibi_slopes: torch.Tensor | None,
    is_causal: bool,
    softmax_scale: float | None,
    fxp_int_bits: int,
    fxp_frac_bits: int,
    logit_softcap: float,
    window_size: int,
    num_kv_splits: int,
) -> None:
    what = "unified_attention_mx4_fxp"
    meta = (query_start_loc, seq_lens, block_table)
    if not (q.is_cuda and o.is_cuda and all(t.is_cuda for t in meta)):
        raise RuntimeError(f"{what}: tensors must be CUDA")
    _check_cache(what, kv_codes, kv_scales)
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError(f"{what}: unsupported q dtype {q.dtype}; expected float16 or bfloat16")
    if o.dtype != q.dtype:
        raise TypeError(f"{what}: o must share dtype with q")
    for name, t in zip(("query_start_loc", "seq_lens", "block_table"), meta):
        if t.dtype != torch.int32:
            raise TypeError(f"{name} must be int32")
    if num_kv_splits < 0:
        raise ValueError(f"num_kv_splits must be >= 0, got {num_kv_splits}")
    has_alibi = alibi_slopes is not None and alibi_slopes.numel() > 0
    if has_alibi and alibi_slopes.dtype != torch.float32:
        raise TypeError("alibi_slopes must be float32")
    fxp_constants(int(fxp_int_bits), int(fxp_frac_bits))
    _same_device(what, q, kv_codes, kv_scales, o, *meta, *([alibi_slopes] if has_alibi else []))
    num_blocks, _, page_size, num_kv_heads, code = kv_codes.shape
    if q.dim() != 3:
        raise ValueError("q must be (num_tokens, num_heads, head_dim)")
    num_tokens, num_heads, head_dim = q.shape
    if num_kv_heads == 0 or num_heads == 0 or num_heads % num_kv_heads != 0:
        raise ValueError("num_heads must be divisible by num_kv_heads")
    if 2 * code != head_dim or o.shape != q.shape:
        raise ValueError("q, o and the cache's head sizes must agree")
    if page_size < 16 or page_size & (page_size - 1):
        raise ValueError(f"{what}: the cache's block_size must be a power of two, 16 or more, got {page_size}")
    if has_alibi and alibi_slopes.numel() != num_heads:
        raise ValueError("alibi_slopes must have one slope per head")
    if seq_lens.dim() != 1 or query_start_loc.dim() != 1 or query_start_loc.shape[0] != seq_lens.shape[0] + 1:
        raise ValueError("query_start_loc must be 1-D with one more element than seq_lens")
    num_requests = seq_lens.shape[0]
    if num_requests == 0 or num_tokens == 0:
        return
    if block_table.numel() % num_requests or (block_table.dim() == 2 and block_table.shape[0] < num_requests):
        raise ValueError("block_table must have a row per request")
    q = _rows(q)
    # (rows of no request stay as they are)
    out = o if o.stride(2) == 1 else o.clone(memory_format=torch.contiguous_format)
    bt = block_table if block_table.dim() == 2 else block_table.reshape(num_requests, -1)
    if bt.stride(1) != 1:
        bt = bt.contiguous()
    qsl, sl = query_start_loc.contiguous(), seq_lens.contiguous()
    alibi = alibi_slopes.contiguous() if has_alibi else None
    scale = softmax_scale if softmax_scale is not None else 1.0 / math.sqrt(head_dim)
    softcap = float(logit_softcap) * _RCP_LN2 if float(logit_softcap) > 0.0 else 0.0
    window, max_query_len = (min(max(0, int(x)), 0x7FFFFFFF) for x in (window_size, max_query_len))
    num_kv_splits = min(num_kv_splits, 0x7FFFFFFF)
    lib = _hip.load()
    with torch.cuda.device(q.device):
        n = lib.fxpr_attention_mx4_plan(num_requests, num_tokens, num_heads, num_kv_heads, head_dim, page_size,
                                        max_query_len, bt.shape[1], window, int(fxp_int_bits), num_kv_splits,
                                        None)
        ws = torch.empty(n, device=q.device, dtype=torch.uint8) if n > 0 else None
        _hip.call(
            "fxpr_unified_attention_mx4", q.data_ptr(), kv_codes.data_ptr(), kv_scales.data_ptr(), out.data_ptr(),
            _hip.DTYPE_CODE[q.dtype], qsl.data_ptr(), sl.data_ptr(), bt.data_ptr(), _hip.ptr(alibi), num_requests,
            num_tokens, num_heads, num_kv_heads, head_dim, page_size, max_query_len, bt.shape[1], num_blocks,
            q.stride(0), q.stride(1), *kv_codes.stride()[:4], *kv_scales.stride()[:4], out.stride(0), out.stride(1),
            bt.stride(0), int(bool(is_causal)), float(scale) * _RCP_LN2, softcap, window, int(fxp_int_bits),
            int(fxp_frac_bits), num_kv_splits, _hip.ptr(ws), n, _hip.stream_ptr(q.device),
        )
    if out is not o:
        o.copy_(out)
