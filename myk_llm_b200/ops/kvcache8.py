"""Key/value cache held in 8 bits, with the attention that reads it.

``KVCache8`` keeps keys and values as e4m3 or int8, head-major (batch, kv_heads, capacity,
head_dim), and one scale for each block of ``block`` tokens of each sequence and head.  A
scale is the smallest power of two that brings the block's largest magnitude within the
8-bit type's range (448 or 127), stored as a byte ``log2(scale) + 127`` (at least 27).

* ``kv8_append`` quantises new tokens as they are written at ``cache_seqlens[b]``.  A block
  that already holds tokens keeps its scale unless the new ones need a larger one; then its
  old tokens move to the new scale, which rounds them once more.  With ``block=1`` nothing is
  ever moved, so the cache does not depend on how the tokens were split into calls (nor on
  drafts that were rejected and overwritten).  A block that is given a NaN or an infinity
  reads back as NaN until it is written again from its first token on.
* ``kv8_read`` returns a range of the cache in bf16 (exact: 8-bit values times powers of two).
* ``flash_attn_with_kvcache8`` is :func:`~myk_llm_b200.ops.attention.flash_attn_with_kvcache`
  over such a cache: same alignment of queries, windows and empty rows.  A query that sees a
  block holding a NaN or an infinity gets NaN, no other does.  Calls of many queries (where it
  is faster, by a rule on sizes) read the cache's whole capacity back to bf16 for the time of
  the call and round the weights to 8 bits instead of 11.

As for the bf16 cache, nothing synchronises with the host, tokens past the capacity are
dropped, the caller advances ``cache_seqlens``, and there is no backward pass.  On CUDA the
kernels are ``csrc/kv8_cache.cu`` and ``csrc/kv8_attention.cu``.
"""

from __future__ import annotations

import math
from dataclasses import dataclass

import torch

from . import reference as ref
from ._ext import ext
from .attention import SUPPORTED_HEAD_DIMS, _window

KV8_DTYPES = (torch.float8_e4m3fn, torch.int8)


@dataclass
class KVCache8:
    keys: torch.Tensor  # (batch, kv_heads, capacity, head_dim) float8_e4m3fn or int8
    values: torch.Tensor
    key_scales: torch.Tensor  # (batch, kv_heads, ceil(capacity / block)) uint8
    value_scales: torch.Tensor
    block: int = 16


def kv8_cache(batch: int, capacity: int, kv_heads: int, head_dim: int, *, dtype: torch.dtype = torch.float8_e4m3fn,
              block: int = 16, device=None) -> KVCache8:
    """An empty 8-bit cache."""
    if dtype not in KV8_DTYPES:
        raise TypeError(f"8-bit cache dtype must be one of {KV8_DTYPES}; got {dtype}")
    if head_dim not in SUPPORTED_HEAD_DIMS:
        raise ValueError(f"head_dim must be one of {SUPPORTED_HEAD_DIMS}; got {head_dim}")
    if block < 1 or block > 1024 or block & (block - 1):
        raise ValueError(f"block must be a power of two up to 1024; got {block}")
    data = [torch.zeros(batch, kv_heads, capacity, head_dim, dtype=torch.uint8, device=device).view(dtype)
            for _ in range(2)]
    scales = [torch.zeros(batch, kv_heads, -(-capacity // block), dtype=torch.uint8, device=device) for _ in range(2)]
    return KVCache8(*data, *scales, block)


def _int32(t: torch.Tensor) -> torch.Tensor:
    return t if t.dtype == torch.int32 else t.to(torch.int32)


def kv8_append(cache: KVCache8, k: torch.Tensor, v: torch.Tensor, *, cache_seqlens: torch.Tensor) -> None:
    """Write k/v (batch, new, kv_heads, head_dim) at positions ``cache_seqlens[b]`` onward."""
    if not cache.keys.is_cuda:
        ref.kv8_append_ref(cache.keys, cache.key_scales, cache.block, k, cache_seqlens)
        ref.kv8_append_ref(cache.values, cache.value_scales, cache.block, v, cache_seqlens)
        return
    ext().kv8_append(cache.keys, cache.values, cache.key_scales, cache.value_scales, cache.block, k, v,
                     _int32(cache_seqlens))


def kv8_read(cache: KVCache8, *, cache_seqlens: torch.Tensor, start: int | torch.Tensor = 0,
             length: int | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """bf16 (batch, length, kv_heads, head_dim) keys and values of tokens ``start`` (one for
    all sequences or one each) onward; tokens from ``cache_seqlens[b]`` on read as 0.
    ``length`` defaults to the rest of the capacity."""
    each = isinstance(start, torch.Tensor)
    if length is None:
        length = cache.keys.shape[2] - (0 if each else start)
    if length < 0 or (not each and start < 0):
        raise ValueError(f"start and length must not be negative; got {start}, {length}")
    if not cache.keys.is_cuda:
        return (ref.kv8_read_ref(cache.keys, cache.key_scales, cache.block, cache_seqlens, start, length),
                ref.kv8_read_ref(cache.values, cache.value_scales, cache.block, cache_seqlens, start, length))
    k, v = ext().kv8_read(cache.keys, cache.values, cache.key_scales, cache.value_scales, cache.block,
                          _int32(cache_seqlens), _int32(start) if each else None, 0 if each else start, length)
    return k, v


def flash_attn_with_kvcache8(q: torch.Tensor, cache: KVCache8, k: torch.Tensor | None = None,
                             v: torch.Tensor | None = None, *, cache_seqlens: torch.Tensor, causal: bool = False,
                             window_size=(-1, -1), softmax_scale=None) -> torch.Tensor:
    """Append k/v (batch, new, kv_heads, d), if given, then attend q (batch, Lq, heads, d)
    over the ``cache_seqlens[b] + new`` tokens the cache then holds.  Forward only."""
    scale = softmax_scale if softmax_scale is not None else 1.0 / math.sqrt(q.shape[-1])
    left, right = _window(causal, window_size)
    if not q.is_cuda:
        if (k is None) != (v is None):
            raise ValueError("new keys and values come together")
        used = cache_seqlens.clamp(min=0)
        if k is not None:
            kv8_append(cache, k, v, cache_seqlens=cache_seqlens)
            used = used + k.shape[1]
        return ref.kv8_attention_ref(q, cache.keys, cache.key_scales, cache.values, cache.value_scales, cache.block,
                                     used.clamp(max=cache.keys.shape[2]), (left, right), scale)
    return ext().kv8_attend(q, cache.keys, cache.values, cache.key_scales, cache.value_scales, cache.block, k, v,
                            _int32(cache_seqlens), float(scale), left, right)
