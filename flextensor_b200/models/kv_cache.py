"""Per-layer key/value caches of the decoder models: bf16, or 8 bits with block scales.

A bf16 cache is a plain ``(k_cache, v_cache)`` pair of ``[B, L, Hk, D]`` tensors. An 8-bit cache is a
:class:`QuantizedKV`: codes of the same shape and one scale per block of tokens and head, half the
memory and half the bytes a decode step reads. :func:`store` and :func:`attend` serve both.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

QUANTIZED_DTYPES = (torch.int8, torch.float8_e4m3fn)


class QuantizedKV(NamedTuple):
    k: torch.Tensor          # codes [B, L, Hk, 128]
    v: torch.Tensor
    k_scale: torch.Tensor    # fp32 [B, ceil(L / block), Hk]
    v_scale: torch.Tensor
    block: int = 64


def new_layer_cache(batch: int, max_len: int, heads: int, head_dim: int, device, dtype=torch.bfloat16, block: int = 64):
    """An empty cache of one layer; ``dtype`` int8 or float8_e4m3fn makes it a :class:`QuantizedKV`."""
    shape = (batch, max_len, heads, head_dim)
    if dtype not in QUANTIZED_DTYPES:
        return torch.empty(shape, device=device, dtype=dtype), torch.empty(shape, device=device, dtype=dtype)
    scales = (batch, -(-max_len // block), heads)
    return QuantizedKV(torch.zeros(shape, device=device, dtype=dtype), torch.zeros(shape, device=device, dtype=dtype),
                       torch.zeros(scales, device=device), torch.zeros(scales, device=device), block)


def store(cache, k: torch.Tensor, v: torch.Tensor, pos: int) -> None:
    """Put ``k`` / ``v [B, S, Hk, D]`` at positions ``[pos, pos + S)``."""
    if isinstance(cache, QuantizedKV):
        from flextensor_b200 import ops

        ops.kv_append_q8(k, v, cache.k, cache.v, cache.k_scale, cache.v_scale, pos, block=cache.block)
        return
    kc, vc = cache
    S = k.shape[1]
    kc[:, pos:pos + S].copy_(k)
    vc[:, pos:pos + S].copy_(v)


def check_draft(token: torch.Tensor, cache) -> int:
    """Tokens per sequence of a decode step's ``token`` (``[B]`` or ``[B, S]``)."""
    S = 1 if token.dim() == 1 else token.shape[1]
    if S != 1 and not isinstance(cache[0], QuantizedKV):
        raise ValueError("several tokens a step need an 8-bit cache (dtype=torch.int8 or torch.float8_e4m3fn)")
    return S


def attend(cache, q: torch.Tensor, kv_len: int) -> torch.Tensor:
    """Attention of the last ``S`` tokens' queries ``q [B, S, Hq, D]`` over keys ``[0, kv_len)`` (S > 1,
    causal among themselves, on an 8-bit cache only)."""
    from flextensor_b200 import ops

    if isinstance(cache, QuantizedKV):
        return ops.decode_attention_q8(q, cache.k, cache.v, cache.k_scale, cache.v_scale, kv_len, block=cache.block)
    return ops.decode_attention(q, cache[0], cache[1], kv_len)
