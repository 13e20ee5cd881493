"""Per-layer key/value caches of the decoder models: bf16, or 8 bits with block scales.

A bf16 cache is a plain ``(k_cache, v_cache)`` pair of ``[B, L, Hk, D]`` tensors. An 8-bit cache is a
:class:`QuantizedKV`: codes of the same shape and one scale per block of tokens and head, half the
memory and half the bytes a decode step reads. :func:`store` and :func:`attend` serve both.

A step of several tokens (a draft to check) joins the open block of an 8-bit cache like any others: a
larger one among them raises the block's scale, and the codes of the tokens before it are rounded again.
:func:`rewind` takes the rejected ones back as if they had never been stored.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

QUANTIZED_DTYPES = (torch.int8, torch.float8_e4m3fn)
DRAFT_TOKENS = 16  # a step of 2 to this many tokens can be taken back


class Draft:
    """The last step of several tokens in an 8-bit cache (``of``: its key codes): positions ``[pos, end)``, the
    tokens as they came (keys and values, ``[2, B, S, Hk, 128]`` bf16), and the open block before them (codes
    of its tokens and scales; None where ``pos`` begins a block)."""

    __slots__ = ("of", "pos", "end", "new", "codes", "scales")  # no __dict__: walks over tensors pass it by

    def __init__(self):
        self.forget()

    def forget(self):
        self.of = self.pos = self.end = self.new = self.codes = self.scales = None


class QuantizedKV(NamedTuple):
    k: torch.Tensor          # codes [B, L, Hk, 128]
    v: torch.Tensor
    k_scale: torch.Tensor    # fp32 [B, ceil(L / block), Hk]
    v_scale: torch.Tensor
    block: int = 64
    draft: Draft | None = None


def new_layer_cache(batch: int, max_len: int, heads: int, head_dim: int, device, dtype=torch.bfloat16, block: int = 64):
    """An empty cache of one layer; ``dtype`` int8 or float8_e4m3fn makes it a :class:`QuantizedKV`."""
    shape = (batch, max_len, heads, head_dim)
    if dtype not in QUANTIZED_DTYPES:
        return torch.empty(shape, device=device, dtype=dtype), torch.empty(shape, device=device, dtype=dtype)
    scales = (batch, -(-max_len // block), heads)
    return QuantizedKV(torch.zeros(shape, device=device, dtype=dtype), torch.zeros(shape, device=device, dtype=dtype),
                       torch.zeros(scales, device=device), torch.zeros(scales, device=device), block, Draft())


def store(cache, k: torch.Tensor, v: torch.Tensor, pos: int) -> None:
    """Put ``k`` / ``v [B, S, Hk, D]`` at positions ``[pos, pos + S)``."""
    if isinstance(cache, QuantizedKV):
        from flextensor_b200 import ops

        S, draft = k.shape[1], cache.draft
        if draft is not None:
            draft.forget()
            if pos > 0 and 1 < S <= DRAFT_TOKENS and pos + S <= cache.k.shape[1]:
                draft.new = torch.stack((k, v))
                if pos % cache.block:
                    codes, scales = _open_block(cache, pos)
                    draft.codes, draft.scales = torch.stack(codes), torch.stack(scales)
        ops.kv_append_q8(k, v, cache.k, cache.v, cache.k_scale, cache.v_scale, pos, block=cache.block)
        if draft is not None and draft.new is not None:
            draft.of, draft.pos, draft.end = cache.k, pos, pos + S
        return
    kc, vc = cache
    S = k.shape[1]
    kc[:, pos:pos + S].copy_(k)
    vc[:, pos:pos + S].copy_(v)


def _open_block(cache: QuantizedKV, pos: int):
    """Views of the block that ``pos`` lies in: the codes of its tokens before ``pos``, and its scales."""
    j = pos // cache.block
    return ([c.view(torch.int8)[:, j * cache.block:pos] for c in (cache.k, cache.v)],
            [s[:, j] for s in (cache.k_scale, cache.v_scale)])


def rewind(cache, pos: int) -> None:
    """Take back the tokens that the last step stored from position ``pos`` on, in every layer of ``cache`` (a
    list as ``new_cache`` makes it): the codes of the tokens before ``pos`` are as if the step had ended there
    (the accepted ones' keys and values are what the step computed). The step must have held 2 to
    ``DRAFT_TOKENS`` tokens, with ``pos`` among them or just behind. Earlier steps stay. A bf16 cache holds every
    token by itself: nothing is to be done, its positions may be written again."""
    from flextensor_b200 import ops

    layers = [c for c in cache if isinstance(c, QuantizedKV)]
    for c in layers:
        d = c.draft
        if d is None or d.of is not c.k:
            raise ValueError(f"rewind: the last step on this 8-bit cache was not one of 2 to {DRAFT_TOKENS} tokens")
        if not d.pos <= pos <= d.end:
            raise ValueError(f"rewind: position {pos} is not in the last step's [{d.pos}, {d.end}]")
    for c in layers:
        d = c.draft
        if pos == d.end:
            continue
        for t in (d.new, d.codes, d.scales):
            if t is not None and t.is_cuda:  # this may be another stream than the step's
                t.record_stream(torch.cuda.current_stream(t.device))
        if d.codes is not None:
            codes, scales = _open_block(c, d.pos)
            for view, kept in zip((*codes, *scales), (*d.codes, *d.scales)):
                view.copy_(kept)
        if pos > d.pos:
            n = pos - d.pos
            ops.kv_append_q8(d.new[0, :, :n], d.new[1, :, :n], c.k, c.v, c.k_scale, c.v_scale, d.pos, block=c.block)
        d.end = pos


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
