"""Mixtral-8x22B-shape sparse-MoE decoder (GQA attention + top-2 of 8 SwiGLU experts).

Attention is the Llama block (``models/llama.py``, native kernels). The MoE feed-forward:
router logits -> top-2 -> softmax over the two; each expert is a SwiGLU FFN whose gate/up
rows are interleaved (one GEMM with the SwiGLU epilogue) followed by the down GEMM.

Four MoE paths share one parameter tree:

* single GPU (``ep=None``): per-expert gather -> fused GEMMs -> weighted scatter-add;
* single GPU, few tokens (``MixtralConfig.moe_decode``): the whole layer in one call without host
  synchronisation (``ops.moe_decode``);
* expert parallel, fused (``ep=ExpertParallel``): each rank keeps its own tokens and owns
  ``E/world`` experts; dispatch / combine run inside the expert GEMM kernels over NVLink
  (``parallel/ep.py``, ``ops/csrc/moe_sm100.cu``);
* expert parallel, NCCL (``ep=NcclExpertParallel``): all-to-all around the same GEMMs.

``layers.*`` are the offload units: with expert parallelism a rank's unit holds only its own
experts' weights, which is what the runtime streams from host memory.
"""

from __future__ import annotations

import zlib
from dataclasses import dataclass

import torch
import torch.nn.functional as F
from torch import nn

from flextensor_b200.models.kv_cache import check_draft, new_layer_cache, rewind
from flextensor_b200.models.llama import LlamaConfig, LlamaLayer, _rms_torch, rope_tables_1d


@dataclass
class MixtralConfig(LlamaConfig):
    dim: int = 6144
    n_layers: int = 56
    n_heads: int = 48
    n_kv_heads: int = 8
    ffn_dim: int = 16384
    vocab: int = 32768
    rope_theta: float = 1000000.0
    n_experts: int = 8
    topk: int = 2
    # single GPU, native path: steps of at most 64 tokens take ops.moe_decode (with at most 128 experts, 8 a token)
    moe_decode: bool = False


MIXTRAL_8X22B = MixtralConfig()


def tiny_mixtral(**kw) -> MixtralConfig:
    base = dict(dim=256, n_layers=2, n_heads=2, n_kv_heads=2, ffn_dim=256, vocab=512, n_experts=4, topk=2)
    base.update(kw)
    return MixtralConfig(**base)


class Expert(nn.Module):
    def __init__(self, d: int, f: int):
        super().__init__()
        self.w_gate_up = nn.Parameter(torch.empty(2 * f, d))
        self.w_down = nn.Parameter(torch.empty(d, f))


class MixtralLayer(nn.Module):
    def __init__(self, cfg: MixtralConfig, expert_ids: list[int] | None = None):
        super().__init__()
        self.cfg = cfg
        self.attn = LlamaLayer(cfg, ffn=1)   # attention weights (its 1-wide dense FFN is unused)
        self.ffn_norm = nn.Parameter(torch.ones(cfg.dim))
        self.router = nn.Parameter(torch.empty(cfg.n_experts, cfg.dim))
        self.expert_ids = list(range(cfg.n_experts)) if expert_ids is None else list(expert_ids)
        self.experts = nn.ModuleList([Expert(cfg.dim, cfg.ffn_dim) for _ in self.expert_ids])

    def all_experts(self):
        """The experts in the order of the router's rows; None if some are not here."""
        ids = list(range(self.cfg.n_experts))
        if self.expert_ids == ids:
            return self.experts
        at = dict(zip(self.expert_ids, self.experts))
        return [at[e] for e in ids] if sorted(self.expert_ids) == ids else None

    def moe_single(self, h: torch.Tensor, ids: torch.Tensor, wts: torch.Tensor, out: torch.Tensor, impl: str):
        from flextensor_b200 import ops

        acc = out.float()
        for j, e in enumerate(self.expert_ids):
            hit = (ids == e)
            rows = hit.any(-1).nonzero().squeeze(-1)
            if rows.numel() == 0:
                continue
            w = (wts * hit).sum(-1)[rows]
            xe = h.index_select(0, rows)
            ex = self.experts[j]
            if impl == "fused":
                y = ops.linear(ops.linear_swiglu(xe, ex.w_gate_up), ex.w_down, None, epi="none")
            else:
                gu = F.linear(xe, ex.w_gate_up)
                y = F.linear(F.silu(gu[:, 0::2]) * gu[:, 1::2], ex.w_down)
            acc.index_add_(0, rows, y.float() * w[:, None])
        out.copy_(acc.to(out.dtype))
        return out

    def forward(self, x, B, S, rope, impl: str = "fused", ep=None, cache=None, pos: int = 0):
        """``cache`` = (k_cache, v_cache) of this layer: prefill (``pos == 0``) fills positions
        [0, S); a decode step (S == 1) appends position ``pos`` and attends over [0, pos] with the
        split-KV decode kernel (native path only)."""
        from flextensor_b200 import ops
        from flextensor_b200.parallel.ep import NcclExpertParallel, route_topk

        cfg = self.cfg
        if impl == "fused":
            x = self.attn.attention_fused(x, B, S, rope, cache, pos)
        else:
            x = self.attn.attention_torch(x, B, S, rope)
        h = ops.rmsnorm(x, self.ffn_norm, eps=cfg.eps) if impl == "fused" else _rms_torch(x, self.ffn_norm, cfg.eps)
        if ep is None and impl == "fused" and cfg.moe_decode and h.shape[0] <= ops.MOE_DECODE_MAX_TOKENS:
            experts = self.all_experts()
            if experts is not None and cfg.n_experts <= ops.MOE_DECODE_MAX_EXPERTS and cfg.topk <= ops.MOE_DECODE_MAX_TOPK:
                return ops.moe_decode(h, self.router, [e.w_gate_up for e in experts], [e.w_down for e in experts],
                                      cfg.topk, residual=x, out=x)
        ids, wts = route_topk(h, self.router, cfg.topk)
        if ep is None:
            return self.moe_single(h, ids, wts, x, impl)
        if isinstance(ep, NcclExpertParallel):
            return ep(h, ids, wts, [e.w_gate_up for e in self.experts], [e.w_down for e in self.experts], x)
        slots = ep.dispatch(h, ids)
        ep.experts([e.w_gate_up for e in self.experts], [e.w_down for e in self.experts])
        return ep.combine(slots, wts, residual=x, out=x)


class MixtralModel(nn.Module):
    def __init__(self, cfg: MixtralConfig = MIXTRAL_8X22B, impl: str = "fused", rank: int = 0, world: int = 1,
                 layers: int | None = None):
        super().__init__()
        self.cfg, self.impl = cfg, impl
        el = cfg.n_experts // world
        mine = list(range(rank * el, (rank + 1) * el))
        self.embed = nn.Embedding(cfg.vocab, cfg.dim)
        self.layers = nn.ModuleList([MixtralLayer(cfg, mine) for _ in range(layers or cfg.n_layers)])
        self.norm = nn.Parameter(torch.ones(cfg.dim))
        self.lm_head = nn.Parameter(torch.empty(cfg.vocab, cfg.dim))
        self._rope = {}

    def rope(self, S, device):
        key = (S, str(device))
        if key not in self._rope:
            self._rope[key] = rope_tables_1d(S, self.cfg.head_dim, self.cfg.rope_theta, device)
        return self._rope[key]

    def hidden(self, tokens: torch.Tensor, ep=None) -> torch.Tensor:
        B, S = tokens.shape
        x = self.embed(tokens).reshape(B * S, -1).contiguous()
        rope = self.rope(S, x.device)
        for layer in self.layers:
            x = layer(x, B, S, rope, self.impl, ep=ep)
        return x

    def forward(self, tokens: torch.Tensor, ep=None) -> torch.Tensor:
        B, S = tokens.shape
        x = self.hidden(tokens, ep)
        h = _rms_torch(x.view(B, S, -1)[:, -1], self.norm, self.cfg.eps)
        return F.linear(h, self.lm_head)

    # ---------------------------------------------------------------- KV-cache generation
    def new_cache(self, batch: int, max_len: int, device=None, dtype=torch.bfloat16):
        """One cache a layer, bf16 or 8 bits (``dtype`` ``torch.int8`` / ``torch.float8_e4m3fn``)."""
        cfg = self.cfg
        dev = device or self.lm_head.device
        return [new_layer_cache(batch, max_len, cfg.n_kv_heads, cfg.head_dim, dev, dtype) for _ in self.layers]

    def _logits(self, h_last):
        return F.linear(_rms_torch(h_last, self.norm, self.cfg.eps), self.lm_head)

    @torch.no_grad()
    def prefill(self, tokens: torch.Tensor, cache, ep=None) -> torch.Tensor:
        """Run the prompts (native path), fill the cache, return last-position logits."""
        B, S = tokens.shape
        x = self.embed(tokens).reshape(B * S, -1).contiguous()
        cos, sin = self.rope(cache[0][0].shape[1], x.device)
        rope_s = (cos[:S], sin[:S])
        for layer, c in zip(self.layers, cache):
            x = layer(x, B, S, rope_s, self.impl, ep=ep, cache=c, pos=0)
        return self._logits(x.view(B, S, -1)[:, -1])

    @torch.no_grad()
    def decode_step(self, token: torch.Tensor, cache, pos: int, ep=None) -> torch.Tensor:
        """One new token per sequence at position ``pos``; returns its logits ``[B, vocab]``. On an 8-bit
        cache ``token`` may be ``[B, S]``, S > 1 (a draft to check); the logits are then ``[B, S, vocab]``.
        Where only the first are accepted, :meth:`rewind` takes the others back before the next step: left
        there, they would keep the scale of the block they share with the tokens before them."""
        B = token.shape[0]
        S = check_draft(token, cache)
        x = self.embed(token.reshape(B * S)).contiguous()
        cos, sin = self.rope(cache[0][0].shape[1], x.device)
        rope_p = (cos[pos:pos + S].contiguous(), sin[pos:pos + S].contiguous())
        for layer, c in zip(self.layers, cache):
            x = layer(x, B, S, rope_p, self.impl, ep=ep, cache=c, pos=pos)
        logits = self._logits(x)
        return logits if S == 1 else logits.view(B, S, -1)

    @torch.no_grad()
    def rewind(self, cache, pos: int) -> None:
        """Take back the tokens from position ``pos`` on of the last :meth:`decode_step`, a draft of 2 to 16
        tokens of which only the first were accepted (:func:`flextensor_b200.models.kv_cache.rewind`)."""
        rewind(cache, pos)

    @torch.no_grad()
    def generate(self, tokens: torch.Tensor, max_new: int, ep=None, cache_dtype=torch.bfloat16) -> torch.Tensor:
        """Greedy continuation ``[B, max_new]`` with a KV cache of ``cache_dtype``."""
        B, S = tokens.shape
        cache = self.new_cache(B, S + max_new, tokens.device, cache_dtype)
        logits = self.prefill(tokens, cache, ep)
        out = []
        for i in range(max_new):
            nxt = logits.argmax(-1)
            out.append(nxt)
            if i + 1 < max_new:
                logits = self.decode_step(nxt, cache, S + i, ep)
        return torch.stack(out, dim=1)


class MixtralStack(nn.Module):
    """The decoder layers alone (no embedding / head): the offloadable body for end-to-end runs.
    ``ep``: an :class:`~flextensor_b200.parallel.ep.ExpertParallel` per token-row count (e.g. the
    prefill's and the decode step's), chosen by the rows of ``x``."""

    def __init__(self, cfg: MixtralConfig = MIXTRAL_8X22B, rank: int = 0, world: int = 1, layers: int | None = None):
        super().__init__()
        self.cfg = cfg
        el = cfg.n_experts // world
        mine = list(range(rank * el, (rank + 1) * el))
        self.layers = nn.ModuleList([MixtralLayer(cfg, mine) for _ in range(layers or cfg.n_layers)])

    def new_cache(self, batch: int, max_len: int, device=None, dtype=torch.bfloat16):
        c = self.cfg
        dev = device or torch.device("cuda", torch.cuda.current_device())
        return [new_layer_cache(batch, max_len, c.n_kv_heads, c.head_dim, dev, dtype) for _ in self.layers]

    def forward(self, x, B, S, rope, ep: dict | None = None, cache=None, pos: int = 0):
        e = None if not ep else ep.get(x.shape[0])
        for i, L in enumerate(self.layers):
            x = L(x, B, S, rope, "fused", ep=e, cache=None if cache is None else cache[i], pos=pos)
        return x


@torch.no_grad()
def init_mixtral_params_(model: nn.Module, seed: int = 0, std: float = 0.02, full_experts: int | None = None) -> None:
    """Deterministic init; an expert's weights depend only on (seed, layer, global expert id),
    so expert-parallel shards match the single-GPU model."""
    dev = next(model.parameters()).device
    g = torch.Generator(device=dev)
    for name, p in model.named_parameters():
        if ".experts." in name:
            continue
        g.manual_seed(seed * 1000003 + zlib.crc32(name.encode()))
        if name.endswith("norm") or name.endswith("attn_norm") or name.endswith("ffn_norm"):
            p.fill_(1.0)
        else:
            p.normal_(0.0, std, generator=g)
    for li, layer in enumerate(model.layers):
        for j, e in enumerate(layer.expert_ids):
            ex = layer.experts[j]
            g.manual_seed(seed * 7919 + li * 131 + e)
            ex.w_gate_up.normal_(0.0, std, generator=g)
            ex.w_down.normal_(0.0, std, generator=g)
