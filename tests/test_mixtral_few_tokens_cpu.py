"""Which of a Mixtral layer's paths a step takes (``MixtralConfig.moe_decode``): the whole layer in one call
where that holds the config, else the expert loop. The kernels are replaced by recorders."""

import pytest
import torch

from flextensor_b200 import ops
from flextensor_b200.models.mixtral import MixtralLayer, tiny_mixtral


@pytest.fixture
def step(monkeypatch):
    """step(layer, tokens) -> ("decode", weights) or ("loop", None)"""
    monkeypatch.setattr(ops, "rmsnorm", lambda x, w, eps: x)

    def run(layer, tokens):
        monkeypatch.setattr(layer.attn, "attention_fused", lambda x, *a: x)
        monkeypatch.setattr(layer, "moe_single", lambda *a: ("loop", None))
        monkeypatch.setattr(ops, "moe_decode", lambda h, router, gu, dn, topk, **kw: ("decode", list(zip(gu, dn))))
        x = torch.randn(tokens, layer.cfg.dim, generator=torch.Generator().manual_seed(0))
        with torch.no_grad():
            return layer(x, 1, tokens, None)

    return run


def layer(expert_ids=None, **kw):
    m = MixtralLayer(tiny_mixtral(dim=128, n_heads=1, n_kv_heads=1, ffn_dim=8, moe_decode=True, **kw), expert_ids)
    for p in m.parameters():
        torch.nn.init.normal_(p)
    return m


@pytest.mark.parametrize("tokens,kw,path", [
    (1, {}, "decode"), (64, {}, "decode"), (65, {}, "loop"),
    (1, dict(n_experts=128), "decode"), (1, dict(n_experts=129), "loop"), (64, dict(n_experts=160, topk=6), "loop"),
    (1, dict(n_experts=16, topk=8), "decode"), (1, dict(n_experts=16, topk=9), "loop"),
])
def test_path(step, tokens, kw, path):
    m = layer(**kw)
    assert step(m, tokens)[0] == path
    m.cfg.moe_decode = False
    assert step(m, tokens)[0] == "loop"
