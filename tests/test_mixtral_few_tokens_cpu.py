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


def test_experts_go_by_their_ids(step):
    """The router's row e belongs to the expert whose id is e, wherever the layer keeps it."""
    m = layer(expert_ids=[2, 0, 3, 1])
    path, weights = step(m, 3)
    assert path == "decode"
    for e, (gate_up, down) in enumerate(weights):
        mine = m.experts[m.expert_ids.index(e)]
        assert gate_up is mine.w_gate_up and down is mine.w_down
    assert step(layer(expert_ids=[0, 1]), 3)[0] == "loop"
    assert step(layer(expert_ids=[0, 1, 1, 2]), 3)[0] == "loop"
