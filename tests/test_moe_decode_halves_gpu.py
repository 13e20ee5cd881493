"""``ops.moe_decode`` within the bounds of a kernel that keeps h in two bf16 halves (``helpers/moe_layer.py``):
its error is the output's own rounding. Dropping, shifting or mixing up the low halves fails these."""

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("needs a CUDA device", allow_module_level=True)

from flextensor_b200 import ops  # noqa: E402
from flextensor_b200.ops import native  # noqa: E402
from helpers.moe_layer import cancelling_layer, layer, norm_ratio, random_layer  # noqa: E402

DEV = "cuda"


def check(p, topk, norm=True, **kw):
    want, bound = layer(**p, topk=topk, **kw)
    got = ops.moe_decode(**p, topk=topk, **kw)
    torch.cuda.synchronize()
    assert native.device_error(reset=True) == 0
    assert bool(((got.double() - want).abs() <= bound).all())
    if norm:
        ratio, most = norm_ratio(got, want)
        assert ratio <= most, ratio


@pytest.mark.parametrize("T,D,F,E,topk", [
    (3, 1000, 1416, 5, 2), (1, 2048, 1024, 8, 2), (7, 2048, 1024, 64, 6), (17, 256, 256, 4, 2), (64, 512, 520, 8, 3),
    (64, 136, 72, 128, 8), (33, 128, 4096, 2, 1), (16, 4096, 256, 33, 4), (64, 1024, 2048, 2, 2), (2, 1024, 16384, 8, 2)])
@pytest.mark.parametrize("stacked", [True, False])
def test_random_layers(T, D, F, E, topk, stacked):
    p = random_layer(T, D, F, E, seed=T + D, device=DEV)
    if not stacked:
        p.update({k: [w.clone() for w in p[k]] for k in ("w_gate_up", "w_down")})
    check(p, topk)
    res = torch.randn(T, D, device=DEV, generator=torch.Generator(device=DEV).manual_seed(T)).bfloat16()
    check(p, topk, residual=res)


@pytest.mark.parametrize("T", [1, 5, 16, 17, 64])
def test_cancelling_layers(T):
    check(cancelling_layer(T, DEV), 2, norm=False)
