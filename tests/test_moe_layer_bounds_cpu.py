"""The bounds that ``ops.moe_decode`` is held to (``helpers/moe_layer.py``) tell two bf16 halves of h from one,
and from a wrong second one: mistakes are planted in the oracle."""

import pytest
import torch

from helpers.moe_layer import cancelling_layer, layer, norm_ratio, random_layer

SPOILED = {
    "both halves": lambda hi, lo: hi + lo,
    "no low half": lambda hi, lo: hi,
    "another row's low half": lambda hi, lo: hi + lo.roll(1, 0) if len(lo) > 1 else hi + lo.roll(1, 1),
    "shifted low half": lambda hi, lo: hi + lo.roll(8, 1),
    "low half twice": lambda hi, lo: hi + 2 * lo,
}


@pytest.mark.parametrize("how", SPOILED)
@pytest.mark.parametrize("shape", [(3, 1000, 1416, 5, 2), (7, 512, 256, 16, 6), (1, 2048, 1024, 8, 2)])
def test_norm(how, shape):
    T, D, F, E, topk = shape
    p = random_layer(T, D, F, E, seed=1)
    want, bound = layer(**p, topk=topk)
    got, _ = layer(**p, topk=topk, spoil=SPOILED[how])
    ratio, most = norm_ratio(got, want)
    assert (ratio <= most) == (how == "both halves"), ratio
    if how == "both halves":
        assert bool(((got - want).abs() <= bound).all())


@pytest.mark.parametrize("how", SPOILED)
def test_elements(how):
    p = cancelling_layer(5)
    want, bound = layer(**p, topk=2)
    got, _ = layer(**p, topk=2, spoil=SPOILED[how])
    assert bool(((got - want).abs() <= bound).all()) == (how == "both halves")
