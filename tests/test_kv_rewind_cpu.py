"""Taking a draft's rejected tokens back out of an 8-bit cache (``models/kv_cache.rewind``), with the append
kernel replaced by its definition in plain torch."""

import pytest
import torch

from flextensor_b200 import ops
from flextensor_b200.models.kv_cache import DRAFT_TOKENS, new_layer_cache, rewind, store

B, L, HK, BLOCK = 2, 100, 2, 16


def append(k, v, kc, vc, ks, vs, pos, *, block):
    for x, codes, scales in ((k, kc, ks), (v, vc, vs)):
        lo, end = pos, pos + k.shape[1]
        while lo < end:
            j = lo // block
            hi = min(end, (j + 1) * block)
            rows = x[:, lo - pos:hi - pos].double()
            a = rows.abs().amax(dim=(1, 3))
            m, e = torch.frexp(a / 127)
            s = torch.where(a > 0, torch.ldexp(torch.ones_like(a), e - (m == 0.5).int()), torch.zeros_like(a))
            s = torch.where(a.isfinite(), s, torch.full_like(s, float("nan")))
            if lo > j * block:
                s0 = scales[:, j].double()
                s = torch.maximum(s, s0)
                again = codes[:, j * block:lo].double() * (s0 / s)[:, None, :, None]
                codes[:, j * block:lo] = torch.nan_to_num(again).round().to(torch.int8)
            codes[:, lo:hi] = torch.nan_to_num(rows / s[:, None, :, None], posinf=0, neginf=0).round().to(torch.int8)
            scales[:, j] = s.float()
            lo = hi


@pytest.fixture(autouse=True)
def plain(monkeypatch):
    monkeypatch.setattr(ops, "kv_append_q8", append)


def tokens(n, seed=0, size=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(B, n, HK, 128, generator=g) * size).bfloat16() for _ in range(2)]


def filled(pos):
    c = new_layer_cache(B, L, HK, 128, "cpu", torch.int8, BLOCK)
    if pos:
        store(c, *tokens(pos), 0)
    return c


def same_until(a, b, pos):
    blocks = -(-pos // BLOCK)
    return all(torch.equal(x[:, :pos], y[:, :pos]) for x, y in zip(a[:2], b[:2])) and \
        all(torch.equal(x[:, :blocks], y[:, :blocks]) for x, y in zip(a[2:4], b[2:4]))


@pytest.mark.parametrize("pos", [1, 15, 16, 17, 31, 40])
@pytest.mark.parametrize("n", [2, 5, DRAFT_TOKENS])
@pytest.mark.parametrize("size", [64.0, float("nan")])
def test_rejected_tokens_leave_no_trace(pos, n, size):
    for accepted in {0, 1, n - 1, n}:
        cache, want = filled(pos), filled(pos)
        k, v = tokens(n, 1)
        for x in (k, v):
            x[:, accepted:] *= size
        store(cache, k, v, pos)
        if accepted < n and pos % BLOCK and (pos + accepted) // BLOCK == pos // BLOCK:  # a large token joins older ones
            assert not same_until(cache, want, pos)
        if accepted:
            store(want, k[:, :accepted], v[:, :accepted], pos)
        rewind([cache], pos + accepted)
        assert same_until(cache, want, pos + accepted)
        one = tokens(1, 2)
        for c in (cache, want):
            store(c, *one, pos + accepted)
        assert same_until(cache, want, pos + accepted + 1)


def test_rewinding_twice():
    cache, want = filled(20), filled(20)
    k, v = tokens(6, 1, 50.0)
    store(cache, k, v, 20)
    rewind([cache], 24)
    rewind([cache], 21)
    store(want, k[:, :1], v[:, :1], 20)
    assert same_until(cache, want, 21)
    with pytest.raises(ValueError, match="not in the last step"):
        rewind([cache], 22)  # taken back already


def test_refusals():
    cache = filled(20)
    with pytest.raises(ValueError, match="not one of 2 to"):
        rewind([cache], 20)  # a prompt
    store(cache, *tokens(3), 20)
    for pos in (19, 24):
        with pytest.raises(ValueError, match="not in the last step"):
            rewind([cache], pos)
    with pytest.raises(ValueError, match="not one of 2 to"):
        rewind([cache._replace(k=cache.k.clone())], 21)  # another cache's step
    store(cache, *tokens(1), 23)
    with pytest.raises(ValueError, match="not one of 2 to"):
        rewind([cache], 23)
    store(cache, *tokens(DRAFT_TOKENS + 1), 24)
    with pytest.raises(ValueError, match="not one of 2 to"):
        rewind([cache], 30)


def test_a_bf16_cache_needs_nothing():
    c = new_layer_cache(B, L, HK, 128, "cpu")
    store(c, *tokens(5), 0)
    before = [t.clone() for t in c]
    rewind([c], 3)
    assert all(torch.equal(a[:, :5], b[:, :5]) for a, b in zip(c, before))
