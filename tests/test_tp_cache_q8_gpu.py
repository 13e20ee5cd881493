"""Tensor-parallel Llama layers on 8-bit caches, each rank with its own heads' cache. Two ranks on one GPU:
two threads on one stream whose collectives are host barriers around plain torch sums, so that no kernel
waits for another (the collectives themselves are tested on two GPUs elsewhere).

Both sides round every operator's output to bf16 and store codes; a model of three layers with some ten
operators each is compared in the 2-norm at 10 * 2^-8 a layer."""

import threading

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("needs a CUDA device", allow_module_level=True)

from flextensor_b200.models.kv_cache import QuantizedKV, rewind  # noqa: E402
from flextensor_b200.models.llama import LlamaModel, LlamaTP, init_llama_params_, tiny_llama  # noqa: E402
from flextensor_b200.ops import native  # noqa: E402

DEV = torch.device("cuda", 0)
W = 2


class HostCollectives:
    def __init__(self):
        self.barrier, self.parts = threading.Barrier(W, timeout=60), [None] * W

    def exchange(self, rank, t):
        self.parts[rank] = t
        self.barrier.wait()
        got = list(self.parts)
        self.barrier.wait()  # nobody overwrites a part before all have it
        return got


class Rank:
    def __init__(self, shared, rank):
        self.shared, self.rank = shared, rank

    def all_gather(self, t):
        return torch.cat(self.shared.exchange(self.rank, t.contiguous()))

    def reduce_scatter(self, t):
        total = sum(p.float() for p in self.shared.exchange(self.rank, t))
        return total.chunk(W)[self.rank].to(t.dtype)


def on_ranks(fn):
    """fn(rank) in a thread each; their results in order."""
    out, errors = [None] * W, []

    def go(r):
        try:
            with torch.no_grad():
                out[r] = fn(r)
        except BaseException as e:  # noqa: BLE001
            errors.append(e)

    ts = [threading.Thread(target=go, args=(r,)) for r in range(W)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    if errors:
        raise errors[0]
    return out


def values(c, heads=slice(None)):
    of = torch.arange(c.k.shape[1], device=DEV) // c.block
    return [x[:, :, heads].float() * s[:, of][:, :, heads, None] for x, s in ((c.k, c.k_scale), (c.v, c.v_scale))]


def rel(a, b):
    return float((a.float() - b.float()).norm() / b.float().norm())


@torch.no_grad()
@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn])
def test_two_ranks(dtype):
    torch.manual_seed(0)
    cfg = tiny_llama(n_layers=3)
    full = LlamaModel(cfg).to(DEV)
    init_llama_params_(full, seed=1)
    full = full.to(torch.bfloat16)
    B, S, L = 4, 70, 80
    hk = cfg.n_kv_heads // W
    shared = HostCollectives()
    ranks = []
    for r in range(W):
        tp = LlamaTP(cfg, r, W).to(DEV).to(torch.bfloat16).load_from_full(full)
        tp.collective, tp._nccl = "nccl", Rank(shared, r)
        tp._by_rows = {rows: (None, None) for rows in (B * S, B, B * 4)}
        ranks.append(tp)
    caches = [tp.new_cache(B, L, DEV, dtype) for tp in ranks]
    whole = full.new_cache(B, L, dtype=dtype)
    for c in caches:
        assert all(isinstance(x, QuantizedKV) and x.k.shape == (B, L, hk, cfg.head_dim) and x.k.dtype == dtype for x in c)
    cos, sin = full.rope(L, DEV)
    g = torch.Generator(device=DEV).manual_seed(2)

    def step(pos, n):
        x = torch.randn(B * n, cfg.dim, device=DEV, generator=g).bfloat16()
        rope = (cos[pos:pos + n].contiguous(), sin[pos:pos + n].contiguous())
        want = x.clone()
        for layer, c in zip(full.layers, whole):
            want = layer(want, B, n, rope, cache=c, pos=pos)
        got = torch.cat(on_ranks(lambda r: ranks[r](x.chunk(W)[r].clone(), B, n, rope, cache=caches[r], pos=pos)))
        assert rel(got, want) <= 3 * 10 * 2 ** -8, (pos, n)
        for r in range(W):  # the first layer's codes stand for the same heads' values
            for a, b in zip(values(caches[r][0]), values(whole[0], slice(r * hk, (r + 1) * hk))):
                assert rel(a, b) <= 2 ** -6

    step(0, S)          # a prompt
    step(S, 1)          # single tokens
    step(S + 1, 1)
    step(S + 2, 4)      # a draft, of which two are accepted
    for c in (*caches, whole):
        rewind(c, S + 4)
    step(S + 4, 1)
    assert native.device_error(reset=True) == 0
