"""``ops.moe_decode`` against the layer's definition in 64 bits.

Tolerance: h is rounded to bf16 (at most 2^-8 of each element) before the down product, the output
once more. Element by element that is at most 2^-8 |out| + 2^-8 A with A = sum_k w_k sum_f |W_down| |h|;
fp32 sums and the exponential's approximation add less than 2^-12 A (at most 2^10 terms in a row of
fp32 additions at 2^-24 here, and 2^-21 from exp). In the 2-norm over random weights both roundings
are independent with a root mean square of at most 2^-8 / sqrt(3) of the value, so the relative
error stays below sqrt(2/3) 2^-8, checked at 2^-8."""

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("needs a CUDA device", allow_module_level=True)

from flextensor_b200 import ops  # noqa: E402
from flextensor_b200.ops import native  # noqa: E402

DEV = "cuda"


def make(T, D, F, E, seed=0, stacked=True):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s, std=1.0: (torch.randn(*s, device=DEV, generator=g) * std).bfloat16()  # noqa: E731
    gu, dn = r(E, 2 * F, D, std=D ** -0.5), r(E, D, F, std=F ** -0.5)
    if not stacked:
        gu, dn = [w.clone() for w in gu], [w.clone() for w in dn]
    return dict(x=r(T, D), router=r(E, D, std=2 * D ** -0.5), w_gate_up=gu, w_down=dn), r(T, D)


def reference(x, router, w_gate_up, w_down, topk, residual=None):
    x64 = x.double()
    val, ids = torch.sort(x64 @ router.double().t(), dim=-1, descending=True, stable=True)
    val, ids = val[:, :topk], ids[:, :topk]
    w = torch.softmax(val, -1)
    y, A = torch.zeros_like(x64), torch.zeros_like(x64)
    for e in range(router.shape[0]):
        t, k = (ids == e).nonzero(as_tuple=True)
        if t.numel() == 0:
            continue
        z = x64[t] @ w_gate_up[e].double().t()
        h = torch.nn.functional.silu(z[:, 0::2]) * z[:, 1::2]
        d = w_down[e].double().t()
        y.index_add_(0, t, h @ d * w[t, k][:, None])
        A.index_add_(0, t, h.abs() @ d.abs() * w[t, k][:, None])
    return y if residual is None else y + residual.double(), A


def check(p, topk, residual=None, out=None):
    want, A = reference(**p, topk=topk, residual=residual)
    got = ops.moe_decode(**p, topk=topk, residual=residual, out=out)
    torch.cuda.synchronize()
    assert native.device_error(reset=True) == 0
    err = (got.double() - want).abs()
    assert bool((err <= want.abs() * 2 ** -8 + A * (2 ** -8 + 2 ** -12)).all())
    assert float(err.norm() / want.norm()) <= 2 ** -8
    return got


@pytest.mark.parametrize("T,D,F,E,topk", [
    (1, 8, 8, 1, 1), (1, 64, 32, 4, 2), (2, 72, 200, 3, 3), (3, 1000, 1416, 5, 2), (17, 256, 256, 4, 2), (64, 512, 520, 8, 3),
    (64, 136, 72, 128, 8), (5, 2048, 1024, 64, 6), (33, 128, 4096, 2, 1), (1, 128, 16384, 8, 2), (16, 4096, 256, 33, 4)])
@pytest.mark.parametrize("stacked", [True, False])
def test_shapes(T, D, F, E, topk, stacked):
    p, res = make(T, D, F, E, seed=T + D, stacked=stacked)
    a = check(p, topk)
    b = check(p, topk, residual=res)
    assert torch.equal(a, ops.moe_decode(**p, topk=topk)) and torch.equal(b, ops.moe_decode(**p, topk=topk, residual=res))


def test_strides_and_aliases():
    p, res = make(9, 256, 192, 4, seed=1)
    wide = torch.zeros(9, 512, device=DEV, dtype=torch.bfloat16)
    wide[:, 256:] = p["x"]
    wgu = torch.zeros(4, 384, 264, device=DEV, dtype=torch.bfloat16)
    wgu[..., :256] = p["w_gate_up"]
    q = dict(p, x=wide[:, 256:], w_gate_up=wgu[..., :256], router=torch.cat([p["router"], p["router"]], 1)[:, :256])
    want = check(p, 2, residual=res)
    assert torch.equal(check(q, 2, residual=res), want)
    acc = res.clone()
    assert ops.moe_decode(**p, topk=2, residual=acc, out=acc) is acc and torch.equal(acc, want)
    x = p["x"].clone()
    assert torch.equal(ops.moe_decode(**dict(p, x=x), topk=2, residual=res, out=x), want)
    one = torch.zeros(1, 256, device=DEV, dtype=torch.bfloat16).expand(9, 256)
    assert torch.equal(ops.moe_decode(**p, topk=2, residual=one), ops.moe_decode(**p, topk=2))
    single = dict(p, x=p["x"][:1])  # a single row may have any row stride
    assert torch.equal(ops.moe_decode(**dict(p, x=p["x"].as_strided((1, 256), (0, 1))), topk=2), check(single, 2))


def test_shared_and_scattered_experts():
    """The same weights for every expert, and experts in no order of memory."""
    p, res = make(5, 256, 192, 4, seed=7)
    check(dict(p, w_gate_up=[p["w_gate_up"][0]] * 4, w_down=[p["w_down"][3]] * 4), 2, residual=res)
    order = [2, 0, 3, 1]
    check(dict(p, w_gate_up=[p["w_gate_up"][i] for i in order], w_down=[p["w_down"][i] for i in order]), 3)


def test_routing_corners():
    """All tokens on one expert; equal logits go to the lowest expert; a NaN token stays alone; weights
    that are NaN for an expert that nobody chose are not touched."""
    p, res = make(48, 128, 256, 6, seed=2)
    p["x"][:, 0] = 8.0
    p["router"].zero_()
    p["router"][4, 0] = 4.0
    check(p, 1)
    check(p, 3)  # experts 4, 0, 1
    p["w_gate_up"][5], p["w_down"][2] = float("nan"), float("nan")
    check(p, 2)
    clean = check(p, 2, residual=res)
    p["x"][7] = float("nan")
    got = ops.moe_decode(**p, topk=2, residual=res)
    assert got[7].isnan().all()
    keep = torch.arange(48, device=DEV) != 7
    assert torch.equal(got[keep], clean[keep])
    p["x"][7] = float("inf")
    got = ops.moe_decode(**p, topk=2, residual=res)
    assert got[7].isnan().any() and torch.equal(got[keep], clean[keep])


def test_empty():
    p, res = make(4, 64, 32, 4)
    assert ops.moe_decode(**dict(p, x=p["x"][:0]), topk=2).shape == (0, 64)


def test_streams_and_graphs():
    """A side stream, and a captured call replayed with new tokens while eager calls run on another
    stream (each has its own workspace)."""
    p, res = make(6, 512, 1024, 8, seed=3)
    want = check(p, 2, residual=res)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(ops.moe_decode(**p, topk=2, residual=res), want)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    x = p["x"].clone()
    with torch.cuda.graph(g):
        got = ops.moe_decode(**dict(p, x=x), topk=2, residual=res)
    for seed in (5, 6):
        fresh = make(6, 512, 1024, 8, seed=seed)[0]["x"]
        x.copy_(fresh)
        side.wait_stream(torch.cuda.current_stream())
        g.replay()
        with torch.cuda.stream(side):
            again = [ops.moe_decode(**p, topk=2, residual=res) for _ in range(3)]
        torch.cuda.synchronize()
        assert all(torch.equal(a, want) for a in again)
        assert torch.equal(got, ops.moe_decode(**dict(p, x=fresh), topk=2, residual=res))
    assert native.device_error(reset=True) == 0


def test_single_row_of_any_stride():
    p, res = make(1, 256, 192, 1, seed=8)
    odd = lambda t: t.as_strided(t.shape, (3, 1))  # noqa: E731
    want = check(p, 1, residual=res)
    got = ops.moe_decode(**dict(p, x=odd(p["x"]), router=odd(p["router"])), topk=1, residual=odd(res), out=odd(torch.zeros_like(res)))
    assert torch.equal(got, want)


def test_halves_of_a_wide_buffer():
    """The output beside the residual in one buffer: columns side by side share no memory."""
    p, res = make(9, 256, 192, 4, seed=9)
    want = check(p, 2, residual=res)
    wide = torch.zeros(9, 512, device=DEV, dtype=torch.bfloat16)
    wide[:, 256:] = res
    assert torch.equal(ops.moe_decode(**p, topk=2, residual=wide[:, 256:], out=wide[:, :256]), want)
    assert torch.equal(wide[:, 256:], res)
