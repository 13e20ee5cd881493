"""Refusals of ``ops.moe_decode`` (checked before the device, so on CPU tensors), and a model in
Python of how its products divide the stream of weight tiles among CTAs."""

import random

import pytest
import torch

from flextensor_b200 import ops
from flextensor_b200.ops import native

T, D, F, E = 3, 64, 32, 4


def args(t=T, d=D, f=F, e=E):
    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731
    return dict(x=z(t, d), router=z(e, d), w_gate_up=[z(2 * f, d) for _ in range(e)], w_down=[z(d, f) for _ in range(e)], topk=2)


def bf(*s):
    return torch.zeros(*s, dtype=torch.bfloat16)


@pytest.mark.skipif(not native.available(), reason="native extension not built")
@pytest.mark.parametrize("change,match", [
    ({}, "CUDA device"),
    (dict(x=torch.zeros(T, D)), "x must be bfloat16"),
    (dict(x=bf(T, D, 1)), r"x must be \[T, D\]"),
    (dict(x=bf(65, D)), "at most 64 tokens"),
    (dict(router=bf(E, D + 8)), "router must be"),
    (dict(router=bf(0, D)), "experts"),
    (dict(topk=0), "topk"),
    (dict(topk=5), "topk"),
    (dict(w_down=[bf(D, F)] * 3), "one w_gate_up and one w_down"),
    (dict(w_gate_up=[bf(2 * F, D)] * 3 + [bf(2 * F + 2, D)]), "w_gate_up must be"),
    (dict(w_gate_up=[bf(2 * F, D)] * 3 + [bf(2 * F, D).float()]), "w_gate_up must be"),
    (dict(w_gate_up=[bf(2 * F, D)] * 3 + [bf(2 * F, 2 * D)[:, :D]]), "one row stride"),
    (dict(w_down=[bf(D, F)] * 3 + [bf(F, D).t()]), "16-byte"),
    (dict(w_down=[bf(D, F)] * 3 + [bf(D * F + 1)[1:].view(D, F)]), "16-byte"),
    (dict(residual=bf(T, D + 8)), "residual must be"),
    (dict(out=bf(T + 1, D)), "out must be"),
    (dict(out=bf(1, D).expand(T, D)), "overlap"),
    (dict(x=bf(1, D).expand(T, D)), "rows of x must not overlap"),
    (dict(w_down=[bf(1, F).expand(D, F)] * 4), "rows of w_down must not overlap"),
])
def test_refusals(change, match):
    a = args()
    a.update(change)
    with pytest.raises(RuntimeError, match=match):
        ops.moe_decode(**a)


@pytest.mark.skipif(not native.available(), reason="native extension not built")
def test_refuses_odd_sizes_and_partial_overlap():
    with pytest.raises(RuntimeError, match="multiples of 8"):
        ops.moe_decode(**args(d=60))
    with pytest.raises(RuntimeError, match="multiples of 8"):
        ops.moe_decode(**args(f=36))
    buf = bf(T + 1, D)
    with pytest.raises(RuntimeError, match="overlap|memory"):
        ops.moe_decode(**dict(args(), residual=buf[:T], out=buf[1:]))


def splits(D_, F_, topk, sms, min_chunks=4):
    rt, kc = -(-D_ // 128), -(-F_ // 64)
    m = max(min_chunks, rt * kc * topk // sms)
    return (kc - 1 + m - 1) // m + 1


def test_stream_partition_model():
    """Runs cover the stream once, a run cuts at most two tiles, ``owner`` finds the run of a tile, and
    the number of CTAs on one row tile stays within what the workspace holds."""
    rng = random.Random(0)
    for _ in range(400):
        D_, F_, topk = 8 * rng.randint(1, 800), 8 * rng.randint(1, 2100), rng.randint(1, 8)
        n_act, sms = rng.randint(topk, 64), rng.choice([148, 132, 7])
        rt, kc = -(-D_ // 128), -(-F_ // 64)
        total = n_act * rt * kc
        ctas = min(sms, max(1, total // 4))
        base, rem = divmod(total, ctas)
        begin = lambda c: c * base + min(c, rem)  # noqa: E731
        longer = rem * (base + 1)
        owner = lambda i: i // (base + 1) if i < longer else rem + (i - longer) // base  # noqa: E731
        assert begin(0) == 0 and begin(ctas) == total
        for c in range(ctas):
            assert begin(c) < begin(c + 1) and owner(begin(c)) == c == owner(begin(c + 1) - 1)
        for it in [rng.randrange(n_act * rt) for _ in range(20)]:
            c0, c1 = owner(it * kc), owner((it + 1) * kc - 1)
            assert c1 - c0 + 1 <= splits(D_, F_, topk, sms)
            for c in range(c0, c1 + 1 if c1 > c0 else c0):  # a tile that several share is each one's first or last
                assert begin(c) // kc == it or (begin(c + 1) - 1) // kc == it


@pytest.mark.skipif(not native.available(), reason="native extension not built")
@pytest.mark.parametrize("out", [
    torch.zeros(T * D, dtype=torch.bfloat16).as_strided((T, D), (8, 1)),
    torch.zeros(T * D, dtype=torch.bfloat16).as_strided((T, D), (0, 1)),
    torch.zeros(T * D, dtype=torch.bfloat16).as_strided((T, D), (D - 8, 1)),
])
def test_refuses_outputs_whose_rows_overlap(out):
    with pytest.raises(RuntimeError, match="overlap itself"):
        ops.moe_decode(**dict(args(), out=out))


@pytest.mark.skipif(not native.available(), reason="native extension not built")
@pytest.mark.parametrize("out,residual,refused", [
    ((0, 2 * D), (2 * D, 2 * D), True),     # one row later in a wide buffer
    ((0, 2 * D), (8, 2 * D), True),         # columns that overlap
    ((0, 2 * D), (3 * D, 2 * D), False),    # the other half of the columns, one row later
    ((0, 2 * D), (D, 2 * D), False),        # the other half of the columns
    ((0, 2 * D), (0, 2 * D), False),        # the same
    ((0, 2 * D), (6 * D, 2 * D), False),    # the rows behind
    ((0, 2 * D), (0, D), True),             # the same memory with other strides
    ((0, D), (0, 0), True),                 # one row of it for all
    ((0, D), (2 * D, D), True), ((D, D), (0, D), True), ((0, D), (3 * D, D), False),
])
def test_outputs_and_residuals_of_one_buffer(out, residual, refused):
    buf = bf(20 * D)
    view = lambda at, stride: buf[at:].as_strided((T, D), (stride, 1), buf.storage_offset() + at)  # noqa: E731
    with pytest.raises(RuntimeError, match="overlap it otherwise" if refused else "CUDA device"):
        ops.moe_decode(**dict(args(), out=view(*out), residual=view(*residual)))


def test_overlap_model():
    """The rule of the binding's check against a count of shared elements, for random views of one buffer."""
    rng = random.Random(1)

    def reaches(d, rest):
        if not d:
            return rest == 0
        (stride, size), low = d[0], d[1:]
        below = sum((n - 1) * s for s, n in low)
        quotient = int((rest - below) / stride)  # towards zero, as in C++
        return any(abs(k) < size and abs(rest - k * stride) <= below and reaches(low, rest - k * stride)
                   for k in range(quotient - 1, (rest + below) // stride + 1))

    for _ in range(2000):
        dims, reach = [], 1
        for _ in range(rng.randint(1, 4)):
            n, s = rng.randint(2, 5), reach + rng.choice([0, 0, 1, 3, reach])
            dims.append((s, n))
            reach += (n - 1) * s
        dims.sort(reverse=True)
        offsets = {0}
        for s, n in dims:
            offsets = {o + k * s for o in offsets for k in range(n)}
        d = rng.randint(-reach, reach)
        assert reaches(dims, d) == bool(offsets & {o + d for o in offsets}), (dims, d)


@pytest.mark.skipif(not native.available(), reason="native extension not built")
@pytest.mark.parametrize("stride", [0, 1, 3])
def test_a_single_row_may_have_any_stride(stride):
    row = lambda: bf(1, D).as_strided((1, D), (stride, 1))  # noqa: E731
    a = dict(args(t=1, e=1), topk=1)
    a.update(x=row(), router=row(), residual=row(), out=row())
    with pytest.raises(RuntimeError, match="CUDA device"):
        ops.moe_decode(**a)


@pytest.mark.skipif(not native.available(), reason="native extension not built")
@pytest.mark.parametrize("distances,one", [
    ([], True), ([1 << 20] * 7, True), ([16] * 3, True), ([(1 << 40) - 16], True),
    ([1 << 40], False), ([1 << 41] * 3, False),           # farther than a tensor map's stride reaches
    ([1 << 20, 1 << 20, 1 << 21], False), ([-(1 << 20)] * 3, False), ([0, 0], False), ([8], False),
])
def test_one_tensor_map_for_all_experts(distances, one):
    w = [1 << 44]
    for d in distances:
        w.append(w[-1] + d)
    assert native.lib().moe_decode_one_map(w) == one


def test_model_constants_are_the_kernel_s():
    import os
    import re

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    text = open(os.path.join(root, "flextensor_b200", "ops", "csrc", "moe_decode_sm100.cu")).read()
    value = lambda name: int(re.search(rf"constexpr int {name} = (\d+);", text).group(1))  # noqa: E731
    assert (value("BM"), value("BK"), value("MIN_CHUNKS")) == (128, 64, 4)
    head = open(os.path.join(root, "flextensor_b200", "ops", "csrc", "ft_moe_decode.h")).read()
    limit = lambda name: int(re.search(rf"constexpr int {name} = (\d+);", head).group(1))  # noqa: E731
    assert (ops.MOE_DECODE_MAX_TOKENS, ops.MOE_DECODE_MAX_EXPERTS, ops.MOE_DECODE_MAX_TOPK) == \
        (limit("kMoeDecMaxTokens"), limit("kMoeDecMaxExperts"), limit("kMoeDecMaxTopk"))
