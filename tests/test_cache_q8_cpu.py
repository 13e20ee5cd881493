"""Refusals of the 8-bit cache entry points: every malformed call raises before anything is
launched (the checks of shapes, types and strides come before the device check, so they run on
CPU tensors)."""

import pytest
import torch

from flextensor_b200 import ops
from flextensor_b200.ops import native

pytestmark = pytest.mark.skipif(not native.available(), reason="native extension not built")

B, L, HK, S, BLOCK = 2, 100, 2, 5, 32


def cache(dtype=torch.int8, b=B, l=L, hk=HK, block=BLOCK):
    nb = -(-l // block)
    return [torch.zeros(b, l, hk, 128, dtype=dtype), torch.zeros(b, l, hk, 128, dtype=dtype),
            torch.zeros(b, nb, hk), torch.zeros(b, nb, hk)]


def new(b=B, s=S, hk=HK, dtype=torch.bfloat16):
    return torch.zeros(b, s, hk, 128, dtype=dtype)


def lens(*v):
    return torch.tensor(v, dtype=torch.int32)


def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError, match="CUDA device"):
        ops.kv_append_q8(new(), new(), *cache(), 0, block=BLOCK)
    with pytest.raises(RuntimeError, match="CUDA device"):
        ops.decode_attention_q8(torch.zeros(B, 4, 128, dtype=torch.bfloat16), *cache(), L, block=BLOCK)


@pytest.mark.parametrize("change,match", [
    (lambda c: c.__setitem__(0, c[0].to(torch.uint8)), "int8 or both float8"),
    (lambda c: c.__setitem__(1, c[1].to(torch.float8_e4m3fn)), "int8 or both float8"),
    (lambda c: c.__setitem__(1, c[1][:, :-1]), "of one shape"),
    (lambda c: c.__setitem__(0, c[0][..., :64]), "of one shape"),
    (lambda c: c.__setitem__(2, c[2][:, :-1]), "scales must be"),
    (lambda c: c.__setitem__(3, c[3].half()), "scales must be"),
    (lambda c: c.__setitem__(3, c[3][..., :1]), "scales must be"),
    (lambda c: c.__setitem__(0, torch.zeros(B, L, 128, HK, dtype=torch.int8).transpose(2, 3)), "16-byte"),
    (lambda c: c.__setitem__(0, torch.zeros(B * L * HK * 128 + 1, dtype=torch.int8)[1:].view(B, L, HK, 128)), "16-byte"),
    (lambda c: c.__setitem__(1, torch.zeros(B, L, HK * 128 + 8, dtype=torch.int8)[..., :HK * 128].unflatten(2, (HK, 128))), "16-byte"),
])
def test_malformed_caches_are_refused(change, match):
    c = cache()
    change(c)
    with pytest.raises(RuntimeError, match=match):
        ops.kv_append_q8(new(), new(), *c, 0, block=BLOCK)
    with pytest.raises(RuntimeError, match=match):
        ops.decode_attention_q8(torch.zeros(B, 4, 128, dtype=torch.bfloat16), *c, L, block=BLOCK)


@pytest.mark.parametrize("block", [0, 8, 24, 48, 512, -64])
def test_block_sizes(block):
    with pytest.raises(RuntimeError, match="block must be"):
        ops.kv_append_q8(new(), new(), *cache(), 0, block=block)


@pytest.mark.parametrize("args,kw,match", [
    ((new(dtype=torch.float16), new(), 0), {}, "bfloat16"),
    ((new(), new(s=S + 1), 0), {}, "k and v must be"),
    ((new(hk=1), new(hk=1), 0), {}, "k and v must be"),
    ((new(b=1), new(b=1), 0), {}, "k and v must be"),
    ((new().transpose(1, 3).contiguous().transpose(1, 3), new(), 0), {}, "16-byte"),
    ((new(), new(), -1), {}, "do not fit"),
    ((new(), new(), L - S + 1), {}, "do not fit"),
    ((new(s=L + 1), new(s=L + 1), 0), {}, "do not fit"),
    ((new(s=L + 1), new(s=L + 1), lens(0, 0)), {}, "do not fit"),
    ((new(), new(), lens(0)), {}, "one number per sequence"),
    ((new(), new(), lens(0, 0).long()), {}, "one number per sequence"),
    ((new(), new(), 0), {"n_new": lens(1, 1, 1)}, "one number per sequence"),
    ((new(), new(), 0), {"n_new": torch.zeros(B, 1, dtype=torch.int32)}, "one number per sequence"),
])
def test_append_refusals(args, kw, match):
    k, v, pos = args
    with pytest.raises(RuntimeError, match=match):
        ops.kv_append_q8(k, v, *cache(), pos, block=BLOCK, **kw)


def test_append_refuses_a_cache_that_overlaps_itself():
    c = cache()
    c[0] = torch.zeros(1, L, HK, 128, dtype=torch.int8).expand(B, L, HK, 128)
    with pytest.raises(RuntimeError, match="overlap"):
        ops.kv_append_q8(new(), new(), *c, 0, block=BLOCK)
    c = cache()
    c[1] = c[0]
    with pytest.raises(RuntimeError, match="[Oo]verlap|memory"):
        ops.kv_append_q8(new(), new(), *c, 0, block=BLOCK)


@pytest.mark.parametrize("q,kv_len,kw,match", [
    (torch.zeros(B, 4, 128), L, {}, "bfloat16"),
    (torch.zeros(B, 4, 64, dtype=torch.bfloat16), L, {}, "128"),
    (torch.zeros(B, 3, 128, dtype=torch.bfloat16), L, {}, "multiple of kv heads"),
    (torch.zeros(B + 1, 4, 128, dtype=torch.bfloat16), L, {}, "sequences"),
    (torch.zeros(B, 4, 128, dtype=torch.bfloat16), L + 1, {}, "lengths must lie"),
    (torch.zeros(B, 4, 128, dtype=torch.bfloat16), -1, {}, "lengths must lie"),
    (torch.zeros(B, 4, 128, dtype=torch.bfloat16), lens(1, 1), {"max_len": L + 1}, "lengths must lie"),
    (torch.zeros(B, 4, 128, dtype=torch.bfloat16), lens(1), {}, "one number per sequence"),
    (torch.zeros(B, 4, 128, dtype=torch.bfloat16), L, {"out": torch.zeros(B, 2, 128, dtype=torch.bfloat16)}, "shape of q"),
    (torch.zeros(B, 4, 128, dtype=torch.bfloat16), L, {"out": torch.zeros(B, 1, 128, dtype=torch.bfloat16).expand(B, 4, 128)}, "overlap"),
    (torch.zeros(B, 4, 129, dtype=torch.bfloat16)[..., 1:], L, {}, "16-byte"),
])
def test_attention_refusals(q, kv_len, kw, match):
    with pytest.raises(RuntimeError, match=match):
        ops.decode_attention_q8(q, *cache(), kv_len, block=BLOCK, **kw)


def codes(at, strides, l=L):
    buf = torch.zeros(4 * B * L * HK * 128, dtype=torch.int8)
    return buf[at:].as_strided((B, l, HK, 128), (*strides, 1), buf.storage_offset() + at), buf


@pytest.mark.parametrize("strides,refused", [
    ((L * HK * 128, HK * 128, 64), True),       # heads half on one another
    ((L * HK * 128, 128, 128), True),           # a token's second head is the next one's first
    ((128, 2 * HK * 128, 128), True),           # sequences
    ((L * HK * 128, 128, L * 128), False),      # heads first
    ((HK * 128, B * HK * 128, 128), False),     # tokens first
    ((L * HK * 256, HK * 256, 256), False),     # rows with gaps
])
def test_append_refuses_strided_caches_that_overlap_themselves(strides, refused):
    c = cache()
    c[0], _ = codes(0, strides)
    with pytest.raises(RuntimeError, match="overlap itself" if refused else "CUDA device"):
        ops.kv_append_q8(new(), new(), *c, 0, block=BLOCK)
    c = cache()
    c[2] = torch.zeros(64).as_strided((B, 4, HK), (8, 1, 2) if refused else (8, 2, 1))
    with pytest.raises(RuntimeError, match="overlap itself" if refused else "CUDA device"):
        ops.kv_append_q8(new(), new(), *c, 0, block=BLOCK)


@pytest.mark.parametrize("gap,refused", [(HK * 128, False), (128, True), (0, True), (2 * HK * 128, True), (B * L * 2 * HK * 128, False),
                                         (L * 2 * HK * 128 + 128, True), (3 * HK * 128, False)])
def test_append_refuses_strided_caches_that_overlap_one_another(gap, refused):
    """Keys and values as views of one buffer, [B, L, 2, Hk, 128] where they are side by side."""
    strides = (L * 2 * HK * 128, 2 * HK * 128, 128)
    c = cache()
    c[0], buf = codes(0, strides)
    c[1] = buf.as_strided((B, L, HK, 128), (*strides, 1), gap)
    with pytest.raises(RuntimeError, match="must not overlap" if refused else "CUDA device"):
        ops.kv_append_q8(new(), new(), *c, 0, block=BLOCK)
    c = cache()
    both = torch.zeros(B, 4, 2, HK)
    c[2], c[3] = both[:, :, 0], both[:, :, 1]
    with pytest.raises(RuntimeError, match="CUDA device"):
        ops.kv_append_q8(new(), new(), *c, 0, block=BLOCK)
    c[3] = both[:, :, 0]
    with pytest.raises(RuntimeError, match="must not overlap"):
        ops.kv_append_q8(new(), new(), *c, 0, block=BLOCK)


@pytest.mark.parametrize("shape,strides,refused", [
    ((B, 4, 128), (4 * 128, 120, 1), True), ((B, 4, 128), (128, 128, 1), True), ((B, 4, 128), (128, 256, 1), False),
    ((B, 3, 4, 128), (1536, 128, 128, 1), True), ((B, 3, 4, 128), (1536, 128, 384, 1), False),
])
def test_attention_refuses_strided_outputs_that_overlap_themselves(shape, strides, refused):
    q = torch.zeros(shape, dtype=torch.bfloat16)
    out = torch.zeros(8192, dtype=torch.bfloat16).as_strided(shape, strides)
    with pytest.raises(RuntimeError, match="overlap itself" if refused else "CUDA device"):
        ops.decode_attention_q8(q, *cache(), L, block=BLOCK, out=out)


@pytest.mark.parametrize("pos", [2 ** 63 - 1, 2 ** 63 - S, 2 ** 31, -2 ** 63])
def test_append_refuses_positions_past_any_cache(pos):
    with pytest.raises(RuntimeError, match="do not fit"):
        ops.kv_append_q8(new(), new(), *cache(), pos, block=BLOCK)


def test_single_entries_may_have_any_stride():
    """A dimension of one entry is never stepped over: its stride does not matter (contiguous() leaves it
    as it is, so a caller could not mend it)."""
    odd = lambda t: t.as_strided(t.shape, [3 if n == 1 else s for n, s in zip(t.shape, t.stride())])  # noqa: E731
    c = [odd(t) if t.dim() == 4 else t for t in cache(b=1, l=1, hk=1)]
    x = odd(new(b=1, s=1, hk=1))
    with pytest.raises(RuntimeError, match="CUDA device"):
        ops.kv_append_q8(x, x, *c, 0, block=BLOCK)
    for q in (odd(torch.zeros(1, 1, 128, dtype=torch.bfloat16)), x):
        with pytest.raises(RuntimeError, match="CUDA device"):
            ops.decode_attention_q8(q, *c, 1, block=BLOCK, out=odd(torch.zeros_like(q)))
