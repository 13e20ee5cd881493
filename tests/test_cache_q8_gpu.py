"""The 8-bit key/value cache on the GPU: what ``kv_append_q8`` writes, bit for bit against the
definition in 64 bits, and ``decode_attention_q8`` against softmax attention in 64 bits over the
values that the codes stand for.

Attention's tolerance, per output element, with A = sum_k p_k |v_k| (the weights of the row):
the output's rounding to bf16 is 2^-8 |o|; each weight is rounded to f16, 2^-11 p, so 2^-11 A;
the sum that divides holds the weights in fp32. Scores are sums of 128 products in fp32 with
|q . k| * scale below 64 in every test, at most 128 roundings of 2^-24 on them: 64 * 128 * 2^-24 =
2^-11 in the exponent at the very worst, as a relative error of p: 2^-11 A again, and 2^-11 A for
the quotient's. Together 2^-8 |o| + 3 * 2^-11 A, taken as 2^-8 |o| + 2^-9 A."""

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("needs a CUDA device", allow_module_level=True)

from flextensor_b200 import ops  # noqa: E402
from flextensor_b200.ops import native  # noqa: E402

DEV = "cuda"
FMT = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
QMAX = {"int8": 127.0, "e4m3": 448.0}


def new_cache(fmt, B, L, Hk, block, heads_first=False):
    nb = -(-L // block)
    out = []
    for _ in range(2):
        c = torch.zeros((B, Hk, L, 128) if heads_first else (B, L, Hk, 128), dtype=FMT[fmt], device=DEV)
        out.append(c.transpose(1, 2) if heads_first else c)
    return out + [torch.zeros(B, nb, Hk, device=DEV) for _ in range(2)]


def junk_cache(fmt, B, L, Hk, block, seed, scale=0.03):
    """Random codes everywhere and power-of-two scales of different sizes."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    c = new_cache(fmt, B, L, Hk, block)
    for i in range(2):
        x = torch.randn(B, L, Hk, 128, device=DEV, generator=g) * QMAX[fmt] / 4
        c[i].copy_(x.clamp(-QMAX[fmt], QMAX[fmt]).round().to(FMT[fmt]) if fmt == "int8" else x.clamp(-448, 448).to(FMT[fmt]))
        e = torch.randint(-2, 3, c[2 + i].shape, device=DEV, generator=g)
        c[2 + i].copy_(torch.ldexp(torch.full(e.shape, 4 / QMAX[fmt] * scale * 32, device=DEV), e))
    return c


def bf16(seed, *shape, spread=True):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(*shape, device=DEV, generator=g)
    if spread:  # tokens of very different sizes, so that blocks' scales grow
        x *= torch.exp2(torch.randint(-4, 5, shape[:2], device=DEV, generator=g).float())[..., None, None]
    return x.bfloat16()


def ref_append(x, codes, scales, pos, count, block, fmt):
    """The definition, block by block in float64: (codes, scales) as float64."""
    codes, scales = codes.double().clone(), scales.double().clone()
    for b in range(x.shape[0]):
        lo, end = pos[b], pos[b] + count[b]
        while lo < end:
            j = lo // block
            hi = min(end, (j + 1) * block)
            r = x[b, lo - pos[b]:hi - pos[b]].double()
            a = r.abs().amax(dim=(0, 2))
            m, e = torch.frexp(a / QMAX[fmt])
            s = torch.where(a > 0, torch.ldexp(torch.ones_like(a), (e - (m == 0.5).int()).clamp(min=-120)), torch.zeros_like(a))
            s = torch.where(torch.isfinite(a), s, torch.full_like(a, float("nan")))
            if lo > j * block:
                s0 = scales[b, j]
                s = torch.maximum(s, s0)
                grown = ~(s == s0)
                old = codes[b, j * block:lo] * torch.where(s > 0, s0 / s, torch.zeros_like(s))[None, :, None]
                old = torch.nan_to_num(old).round() if fmt == "int8" else torch.nan_to_num(old).float().to(FMT[fmt]).double()
                codes[b, j * block:lo] = torch.where(grown[None, :, None], old, codes[b, j * block:lo])
            inv = torch.where(s > 0, 1 / s, torch.zeros_like(s))
            c = torch.nan_to_num(r * inv[None, :, None], posinf=0, neginf=0)
            c = c * torch.isfinite(s)[None, :, None]
            codes[b, lo:hi] = c.round() if fmt == "int8" else c.float().to(FMT[fmt]).double()
            scales[b, j] = s
            lo = hi
    return codes, scales


def check_append(k, v, cache, pos, count, block, fmt, **kw):
    want = [ref_append(x, cache[i], cache[2 + i], pos, count, block, fmt) for i, x in enumerate((k, v))]
    ops.kv_append_q8(k, v, *cache, kw.pop("pos_arg"), block=block, **kw)
    torch.cuda.synchronize()
    for i in range(2):
        assert torch.equal(torch.nan_to_num(cache[2 + i].double(), nan=-1.0), torch.nan_to_num(want[i][1], nan=-1.0))
        assert torch.equal(cache[i].double(), want[i][0])
    assert native.device_error(reset=True) == 0


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("block", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("B,S,L,Hk,pos", [(1, 1, 1, 1, 0), (2, 1, 300, 3, 77), (3, 130, 300, 2, 0), (2, 299, 300, 1, 1), (1, 515, 777, 5, 250)])
def test_append_codes(fmt, block, B, S, L, Hk, pos):
    cache = junk_cache(fmt, B, L, Hk, block, 3)
    k, v = bf16(1, B, S, Hk, 128), bf16(2, B, S, Hk, 128)
    check_append(k, v, cache, [pos] * B, [S] * B, block, fmt, pos_arg=pos)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_append_padded_batch(fmt):
    """Each sequence at its own position with its own count; padding rows hold NaN and are not read."""
    B, S, L, Hk, block = 6, 70, 200, 2, 32
    cache = junk_cache(fmt, B, L, Hk, block, 4)
    k, v = bf16(5, B, S, Hk, 128), bf16(6, B, S, Hk, 128)
    pos, count = [0, 31, 64, 130, 200, 17], [70, 1, 33, 70, 0, 0]
    for b in range(B):
        k[b, count[b]:] = float("nan")
        v[b, count[b]:] = float("inf")
    check_append(k, v, cache, pos, count, block, fmt, pos_arg=torch.tensor(pos, dtype=torch.int32, device=DEV),
                 n_new=torch.tensor(count, dtype=torch.int32, device=DEV))


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_append_token_by_token(fmt):
    """70 single tokens, the scales growing on the way; strided new tokens (a slice of a fused
    projection) and a heads-first cache."""
    B, Hk, L, block = 2, 2, 75, 64
    qkv = bf16(7, B, 70, 12, 128) * torch.exp2(torch.arange(70, device=DEV) / 9.0).bfloat16()[None, :, None, None]
    cache = new_cache(fmt, B, L, Hk, block, heads_first=True)
    for t in range(70):
        check_append(qkv[:, t:t + 1, 8:10], qkv[:, t:t + 1, 10:12], cache, [t] * B, [1] * B, block, fmt, pos_arg=t)
    # every value lies within one step of its code's (half a step for each time the scale doubled: 1/2 + 1/4 + ...)
    if fmt == "int8":
        s = cache[2].repeat_interleave(block, 1)[:, :70, :, None]
        assert bool(((cache[0][:, :70].float() * s - qkv[:, :, 8:10].float()).abs() <= s).all())


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_append_special_values(fmt):
    B, S, Hk, L, block = 1, 64, 1, 128, 16
    k, v = bf16(8, B, S, Hk, 128, spread=False), bf16(9, B, S, Hk, 128, spread=False)
    k[:, :16] = 0.0                                   # a block of zeros
    k[:, 16:32] = k[:, 16:32] * 2.0 ** -126           # below the smallest scale
    k[0, 40, 0, 5] = float("nan")
    v[0, 63, 0, 127] = float("-inf")
    v[:, :16] = torch.finfo(torch.bfloat16).max       # the type's largest
    v[:, 16:32] = torch.finfo(torch.bfloat16).min
    cache = junk_cache(fmt, B, L, Hk, block, 5)
    check_append(k, v, cache, [0], [S], block, fmt, pos_arg=0)
    assert cache[2].isnan().nonzero().tolist() == [[0, 2, 0]] and cache[3].isnan().nonzero().tolist() == [[0, 3, 0]]
    check_append(k[:, :1], v[:, :1], cache, [41], [1], block, fmt, pos_arg=41)  # NaN stays until the block starts afresh
    assert cache[2][0, 2, 0].isnan()
    check_append(v[:, 40:56], v[:, 40:56], cache, [32], [16], block, fmt, pos_arg=32)
    assert not cache[2][0, 2, 0].isnan()


def test_append_leaves_sequences_that_do_not_fit():
    B, S, L, Hk, block = 4, 5, 40, 2, 16
    cache = junk_cache("int8", B, L, Hk, block, 6)
    before = [c.clone() for c in cache]
    k, v = bf16(10, B, S, Hk, 128), bf16(11, B, S, Hk, 128)
    pos = torch.tensor([36, -1, 3, 3], dtype=torch.int32, device=DEV)
    n = torch.tensor([5, 5, 6, -2], dtype=torch.int32, device=DEV)
    ops.kv_append_q8(k, v, *cache, pos, block=block, n_new=n)
    torch.cuda.synchronize()
    assert native.device_error(reset=True) != 0
    assert all(torch.equal(a.float(), b.float()) for a, b in zip(cache, before))


# ----------------------------------------------------------------------------- attention
def ref_attend(q, cache, lens, block):
    """(output, sum of p |v|) in float64."""
    kc, vc, ks, vs = cache
    B, Sq, Hq, _ = q.shape
    Hk = kc.shape[2]
    o = torch.zeros(B, Sq, Hq, 128, dtype=torch.float64, device=DEV)
    A = torch.zeros_like(o)
    for b in range(B):
        n = int(lens[b])
        j = torch.arange(n, device=DEV) // block
        k = kc[b, :n].double() * ks[b, j].double()[..., None]
        v = vc[b, :n].double() * vs[b, j].double()[..., None]
        for i in range(Sq):
            m = n - Sq + 1 + i
            if m <= 0:
                continue
            for h in range(Hq):
                hk = h // (Hq // Hk)
                p = torch.softmax(k[:m, hk] @ q[b, i, h].double() * 128 ** -0.5, 0)
                o[b, i, h], A[b, i, h] = p @ v[:m, hk], p @ v[:m, hk].abs()
    return o, A


def check_attend(q, cache, lens, block, kv_len, **kw):
    want, A = ref_attend(q if q.dim() == 4 else q[:, None], cache, lens, block)
    got = ops.decode_attention_q8(q, *cache, kv_len, block=block, **kw)
    torch.cuda.synchronize()
    assert native.device_error(reset=True) == 0 and got.shape == q.shape
    err = (got.double().view(want.shape) - want).abs()
    assert bool((err <= want.abs() * 2 ** -8 + A * 2 ** -9).all()), float((err / (A + 1e-30)).max())
    return got


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("B,Sq,L,Hq,Hk,block", [
    (1, 1, 1, 1, 1, 16), (2, 1, 33, 8, 1, 32), (3, 1, 300, 8, 8, 64), (2, 1, 1000, 48, 8, 64), (1, 1, 5000, 16, 1, 128),
    (4, 1, 130, 5, 5, 256), (1, 1, 777, 64, 2, 64), (2, 1, 257, 96, 2, 16), (2, 3, 300, 16, 4, 64), (1, 8, 520, 24, 4, 32),
    (3, 5, 65, 3, 1, 16), (1, 40, 100, 4, 2, 64)])
def test_attention(fmt, B, Sq, L, Hq, Hk, block):
    """Groups of 1 to 48 heads, one and several queries, full and ragged lengths; codes past each
    length are e4m3 NaN / int8 -128 and their blocks' scales NaN."""
    cache = junk_cache(fmt, B, L, Hk, block, B * 31 + L)
    q = bf16(12, B, Sq, Hq, 128, spread=False)
    check_attend(q if Sq > 1 else q[:, 0], cache, [L] * B, block, L)
    lens = torch.randint(0, L + 1, (B,), generator=torch.Generator().manual_seed(L)).tolist()
    lens[0] = max(1, L - 1)
    for b in range(B):
        for i in range(2):
            cache[i][b].view(torch.uint8)[lens[b]:] = 0x80 if fmt == "int8" else 0x7f
            cache[2 + i][b, -(-lens[b] // block):] = float("nan")
    check_attend(q, cache, lens, block, torch.tensor(lens, dtype=torch.int32, device=DEV))


def test_attention_bounds_and_strides():
    """max_len cuts longer lengths, lengths below zero count as none; a heads-first cache, a prefix
    view of a longer one, strided q and out."""
    B, L, Hq, Hk, block = 4, 200, 8, 2, 32
    cache = junk_cache("int8", B, L + 56, Hk, block, 9)
    lens = torch.tensor([200, 150, -3, 0], dtype=torch.int32, device=DEV)
    q = bf16(13, B, 3, Hq, 128, spread=False)[:, 1]
    out = torch.zeros(B, Hq, 256, device=DEV, dtype=torch.bfloat16)[..., 128:]
    got = check_attend(q, cache, [160, 150, 0, 0], block, lens, max_len=160, out=out)
    assert got.data_ptr() == out.data_ptr() and bool((got[2:] == 0).all())
    hf = [c.transpose(1, 2).contiguous().transpose(1, 2) for c in cache]
    view = [hf[0][:, :L], hf[1][:, :L], hf[2][:, :7], hf[3][:, :7]]
    check_attend(q, view, [L] * B, block, L)


def test_attention_over_a_shared_cache():
    """A cache expanded over sequences (one prompt for several), or over heads; q expanded too; out = q."""
    B, L, Hq, Hk, block = 5, 230, 16, 2, 64
    lens = torch.tensor([230, 1, 64, 100, 0], dtype=torch.int32, device=DEV)
    one = junk_cache("e4m3", 1, L, Hk, block, 21)
    q = bf16(22, B, Hq, 128, spread=False)
    check_attend(q, [c.expand(B, *c.shape[1:]) for c in one], lens, block, lens)
    narrow = junk_cache("int8", B, L, 1, block, 23)
    wide = [narrow[0].expand(B, L, Hk, 128), narrow[1].expand(B, L, Hk, 128), narrow[2].expand(B, -1, Hk), narrow[3].expand(B, -1, Hk)]
    want = check_attend(q[:1].expand(B, Hq, 128), wide, lens, block, lens)
    mine = q[:1].expand(B, Hq, 128).contiguous()
    assert torch.equal(ops.decode_attention_q8(mine, *wide, lens, block=block, out=mine), want)


def test_attention_scales_and_magnitudes():
    """Value scales 2^40 apart between blocks, zero scales, queries near the type's limits."""
    B, L, Hq, Hk, block = 1, 128, 8, 1, 16
    cache = junk_cache("int8", B, L, Hk, block, 10)
    q = bf16(14, B, Hq, 128, spread=False)
    cache[3][0, :, 0] = torch.tensor([2.0 ** -20, 2.0 ** 20, 0, 1, 2.0 ** -20, 0, 1, 2.0 ** 10], device=DEV)
    check_attend(q, cache, [L], block, L)
    cache[3].zero_()
    assert bool((check_attend(q, cache, [L], block, L) == 0).all())
    cache[3].fill_(0.5)
    cache[2].zero_()  # every score 0: the mean of the values
    check_attend(q, cache, [L], block, L)
    cache[2].fill_(2.0 ** -100)
    check_attend((q.float() * 2.0 ** 98).bfloat16(), cache, [L], block, L)
    cache[2].fill_(2.0 ** 100)
    check_attend((q.float() * 2.0 ** -108).bfloat16(), cache, [L], block, L)


@pytest.mark.parametrize("scale", [2.0 ** 115, 2.0 ** 60, 2.0 ** -70])
def test_attention_far_value_scales(scale):
    """All values huge or tiny, a third of them zero up to 2^60 (their sum and the zeros' are far apart in size)."""
    L, block = 384, 32
    cache = junk_cache("int8", 2, L, 2, block, 41)
    cache[3].fill_(scale)
    if scale == 2.0 ** 60:
        cache[3][:, ::3] = 0
    check_attend(bf16(42, 2, 8, 128, spread=False), cache, [L, 200], block, torch.tensor([L, 200], dtype=torch.int32, device=DEV))


def test_attention_zeros_before_values():
    """12288 keys with zero values, all but the first of them e^5.5 heavier, then 4096 with values: the
    zeros only divide. One warp passes over a whole sequence here (more sequences than SMs)."""
    B, L, Hk, block = 160, 16384, 8, 64
    one = new_cache("int8", 1, L, Hk, block)
    one[0][:, block:, :, 0] = 64
    one[1][:, 12288:] = 64
    one[2].fill_(2.0 ** -6)
    one[3][:, 12288 // block:] = 2.0 ** -6
    q = torch.zeros(B, Hk, 128, device=DEV, dtype=torch.bfloat16)
    q[..., 0] = 5.5 * 128 ** 0.5
    got = ops.decode_attention_q8(q, *[c.expand(B, *c.shape[1:]) for c in one], L, block=block)
    torch.cuda.synchronize()
    want, A = ref_attend(q[:1, None], one, [L], block)
    assert bool(((got.double() - want[0]).abs() <= want[0].abs() * 2 ** -8 + A[0] * 2 ** -9).all())


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_attention_many_small_weights(fmt):
    """One key outweighs each of 131071 others by e^18 = 2^26, and its value is zero: the output is what
    the others add up to, although each of their weights is below f16's steps next to 1."""
    L, block = 131072, 256
    cache = new_cache(fmt, 1, L, 1, block)
    one = 64 if fmt == "int8" else 64.0
    cache[0][..., 0] = one                        # every key: 64 in dim 0 ...
    cache[0][0, 70001, 0, 1] = one                # ... the heavy one 64 in dim 1 too
    cache[1].copy_(torch.full((), one, device=DEV).expand(1, L, 1, 128).to(FMT[fmt]))
    cache[1][0, 70001] = 0
    cache[2].fill_(2.0 ** -6)
    cache[3].fill_(2.0 ** -6)
    q = torch.zeros(1, 8, 128, device=DEV, dtype=torch.bfloat16)
    q[..., 0] = 1.0
    q[..., 1] = 18.0 * 128 ** 0.5
    got = check_attend(q, cache, [L], block, L)
    assert 1e-3 < float(got.min()) and float(got.max()) < 3e-3


def test_attention_keeps_nan():
    """A NaN block reaches exactly the rows that see it, through keys or values alike."""
    B, Sq, L, Hq, Hk, block = 2, 3, 96, 4, 1, 32
    for side in (2, 3):
        cache = junk_cache("int8", B, L, Hk, block, 11)
        cache[side][0, 2] = float("nan")
        q = bf16(15, B, Sq, Hq, 128, spread=False)
        lens = torch.tensor([66, 66], dtype=torch.int32, device=DEV)  # query 0 sees 64 keys, none of block 2
        got = ops.decode_attention_q8(q, *cache, lens, block=block)
        assert not got[0, 0].isnan().any() and got[0, 1:].isnan().all() and not got[1].isnan().any()
        cache[side][:] = float("nan")
        assert ops.decode_attention_q8(q, *cache, lens, block=block).isnan().all()
    q[0, 0, 0, 0] = float("nan")
    cache = junk_cache("int8", B, L, Hk, block, 11)
    got = ops.decode_attention_q8(q, *cache, lens, block=block)
    assert got[0, 0, 0].isnan().all() and not got[0, 0, 1:].isnan().any() and not got[1].isnan().any()


def test_attention_past_two_gigabytes():
    """Offsets past 32 bits: a cache of 2.3 GB a side, read near its end."""
    B, L, Hk, block = 1, 2_250_000, 8, 256
    g = torch.Generator(device=DEV).manual_seed(1)
    cache = [torch.empty(B, L, Hk, 128, dtype=torch.int8, device=DEV).random_(-127, 128, generator=g) for _ in range(2)]
    cache += [torch.full((B, -(-L // block), Hk), 0.01, device=DEV) for _ in range(2)]
    k, v = bf16(16, B, 3, Hk, 128, spread=False), bf16(17, B, 3, Hk, 128, spread=False)
    ops.kv_append_q8(k * 8, v, *cache, L - 3, block=block)
    q = (k[:, 1] * 4).contiguous()  # each head finds its own new key
    got = ops.decode_attention_q8(q, *cache, L, block=block)
    torch.cuda.synchronize()
    for h in (0, Hk - 1):
        s = torch.cat([(cache[0][0, i:i + 250_000, h].float() * 0.01) @ q[0, h].float() for i in range(0, L, 250_000)])
        s[-3:] = (cache[0][0, -3:, h].float() * cache[2][0, -1, h]) @ q[0, h].float()
        p = torch.softmax(s.double() * 128 ** -0.5, 0)
        assert float(p[-2]) > 0.5
        want = sum((p[i:i + 250_000] @ (cache[1][0, i:i + 250_000, h].double() * 0.01)) for i in range(0, L - 250_000, 250_000))
        tail = cache[1][0, L - 250_000:, h].double() * 0.01
        first = (L - 1) // block * block - (L - 250_000)
        tail[first:] = cache[1][0, L - 250_000 + first:, h].double() * cache[3][0, -1, h].double()
        want = want + p[L - 250_000:] @ tail
        err = (got[0, h].double() - want).abs()
        assert bool((err <= want.abs() * 2 ** -8 + 3 * 2 ** -9).all())  # A <= the largest |v| here, below 3


def test_streams_and_graphs():
    """A side stream; a decode step captured once and replayed at new lengths beside an eager call."""
    B, L, Hq, Hk, block = 3, 400, 8, 2, 64
    cache = junk_cache("e4m3", B, L, Hk, block, 12)
    k, v, q = bf16(18, B, 1, Hk, 128), bf16(19, B, 1, Hk, 128), bf16(20, B, Hq, 128, spread=False)
    pos = torch.tensor([5, 200, 398], dtype=torch.int32, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    n = torch.empty_like(pos)

    def step():
        ops.kv_append_q8(k, v, *cache, pos, block=block)
        torch.add(pos, 1, out=n)
        return ops.decode_attention_q8(q, *cache, n, block=block)

    with torch.cuda.stream(side):
        check_attend(q, cache, [L] * B, block, L)
        before = [c.clone() for c in cache]
        step()
        for c, o in zip(cache, before):
            c.copy_(o)
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        got = step()
    for at in ([0, 63, 64], [399, 1, 128]):
        for c, o in zip(cache, before):
            c.copy_(o)
        pos.copy_(torch.tensor(at, dtype=torch.int32))
        graph.replay()
        eager = ops.decode_attention_q8(q, *before, L, block=block)  # its own workspace, in flight beside the replay's
        torch.cuda.synchronize()
        want_c = [c.clone() for c in before]
        ops.kv_append_q8(k, v, *want_c, pos, block=block)
        assert all(torch.equal(a.float(), b.float()) for a, b in zip(cache, want_c))
        assert torch.equal(got, ops.decode_attention_q8(q, *want_c, n, block=block))
        assert torch.equal(eager, ops.decode_attention_q8(q, *before, L, block=block))


def test_empty_calls():
    cache = junk_cache("int8", 2, 64, 2, 64, 13)
    before = [c.clone() for c in cache]
    ops.kv_append_q8(bf16(1, 2, 0, 2, 128), bf16(1, 2, 0, 2, 128), *cache, 64)
    assert all(torch.equal(a, b) for a, b in zip(cache, before))
    assert bool((ops.decode_attention_q8(bf16(1, 2, 4, 128, spread=False), *cache, 0) == 0).all())
    none = junk_cache("int8", 1, 0, 2, 64, 13)
    assert bool((ops.decode_attention_q8(bf16(1, 1, 4, 128, spread=False), *none, 0) == 0).all())


def test_attention_without_keys_takes_the_merge_alone():
    """No key may count (a cache of length 0, or max_len 0): no tensor map is made of it and the first
    kernel is not launched; the lengths on the device have no say."""
    q = bf16(1, 1, 3, 4, 128, spread=False)
    for L, kv_len in ((0, 0), (0, torch.tensor([7], dtype=torch.int32, device=DEV)), (40, 0),
                      (40, torch.tensor([40], dtype=torch.int32, device=DEV))):
        cache = junk_cache("int8", 1, L, 2, 64, 13)
        before = ops.launch_count()
        got = ops.decode_attention_q8(q, *cache, kv_len, max_len=0, out=torch.full_like(q, 7.0))
        assert ops.launch_count() - before == 1 and bool((got == 0).all())
    assert native.device_error(reset=True) == 0


@pytest.mark.parametrize("scale,top", [(2.0 ** 121, 60), (2.0 ** 122, 60), (2.0 ** 126, 3), (2.0 ** 127, 1)])
def test_attention_largest_value_scales(scale, top):
    """The largest scales that the append makes (2^122: int8 codes of bf16's largest values) and larger
    ones. 64 keys of weight 1, then 64 of up to 2^8: a weight of the second tile is as far above the first
    tile's reference as it may be without moving it. More sequences than SMs, so that a warp passes over
    both tiles."""
    B, L, Hk, block = 160, 128, 8, 64
    g = torch.Generator(device=DEV).manual_seed(3)
    one = new_cache("int8", 1, L, Hk, block)
    one[0][:, block:, :, 0] = 64
    one[1].copy_(torch.randint(-top, top + 1, one[1].shape, device=DEV, generator=g))
    one[2].fill_(2.0 ** -6)
    one[3].fill_(scale)
    q = torch.zeros(B, Hk, 128, device=DEV, dtype=torch.bfloat16)
    q[..., 0] = torch.tensor([8.0, 7.96875, 7.5, 6.0, 4.0, 2.0, 0.0, -8.0], device=DEV)
    ln2 = 0.6931471805599453  # scores in units of log2
    got = ops.decode_attention_q8(q, *[c.expand(B, *c.shape[1:]) for c in one], L, block=block, scale=ln2)
    torch.cuda.synchronize()
    want, A = ref_attend((q[:1, None].double() * (ln2 * 128 ** 0.5)), one, [L], block)
    assert bool(((got.double() - want[0]).abs() <= want[0].abs() * 2 ** -8 + A[0] * 2 ** -9).all())
    assert native.device_error(reset=True) == 0


@pytest.mark.parametrize("scale", [1.0, 2.0 ** 100, 2.0 ** 121, 2.0 ** 126])
def test_attention_small_weights_of_large_values(scale):
    """16383 keys, each 2^18 lighter than the first, whose value is zero: together 1/16 of its weight, at any
    size of the values. One warp passes over a whole sequence (more sequences than SMs)."""
    B, L, Hk, block = 160, 16384, 8, 64
    one = new_cache("int8", 1, L, Hk, block)
    one[0][:, 0, :, 0] = 64
    one[1][:, 1:] = 3
    one[2].fill_(2.0 ** -6)
    one[3].fill_(scale)
    q = torch.zeros(B, Hk, 128, device=DEV, dtype=torch.bfloat16)
    q[..., 0] = 18.0
    ln2 = 0.6931471805599453
    got = ops.decode_attention_q8(q, *[c.expand(B, *c.shape[1:]) for c in one], L, block=block, scale=ln2)
    torch.cuda.synchronize()
    want, A = ref_attend((q[:1, None].double() * (ln2 * 128 ** 0.5)), one, [L], block)
    assert float(want.min()) > 0.17 * scale
    assert bool(((got.double() - want[0]).abs() <= want[0].abs() * 2 ** -8 + A[0] * 2 ** -9).all())


def test_attention_infinite_value_scales_stay():
    """A block of an infinite value scale makes the rows that see it infinite or NaN and no others."""
    B, Sq, L, Hk, block = 1, 2, 96, 1, 16
    cache = junk_cache("int8", B, L, Hk, block, 43)
    cache[1][:, 48:64] = 1
    cache[3][0, 3] = float("inf")
    q = bf16(44, B, Sq, 4, 128, spread=False)
    clean = [c.clone() for c in cache]
    clean[3][0, 3] = 0
    n = torch.tensor([49], dtype=torch.int32, device=DEV)  # query 0 sees 48 keys, none of block 3
    got = ops.decode_attention_q8(q, *cache, n, block=block)
    assert torch.equal(got[:, :1], ops.decode_attention_q8(q, *clean, n, block=block)[:, :1]) and not got[:, 1:].isfinite().any()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_single_entries_may_have_any_stride(fmt):
    """One sequence, head, token: strides of those dimensions that no access could take."""
    odd = lambda t: t.as_strided(t.shape, [3 if n == 1 else s for n, s in zip(t.shape, t.stride())])  # noqa: E731
    for B, L, Hk, S in ((1, 1, 1, 1), (1, 100, 2, 1), (2, 70, 1, 3)):
        cache = [odd(c) for c in junk_cache(fmt, B, L, Hk, 32, 45)]
        k, v = odd(bf16(46, B, S, Hk, 128)), odd(bf16(47, B, S, Hk, 128))
        check_append(k, v, cache, [L - S] * B, [S] * B, 32, fmt, pos_arg=L - S)
        q = odd(bf16(48, B, S, 2 * Hk, 128, spread=False))
        check_attend(q, cache, [L] * B, 32, L, out=odd(torch.zeros(q.shape, device=DEV, dtype=torch.bfloat16)))


@pytest.mark.parametrize("ragged", [False, True])
def test_attention_of_many_queries(ragged):
    """1000 queries a sequence, as where a prompt is continued: the workspace stays below 256 MB (one launch
    for all would take 512 MB), and lengths shorter than the queries leave rows without keys."""
    B, Sq, L, Hq, Hk, block = 16, 1000, 1100, 64, 8, 64
    cache = junk_cache("int8", B, L, Hk, block, 51)
    q = bf16(52, B, Sq, Hq, 128, spread=False)
    lens = [L] * B
    if ragged:
        lens = torch.randint(0, L + 1, (B,), generator=torch.Generator().manual_seed(4)).tolist()
        lens[:4] = [0, 1, 999, 1000]
    kv_len = torch.tensor(lens, dtype=torch.int32, device=DEV) if ragged else L
    out = torch.empty_like(q)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before, launches = torch.cuda.memory_allocated(), ops.launch_count()
    ops.decode_attention_q8(q, *cache, kv_len, block=block, out=out)
    assert torch.cuda.max_memory_allocated() - before <= 257 << 20
    assert ops.launch_count() - launches > 2
    g = torch.Generator().manual_seed(5)
    for b in range(B):
        j = torch.arange(lens[b], device=DEV) // block
        for i in torch.randint(0, Sq, (4,), generator=g).tolist() + [0, Sq - 1]:
            m, h = lens[b] - Sq + 1 + i, int(torch.randint(0, Hq, (1,), generator=g))
            if m <= 0:
                assert bool((out[b, i] == 0).all())
                continue
            k = cache[0][b, :m, h // 8].double() * cache[2][b, j[:m], h // 8].double()[:, None]
            v = cache[1][b, :m, h // 8].double() * cache[3][b, j[:m], h // 8].double()[:, None]
            p = torch.softmax(k @ q[b, i, h].double() * 128 ** -0.5, 0)
            err = (out[b, i, h].double() - p @ v).abs()
            assert bool((err <= (p @ v).abs() * 2 ** -8 + (p @ v.abs()) * 2 ** -9).all())
    assert native.device_error(reset=True) == 0


def test_attention_of_many_queries_in_place():
    """Several launches: out may be q itself; another overlap is refused."""
    B, Sq, L, Hq, Hk, block = 32, 300, 320, 64, 1, 64
    cache = junk_cache("e4m3", B, L, Hk, block, 53)
    buf = torch.randn(B * Sq * Hq * 128 + 128, device=DEV, generator=torch.Generator(device=DEV).manual_seed(54)).bfloat16()
    q, shifted = buf[:-128].view(B, Sq, Hq, 128), buf[128:].view(B, Sq, Hq, 128)
    launches = ops.launch_count()
    want = ops.decode_attention_q8(q, *cache, L, block=block)
    assert ops.launch_count() - launches > 2
    with pytest.raises(RuntimeError, match="overlap it otherwise"):
        ops.decode_attention_q8(q, *cache, L, block=block, out=shifted)
    assert torch.equal(ops.decode_attention_q8(q, *cache, L, block=block, out=q), want)


def test_attention_of_many_queries_of_one_head():
    """Launches of 502 queries (32 groups of rows, eight side by side) and a last one of 494 (31, one by one), whose
    workspace is the larger."""
    B, Sq, L, block = 64, 8024, 8100, 256
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    queries, _ = native.lib().decode_attention_q8_plan(B, Sq, 1, 1, sms)
    assert len(set(queries)) > 1
    cache = junk_cache("int8", 1, L, 1, block, 55)
    shared = [c.expand(B, *c.shape[1:]) for c in cache]
    q = bf16(56, 1, Sq, 1, 128, spread=False)
    got = ops.decode_attention_q8(q.expand(B, Sq, 1, 128), *shared, L, block=block)
    torch.cuda.synchronize()
    assert native.device_error(reset=True) == 0
    of = torch.arange(L, device=DEV) // block
    k, v = (cache[i][0, :, 0].double() * cache[2 + i][0, of, 0].double()[:, None] for i in (0, 1))
    for i in (0, 1, 501, 502, 4000, 7529, 7530, 7531, Sq - 1):
        m = L - Sq + 1 + i
        p = torch.softmax(k[:m] @ q[0, i, 0].double() * 128 ** -0.5, 0)
        err = (got[:, i, 0].double() - p @ v[:m]).abs()
        assert bool((err <= (p @ v[:m]).abs() * 2 ** -8 + (p @ v[:m].abs()) * 2 ** -9).all())
