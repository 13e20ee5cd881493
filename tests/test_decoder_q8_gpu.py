"""Decoder models on an 8-bit cache and the few-token MoE layer together, as a decode step uses them.

The codes' values are bf16 numbers (a code has at most 8 significant bits and scales are powers of
two), so the same step over a bf16 cache holding those values is the same mathematics; the two paths
differ by roundings of their own: weights to bf16 in one, to f16 in the other (2^-8 and 2^-11 of the
weighted |v|), outputs to bf16 (2^-8). A model step adds the bf16 roundings of some ten operators
(2^-8 each) and is compared in the 2-norm at 10 * 2^-8."""

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("needs a CUDA device", allow_module_level=True)

import flextensor_b200 as ft  # noqa: E402
from flextensor_b200 import ops  # noqa: E402
from flextensor_b200.models.kv_cache import QuantizedKV  # noqa: E402
from flextensor_b200.models.kv_cache import new_layer_cache, rewind, store  # noqa: E402
from flextensor_b200.models.llama import LlamaModel, init_llama_params_, tiny_llama  # noqa: E402
from flextensor_b200.models.mixtral import MixtralModel, MixtralStack, init_mixtral_params_, tiny_mixtral  # noqa: E402
from flextensor_b200.ops import native  # noqa: E402
from flextensor_b200.planner import NthLayerStrategy  # noqa: E402

DEV = torch.device("cuda", 0)
DTYPES = [torch.int8, torch.float8_e4m3fn]


def build(family, **kw):
    torch.manual_seed(0)
    if family == "llama":
        m = LlamaModel(tiny_llama(**kw)).to(DEV)
        init_llama_params_(m, seed=1)
    else:
        m = MixtralModel(tiny_mixtral(dim=512, n_heads=4, n_kv_heads=2, moe_decode=True, **kw)).to(DEV)
        init_mixtral_params_(m, seed=1)
    return m.to(torch.bfloat16)


def dequantized(cache):
    out = []
    for c in cache:
        of = torch.arange(c.k.shape[1], device=DEV) // c.block
        out.append(tuple((x.float() * s[:, of][..., None]).bfloat16() for x, s in ((c.k, c.k_scale), (c.v, c.v_scale))))
    return out


def near(a, b, tol=10 * 2 ** -8):
    return float((a.float() - b.float()).norm() / b.float().norm()) <= tol


@torch.no_grad()
@pytest.mark.parametrize("family", ["llama", "mixtral"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_decode_steps_follow_the_cache(family, dtype):
    """Prompt, then single tokens and a draft of three: every step equals the step over a bf16 cache that
    holds the codes' values."""
    m = build(family)
    cfg = m.cfg
    B, S, new = 3, 70, 4
    g = torch.Generator(device=DEV).manual_seed(2)
    tokens = torch.randint(0, cfg.vocab, (B, S + new + 3), device=DEV, generator=g)
    cache = m.new_cache(B, S + new + 3, dtype=dtype)
    assert all(isinstance(c, QuantizedKV) for c in cache)
    plain = m.new_cache(B, S + new + 3)
    assert near(m.prefill(tokens[:, :S], cache), m.prefill(tokens[:, :S], plain), 2 ** -8)
    for i in range(new):
        values = dequantized(cache)
        got = m.decode_step(tokens[:, S + i], cache, S + i)
        # the new token joins with its own bf16 value there, with its code's here
        now = dequantized(cache)
        for (k, v), (k8, v8) in zip(values, now):
            k[:, :S + i + 1], v[:, :S + i + 1] = k8[:, :S + i + 1], v8[:, :S + i + 1]
        want = step_over(m, tokens[:, S + i], values, S + i)
        assert near(got, want), i
    before = [QuantizedKV(*(t.clone() for t in c[:4]), c.block) for c in cache]
    drafts = m.decode_step(tokens[:, S + new:], cache, S + new)
    assert drafts.shape == (B, 3, cfg.vocab)
    for i in range(3):
        one = m.decode_step(tokens[:, S + new + i], before, S + new + i)
        assert near(drafts[:, i], one, 0.1)  # a later draft may have grown a block's scale: other codes, half a step each
    with pytest.raises(ValueError, match="8-bit cache"):
        m.decode_step(tokens[:, S + new:], plain, S + new)
    assert native.device_error(reset=True) == 0


def step_over(m, token, values, pos):
    """decode_step over bf16 caches that already hold position ``pos``."""
    import flextensor_b200.models.llama as llama

    keep, llama.store = llama.store, lambda *a: None
    try:
        return m.decode_step(token, values, pos)
    finally:
        llama.store = keep


@pytest.mark.parametrize("dtype", DTYPES)
def test_generate(dtype):
    for family in ("llama", "mixtral"):
        m = build(family)
        tokens = torch.randint(0, m.cfg.vocab, (2, 33), device=DEV, generator=torch.Generator(device=DEV).manual_seed(3))
        out = m.generate(tokens, 5, cache_dtype=dtype)
        assert out.shape == (2, 5) and torch.equal(out, m.generate(tokens, 5, cache_dtype=dtype))
    assert native.device_error(reset=True) == 0


@torch.no_grad()
def test_moe_decode_path_matches_the_expert_loop():
    m = build("mixtral")
    tokens = torch.randint(0, m.cfg.vocab, (5, 7), device=DEV, generator=torch.Generator(device=DEV).manual_seed(4))
    launches = ops.launch_count()
    a = m(tokens)          # 35 rows: the few-token layer
    few = ops.launch_count() - launches
    m.cfg.moe_decode = False
    launches = ops.launch_count()
    b = m(tokens)
    assert few != ops.launch_count() - launches and near(a, b)
    m.cfg.moe_decode = True
    long = torch.randint(0, m.cfg.vocab, (1, 80), device=DEV)
    a = m(long)            # 80 rows: the expert loop either way
    m.cfg.moe_decode = False
    assert torch.equal(a, m(long))
    assert native.device_error(reset=True) == 0


def test_streamed_decode_is_bitwise():
    """Prefill and decode steps of a streamed stack (int8 cache, few-token MoE) equal the resident one's."""
    from flextensor_b200.models.llama import rope_tables_1d

    cfg = tiny_mixtral(dim=512, n_heads=4, n_kv_heads=2, n_layers=3, moe_decode=True)
    ref = MixtralStack(cfg).to(DEV)
    init_mixtral_params_(ref, seed=5)
    ref = ref.to(torch.bfloat16)
    m = MixtralStack(cfg).to(DEV).to(torch.bfloat16)
    m.load_state_dict(ref.state_dict())
    B, S, steps = 2, 40, 3
    g = torch.Generator(device=DEV).manual_seed(6)
    xs = [torch.randn(B * S, cfg.dim, device=DEV, generator=g).bfloat16()] + \
         [torch.randn(B, cfg.dim, device=DEV, generator=g).bfloat16() for _ in range(steps)]
    cos, sin = rope_tables_1d(S + steps, cfg.head_dim, cfg.rope_theta, DEV)

    def go(model):
        cache = ref.new_cache(B, S + steps, DEV, torch.int8)
        out = []
        for i, x in enumerate(xs):
            pos, n = (0, S) if i == 0 else (S + i - 1, 1)
            out.append(model(x.clone(), B, n, (cos[pos:pos + n].contiguous(), sin[pos:pos + n].contiguous()), cache=cache, pos=pos))
        return out

    with torch.no_grad():
        want = go(ref)
        mm = ft.offload(m, ft.OffloadConfig(include_patterns=["layers.*"], profiling_iters=1, num_blocks=2, min_blocks=2,
                                            skip_discovery=True,
                                            load_strategy=NthLayerStrategy(1, threshold_mb=0.0, n_blocks=2, cyclic=True)))
        om = ft.get_offload_manager()
        for _ in range(om.iters_before_inference + 2):
            for a, b in zip(go(mm), want):
                assert torch.equal(a, b)
    assert om.phase.value == "inference"
    assert native.device_error(reset=True) == 0


@torch.no_grad()
@pytest.mark.parametrize("kw,ids", [(dict(n_experts=4), [2, 0, 3, 1]), (dict(n_experts=130, ffn_dim=64), None),
                                    (dict(n_experts=12, topk=10), None)])
def test_layers_with_and_without_the_few_token_path(kw, ids):
    """Experts kept in another order than their ids; more experts, or more a token, than the one call takes."""
    from flextensor_b200.models.llama import rope_tables_1d
    from flextensor_b200.models.mixtral import MixtralLayer

    cfg = tiny_mixtral(dim=256, n_heads=2, n_kv_heads=1, moe_decode=True, **kw)
    m = MixtralLayer(cfg, ids).to(DEV)
    g = torch.Generator(device=DEV).manual_seed(8)
    for p in m.parameters():
        p.normal_(0.0, 0.06, generator=g)
    m = m.to(torch.bfloat16)
    x = torch.randn(9, cfg.dim, device=DEV, generator=g).bfloat16()
    rope = rope_tables_1d(9, cfg.head_dim, cfg.rope_theta, DEV)
    a = m(x.clone(), 1, 9, rope)
    cfg.moe_decode = False
    b = m(x.clone(), 1, 9, rope)
    assert near(a, b, 2 ** -7)  # one rounding of each path's output, and of the loop's h
    assert native.device_error(reset=True) == 0


def same_until(a, b, pos, block=64):
    """The codes and scales of the tokens before ``pos``, bit for bit."""
    blocks = -(-pos // block)
    return all(torch.equal(x[:, :pos].view(torch.int8), y[:, :pos].view(torch.int8)) for x, y in zip(a[:2], b[:2])) and \
        all(torch.equal(x[:, :blocks], y[:, :blocks]) for x, y in zip(a[2:4], b[2:4]))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("pos,n", [(70, 4), (64, 3), (1, 16), (62, 6)])
@pytest.mark.parametrize("size", [100.0, float("nan")])
def test_rejected_tokens_leave_no_trace(dtype, pos, n, size):
    """Rejected tokens far larger than those before, or NaN: codes and scales as without them."""
    g = torch.Generator(device=DEV).manual_seed(9)
    old, new, one = ([torch.randn(2, s, 3, 128, device=DEV, generator=g).bfloat16() for _ in range(2)] for s in (pos, n, 1))
    for accepted in (0, 1, n):
        cache, want = (new_layer_cache(2, pos + n + 1, 3, 128, DEV, dtype) for _ in range(2))
        k, v = (x.clone() for x in new)
        for x in (k, v):
            x[:, accepted:] *= size
        for c in (cache, want):
            store(c, *old, 0)
        store(cache, k, v, pos)
        if accepted:
            store(want, k[:, :accepted], v[:, :accepted], pos)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            rewind([cache], pos + accepted)
        torch.cuda.current_stream().wait_stream(side)
        assert same_until(cache, want, pos + accepted)
        for c in (cache, want):
            store(c, *one, pos + accepted)
        assert same_until(cache, want, pos + accepted + 1)
    assert native.device_error(reset=True) == 0


@torch.no_grad()
@pytest.mark.parametrize("family", ["llama", "mixtral"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_a_rejected_draft_costs_nothing(family, dtype):
    """A draft of large keys and values (its pass runs with larger norm weights), rejected: the steps after it
    are bit for bit those of a run without it, and nothing like them where it is left in the cache."""
    m = build(family)
    g = torch.Generator(device=DEV).manual_seed(10)
    S, n = 70, 4
    tokens = torch.randint(0, m.cfg.vocab, (3, S + n + 2), device=DEV, generator=g)
    norms = [(layer if family == "llama" else layer.attn).attn_norm for layer in m.layers]

    def run(draft, back):
        cache = m.new_cache(3, S + n + 2, dtype=dtype)
        m.prefill(tokens[:, :S], cache)
        if draft:
            for w in norms:
                w *= 64
            m.decode_step(tokens[:, S:S + n], cache, S)
            for w in norms:
                w /= 64
        if back:
            m.rewind(cache, S)
        return [m.decode_step(tokens[:, S + n + i], cache, S + i) for i in range(2)], cache

    want, clean = run(False, False)
    got, cache = run(True, True)
    assert all(same_until(a, b, S + 2) for a, b in zip(cache, clean))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    left, cache = run(True, False)
    assert not same_until(cache[0], clean[0], S)
    plain = m.new_cache(3, S + n + 2)
    m.rewind(plain, 5)  # bf16: nothing to do
    assert native.device_error(reset=True) == 0
