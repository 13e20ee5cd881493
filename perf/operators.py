"""Workloads of the operators of a decode step that is bound by bytes: a key/value cache held in
8 bits (written by ``ops.kv_append_q8``, read by ``ops.decode_attention_q8``) and a whole
mixture-of-experts feed-forward for a few tokens (``ops.moe_decode``).

Each workload is a case: plain values from which ``prepare`` makes the inputs, ``run`` makes one
pass (the framework's calls where ``own`` is true, else the same operator in elementary torch
operations), ``exact`` the result in 64 bits and ``work`` the bytes and operations that the pass
cannot do without.
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
HEAD = 128                                      # head size of every decoder in this repository
QMAX = {"int8": 127.0, "e4m3": 448.0}           # largest magnitude a code holds
MIN_SCALE = 2.0 ** -120
CAP_CACHE = 131072 * 8                          # tokens x KV heads of the largest cache
CAP_EXPERTS = 8 * 6144 * 16384                  # experts x dim x width of the largest layer


# ----------------------------------------------------------------------------- cases
def listed():
    return [
        # the prompts of a Llama-70B-shape batch, written to the cache after the prefill
        dict(name="append-prompt", op="append", fmt="int8", B=32, S=2048, L=2304, Hk=8, block=64, at="zero", ragged=False),
        # a padded batch of unequal prompts, each continuing its own history at an odd position
        dict(name="append-ragged", op="append", fmt="e4m3", B=5, S=777, L=2001, Hk=8, block=32, at="any", ragged=True),
        # one token a sequence, every sequence at its own length: what each layer of a decode step does
        dict(name="append-token", op="append", fmt="int8", B=32, S=1, L=2304, Hk=8, block=64, at="any", ragged=False),
        # a decode step of a Llama-70B-shape layer: 64 query heads on 8 KV heads, 2304 tokens
        dict(name="decode-llama", op="attend", fmt="int8", B=32, Sq=1, L=2304, Hq=64, Hk=8, block=64, ragged=False),
        # the same step on one rank of eight (8 query heads on one KV head)
        dict(name="decode-llama-tp8", op="attend", fmt="e4m3", B=32, Sq=1, L=2304, Hq=8, Hk=1, block=64, ragged=False),
        # the attention half of a Mixtral-shape step: the new token joins the cache, then attends; unequal lengths
        dict(name="step-mixtral", op="step", fmt="int8", B=64, Sq=1, L=1152, Hq=48, Hk=8, block=64, ragged=True),
        # one long conversation
        dict(name="decode-long", op="attend", fmt="e4m3", B=1, Sq=1, L=131071, Hq=64, Hk=8, block=128, ragged=False),
        # four drafted tokens a sequence, checked in one pass, short unequal contexts
        dict(name="decode-drafts", op="attend", fmt="int8", B=3, Sq=4, L=515, Hq=16, Hk=4, block=32, ragged=True),
        # a single conversation through a Mixtral-8x22B-shape layer: two experts of eight
        dict(name="moe-one", op="moe", T=1, D=6144, F=16384, E=8, topk=2, residual=True),
        # a batch of 64 sequences through the same layer: every expert
        dict(name="moe-batch", op="moe", T=64, D=6144, F=16384, E=8, topk=2, residual=True),
        # many small experts, a few tokens
        dict(name="moe-many", op="moe", T=7, D=2048, F=1024, E=64, topk=6, residual=False),
        # a small layer of odd sizes, where the launch counts
        dict(name="moe-small", op="moe", T=3, D=1000, F=1416, E=5, topk=2, residual=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["append", "attend", "step", "moe"])
    if op == "moe":
        E = rng.choice([4, 5, 8, 16, 31, 64])
        D = 8 * _log(rng, 32, 768)
        F = 8 * _log(rng, 32, 2048)
        while E * D * F > CAP_EXPERTS:
            F = 8 * max(32, F // 16)
        return dict(op=op, T=_log(rng, 1, 64), D=D, F=F, E=E, topk=rng.randint(1, min(8, E)), residual=rng.random() < 0.5)
    fmt, block, Hk = rng.choice(["int8", "e4m3"]), rng.choice([16, 32, 64, 128, 256]), rng.choice([1, 2, 3, 4, 8])
    B = _log(rng, 1, 64)
    if op == "append":
        S = _log(rng, 1, max(1, min(4096, CAP_CACHE // 2 // (B * Hk))))
        return dict(op=op, fmt=fmt, B=B, S=S, L=S + _log(rng, 1, 1024), Hk=Hk, block=block,
                    at=rng.choice(["zero", "any"]), ragged=rng.random() < 0.5)
    Sq = 1 if op == "step" else rng.choice([1, 1, 1, 2, 5, 8])
    L = max(Sq, _log(rng, 1, max(1, min(131072, CAP_CACHE // (B * Hk)))))
    return dict(op=op, fmt=fmt, B=B, Sq=Sq, L=L, Hq=Hk * rng.choice([1, 2, 4, 5, 6, 8, 16]), Hk=Hk, block=block,
                ragged=rng.random() < 0.5)


# ----------------------------------------------------------------------------- inputs
def _activations(g, *shape, heads=None):
    """bf16 values with a width of their own per head, as projections have."""
    x = torch.randn(*shape, device=DEV, generator=g)
    if heads is not None:
        x *= (0.5 + 2.0 * torch.rand(shape[heads], device=DEV, generator=g)).view([-1 if i == heads else 1 for i in range(len(shape))])
    return x.bfloat16()


def _codes(g, fmt, *shape):
    """A cache's codes: roughly normal, within the format."""
    x = torch.randn(*shape, device=DEV, generator=g, dtype=torch.float16)
    if fmt == "int8":
        return (x * 32).round_().clamp_(-127, 127).to(torch.int8)
    return (x * 112).clamp_(-448, 448).to(torch.float8_e4m3fn)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(1000003 * (seed % 2000003) + 17)
    c = dict(case)
    if c["op"] == "moe":
        T, D, F, E = c["T"], c["D"], c["F"], c["E"]
        s = dict(c, x=torch.randn(T, D, device=DEV, generator=g).bfloat16(),
                 router=(torch.randn(E, D, device=DEV, generator=g) * D ** -0.5).bfloat16(),
                 gate_up=torch.empty(E, 2 * F, D, device=DEV, dtype=torch.bfloat16).normal_(0, D ** -0.5, generator=g),
                 down=torch.empty(E, D, F, device=DEV, dtype=torch.bfloat16).normal_(0, F ** -0.5, generator=g),
                 res=torch.randn(T, D, device=DEV, generator=g).bfloat16() if c["residual"] else None)
        s["gate_up_list"], s["down_list"] = list(s["gate_up"].unbind(0)), list(s["down"].unbind(0))  # one tensor an expert, as the layers hold them
        return s
    B, L, Hk, block = c["B"], c["L"], c["Hk"], c["block"]
    nb = -(-L // block)
    kc, vc = _codes(g, c["fmt"], B, L, Hk, HEAD), _codes(g, c["fmt"], B, L, Hk, HEAD)
    top = 0.04 if c["fmt"] == "int8" else 0.012
    ks, vs = ((top * (0.4 + torch.rand(B, nb, Hk, device=DEV, generator=g))).view(torch.int32).bitwise_and_(0x7F800000).view(torch.float32)
              for _ in range(2))  # powers of two
    s = dict(c, kc=kc, vc=vc, ks=ks, vs=vs)
    if c["op"] == "append":
        S = c["S"]
        s["k"], s["v"] = _activations(g, B, S, Hk, HEAD, heads=2), _activations(g, B, S, Hk, HEAD, heads=2)
        s["pos"] = 0 if c["at"] == "zero" else torch.randint(0, L - S + 1, (B,), device=DEV, generator=g, dtype=torch.int32)
        s["n_new"] = torch.randint(0, S + 1, (B,), device=DEV, generator=g, dtype=torch.int32) if c["ragged"] else None
        return s
    s["q"] = _activations(g, B, c["Sq"], c["Hq"], HEAD, heads=2)
    if c["ragged"]:  # lengths from a single query's own keys to the whole cache
        s["kv_len"] = torch.randint(c["Sq"], L + 1, (B,), device=DEV, generator=g, dtype=torch.int32)
    else:
        s["kv_len"] = L
    if c["op"] == "step":
        s["k"], s["v"] = _activations(g, B, 1, Hk, HEAD, heads=2), _activations(g, B, 1, Hk, HEAD, heads=2)
        s["pos"] = s["kv_len"] - 1
        s["n_new"] = None
    return s


# ----------------------------------------------------------------------------- plain forms
def _pow2_scale(amax, fmt):
    """The smallest power of two s with amax <= qmax * s (0 for 0; never below 2^-120)."""
    m, e = torch.frexp(amax)
    lim, down = (127.0 / 128.0, 7) if fmt == "int8" else (448.0 / 512.0, 9)
    s = ((e - down + (m > lim).int() + 127).clamp(min=7) << 23).view(torch.float32)  # 2^k by its bits
    s = torch.where(amax > 0, s, torch.zeros_like(s))
    return torch.where(torch.isfinite(amax), s, torch.full_like(s, float("nan")))


def _to_codes(x, fmt):
    if fmt == "int8":
        return torch.nan_to_num(x.round()).to(torch.int8)
    return torch.nan_to_num(x).to(torch.float8_e4m3fn)


def _plain_append_one(x, cache, scale, pos, n_new, block, fmt):
    B, S, Hk, _ = x.shape
    L, nb = cache.shape[1], scale.shape[1]
    W = min(nb, (S + block - 2) // block + 1)             # blocks a sequence can touch
    rows = torch.arange(B, device=DEV)[:, None]
    p = (pos if isinstance(pos, torch.Tensor) else torch.full((B,), pos, device=DEV)).long()[:, None]
    n = (n_new.long() if n_new is not None else torch.full((B,), S, device=DEV))[:, None]
    first = (p // block).clamp(max=nb - W)
    blk = first + torch.arange(W, device=DEV)[None]       # [B, W]
    t = (first * block + torch.arange(W * block, device=DEV)[None]).clamp(max=L - 1)
    new = (t >= p) & (t < p + n)
    xf = x[rows, (t - p).clamp(0, S - 1)].float() * new[..., None, None]
    amax = xf.abs().view(B, W, block, Hk, HEAD).amax(dim=(2, 4))
    history = ((blk * block < p) & (p < (blk + 1) * block) & (n > 0))[..., None]
    touched = new.view(B, W, block).any(2)[..., None]
    before = scale[rows, blk]
    old = torch.where(history, before, torch.zeros_like(before))
    s = torch.maximum(old, _pow2_scale(amax, fmt))
    st = s.repeat_interleave(block, 1)[..., None]
    inv = torch.where(st > 0, 1.0 / st, torch.zeros_like(st))
    codes = cache[rows, t]
    again = _to_codes(codes.float() * (old.repeat_interleave(block, 1)[..., None] * inv), fmt)
    grown = (touched & history & ~(s == old)).repeat_interleave(block, 1)[..., None] & (t < p)[..., None, None]
    codes = torch.where(new[..., None, None], _to_codes(xf * inv, fmt).float(), torch.where(grown, again.float(), codes.float()))
    cache[rows, t] = codes.to(cache.dtype)
    scale[rows, blk] = torch.where(touched, s, before)


def _plain_attend(q, kc, vc, ks, vs, kv_len, block):
    B, Sq, Hq, _ = q.shape
    L, Hk = kc.shape[1], kc.shape[2]
    of = torch.arange(L, device=DEV) // block
    k = kc.float() * ks[:, of][..., None]
    v = vc.float() * vs[:, of][..., None]
    s = torch.einsum("bihgd,blhd->bhgil", q.float().view(B, Sq, Hk, Hq // Hk, HEAD), k) * HEAD ** -0.5
    n = (kv_len if isinstance(kv_len, torch.Tensor) else torch.full((B,), kv_len, device=DEV)).long()
    sees = (n[:, None] - Sq + 1 + torch.arange(Sq, device=DEV)[None]).clamp(min=0)              # [B, Sq] keys
    seen = torch.arange(L, device=DEV)[None, None] < sees[..., None]                            # [B, Sq, L]
    s = s.masked_fill(~seen[:, None, None], float("-inf"))
    p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-3e38))
    total = p.sum(-1, keepdim=True)
    o = torch.einsum("bhgil,blhd->bihgd", p / total.clamp(min=1e-37), v)
    return o.reshape(B, Sq, Hq, HEAD).bfloat16()


def _plain_moe(s):
    T, topk, E = s["T"], s["topk"], s["E"]
    x = s["x"].float()
    val, ids = torch.topk(x @ s["router"].float().t(), topk, dim=-1)
    w = torch.softmax(val, -1)
    if T * topk <= E:  # only the chosen experts' weights
        gu = torch.einsum("tkfd,td->tkf", s["gate_up"][ids].float(), x)
        h = gu[..., 0::2] * torch.sigmoid(gu[..., 0::2]) * gu[..., 1::2]
        y = torch.einsum("tkdf,tkf,tk->td", s["down"][ids].float(), h, w)
    else:              # every expert on every token, weighted by 0 where it was not chosen
        gu = torch.einsum("efd,td->etf", s["gate_up"].float(), x)
        h = gu[..., 0::2] * torch.sigmoid(gu[..., 0::2]) * gu[..., 1::2]
        h = h * torch.zeros(T, E, device=DEV).scatter_(1, ids, w).t()[..., None]
        y = torch.einsum("edf,etf->td", s["down"].float(), h)
    return (y if s["res"] is None else y + s["res"].float()).bfloat16()


# ----------------------------------------------------------------------------- one pass
def run(s):
    if own:
        from flextensor_b200 import ops

        if s["op"] == "moe":
            return ops.moe_decode(s["x"], s["router"], s["gate_up_list"], s["down_list"], s["topk"], residual=s["res"])
        cache = (s["kc"], s["vc"], s["ks"], s["vs"])
        if s["op"] != "attend":
            ops.kv_append_q8(s["k"], s["v"], *cache, s["pos"], block=s["block"], n_new=s["n_new"])
        if s["op"] == "append":
            return cache
        o = ops.decode_attention_q8(s["q"], *cache, s["kv_len"], block=s["block"], max_len=s["L"])
        return o if s["op"] == "attend" else (o, *cache)
    if s["op"] == "moe":
        return _plain_moe(s)
    cache = (s["kc"], s["vc"], s["ks"], s["vs"])
    if s["op"] != "attend":
        _plain_append_one(s["k"], s["kc"], s["ks"], s["pos"], s["n_new"], s["block"], s["fmt"])
        _plain_append_one(s["v"], s["vc"], s["vs"], s["pos"], s["n_new"], s["block"], s["fmt"])
    if s["op"] == "append":
        return cache  # codes and scales: both have to be equal, bit for bit
    o = _plain_attend(s["q"], *cache, s["kv_len"], s["block"])
    return o if s["op"] == "attend" else (o, *cache)


# ----------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    def append(x, cache, scale, pos, n_new, block, fmt):
        """Sequence by sequence and block by block, as the cache's definition reads."""
        B, S = x.shape[:2]
        at = pos.tolist() if isinstance(pos, torch.Tensor) else [pos] * B
        count = n_new.tolist() if n_new is not None else [S] * B
        qmax = QMAX[fmt]
        codes, scales = cache.double(), scale.double()
        for b in range(B):
            lo, end = at[b], at[b] + count[b]
            while lo < end:
                j = lo // block
                hi = min(end, (j + 1) * block)
                rows = x[b, lo - at[b]:hi - at[b]].double()                       # [n, Hk, 128]
                a = rows.abs().amax(dim=(0, 2))
                m, e = torch.frexp(a / qmax)
                s = ((e.long() - (m == 0.5).long() + 1023) << 52).view(torch.float64)    # the power of two at or above
                s = torch.where(a > 0, s.clamp(min=MIN_SCALE), torch.zeros_like(a))
                if lo > j * block:
                    s0 = scales[b, j]
                    s = torch.maximum(s, s0)
                    kept = codes[b, j * block:lo] * (s0 / s.clamp(min=MIN_SCALE))[None, :, None]
                    codes[b, j * block:lo] = kept.round() if fmt == "int8" else kept.to(torch.float8_e4m3fn).double()
                r = rows / s.clamp(min=MIN_SCALE)[None, :, None]
                codes[b, lo:hi] = r.round() if fmt == "int8" else r.float().to(torch.float8_e4m3fn).double()
                scales[b, j] = s
                lo = hi
        return codes, scales

    def attend(q, kc, vc, ks, vs, kv_len, block):
        B, Sq, Hq, _ = q.shape
        L, Hk = kc.shape[1], kc.shape[2]
        G = Hq // Hk
        lens = kv_len.tolist() if isinstance(kv_len, torch.Tensor) else [kv_len] * B
        o = torch.zeros(B, Sq, Hq, HEAD, dtype=torch.float64, device=DEV)
        for b in range(B):
            n = lens[b]
            j = torch.arange(n, device=DEV) // block
            for h in range(Hk):
                k = kc[b, :n, h].double() * ks[b, j, h].double()[:, None]
                v = vc[b, :n, h].double() * vs[b, j, h].double()[:, None]
                for i in range(Sq):
                    m = n - Sq + 1 + i
                    if m > 0:
                        z = q[b, i, h * G:(h + 1) * G].double() @ k[:m].t() / math.sqrt(HEAD)
                        o[b, i, h * G:(h + 1) * G] = torch.softmax(z, -1) @ v[:m]
        return o

    s = prepare(case, seed)
    if s["op"] == "moe":
        x = s["x"].double()
        val, ids = torch.sort(x @ s["router"].double().t(), dim=-1, descending=True, stable=True)
        val, ids = val[:, :s["topk"]], ids[:, :s["topk"]]
        w = torch.exp(val - val[:, :1])
        w = w / w.sum(-1, keepdim=True)
        y = torch.zeros_like(x) if s["res"] is None else s["res"].double()
        for e in range(s["E"]):
            t, k = (ids == e).nonzero(as_tuple=True)
            if t.numel():
                z = x[t] @ s["gate_up"][e].double().t()
                gate, up = z[:, 0::2], z[:, 1::2]
                y.index_add_(0, t, (gate / (1 + torch.exp(-gate)) * up) @ s["down"][e].double().t() * w[t, k][:, None])
        return y
    cache = [s["kc"], s["vc"], s["ks"], s["vs"]]
    if s["op"] != "attend":
        cache[0], cache[2] = append(s["k"], s["kc"], s["ks"], s["pos"], s["n_new"], s["block"], s["fmt"])
        cache[1], cache[3] = append(s["v"], s["vc"], s["vs"], s["pos"], s["n_new"], s["block"], s["fmt"])
        if s["fmt"] == "int8":
            codes = [c.to(torch.int64).to(torch.int8) for c in cache[:2]]
        else:
            codes = cache[:2]
        if s["op"] == "append":
            return (*codes, *cache[2:])
    o = attend(s["q"], *cache, s["kv_len"], s["block"])
    return o if s["op"] == "attend" else (o, *codes, *cache[2:])


# ----------------------------------------------------------------------------- least work
def _expected_experts(c):
    """Experts that T tokens with topk different choices each reach, on average."""
    return c["E"] * (1.0 - (1.0 - c["topk"] / c["E"]) ** c["T"])


def work(case):
    c = case
    if c["op"] == "moe":
        T, D, F = c["T"], c["D"], c["F"]
        rows = T * (3 if c["residual"] else 2) * D * 2
        return {"bytes": _expected_experts(c) * 3 * D * F * 2 + c["E"] * D * 2 + rows,
                "flops": 2.0 * T * c["topk"] * 3 * D * F + 2.0 * T * c["E"] * D}
    B, L, Hk = c["B"], c["L"], c["Hk"]
    new = c["B"] * (c.get("S", 1) * (0.5 if c["ragged"] and c["op"] == "append" else 1.0)) * Hk * HEAD * 2  # values of k and v
    append = {"bytes": new * 3 + new / HEAD / min(c["block"], c.get("S", 1)) * 4, "flops": 3.0 * new}
    if c["op"] == "append":
        return append
    tokens = B * ((L + c["Sq"]) / 2 if c["ragged"] else L)
    reads = tokens * Hk * (HEAD + 4.0 / c["block"]) * 2
    attend = {"bytes": reads + 2.0 * B * c["Sq"] * c["Hq"] * HEAD * 2, "flops": 4.0 * tokens * c["Sq"] * c["Hq"] * HEAD}
    return attend if c["op"] == "attend" else {k: attend[k] + append[k] for k in attend}
