"""A mixture-of-experts layer in 64 bits, with what a kernel may be off by that keeps h in two bf16 halves.

Element by element the output may differ by its own rounding, 2^-8 |out|, and by

* h as two bf16 numbers: 2^-8 of a rest that is 2^-8 |h|, so 2^-16 |h|; SwiGLU in fp32, 2^-20 |h|;
* gate and up, sums of D products: one rounding (or truncation, 2^-23) for each 16 products, and eight more
  where partial sums are joined, of numbers no larger than sum |x| |w|; through silu, whose slope is
  below 1.1, and the product;
* the down product, sums of 2 F products (both halves): the same of sum |W_down| |h|;
* the choices' weights: logits are sums in fp32 with at most D / 256 + 16 roundings of sum |x| |r|.

Over many elements of random data the roundings of the output are uniform in their steps and dominate:
the 2-norm of the error is that of step / sqrt(12), within 3 / sqrt(n) of it (the norm of n uniform errors has
a deviation of 0.45 / sqrt(n)). An output whose h had one bf16 number instead is about 1.4 times that off."""

import torch


def layer(x, router, w_gate_up, w_down, topk, residual=None, spoil=None):
    """(output, bound of the error element by element), float64. ``spoil(hi, lo)``: what the two bf16 halves
    of h are replaced by (float64 tensors, summed); the output is then rounded as a kernel's would be."""
    x64, D = x.double(), x.shape[1]
    val, ids = torch.sort(x64 @ router.double().t(), dim=-1, descending=True, stable=True)
    val, ids = val[:, :topk], ids[:, :topk]
    w = torch.softmax(val, -1)
    dw = 2 * (D / 256 + 16) * 2 ** -24 * (x64.abs() @ router.double().abs().t()).amax(-1, keepdim=True) + 2 ** -21
    y, bound = torch.zeros_like(x64), torch.zeros_like(x64)
    for e in range(router.shape[0]):
        t, k = (ids == e).nonzero(as_tuple=True)
        if t.numel() == 0:
            continue
        W, d = w_gate_up[e].double().t(), w_down[e].double().t()
        z, dz = x64[t] @ W, (D / 16 + 8) * 2 ** -23 * (x64[t].abs() @ W.abs())
        g, u, dg, du = z[:, 0::2], z[:, 1::2], dz[:, 0::2], dz[:, 1::2]
        silu = torch.nn.functional.silu(g)
        h = silu * u
        if spoil is not None:
            hi = h.bfloat16()
            h = spoil(hi.double(), (h.float() - hi.float()).bfloat16().double())
        dh = 1.1 * dg * u.abs() + silu.abs() * du + 1.1 * dg * du + (2 ** -16 + 2 ** -20) * h.abs()
        wk = w[t, k][:, None]
        y.index_add_(0, t, h @ d * wk)
        A = h.abs() @ d.abs() * wk
        bound.index_add_(0, t, dh @ d.abs() * wk + A * (dw[t] + (2 * d.shape[0] / 16 + 8) * 2 ** -23))
    if residual is not None:
        y += residual.double()
    if spoil is not None:
        y = y.bfloat16().double()
    return y, bound + y.abs() * 2 ** -8


def step(y):
    """The distance of bf16 numbers at y."""
    return torch.ldexp(torch.ones_like(y), torch.frexp(y).exponent - 8)


def norm_ratio(got, want):
    """The error's 2-norm over that of the output's own roundings, and the largest that it may be."""
    err = (got.double() - want).norm() / (step(want).norm() / 12 ** 0.5)
    return float(err), 1 + 3 / want.numel() ** 0.5


def random_layer(T, D, F, E, seed, device="cpu"):
    g = torch.Generator(device=device).manual_seed(seed)
    r = lambda *s, std=1.0: (torch.randn(*s, device=device, generator=g) * std).bfloat16()  # noqa: E731
    return dict(x=r(T, D), router=r(E, D, std=2 * D ** -0.5), w_gate_up=r(E, 2 * F, D, std=D ** -0.5),
                w_down=r(E, D, F, std=F ** -0.5))


def cancelling_layer(T, device="cpu"):
    """Columns of W_down in pairs of opposite sign, h nearly equal in each pair (its up rows differ by 2^-10 or
    less): high halves cancel and what is left is a matter of the low ones."""
    g = torch.Generator(device=device).manual_seed(5)
    D = F = 64
    u = lambda *s: torch.rand(*s, device=device, generator=g)  # noqa: E731
    x = u(T, D) * 0.1
    x[:, 0], x[:, 1] = 1.0, (0.5 + u(T) / 2) * 2 ** -10
    gu = u(2, 2 * F, D) * 0.1
    gu[:, :, 0] += 0.5
    gu[:, 2::4], gu[:, 3::4] = gu[:, 0::4], gu[:, 1::4]
    gu[:, :, 1] = 0.0
    gu[:, 3::4, 1] = 1.0
    dn = 0.5 + u(2, D, F) / 2
    dn[:, :, 1::2] = -dn[:, :, 0::2]
    return dict(x=x.bfloat16(), router=(u(2, D) * 0.1).bfloat16(), w_gate_up=gu.bfloat16(), w_down=dn.bfloat16())
