"""The dense operators in 64 bits, with a bound for each element of a result that is computed with 32-bit sums and with
the stated roundings.

u is half a step of the 16-bit type (bf16 2^-8, fp16 2^-11) and t the absolute error of rounding near zero (half of
fp16's smallest step; bf16 has none above 2^-133).  A sum of n products that is kept in 32 bits is off by at most
n 2^-23 of the sum of their magnitudes (a tensor core's additions may cut instead of round: a whole step each).
The sigmoid, computed in 32 bits, is off by less than 2^-18 of itself for |g| < 32: the exponential's argument is
rounded, |g| 2^-23, and a few steps come on top.  |silu'| < 1.1 and |silu''| <= 0.5."""
from __future__ import annotations

import torch

import moe_testlib  # noqa: F401  (sets sys.path)

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25, torch.float32: 0.0}
FN = 2.0 ** -18
SECOND_ORDER = 1.02  # products of errors; for fp16 and bf16 u^2 is below 2 % of u


def make(tokens, hidden, inter, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s, std: (torch.randn(*s, generator=g) * std).to(dtype).cuda()  # noqa: E731
    return (r(tokens, hidden, std=1.0), r(2 * inter, hidden, std=1.5 / hidden ** 0.5), r(hidden, inter, std=inter ** -0.5),
            r(tokens, hidden, std=1.0))


def product(a, b, ea=None, eb=None):
    """a b^T and the bound of a 32-bit sum of it; ea, eb: bounds of the operands."""
    y, n = a @ b.t(), a.shape[1]
    e = n * 2.0 ** -23 * (a.abs() @ b.abs().t())
    if ea is not None:
        e = e + ea @ b.abs().t()
    if eb is not None:
        e = e + a.abs() @ eb.t()
    return y, e


def rounded(y, e, dtype):
    return e * SECOND_ORDER + U[dtype] * y.abs() * SECOND_ORDER + TINY[dtype]


def gated(x, wg, wu):
    """silu(x wg^T) * (x wu^T) before its rounding, its bound, and what the backward pass needs."""
    (g, eg), (u, eu) = product(x, wg), product(x, wu)
    s = torch.sigmoid(g)
    h = g * s * u
    return h, 1.1 * u.abs() * eg + (g * s).abs() * eu + 2 * FN * h.abs(), (g, u, eg, eu)


def ffn(x, w13, w2):
    """y and its bound."""
    dtype, inter = x.dtype, w2.shape[1]
    x, w13, w2 = x.double(), w13.double(), w2.double()
    h, eh, _ = gated(x, w13[:inter], w13[inter:])
    y, e = product(h, w2, ea=rounded(h, eh, dtype))
    return y, rounded(y, e, dtype)


def ffn_grads(x, w13, w2, dy):
    """(dx, dw13, dw2) and their bounds; between the passes g and u lose the last eight of 24 significant bits, 2^-15 of
    the value at most."""
    dtype, inter = x.dtype, w2.shape[1]
    x, w13, w2, dy = x.double(), w13.double(), w2.double(), dy.double()
    h, eh, (g, u, eg, eu) = gated(x, w13[:inter], w13[inter:])
    eg, eu = eg * SECOND_ORDER + 2.0 ** -15 * g.abs(), eu * SECOND_ORDER + 2.0 ** -15 * u.abs()
    s = torch.sigmoid(g)
    silu, slope = g * s, s * (1 + g * (1 - s))
    dh, edh = product(dy, w2.t())
    dg, du = dh * u * slope, dh * silu
    edg = (u * slope).abs() * edh + (dh * slope).abs() * eu + 0.5 * (dh * u).abs() * eg + 3 * FN * (dh * u).abs() * 1.1
    edu = silu.abs() * edh + dh.abs() * 1.1 * eg + 2 * FN * du.abs()
    dgu, edgu = torch.cat([dg, du], 1), torch.cat([rounded(dg, edg, dtype), rounded(du, edu, dtype)], 1)
    dx, edx = product(dgu, w13.t(), ea=edgu)
    dw13, edw13 = product(dgu.t(), x.t(), ea=edgu.t())
    dw2, edw2 = product(dy.t(), h.t(), eb=rounded(h, eh, dtype).t())
    return [(t, rounded(t, e, dtype)) for t, e in ((dx, edx), (dw13, edw13), (dw2, edw2))]


def assert_within(got, want, bound, what=""):
    assert got.shape == want.shape, what
    over = ((got.double() - want).abs() / bound.clamp_min(1e-300)).nan_to_num(nan=float("inf"))
    over = torch.where(got.double() == want, torch.zeros_like(over), over)
    assert over.numel() == 0 or over.max().item() <= 1.0, f"{what}: {over.max().item():.2f} of the bound"


GRID = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def mx4(x):
    """What x stands for in 4-bit microscaled form, 64 bits, from the definition: the nearest point of the grid, the one
    with the even code where two are as near."""
    v = x.double().unflatten(-1, (-1, 32))
    top = v.abs().amax(-1, keepdim=True)
    bad = ~torch.isfinite(top)
    exponent = torch.frexp(torch.where(bad, torch.ones_like(top), top)).exponent.double() - 1 - 2
    exponent = torch.where(top > 0, exponent, torch.full_like(exponent, -127.0)).clamp(-127, 127)
    scale = torch.exp2(exponent)
    m = v.abs() / scale
    grid = torch.tensor(GRID, dtype=torch.float64, device=x.device)
    distance = (m.unsqueeze(-1) - grid).abs()
    near = distance <= distance.amin(-1, keepdim=True)
    even = near & (torch.arange(8, device=x.device) % 2 == 0)
    pick = torch.where(even.any(-1, keepdim=True), even, near).int().argmax(-1)
    out = torch.copysign(grid[pick], v) * scale
    return torch.where(bad, torch.full_like(out, float("nan")), out).flatten(-2)
