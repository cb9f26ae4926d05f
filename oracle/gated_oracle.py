"""The gated projection h = silu(x Wg^T) * (x Wu^T) in 64 bits, with its gradients, and how far bf16 kernels may be from it.

The bounds count roundings: eps / 2 = 2^-8 relative for each step to bf16, and for each sum of n products in fp32 n 2^-23 of the sum of
their magnitudes (products of bf16 are exact in fp32; the tensor cores' additions may cut off instead of rounding)."""
import torch

HALF = 2.0 ** -8
CUT = 2.0 ** -23
KEPT = 2.0 ** -15          # the 24 bits of a product that wait for the backward, cut off
GATE = 2.0 ** -18          # silu from fp32 sums: estimates of e^x and 1/x, taken to the fourth power at worst


def gate(g):
    """The same for gates of any size.  e^-|g| is the fourth power of 2^-t for t = |g| c, c = log2(e) / 4 in fp32.  t is off by 2^-24 of itself
    from its rounding and by 2^-26 from c's (1.4426950216 for 1.4426950409): |g| c (2^-24 + 2^-26) in the exponent, ln 2 of that in 2^-t, and
    four times in the power, |g| (2^-24 + 2^-26) < |g| 2^-23.6.  A positive gate's factor 1 / (1 + e^-g) hardly has it: e^-g g < 0.4."""
    return GATE + g.clamp(max=0).abs() * 2.0 ** -23.6


def forward(x, wg, wu):
    g, u = x @ wg.t(), x @ wu.t()
    return g * torch.sigmoid(g) * u


def gradients(x, wg, wu, dh):
    """(dx, dwg, dwu) by the formula."""
    g, u = x @ wg.t(), x @ wu.t()
    s = torch.sigmoid(g)
    dg, du = dh * u * s * (1 + g * (1 - s)), dh * g * s
    return dg @ wg + du @ wu, dg.t() @ x, du.t() @ x


def bounds(x, wg, wu, dh):
    """Largest errors of (h, dx, dwg, dwu).  |silu'| <= 1.1 and |silu''| <= 0.5."""
    E, (M, I) = x.shape[1], dh.shape
    g, u = x @ wg.t(), x @ wu.t()
    s = torch.sigmoid(g)
    eg, eu = (E * CUT * (x.abs() @ w.abs().t()) for w in (wg, wu))
    h, f = g * s * u, s * (1 + g * (1 - s))
    bh = 1.1 * eg * u.abs() + (g * s).abs() * eu + 1.1 * eg * eu + (HALF + gate(g)) * h.abs()
    eg, eu = eg + KEPT * (g.abs() + eg), eu + KEPT * (u.abs() + eu)       # as they are kept for the backward
    dg, du = dh * u * f, dh * g * s
    bg = dh.abs() * (0.5 * eg * (u.abs() + eu) + f.abs() * eu)
    bu = dh.abs() * 1.1 * eg
    bg, bu = bg + (HALF + gate(g)) * (dg.abs() + bg), bu + (HALF + gate(g)) * (du.abs() + bu)
    mg, mu = dg.abs() + bg, du.abs() + bu
    out = lambda exact, err: err + HALF * (exact.abs() + err)
    dx, dwg, dwu = dg @ wg + du @ wu, dg.t() @ x, du.t() @ x
    bx = bg @ wg.abs() + bu @ wu.abs() + 2 * I * CUT * (mg @ wg.abs() + mu @ wu.abs())
    bwg, bwu = (b.t() @ x.abs() + M * CUT * (m.t() @ x.abs()) for b, m in ((bg, mg), (bu, mu)))
    return bh, out(dx, bx), out(dwg, bwg), out(dwu, bwu)
