"""Weights in 4 bits in 64 bits: quantisation, what a weight stands for, products with it, and how far fp32 sums may be from them.

Test infrastructure; written from the definition, apart from the library's code."""
import torch

from gated_oracle import gate as gate_error

CUT = 2.0 ** -23       # an addition in fp32 that may cut off instead of rounding


def quantize(w, group, zeros):
    """(whole numbers q in int64 (N, K), scales in w's type, zeros in int64 or None)."""
    N, K = w.shape
    groups = -(-K // group)
    q, scales, zs = torch.zeros(N, K, dtype=torch.int64, device=w.device), [], []
    for j in range(groups):
        part = w[:, j * group:(j + 1) * group].double()
        bad = ~part.isfinite().all(1)
        lo, hi = part.amin(1).clamp(max=0), part.amax(1).clamp(min=0)
        s = (((hi - lo) / 15) if zeros else torch.maximum(-lo, hi) / 7).to(w.dtype)
        s = torch.where(bad, torch.full_like(s, float("nan")), s)
        scales.append(s)
        some = (s > 0) & ~bad
        d = torch.where(some, s.double(), 1.0)
        steps = torch.where(some[:, None], torch.round(part / d[:, None]), 0.0)
        if zeros:
            z = torch.where(some, torch.round(-lo / d).clamp(0, 15), 0.0)
            zs.append(z.to(torch.int64))
            q[:, j * group:(j + 1) * group] = (steps + z[:, None]).clamp(0, 15).to(torch.int64)
        else:
            q[:, j * group:(j + 1) * group] = steps.clamp(-8, 7).to(torch.int64) + 8
    return q, torch.stack(scales, 1), torch.stack(zs, 1) if zeros else None


def unpack(q, K):
    """The whole numbers of packed rows."""
    column = torch.arange(K, device=q.device)
    return (q.long()[:, column // 2] >> (4 * (column % 2))) & 15


def values(q, scales, zeros, K, group):
    """What a weight stands for, in 64 bits."""
    at = torch.arange(K, device=q.device) // group
    zero = 8 if zeros is None else zeros.long()[:, at]
    return (unpack(q, K) - zero).double() * scales.double()[:, at]


def product(x, weight, K, group, half):
    """(x W^T, its largest error): sums of K products and of the groups, each scaled (a rounding), and the result's rounding `half`.
    An fp32 x is taken in three parts, whose sums are three times as long."""
    w = values(*weight, K, group)
    exact = x.double() @ w.t()
    size = x.double().abs() @ w.abs().t()
    terms = (3 if x.dtype == torch.float32 else 1) * min(group, K) + 2 * -(-K // group) + 8
    return exact, terms * CUT * size + half * exact.abs(), terms * CUT * size


def gated(x, gate, up, K, group, half):
    """(silu(g) u, its largest error)."""
    g, _, eg = product(x, gate, K, group, 0.0)
    u, _, eu = product(x, up, K, group, 0.0)
    s = torch.sigmoid(g)
    h = g * s * u
    silu = gate_error(g) if half > 2.0 ** -20 else 2.0 ** -20
    return h, 1.1 * eg * u.abs() + (g * s).abs() * eu + 1.1 * eg * eu + (half + silu) * h.abs()
