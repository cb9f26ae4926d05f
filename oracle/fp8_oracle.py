"""The definitions of the 8-bit operators in 64 bits, written from the formulas (test infrastructure)."""
import torch

BLOCK, TOP = 128, 448.0


def e4m3(v):
    """Nearest e4m3 value in fp64: three mantissa bits down to 2^-6, steps of 2^-9 below; ties to even; |v| <= 464 saturates."""
    _, ex = torch.frexp(v)
    step = torch.ldexp(torch.ones_like(v), (ex - 1).clamp(min=-6) - 3)
    return (torch.round(v / step) * step).clamp(-TOP, TOP)


def scale_of(top):
    """Smallest power of two s >= 2^-126 with top <= 448 s, elementwise, exactly."""
    m, ex = torch.frexp(top.double().clamp(min=TOP * 2.0 ** -126) / TOP)                     # (exact where it matters: top / 448 = 2^e only for top = 448 * 2^e)
    e = torch.where(m > 0.5, ex, ex - 1)
    return torch.ldexp(torch.ones_like(m), e)


def tops(y, tall=1):
    """Largest magnitude of every block."""
    rows, width = y.shape
    down, across = -(-rows // tall), -(-width // BLOCK)
    full = y.new_zeros(down * tall, across * BLOCK)
    full[:rows, :width] = y.abs()
    return full.view(down, tall, across, BLOCK).amax(dim=(1, 3))


def spread(scales, rows, width, tall=1):
    """Scales of blocks as a matrix of the values' shape."""
    return scales.repeat_interleave(tall, 0)[:rows].repeat_interleave(BLOCK, 1)[:, :width]


def pair(y, tall=1):
    y = y.double()
    s = scale_of(tops(y, tall))
    return e4m3(y / spread(s, *y.shape, tall)), s


def value(q, scales, tall=1):
    return q.double() * spread(scales.double(), *q.shape, tall)


def check_pair(q, scales, y, eps, tall=1):
    """(q, scales) is what the definition gives for some values within `eps` (relative) of y: each scale lies between those of
    the block's largest value made smaller and larger by that, each q between the roundings of its value so moved."""
    y = y.double()
    assert q.dtype == torch.float8_e4m3fn and scales.dtype == torch.float8_e8m0fnu and q.shape == y.shape
    top = tops(y, tall)
    s = scales.double()
    assert s.shape == top.shape
    assert bool(((scale_of(top * (1 - eps)) <= s) & (s <= scale_of(top * (1 + eps)))).all())
    v = y / spread(s, *y.shape, tall)
    lo, hi = e4m3(v - v.abs() * eps), e4m3(v + v.abs() * eps)
    got = q.double()
    bad = (got < lo) | (got > hi)
    assert not bool(bad.any()), (int(bad.sum()), got[bad][:4], v[bad][:4])
