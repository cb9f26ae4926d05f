"""CPU: the gated projection's definition against differences, and what the C entry points refuse before they touch a GPU."""
import ctypes

import pytest
import torch

import gated_oracle as ref
import mvpa_host
import mvpa_native as nat
import mvpa_ops as ops


def _inputs(M, E, I, seed=0):
    g = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)
    return rand(M, E), rand(I, E) * E ** -0.5, rand(I, E) * E ** -0.5, rand(M, I)


def test_gradients_against_differences():
    x, wg, wu, dh = ins = _inputs(5, 7, 6)
    grads = ref.gradients(*ins)
    step = 2.0 ** -17                       # error of a central difference: step^2 |f'''| / 6 ~ 1e-11, roundings 1e-16 / step ~ 1e-11
    for i, grad in enumerate(grads):
        for at in range(grad.numel()):
            moved = [t.clone() for t in (x, wg, wu)]
            value = []
            for sign in (1, -1):
                moved[i].view(-1)[at] = ins[i].view(-1)[at] + sign * step
                value.append((ref.forward(*moved) * dh).sum())
            assert abs((value[0] - value[1]) / (2 * step) - grad.view(-1)[at]) < 1e-8


def test_gradients_against_autograd():
    x, wg, wu, dh = _inputs(4, 9, 3, 1)
    leaves = [t.requires_grad_() for t in (x, wg, wu)]
    auto = torch.autograd.grad(ref.forward(*leaves), leaves, dh)
    for a, b in zip(auto, ref.gradients(x.detach(), wg.detach(), wu.detach(), dh)):
        torch.testing.assert_close(a, b, rtol=1e-12, atol=1e-13)


def test_bound_of_the_gates_factor():
    """e^-|g| as the fourth power of 2^(|g| c) in fp32, with an exact power of two: what the argument's rounding alone makes of it, over the gates
    in bf16.  From |g| of some 50 on that is more than 2^-18."""
    g = torch.arange(0x3f80, 0x43ad, dtype=torch.int32).to(torch.int16).view(torch.bfloat16).double()     # 1 to 345
    c = torch.tensor(0.25 * 1.4426950408889634, dtype=torch.float32)
    t = (g.float() * c).double()
    off = (torch.exp2(-4 * t) / torch.exp(-g) - 1).abs()
    assert bool((off <= ref.gate(-g) - ref.GATE).all())
    assert float(off.max()) > 2.0 ** -17 > ref.GATE and bool((off[g < 20] < ref.GATE).all())


def test_entry_points_refuse():
    lib = nat.lib()
    buf = ctypes.create_string_buffer(1 << 16)
    p = (ctypes.addressof(buf) + 15) & ~15
    fwd = lambda x=p, ld_x=64, wg=p, wu=p, h=p, ld_h=64, saved=None, M=4, E=64, I=64: lib.mvpa_gated_linear(
        x, ld_x, wg, wu, h, ld_h, saved, M, E, I, None, None)
    bwd = lambda dh=p, ld=64, saved=p, x=p, dg=p, du=p, dx=p, dwg=p, dwu=p, M=4, E=64, I=64: lib.mvpa_gated_linear_bwd(
        dh, ld, saved, x, 64, p, p, dg, du, dx, dwg, dwu, M, E, I, None, 0, None, None)
    assert lib.mvpa_gated_linear_saved_bytes(5, 24) == 5 * (2 * 48 + 2 * 32) and lib.mvpa_gated_linear_saved_bytes(0, 24) == 0
    shape = (dict(M=0), dict(E=0), dict(I=0), dict(E=60), dict(I=4), dict(M=-1), dict(M=2 ** 31))
    for bad in shape:
        assert fwd(**bad) == bwd(**bad) == -1 and "multiples of 8" in nat.last_error(), bad
    for bad in (dict(x=p + 2), dict(ld_x=63), dict(ld_x=56), dict(wg=None), dict(wu=p + 8), dict(h=None), dict(ld_h=68), dict(saved=p + 8)):
        assert fwd(**bad) not in (0, -1) and "16-byte" in nat.last_error(), bad
    for bad in (dict(dh=None), dict(ld=60), dict(saved=None), dict(du=p + 4), dict(dwg=None), dict(dx=p + 2), dict(x=None)):
        assert bwd(**bad) not in (0, -1) and "16-byte" in nat.last_error(), bad


@pytest.mark.parametrize("name,counts", [("backward", (14,)), ("branches", (14, 15)), ("block_forward", (20,)), ("block_backward", (32,))])
def test_native_calls_count_their_arguments(name, counts):
    call = getattr(mvpa_host.module(), name)
    for count in counts:
        assert call(*[None] * count) is None      # (no tensors: Python's path answers)
    for other in (counts[0] - 1, counts[-1] + 1):
        with pytest.raises(TypeError, match="number of arguments"):
            call(*[None] * other)


def test_more_rows_than_the_kernels_count(monkeypatch):
    """2^31 - 1024 rows and more are served by torch's operations, like everything that the kernels do not take."""
    lib = nat.lib()
    buf = ctypes.create_string_buffer(1 << 12)
    p = (ctypes.addressof(buf) + 15) & ~15
    assert lib.mvpa_gated_linear(p, 8, p, p, p, 8, None, ops._MOST + 1, 8, 8, None, None) == -1 and str(ops._MOST) in nat.last_error()
    monkeypatch.setattr(ops, "_plain", lambda *ts: True)
    monkeypatch.setattr(ops._GatedLinear, "apply", lambda *a: pytest.fail("the kernel was asked for"))
    monkeypatch.setattr(ops, "_MOST", 8)
    monkeypatch.setattr(ops, "swiglu", lambda g, u: torch.nn.functional.silu(g) * u)
    x, w = torch.ones(9, 8, dtype=torch.bfloat16), torch.ones(8, 8, dtype=torch.bfloat16)
    assert ops.gated_linear(x, w, w).shape == (9, 8)
