"""CPU: the 8-bit entry points refuse what they cannot take, in words and before a device is touched; the oracle of their
tests agrees with torch's own e4m3 and e8m0."""
import ctypes

import pytest
import torch

import fp8_oracle as ref
import mvpa_native as nat
import mvpa_ops


def test_oracle_rounds_like_torch():
    v = torch.cat([torch.linspace(-448, 448, 20001), torch.randn(4000) * 2.0 ** -7, torch.tensor([0.0, 2.0 ** -10, 3 * 2.0 ** -10, 17.0, 19.0])])
    assert torch.equal(ref.e4m3(v.double()), v.to(torch.float8_e4m3fn).double())
    tops = torch.tensor([448.0, 448.0000305, 447.99997, 1.0, 1.75, 1.7500001, 0.0, 1e-45, 3e38])
    want = torch.tensor([1.0, 2.0, 1.0, 2.0 ** -8, 2.0 ** -8, 2.0 ** -7, 2.0 ** -126, 2.0 ** -126, 2.0 ** 120])
    got = ref.scale_of(tops)
    assert torch.equal(got, want.double()) and torch.equal(got.float().to(torch.float8_e8m0fnu).double(), got)


@pytest.mark.parametrize("call", [
    lambda x: mvpa_ops.quantize_fp8(x),
    lambda x: mvpa_ops.rmsnorm_fp8(x, x[0], 1e-5),
    lambda x: mvpa_ops.silu_mul_fp8(x, x),
    lambda x: mvpa_ops.matmul_fp8(*[x] * 4),
])
def test_cpu_tensors_are_refused(call):
    with pytest.raises(RuntimeError, match="CUDA device"):
        call(torch.zeros(2, 128))


P = 4096   # an address that is never read: every call below is refused first


def _quantize(x=P, ld_x=128, q=P, ld_q=128, s=P, ld_s=1, rows=2, width=128, block=1, dtype=1):
    return nat.lib().mvpa_quantize_fp8(x, ld_x, q, ld_q, s, ld_s, rows, width, block, dtype, None)


def test_quantize_refusals():
    assert _quantize(rows=0) == 0 and _quantize(width=0) == 0          # nothing to do
    assert _quantize(rows=-1) == -1 and _quantize(block=64) == -1 and "64" in nat.last_error()
    assert _quantize(dtype=2) == -2 and _quantize(dtype=3) == -2
    assert _quantize(q=P + 8) == -3 and _quantize(ld_q=136) == -3 and _quantize(ld_q=112) == -3 and _quantize(s=None) == -3
    assert _quantize(ld_s=0) == -1
    assert _quantize(x=None) == -3 and _quantize(x=P + 1) == -3 and _quantize(ld_x=100) == -3
    assert _quantize(rows=1 << 40) == -1 and "too many" in nat.last_error()
    assert _quantize(rows=(65535 * 128) + 1, block=128) == -1
    assert _quantize(width=0x7fffffff, ld_x=1 << 31, ld_q=1 << 31, ld_s=1 << 24) == -1 and _quantize(rows=1 << 31) == -1


def _norm(x=P, add=None, w=P, h=None, q=P, ld_q=128, s=P, ld_s=1, rows=2, width=128, dtype=1):
    return nat.lib().mvpa_rmsnorm_fp8(x, add, w, h, q, ld_q, s, ld_s, rows, width, 1e-5, dtype, None)


def test_norm_and_gate_refusals():
    assert _norm(rows=0) == 0
    assert _norm(width=4112, ld_q=4112, ld_s=33) == -6 and _norm(width=2064, ld_q=2064, ld_s=17, dtype=0) == -6
    assert _norm(x=None) == -3 and _norm(w=None) == -3 and _norm(add=P + 1) == -3 and _norm(h=P + 1) == -3 and _norm(dtype=5) == -2
    gate = nat.lib().mvpa_silu_mul_fp8
    assert gate(P, P, 128, P, 128, P, 1, 0, 128, 1, None) == 0
    assert gate(P, None, 128, P, 128, P, 1, 2, 128, 1, None) == -3
    assert gate(P, P, 100, P, 128, P, 1, 2, 128, 1, None) == -3
    assert gate(P, P, 128, P, 128, P, 1, 2, 128, 2, None) == -2


def _matmul(a=P, ld_a=128, sa=P, b=P, ld_b=128, sb=P, sdt=3, out=P, ld_out=64, M=2, N=64, K=128, odt=1):
    return nat.lib().mvpa_matmul_fp8(a, ld_a, sa, 1, 1, b, ld_b, sb, 1, 1, sdt, out, ld_out, M, N, K, odt, None, None)


def test_matmul_refusals():
    assert _matmul(M=0) == 0 and _matmul(N=0) == 0
    assert _matmul(M=-1) == -1 and _matmul(K=-1) == -1 and _matmul(M=1 << 31) == -1 and _matmul(K=0x7fffffff, ld_a=1 << 31, ld_b=1 << 31) == -1
    assert _matmul(odt=2) == -2 and _matmul(sdt=1) == -2
    assert _matmul(out=None) == -3 and _matmul(out=P + 1) == -3 and _matmul(ld_out=63) == -3 and _matmul(out=P + 2, odt=0) == -3
    assert _matmul(a=P + 8) == -3 and _matmul(ld_a=136) == -3 and _matmul(ld_b=112) == -3 and _matmul(b=None) == -3
    assert _matmul(sa=None) == -3 and _matmul(sb=P + 2, sdt=0) == -3
