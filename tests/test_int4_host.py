"""CPU: the 4-bit definition against itself, and what the operators and the C entry points refuse before they touch a GPU."""
import ctypes

import pytest
import torch

import int4_oracle as ref
import mvpa_native as nat
import mvpa_ops as ops


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_definition(zeros, dtype):
    """Every value within half a step of what stands for it (a step and a clamp more where the scale was rounded down)."""
    g = torch.Generator().manual_seed(3)
    w = torch.randn(9, 200, generator=g).to(dtype)
    q, s, z = ref.quantize(w, 64, zeros)
    at = torch.arange(200) // 64
    stands = (q - (z[:, at] if zeros else 8)).double() * s.double()[:, at]
    slack = 0.5 + 15 * torch.finfo(dtype).eps
    if zeros:
        slack += 0.5                                   # the zero's own rounding moves both ends of the range
    assert ((stands - w.double()).abs() <= slack * s.double()[:, at]).all()
    assert q.min() >= 0 and q.max() <= 15


def test_operators_refuse_on_the_host():
    w = torch.randn(4, 64)
    q, s = torch.zeros(4, 32, dtype=torch.uint8), torch.ones(4, 1)
    for call in (lambda: ops.quantize_int4(w), lambda: ops.dequantize_int4(q, s, group=64), lambda: ops.matmul_int4(w, q, s, group=64),
                 lambda: ops.gated_linear_int4(w, (q, s), (q, s), group=64)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
    with pytest.raises(RuntimeError, match="gate and up"):
        ops.gated_linear_int4(w, (q,), (q, s))


def test_struct_layout():
    assert ctypes.sizeof(nat.Int4) == 48 and [nat.Int4.q.offset, nat.Int4.scales.offset, nat.Int4.zeros.offset, nat.Int4.ld_q.offset,
                                              nat.Int4.ld_s.offset, nat.Int4.ld_z.offset] == [0, 8, 16, 24, 32, 40]


def test_entry_points_refuse():
    lib = nat.lib()
    buf = ctypes.create_string_buffer(1 << 16)
    p = (ctypes.addressof(buf) + 15) & ~15
    ref_of = lambda **k: ctypes.byref(nat.Int4(**{**dict(q=p, scales=p, zeros=None, ld_q=32, ld_s=1, ld_z=0), **k}))
    quant = lambda w=p, ld=64, to=ref_of(), N=4, K=64, group=64, dtype=0: lib.mvpa_quantize_int4(w, ld, to, N, K, group, dtype, None)
    back = lambda w=ref_of(), sd=0, out=p, ld=64, N=4, K=64, group=64, dtype=0: lib.mvpa_dequantize_int4(w, sd, out, ld, N, K, group, dtype, None)
    mul = lambda x=p, ld_x=64, w=ref_of(), up=None, sd=0, out=p, ld=64, M=2, N=4, K=64, group=64, dtype=0, ws=None, nbytes=0: lib.mvpa_matmul_int4(
        x, ld_x, w, up, sd, out, ld, M, N, K, group, dtype, ws, nbytes, None, None)
    shape, types, alignment = -1, -2, -3
    for bad in (dict(N=-1), dict(K=-1), dict(group=16), dict(group=256), dict(K=2 ** 31 - 1)):
        assert quant(**bad) == back(**bad) == mul(**bad) == shape, bad
    assert mul(M=-1) == mul(M=2 ** 31) == shape
    assert quant(dtype=2) == back(sd=2) == back(dtype=3) == mul(sd=3) == mul(dtype=2) == types
    for w in (ref_of(q=None), ref_of(q=p + 8), ref_of(ld_q=40), ref_of(ld_q=16), ref_of(scales=None), ref_of(scales=p + 2), ref_of(ld_s=0),
              ref_of(zeros=p)):
        assert quant(to=w) == back(w=w) == mul(w=w) == mul(up=w) == alignment
    assert quant(w=None) == quant(w=p + 2) == quant(ld=63) == back(out=None) == back(out=p + 1) == back(ld=63) == alignment
    assert mul(x=None) == mul(x=p + 2) == mul(ld_x=63) == mul(out=None) == mul(out=p + 2) == mul(ld=3) == alignment
    # nothing to do is no error
    assert quant(N=0) == quant(K=0) == back(N=0) == back(K=0) == mul(M=0) == mul(N=0) == 0
    # a workspace where x has to be laid out again, and none where it has not
    need = lib.mvpa_matmul_int4_workspace_bytes
    assert need(p, 64, 0, 64, 0) == 0 and need(p, 64, 9, 64, 1) == 0 and need(p, 64, 9, 60, 0) == 9 * 64 * 2 * 3 and need(p + 2, 64, 9, 60, 1) == 9 * 64 * 2
    assert need(p, 63, 9, 60, 1) == 9 * 64 * 2
    assert mul(M=9) == mul(M=9, ws=p, nbytes=9 * 64 * 6 - 1) == mul(M=9, ws=p + 8, nbytes=1 << 15) == -4
    assert "workspace" in nat.last_error()


def test_entry_points_refuse_no_weight():
    """NULL in the place of a weight is an error like the others, not a crash; where nothing is to be done it is not looked at."""
    lib = nat.lib()
    buf = ctypes.create_string_buffer(1 << 16)
    p = (ctypes.addressof(buf) + 15) & ~15
    assert lib.mvpa_quantize_int4(p, 64, None, 4, 64, 64, 0, None) == -3 and "NULL" in nat.last_error()
    assert lib.mvpa_dequantize_int4(None, 0, p, 64, 4, 64, 64, 0, None) == -3 and "NULL" in nat.last_error()
    assert lib.mvpa_matmul_int4(p, 64, None, None, 0, p, 64, 2, 4, 64, 64, 0, None, 0, None, None) == -3 and "NULL" in nat.last_error()
    assert lib.mvpa_quantize_int4(p, 64, None, 0, 64, 64, 0, None) == 0 and lib.mvpa_dequantize_int4(None, 0, p, 64, 4, 0, 64, 0, None) == 0
