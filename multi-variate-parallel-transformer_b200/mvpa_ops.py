"""Torch-tensor front ends of the C-ABI kernels that surround the attention in an MVPFormer block,
its encoder and its heads (``include/mvpa.h``: mvpa_rmsnorm, mvpa_silu_mul, mvpa_wave_encode,
mvpa_channel_mean, mvpa_contrastive_logits, the backwards mvpa_rmsnorm_bwd, mvpa_silu_mul_bwd, the gated
projection mvpa_gated_linear(_bwd), the block in 8 bits: mvpa_quantize_fp8, mvpa_rmsnorm_fp8,
mvpa_silu_mul_fp8, mvpa_matmul_fp8, and weights in 4 bits: mvpa_quantize_int4, mvpa_dequantize_int4,
mvpa_matmul_int4).  `rmsnorm_train`, `swiglu` and `gated_linear` are differentiable and take any tensor
(torch expressions serve what the kernels do not); the others are forward only, CUDA tensors, bf16 or
fp32 (and their pairs in 8 or 4 bits).
"""
from __future__ import annotations

import ctypes
import functools

import numpy as np
import torch

import mvpa_host as _host
import mvpa_native as _nat
from attentions import attn as _attn


def _code(t: torch.Tensor) -> int:
    if t.dtype == torch.bfloat16:
        return _nat.MVPA_BF16
    if t.dtype == torch.float32:
        return _nat.MVPA_F32
    raise RuntimeError(f"mvpa_ops: dtype {t.dtype} not supported (bfloat16 or float32)")


def _stream(t: torch.Tensor) -> ctypes.c_void_p:
    return ctypes.c_void_p(torch.cuda.current_stream(t.device).cuda_stream)


def _need_cuda(*ts):
    for t in ts:
        if t is not None and not t.is_cuda:
            raise RuntimeError("mvpa_ops: tensors must be on a CUDA device (no CPU path)")


def rmsnorm(x, weight, eps, add=None, sum_out=None, out=None):
    """y = rmsnorm(h) * weight over the last dimension, h = x (+ add).  With `add`, h is written to `sum_out`
    (which may be `x` itself: the update is elementwise).  Returns y."""
    _need_cuda(x, weight, add)
    E = x.shape[-1]
    x2 = x.reshape(-1, E)
    assert x2.is_contiguous() and weight.is_contiguous() and weight.dtype == x.dtype
    y = torch.empty_like(x2) if out is None else out
    if add is not None:
        assert add.dtype == x.dtype and add.reshape(-1, E).is_contiguous()
    with _nat.on_device(x.device):
        st = _nat.lib().mvpa_rmsnorm(x2.data_ptr(), add.data_ptr() if add is not None else None, weight.data_ptr(),
                                     sum_out.data_ptr() if sum_out is not None else None, y.data_ptr(), x2.shape[0], E,
                                     float(eps), _code(x), _stream(x))
    _nat.check(st, "mvpa_rmsnorm")
    return y.view(x.shape)


def silu_mul(gate, up, out):
    """out = silu(gate) * up for 2-D views with unit inner stride (column blocks of wider buffers are fine)."""
    _need_cuda(gate, up, out)
    rows, width = gate.shape
    assert up.shape == gate.shape and out.shape == gate.shape
    assert gate.stride(1) == up.stride(1) == out.stride(1) == 1 and gate.stride(0) == up.stride(0)
    with _nat.on_device(gate.device):
        st = _nat.lib().mvpa_silu_mul(gate.data_ptr(), up.data_ptr(), gate.stride(0), out.data_ptr(), out.stride(0), rows,
                                      width, _code(gate), _stream(gate))
    _nat.check(st, "mvpa_silu_mul")
    return out


def rmsnorm_bwd(x, weight, dy, eps, add=None):
    """Gradients (dx, dweight) of `rmsnorm(x, weight, eps)` (no residual) for the incoming gradient `dy`; `add`, the
    gradient that reaches x on another way (a residual connection), is added to dx."""
    _need_cuda(x, weight, dy, add)
    E = x.shape[-1]
    x2, dy2 = x.reshape(-1, E), dy.reshape(-1, E)
    assert x2.is_contiguous() and dy2.is_contiguous() and weight.is_contiguous()
    assert weight.dtype == x.dtype == dy.dtype and dy.shape == x.shape
    if add is not None:
        assert add.dtype == x.dtype and add.is_contiguous() and add.numel() == x.numel()
    dx, dw = torch.empty(x.shape, dtype=x.dtype, device=x.device), torch.empty_like(weight)
    lib = _nat.lib()
    with _nat.on_device(x.device):   # (the size depends on the device's multiprocessors)
        nbytes = lib.mvpa_rmsnorm_bwd_workspace_bytes(x2.shape[0], E)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
        st = lib.mvpa_rmsnorm_bwd(x2.data_ptr(), weight.data_ptr(), dy2.data_ptr(), add.data_ptr() if add is not None else None,
                                  dx.data_ptr(), dw.data_ptr(), x2.shape[0], E, float(eps), _code(x), ws.data_ptr(), nbytes,
                                  _stream(x))
    _nat.check(st, "mvpa_rmsnorm_bwd")
    return dx, dw


def silu_mul_bwd(gate, up, dout):
    """Gradients (dgate, dup) of silu(gate) * up for 2-D tensors with unit inner stride."""
    _need_cuda(gate, up, dout)
    rows, width = gate.shape
    assert up.shape == gate.shape and dout.shape == gate.shape and gate.dtype == up.dtype == dout.dtype
    assert gate.stride(1) == up.stride(1) == dout.stride(1) == 1 and gate.stride(0) == up.stride(0)
    dgate, dup = (torch.empty((rows, width), dtype=gate.dtype, device=gate.device) for _ in range(2))
    with _nat.on_device(gate.device):
        st = _nat.lib().mvpa_silu_mul_bwd(gate.data_ptr(), up.data_ptr(), gate.stride(0), dout.data_ptr(), dout.stride(0),
                                          dgate.data_ptr(), dup.data_ptr(), width, rows, width, _code(gate), _stream(gate))
    _nat.check(st, "mvpa_silu_mul_bwd")
    return dgate, dup


def _plain(*ts):
    """Tensors that the kernels can take and that nothing traces: ordinary CUDA tensors of one supported dtype,
    contiguous, 16-byte aligned, not empty; no forward-mode level, functorch transform or tracer is active
    (those are served by the differentiable torch expressions)."""
    t0 = ts[0]
    if _host.usable(t0):
        answer = _host.module().plain(*ts)
        if answer >= 0:
            return answer == 1
    # (a function mode is active, or the first tensor is none of ours; types first: a symbolic value answers no question about itself)
    if not all(type(t) in (torch.Tensor, torch.nn.Parameter) for t in ts) or not _nat.untraced() \
            or t0.dtype not in (torch.bfloat16, torch.float32):
        return False
    # (a backward may run on a thread of the autograd engine, where a transform shows on the tensor alone)
    if any(torch._C._functorch.is_functorch_wrapped_tensor(t) or not torch._C._has_storage(t) for t in ts):
        return False
    return all(t.is_cuda and t.dtype == t0.dtype and t.device == t0.device
               and t.is_contiguous() and t.numel() > 0 and t.data_ptr() % 16 == 0 for t in ts)


def _rows_fit(t):
    """The row kernels' widths: whole 16-byte vectors, at most 512 of them."""
    nbytes = t.shape[-1] * t.element_size() if t.dim() else 0
    return nbytes % 16 == 0 and nbytes <= 512 * 16


class _RMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, eps):
        ctx.save_for_backward(x, weight)
        ctx.eps = eps
        y = torch.empty_like(x)          # (not a view of one: the caller may change it in place)
        rmsnorm(x, weight, eps, out=y)
        return y

    @staticmethod
    def backward(ctx, dy):
        x, weight = ctx.saved_tensors
        if not torch.is_grad_enabled() and _plain(x, weight, dy.contiguous()):
            return (*rmsnorm_bwd(x, weight, dy.contiguous(), ctx.eps), None)
        # a graph of the gradient is wanted (or a transform is active): the same formula in torch operations
        xf, wf, g = x.float(), weight.float(), dy.float()
        rstd = torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + ctx.eps)
        xh, gw = xf * rstd, g * wf
        dx = rstd * (gw - xh * (gw * xh).mean(-1, keepdim=True))
        return dx.to(x.dtype), (g * xh).sum(dim=tuple(range(x.dim() - 1))).to(weight.dtype), None


def rmsnorm_train(x, weight, eps):
    """Differentiable `x * rsqrt(mean(x^2) + eps) * weight` over the last dimension, in fp32, rounded once: one
    kernel forward and two backward where the kernels apply, torch operations everywhere else."""
    if _plain(x, weight) and _rows_fit(x) and x.dim() > 0 and weight.shape == x.shape[-1:]:
        return _RMSNorm.apply(x, weight, eps)
    xf = x.float()
    return (xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps) * weight.float()).to(x.dtype)


class _SwiGLU(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gate, up):
        ctx.save_for_backward(gate, up)
        w = gate.shape[-1]
        out = torch.empty_like(gate)     # (not a view of one, as above)
        silu_mul(gate.view(-1, w), up.view(-1, w), out.view(-1, w))
        return out

    @staticmethod
    def backward(ctx, dout):
        gate, up = ctx.saved_tensors
        if not torch.is_grad_enabled() and _plain(gate, up, dout.contiguous()):
            w = gate.shape[-1]
            dgate, dup = silu_mul_bwd(gate.view(-1, w), up.view(-1, w), dout.contiguous().view(-1, w))
            return dgate.view(gate.shape), dup.view(gate.shape)
        gf, d = gate.float(), dout.float()
        s = torch.sigmoid(gf)
        return (d * up.float() * (s * (1 + gf * (1 - s)))).to(gate.dtype), (d * (gf * s)).to(up.dtype)


def swiglu(gate, up):
    """Differentiable silu(gate) * up: one kernel each way where the kernels apply, torch operations elsewhere."""
    if _plain(gate, up) and gate.shape == up.shape and gate.dim() > 0 and gate.shape[-1] * gate.element_size() % 16 == 0:
        return _SwiGLU.apply(gate, up)
    return torch.nn.functional.silu(gate) * up


def _status_word(device):
    """The kernels' status word, or None unless calls look at it."""
    return torch.zeros(64, dtype=torch.int32, device=device) if _attn._CHECK_STATUS else None


def _look_at(status, what, like):
    if status is not None:      # debugging aid: synchronises the stream
        _nat.check(_nat.lib().mvpa_workspace_status(status.data_ptr(), 256, _stream(like)), f"{what} kernel")


def _gated_kernel(x, w_gate, w_up, save):
    """(h, what the backward wants of it, or None unless `save`) by the kernel; x (rows, E)."""
    (rows, E), I = x.shape, w_gate.shape[0]
    h = torch.empty((rows, I), dtype=x.dtype, device=x.device)
    lib = _nat.lib()
    saved = torch.empty(lib.mvpa_gated_linear_saved_bytes(rows, I), dtype=torch.uint8, device=x.device) if save else None
    with _nat.on_device(x.device):
        status = _status_word(x.device)
        st = lib.mvpa_gated_linear(x.data_ptr(), E, w_gate.data_ptr(), w_up.data_ptr(), h.data_ptr(), I, saved.data_ptr() if save else None,
                                   rows, E, I, None if status is None else status.data_ptr(), _stream(x))
        _nat.check(st, "mvpa_gated_linear")
        _look_at(status, "mvpa_gated_linear", x)
    return h, saved


def _gated_kernel_bwd(dh, x, w_gate, w_up, saved, need_x, need_w):
    """(dx, dw_gate, dw_up) by the kernels, None where not needed; x (rows, E)."""
    (rows, E), I = x.shape, w_gate.shape[0]
    dgate, dup = torch.empty_like(dh), torch.empty_like(dh)
    dx = torch.empty((rows, E), dtype=x.dtype, device=x.device) if need_x else None
    dw_gate, dw_up = (torch.empty_like(w_gate), torch.empty_like(w_up)) if need_w else (None, None)
    ptr = lambda t: None if t is None else t.data_ptr()
    with _nat.on_device(x.device):
        status = _status_word(x.device)
        nbytes = _nat.lib().mvpa_gated_linear_bwd_workspace_bytes(rows, E, I)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device) if nbytes else None
        st = _nat.lib().mvpa_gated_linear_bwd(dh.data_ptr(), I, saved.data_ptr(), x.data_ptr(), E, w_gate.data_ptr(), w_up.data_ptr(),
                                              dgate.data_ptr(), dup.data_ptr(), ptr(dx), ptr(dw_gate), ptr(dw_up), rows, E, I, ptr(ws), nbytes,
                                              ptr(status), _stream(x))
        _nat.check(st, "mvpa_gated_linear_bwd")
        _look_at(status, "mvpa_gated_linear_bwd", x)
    return dx, dw_gate, dw_up


class _GatedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up):
        need = any(ctx.needs_input_grad)
        native = _host.module().gated_forward(x, w_gate, w_up, need, _attn._CHECK_STATUS) if _host.usable(x) else None
        h, saved = native or _gated_kernel(x.view(-1, x.shape[-1]), w_gate, w_up, need)
        ctx.save_for_backward(x, w_gate, w_up, saved)
        return h if h.dim() == x.dim() else h.reshape(*x.shape[:-1], w_gate.shape[0])

    @staticmethod
    def backward(ctx, dh):
        x, w_gate, w_up, saved = ctx.saved_tensors
        need = ctx.needs_input_grad
        E, I = x.shape[-1], w_gate.shape[0]
        if not torch.is_grad_enabled():
            if _host.usable(dh):
                native = _host.module().gated_backward(dh, x, w_gate, w_up, saved, need[0] + 2 * need[1] + 4 * need[2], _attn._CHECK_STATUS)
                if native is not None:
                    return native
            d = dh.contiguous()
            if _plain(d, x, w_gate, w_up) and saved.device == x.device and saved.is_contiguous() and saved.data_ptr() % 16 == 0:
                dx, dw_gate, dw_up = _gated_kernel_bwd(d.view(-1, I), x.view(-1, E), w_gate, w_up, saved, need[0], need[1] or need[2])
                return dx.view(x.shape) if need[0] else None, dw_gate if need[1] else None, dw_up if need[2] else None
        # a graph of the gradient is wanted (or a transform is active): the same formula in torch operations, in fp32 as the kernels' sums
        # are and rounded once, whatever region the backward runs in
        with torch.autocast("cuda", enabled=False):
            x2, d, wg, wu = x.reshape(-1, E).float(), dh.reshape(-1, I).float(), w_gate.float(), w_up.float()
            g, u = torch.nn.functional.linear(x2, wg), torch.nn.functional.linear(x2, wu)
            s = torch.sigmoid(g)
            dg, du = d * (s * (1 + g * (1 - s))) * u, d * (g * s)
            return (dg @ wg + du @ wu).to(x.dtype).view(x.shape), (dg.t() @ x2).to(x.dtype), (du.t() @ x2).to(x.dtype)


_MOST = 2 ** 31 - 1025     # rows, columns and features that the gated projection's kernels count (include/mvpa.h)


def gated_linear_kernel(x, w_gate, w_up):
    """`gated_linear` where it is one kernel, else None."""
    if _host.usable(x):
        h = _host.module().gated_linear(x, w_gate, w_up, _attn._CHECK_STATUS)     # (an ordinary call that no gradient flows through)
        if h is not None:
            return h
    # (types first: a symbolic value answers no question about itself)
    if (all(type(t) in (torch.Tensor, torch.nn.Parameter) for t in (x, w_gate, w_up)) and not torch.is_autocast_enabled("cuda")
            and x.dtype == torch.bfloat16 and x.dim() > 1 and w_gate.dim() == 2 and w_gate.shape == w_up.shape
            and x.shape[-1] == w_gate.shape[1] and x.shape[-1] % 8 == 0 and w_gate.shape[0] % 8 == 0):
        if not x.is_contiguous():
            x = x.contiguous()
        if _plain(x, w_gate, w_up) and max(x.numel() // x.shape[-1], *w_gate.shape) <= _MOST:
            return _GatedLinear.apply(x, w_gate, w_up)
    return None


def gated_linear(x, w_gate, w_up):
    """Differentiable silu(x w_gate^T) * (x w_up^T) for x (..., E) and weights (I, E): the MLP up to its down projection.  bf16 with E
    and I multiples of 8: one kernel forward, with both products and the activation in fp32, rounded once; the backward is one for the
    gate and one for each matrix product (the gradient of x, that of both weights), from the two products, of which the forward keeps
    24 bits each where a gradient is wanted.  Everything else, and calls under autocast, by torch operations."""
    h = gated_linear_kernel(x, w_gate, w_up)
    return swiglu(torch.nn.functional.linear(x, w_gate), torch.nn.functional.linear(x, w_up)) if h is None else h


def gated_linear_into(out, x, w_gate, w_up):
    """Inference form of `gated_linear`: no autograd record, and the result goes into `out` (rows, I), which may be a column block of a
    wider buffer.  x (rows, E) and weights (I, E) in bf16 with E and I multiples of 8, contiguous; rows on 16-byte boundaries."""
    _fp8_inputs("gated_linear_into", x, w_gate, w_up, out)
    if not (x.dtype == w_gate.dtype == w_up.dtype == out.dtype == torch.bfloat16):
        raise RuntimeError(f"gated_linear_into: tensors are bfloat16, got {x.dtype}, {w_gate.dtype}, {w_up.dtype}, {out.dtype}")
    if (x.dim() != 2 or w_gate.dim() != 2 or w_up.shape != w_gate.shape or w_gate.shape[1] != x.shape[1] or out.shape != (x.shape[0], w_gate.shape[0])
            or not (x.is_contiguous() and w_gate.is_contiguous() and w_up.is_contiguous())):
        raise RuntimeError("gated_linear_into: shapes do not go together, or x or a weight is not contiguous: "
                           + ", ".join(str(tuple(t.shape)) for t in (out, x, w_gate, w_up)))
    (rows, E), I = x.shape, w_gate.shape[0]
    ld = _fp8_rows("gated_linear_into", out, "out")
    if rows == 0:
        return out
    with _nat.on_device(x.device):
        status = _status_word(x.device)
        st = _nat.lib().mvpa_gated_linear(x.data_ptr(), E, w_gate.data_ptr(), w_up.data_ptr(), out.data_ptr(), ld, None, rows, E, I,
                                          None if status is None else status.data_ptr(), _stream(x))
        _nat.check(st, "mvpa_gated_linear")
        _look_at(status, "mvpa_gated_linear", x)
    return out


@functools.lru_cache(maxsize=None)
def db4_filters():
    """Decomposition filters (dec_lo, dec_hi) of the Daubechies wavelet with four vanishing moments, eight
    taps, derived numerically: |H(w)|^2 = 2 cos^8(w/2) P(sin^2(w/2)), P(y) = 1 + 4y + 10y^2 + 20y^3;
    the roots of P map to z through y = (2 - z - 1/z) / 4, the three roots inside the unit circle give the
    minimum-phase ("extremal phase") scaling filter h, normalised to sum sqrt(2).  Conventions of `pywt`
    (which `models/fftencoder.py:62` takes its filters from): dec_lo = h reversed, dec_hi[k] = -(-1)^k h[k]."""
    y_roots = np.roots([20.0, 10.0, 4.0, 1.0])
    z_roots = []
    for y in y_roots:
        pair = np.roots([1.0, -(2.0 - 4.0 * y), 1.0])
        z_roots.append(pair[np.argmin(np.abs(pair))])
    h = np.poly(np.concatenate([-np.ones(4), np.array(z_roots)])).real
    h *= np.sqrt(2.0) / h.sum()
    dec_lo = h[::-1].copy()
    dec_hi = np.array([-((-1) ** k) * h[k] for k in range(8)])
    return dec_lo.astype(np.float32), dec_hi.astype(np.float32)


def wave_sizes(segment_len: int):
    """(per-level coefficient counts finest first, total row length) of the encoder's transform."""
    levels = (ctypes.c_int32 * 16)()
    total = _nat.lib().mvpa_wave_encode_size(int(segment_len), levels, 16)
    sizes, n = [], segment_len
    while len(sizes) < 16 and levels[len(sizes)] > 0:
        sizes.append(int(levels[len(sizes)]))
    return sizes, int(total)


def wave_encode(x, ln_weight, eps=1e-5, pad_to=None):
    """x (rows, len) fp32 / bf16 -> (rows, pad_to or total) in ln_weight's dtype: wavelet coefficients of every
    level, RMS-normalised and scaled by ln_weight; columns past the coefficient count are zero."""
    _need_cuda(x, ln_weight)
    rows, n = x.shape
    assert x.stride(1) == 1
    _, total = wave_sizes(n)
    ld_out = total if pad_to is None else int(pad_to)
    assert ln_weight.numel() == total and ln_weight.is_contiguous()
    out = torch.empty((rows, ld_out), dtype=ln_weight.dtype, device=x.device)
    lo, hi = db4_filters()
    fp = ctypes.POINTER(ctypes.c_float)
    with _nat.on_device(x.device):
        st = _nat.lib().mvpa_wave_encode(x.data_ptr(), x.stride(0), _code(x), lo.ctypes.data_as(fp), hi.ctypes.data_as(fp),
                                         ln_weight.data_ptr(), out.data_ptr(), ld_out, _code(ln_weight), rows, n,
                                         float(eps), _stream(x))
    _nat.check(st, "mvpa_wave_encode")
    return out


def channel_mean(h):
    """h (B,T,C,E) -> (B,E): mean over the channels of the last time step."""
    _need_cuda(h)
    B, T, C, E = h.shape
    assert h.is_contiguous()
    out = torch.empty((B, E), dtype=h.dtype, device=h.device)
    with _nat.on_device(h.device):
        st = _nat.lib().mvpa_channel_mean(h.data_ptr(), out.data_ptr(), B, T, C, E, _code(h), _stream(h))
    _nat.check(st, "mvpa_channel_mean")
    return out


def contrastive_logits(pred, enc, negatives, temperature):
    """pred, enc (B,T,C,E); negatives (B,T,C,K) int32 rows of enc.view(-1, E).  Returns (B*(T-1)*C, 1+K) fp32."""
    _need_cuda(pred, enc, negatives)
    B, T, C, E = pred.shape
    K = negatives.shape[-1]
    assert enc.shape == pred.shape and pred.is_contiguous() and enc.is_contiguous() and enc.dtype == pred.dtype
    assert negatives.dtype == torch.int32 and negatives.is_contiguous() and negatives.shape[:3] == (B, T, C)
    out = torch.empty((B * (T - 1) * C, K + 1), dtype=torch.float32, device=pred.device)
    with _nat.on_device(pred.device):
        st = _nat.lib().mvpa_contrastive_logits(pred.data_ptr(), enc.data_ptr(), negatives.data_ptr(), out.data_ptr(), B, T,
                                                C, E, K, float(temperature), _code(pred), _stream(pred))
    _nat.check(st, "mvpa_contrastive_logits")
    return out


# ---- the block in 8 bits ----
# A row in 8 bits is a pair (q, scales): q (rows, width) float8_e4m3fn whose rows start on 16-byte boundaries, scales
# (rows, ceil(width / 128)) float8_e8m0fnu, one power of two for each block of 128 neighbours; a weight has one for each block
# of 128 x 128.  The pair stands for q * scale.  scale is the smallest 2^e, e >= -126, with max|y| <= 448 * 2^e over the block,
# q = y / scale rounded once, to nearest, ties to even.  A block that holds an infinity or a NaN is NaN throughout.

FP8_BLOCK = 128
_FP8_SCALES = {torch.float8_e8m0fnu: _nat.MVPA_E8M0, torch.float32: _nat.MVPA_F32}


def _fp8_inputs(what, *ts):
    """Ordinary CUDA tensors on one device that no gradient has to flow through."""
    t0 = ts[0]
    for t in ts:
        if not t.is_cuda:
            raise RuntimeError(f"{what}: tensors must be on a CUDA device (no CPU path)")
        if t.device != t0.device:
            raise RuntimeError(f"{what}: tensors are on {t0.device} and {t.device}")
    if torch.is_grad_enabled() and any(t.requires_grad for t in ts):
        raise RuntimeError(f"{what} has no gradient: call it under torch.no_grad() or on detached tensors")


def _fp8_rows(what, t, name):
    """Leading dimension of a matrix with unit inner stride (that of one row, or of an empty matrix, is never used)."""
    if t.dim() != 2 or (t.stride(1) != 1 and t.shape[1] > 1):
        raise RuntimeError(f"{what}: {name} must be a matrix with unit inner stride, got shape {tuple(t.shape)}, strides {t.stride()}")
    if t.shape[0] < 2 or t.numel() == 0:
        return (t.shape[1] + 15) // 16 * 16
    if t.stride(0) < t.shape[1]:
        raise RuntimeError(f"{what}: the rows of {name} overlap (strides {t.stride()})")
    return t.stride(0)


def _fp8_pair(what, out, rows, width, block_rows, device):
    """(q, scales) to write into: the caller's, or new ones."""
    shape, blocks = (rows, width), (-(-rows // block_rows), -(-width // FP8_BLOCK))
    if out is None:
        ld = (width + 15) // 16 * 16
        q = torch.empty((rows, ld), dtype=torch.float8_e4m3fn, device=device)
        return (q if ld == width else q[:, :width]), torch.empty(blocks, dtype=torch.float8_e8m0fnu, device=device)
    q, scales = out
    if (q.shape != shape or q.dtype != torch.float8_e4m3fn or scales.shape != blocks or scales.dtype != torch.float8_e8m0fnu
            or q.device != device or scales.device != device):
        raise RuntimeError(f"{what}: out must be q {shape} float8_e4m3fn and scales {blocks} float8_e8m0fnu on {device}, got "
                           f"{tuple(q.shape)} {q.dtype} {q.device} and {tuple(scales.shape)} {scales.dtype} {scales.device}")
    return q, scales


def quantize_fp8(x, block_rows=1, out=None):
    """x (rows, width), bf16 or fp32, in 8 bits: (q, scales).  `block_rows=1` gives every row its own scales (activations),
    `block_rows=128` every block of 128 x 128 one (weights).  `out=(q, scales)` writes into the caller's tensors, which may be
    column blocks of wider ones."""
    if _host.usable(x):
        pair = _host.module().quantize_fp8(x, block_rows, None, None) if out is None else _host.module().quantize_fp8(x, block_rows, *out)
        if pair is not None:
            return pair
    _fp8_inputs("quantize_fp8", x)
    if block_rows not in (1, FP8_BLOCK):
        raise RuntimeError(f"quantize_fp8: block_rows is 1 or {FP8_BLOCK}, got {block_rows}")
    ld = _fp8_rows("quantize_fp8", x, "x")
    rows, width = x.shape
    q, scales = _fp8_pair("quantize_fp8", out, rows, width, block_rows, x.device)
    ld_q, ld_s = _fp8_rows("quantize_fp8", q, "q"), _fp8_rows("quantize_fp8", scales, "scales")
    with _nat.on_device(x.device):
        st = _nat.lib().mvpa_quantize_fp8(x.data_ptr(), ld, q.data_ptr(), ld_q, scales.data_ptr(), ld_s, rows, width, block_rows,
                                          _code(x), _stream(x))
    _nat.check(st, "mvpa_quantize_fp8")
    return q, scales


def rmsnorm_fp8(x, weight, eps, add=None, sum_out=None, out=None):
    """`rmsnorm` with the result in 8 bits: (q, scales) of rmsnorm(h) * weight, h = x (+ add), for x (..., E) with all leading
    dimensions as rows.  h is rounded to x's type, as in `rmsnorm`, and written to `sum_out` (which may be `x`); the normalised
    row goes from fp32 to e4m3 in one rounding.  E up to 4096 in bf16, 2048 in fp32."""
    if _host.usable(x):
        pair = _host.module().rmsnorm_fp8(x, weight, eps, add, sum_out, None, None) if out is None else _host.module().rmsnorm_fp8(x, weight, eps, add, sum_out, *out)
        if pair is not None:
            return pair
    extra = [t for t in (add, sum_out) if t is not None]
    _fp8_inputs("rmsnorm_fp8", x, weight, *extra)
    E = x.shape[-1]
    if not all(t.is_contiguous() and t.dtype == x.dtype for t in (x, weight, *extra)):
        raise RuntimeError("rmsnorm_fp8: x, weight, add and sum_out must be contiguous and of one type")
    if weight.shape != (E,) or any(t.numel() != x.numel() or t.shape[-1:] != (E,) for t in extra):
        raise RuntimeError(f"rmsnorm_fp8: shapes do not go together: x {tuple(x.shape)}, weight {tuple(weight.shape)}, "
                           + ", ".join(str(tuple(t.shape)) for t in extra))
    rows = x.numel() // E if E else 0
    q, scales = _fp8_pair("rmsnorm_fp8", out, rows, E, 1, x.device)
    ld_q, ld_s = _fp8_rows("rmsnorm_fp8", q, "q"), _fp8_rows("rmsnorm_fp8", scales, "scales")
    with _nat.on_device(x.device):
        st = _nat.lib().mvpa_rmsnorm_fp8(x.data_ptr(), add.data_ptr() if add is not None else None, weight.data_ptr(),
                                         sum_out.data_ptr() if sum_out is not None else None, q.data_ptr(), ld_q,
                                         scales.data_ptr(), ld_s, rows, E, float(eps), _code(x), _stream(x))
    _nat.check(st, "mvpa_rmsnorm_fp8")
    return q, scales


def silu_mul_fp8(gate, up, out=None):
    """silu(gate) * up in 8 bits: (q, scales).  gate, up (rows, width) with unit inner stride (column blocks of a wider buffer
    are fine).  From fp32 to e4m3 in one rounding; `silu_mul` rounds silu(gate) to the type in between, as eager PyTorch does."""
    if _host.usable(gate):
        pair = _host.module().silu_mul_fp8(gate, up, None, None) if out is None else _host.module().silu_mul_fp8(gate, up, *out)
        if pair is not None:
            return pair
    _fp8_inputs("silu_mul_fp8", gate, up)
    ld = _fp8_rows("silu_mul_fp8", gate, "gate")
    if up.shape != gate.shape or up.dtype != gate.dtype or _fp8_rows("silu_mul_fp8", up, "up") != ld:
        raise RuntimeError(f"silu_mul_fp8: gate and up must have one shape, type and row stride, got {tuple(gate.shape)} {gate.dtype} "
                           f"{gate.stride()} and {tuple(up.shape)} {up.dtype} {up.stride()}")
    rows, width = gate.shape
    q, scales = _fp8_pair("silu_mul_fp8", out, rows, width, 1, gate.device)
    ld_q, ld_s = _fp8_rows("silu_mul_fp8", q, "q"), _fp8_rows("silu_mul_fp8", scales, "scales")
    with _nat.on_device(gate.device):
        st = _nat.lib().mvpa_silu_mul_fp8(gate.data_ptr(), up.data_ptr(), ld, q.data_ptr(), ld_q, scales.data_ptr(), ld_s, rows,
                                          width, _code(gate), _stream(gate))
    _nat.check(st, "mvpa_silu_mul_fp8")
    return q, scales


def matmul_fp8(a, a_scales, b, b_scales, out=None, dtype=torch.bfloat16):
    """a @ b.T for pairs in 8 bits: a (M, K) with scales (M, ceil(K / 128)), b (N, K), a weight, with scales
    (ceil(N / 128), ceil(K / 128)); the result (M, N) in `dtype` (bfloat16 or float32), or in `out`, which may be a column
    block of a wider buffer.  The scales are both float8_e8m0fnu, as the functions above write them, or both float32, with any
    strides.  Products and sums are in fp32, rounded once."""
    if (out is not None or dtype is torch.bfloat16 or dtype is torch.float32) and _host.usable(a):
        done = _host.module().matmul_fp8(a, a_scales, b, b_scales, out, dtype is torch.float32, _attn._CHECK_STATUS)
        if done is not None:
            return done if out is None else out
    what = "matmul_fp8"
    _fp8_inputs(what, a, a_scales, b, b_scales, *(() if out is None else (out,)))
    ld_a, ld_b = _fp8_rows(what, a, "a"), _fp8_rows(what, b, "b")
    (M, K), N = a.shape, b.shape[0]
    kb = -(-K // FP8_BLOCK)
    if a.dtype != torch.float8_e4m3fn or b.dtype != torch.float8_e4m3fn or a_scales.dtype != b_scales.dtype or a_scales.dtype not in _FP8_SCALES:
        raise RuntimeError(f"matmul_fp8: operands are float8_e4m3fn with scales both float8_e8m0fnu or both float32, got {a.dtype}, "
                           f"{a_scales.dtype}, {b.dtype}, {b_scales.dtype}")
    if b.shape[1] != K or a_scales.shape != (M, kb) or b_scales.shape != (-(-N // FP8_BLOCK), kb):
        raise RuntimeError(f"matmul_fp8: shapes do not go together: a {tuple(a.shape)} with scales {tuple(a_scales.shape)}, "
                           f"b {tuple(b.shape)} with scales {tuple(b_scales.shape)}")
    if out is None:
        out = torch.empty((M, N), dtype=dtype, device=a.device)
    elif out.shape != (M, N):
        raise RuntimeError(f"matmul_fp8: out must be {(M, N)}, got {tuple(out.shape)}")
    ld_out = _fp8_rows(what, out, "out")
    status = torch.zeros(64, dtype=torch.int32, device=a.device) if _attn._CHECK_STATUS else None
    with _nat.on_device(a.device):
        st = _nat.lib().mvpa_matmul_fp8(a.data_ptr(), ld_a, a_scales.data_ptr(), *a_scales.stride(), b.data_ptr(), ld_b,
                                        b_scales.data_ptr(), *b_scales.stride(), _FP8_SCALES[a_scales.dtype], out.data_ptr(), ld_out,
                                        M, N, K, _code(out), None if status is None else status.data_ptr(), _stream(a))
        _nat.check(st, "mvpa_matmul_fp8")
        if status is not None:  # debugging aid: synchronises the stream
            _nat.check(_nat.lib().mvpa_workspace_status(status.data_ptr(), 256, _stream(a)), "mvpa_matmul_fp8 kernel")
    return out


# ---- weights in 4 bits ----
# A weight (N, K) in 4 bits is (q, scales) or (q, scales, zeros): q (N, ceil(K / 2)) uint8, two values a byte, the first in its low
# half, whose rows start on 16-byte boundaries; scales (N, ceil(K / group)), one for each group of 32, 64 or 128 neighbours in a row;
# zeros, uint8 from 0 to 15, one for each scale.  It stands for (q - zero) * scale, zero = 8 where there are none.

INT4_GROUPS = (32, 64, 128)


def _int4_weight(what, q, scales, zeros, N, K, group):
    """The weight for the C entry points; N and K from its shape where they are None."""
    if group not in INT4_GROUPS:
        raise RuntimeError(f"{what}: group is 32, 64 or 128, got {group}")
    if q.dtype != torch.uint8 or scales.dtype not in (torch.bfloat16, torch.float32) or (zeros is not None and zeros.dtype != torch.uint8):
        raise RuntimeError(f"{what}: q and zeros are uint8, scales bfloat16 or float32, got {q.dtype}, {scales.dtype}"
                           + ("" if zeros is None else f", {zeros.dtype}"))
    ld_q, ld_s = _fp8_rows(what, q, "q"), _fp8_rows(what, scales, "scales")
    ld_z = 0 if zeros is None else _fp8_rows(what, zeros, "zeros")
    groups = -(-K // group)
    if q.shape != (N, (K + 1) // 2) or scales.shape != (N, groups) or (zeros is not None and zeros.shape != (N, groups)):
        raise RuntimeError(f"{what}: shapes do not go together: q {tuple(q.shape)}, scales {tuple(scales.shape)}"
                           + ("" if zeros is None else f", zeros {tuple(zeros.shape)}") + f" for {N} rows of {K} in groups of {group}")
    return _nat.Int4(q.data_ptr(), scales.data_ptr(), None if zeros is None else zeros.data_ptr(), ld_q, ld_s, ld_z)


def quantize_int4(w, group=128, zeros=False):
    """A weight w (N, K), bf16 or fp32, in 4 bits: (q, scales), or with `zeros` (q, scales, zeros); scales in w's type.  Without zeros
    scale = max|w| / 7 over a group, values -8 to 7; with them scale = (hi - lo) / 15 for lo = min(0, min w) and hi = max(0, max w), and
    the zero is -lo / scale, rounded.  Quotients are exact before they are rounded, halves to even.  A group whose scale rounds to zero
    stands for zeros, one that holds an infinity or a NaN has the scale NaN."""
    if _host.usable(w):
        made = _host.module().quantize_int4(w, group, zeros)
        if made is not None:
            return made
    what = "quantize_int4"
    _fp8_inputs(what, w)
    if group not in INT4_GROUPS:
        raise RuntimeError(f"{what}: group is 32, 64 or 128, got {group}")
    ld, (N, K) = _fp8_rows(what, w, "w"), w.shape
    half, groups = (K + 1) // 2, -(-K // group)
    q = torch.empty((N, (half + 15) // 16 * 16), dtype=torch.uint8, device=w.device)[:, :half]
    scales = torch.empty((N, groups), dtype=w.dtype, device=w.device)
    z = torch.empty((N, groups), dtype=torch.uint8, device=w.device) if zeros else None
    code = _code(w)
    with _nat.on_device(w.device):
        st = _nat.lib().mvpa_quantize_int4(w.data_ptr(), ld, ctypes.byref(_int4_weight(what, q, scales, z, N, K, group)), N, K, group, code,
                                           _stream(w))
    _nat.check(st, "mvpa_quantize_int4")
    return (q, scales, z) if zeros else (q, scales)


def dequantize_int4(q, scales, zeros=None, width=None, group=128, dtype=None):
    """The values (N, width) that a weight in 4 bits stands for, in `dtype` (the scales' type unless given).  `width` is K, which for an
    odd K the shape of q does not tell; 2 * q.shape[1] unless given."""
    if _host.usable(q) and (dtype is None or dtype is torch.bfloat16 or dtype is torch.float32):
        made = _host.module().dequantize_int4(q, scales, zeros, 2 * q.shape[-1] if width is None else width, group,
                                              scales.dtype is torch.float32 if dtype is None else dtype is torch.float32)
        if made is not None:
            return made
    what = "dequantize_int4"
    _fp8_inputs(what, q, scales, *(() if zeros is None else (zeros,)))
    if q.dim() != 2:
        raise RuntimeError(f"{what}: q must be a matrix, got shape {tuple(q.shape)}")
    N, K = q.shape[0], 2 * q.shape[1] if width is None else int(width)
    weight = _int4_weight(what, q, scales, zeros, N, K, group)
    out = torch.empty((N, K), dtype=scales.dtype if dtype is None else dtype, device=q.device)
    code = _code(out)
    with _nat.on_device(q.device):
        st = _nat.lib().mvpa_dequantize_int4(ctypes.byref(weight), _code(scales), out.data_ptr(), K, N, K, group, code, _stream(q))
    _nat.check(st, "mvpa_dequantize_int4")
    return out


def _int4_product(what, x, weight, up, group, out):
    tensors = [t for t in (*weight, *(() if up is None else up)) if t is not None]
    _fp8_inputs(what, x, *tensors, *(() if out is None else (out,)))
    if x.dim() == 0:
        raise RuntimeError(f"{what}: x must have a last dimension")
    K, N = x.shape[-1], weight[0].shape[0] if weight[0].dim() else 0
    x2 = x if x.dim() == 2 else x.reshape(-1, K)
    if x2.dim() == 2 and x2.stride(1) != 1 and K > 1:
        x2 = x2.contiguous()
    first = _int4_weight(what, *weight, *(() if len(weight) == 3 else (None,)), N, K, group)
    second = None if up is None else _int4_weight(what, *up, *(() if len(up) == 3 else (None,)), N, K, group)
    if up is not None and up[1].dtype != weight[1].dtype:
        raise RuntimeError(f"{what}: the scales of both weights are of one type, got {weight[1].dtype} and {up[1].dtype}")
    code, ld_x, M = _code(x), _fp8_rows(what, x2, "x"), x2.shape[0]
    made = out is None
    if made:
        out = torch.empty((M, N), dtype=x.dtype, device=x.device)
    elif out.shape != (M, N) or out.dtype != x.dtype:
        raise RuntimeError(f"{what}: out must be {(M, N)} {x.dtype}, got {tuple(out.shape)} {out.dtype}")
    ld_out = _fp8_rows(what, out, "out")
    lib = _nat.lib()
    with _nat.on_device(x.device):
        nbytes = lib.mvpa_matmul_int4_workspace_bytes(x2.data_ptr(), ld_x, M, K, code)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device) if nbytes else None
        status = _status_word(x.device)
        st = lib.mvpa_matmul_int4(x2.data_ptr(), ld_x, ctypes.byref(first), None if second is None else ctypes.byref(second),
                                  _code(weight[1]), out.data_ptr(), ld_out, M, N, K, group, code, None if ws is None else ws.data_ptr(),
                                  nbytes, None if status is None else status.data_ptr(), _stream(x))
        _nat.check(st, "mvpa_matmul_int4")
        _look_at(status, "mvpa_matmul_int4", x)
    return out.view(*x.shape[:-1], N) if made and x.dim() != 2 else out


def matmul_int4(x, q, scales, zeros=None, group=128, out=None):
    """x @ W.T for a weight W (N, K) in 4 bits and x (..., K), bf16 or fp32; the result in x's type, or in `out` (rows, N), which may be a
    column block of a wider buffer.  No weight is rounded: whole numbers are multiplied and added in fp32 over a group, the groups' sums
    scaled and added in fp32, rounded once."""
    if _host.usable(x):
        done = _host.module().matmul_int4(x, q, scales, zeros, None, None, None, group, out, _attn._CHECK_STATUS)
        if done is not None:
            return done if out is None else out
    return _int4_product("matmul_int4", x, (q, scales, zeros), None, group, out)


def gated_linear_int4(x, gate, up, group=128, out=None):
    """silu(x @ G.T) * (x @ U.T) for weights G and U (N, K) in 4 bits, `gate` and `up` each (q, scales) or (q, scales, zeros): `gated_linear`
    for inference, in one kernel, from x to the result in fp32 and rounded once."""
    what = "gated_linear_int4"
    if len(gate) not in (2, 3) or len(up) not in (2, 3):
        raise RuntimeError(f"{what}: gate and up are (q, scales) or (q, scales, zeros)")
    if _host.usable(x):
        done = _host.module().matmul_int4(x, *(gate if len(gate) == 3 else (*gate, None)), *(up if len(up) == 3 else (*up, None)), group, out,
                                          _attn._CHECK_STATUS)
        if done is not None:
            return done if out is None else out
    return _int4_product(what, x, tuple(gate), tuple(up), group, out)
