"""The gated projection of the MLP, for training and for inference, and the block's projections with weights in 4 bits, as
measurable cases.

gated     h = silu(x Wg^T) * (x Wu^T) for x (M, E), Wg and Wu (I, E), all bf16; a training step adds the gradients of x, Wg and Wu
          for an incoming dh:  with g = x Wg^T, u = x Wu^T, s = 1 / (1 + e^-g),
          dg = dh u s (1 + g (1 - s)),  du = dh g s,   dx = dg Wg + du Wu,  dWg = dg^T x,  dWu = du^T x.
quantize  a weight (N, K) in 4 bits and back: the K values of a row in groups of 32, 64 or 128 neighbours (the last one as long as the
          row leaves it) with one scale each, in the weight's type.  Without zeros a group y has
              scale = max|y| / 7 rounded to the type,   q = 8 + clamp(round(y / scale), -8, 7)     standing for (q - 8) scale,
          with zeros, for lo = min(0, min y) and hi = max(0, max y),
              scale = (hi - lo) / 15 rounded to the type,  z = clamp(round(-lo / scale), 0, 15),  q = clamp(round(y / scale) + z, 0, 15)
          standing for (q - z) scale; halves round to even, and a group whose scale rounds to zero stands for zeros.
          Two values share a byte, the first one in its low half; rows of bytes start on 16-byte boundaries.
matmul4   x W^T for x (M, K) in bf16 or fp32 and such a weight W.
gate4     silu(x Wg^T) * (x Wu^T) for such weights.

Sizes come from the shipped architectures (MVPFormer-S: width 768, 4 kv heads of 64, gate 1728; the generative model: width
2048, 8 kv heads of 128, gate 5632), whose fused projections are N x K = 4736 x 768 and 768 x 2496, 15360 x 2048 and
2048 x 7680, and from the token counts of one segment up to several long recordings.
"""
from __future__ import annotations

import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # one new segment of a 22-channel patient through the gate of MVPFormer-S
        dict(name="gated_segment", kind="gated", M=22, E=768, I=1728, train=False),
        # a long recording through the gate of the generative model
        dict(name="gated_recording", kind="gated", M=16384, E=2048, I=5632, train=False),
        # a training step of MVPFormer-S on a batch of the loader's windows
        dict(name="gated_train_s", kind="gated", M=6400, E=768, I=1728, train=True),
        # a training step of the generative model on a long recording
        dict(name="gated_train_generative", kind="gated", M=16384, E=2048, I=5632, train=True),
        # a training step with sizes that fill no tile
        dict(name="gated_train_ragged", kind="gated", M=2501, E=1000, I=1368, train=True),
        # the fused projection of a generative block, quantised when a checkpoint is loaded
        dict(name="weight_load", kind="quantize", dtype="bf16", N=15360, K=2048, group=128, zeros=False),
        # the output projection of MVPFormer-S with small groups and zeros, from an fp32 checkpoint
        dict(name="weight_zeros", kind="quantize", dtype="fp32", N=768, K=2496, group=32, zeros=True),
        # one token through the fused projection of the generative model: bound by the weight's bytes
        dict(name="int4_token", kind="matmul4", dtype="bf16", M=1, N=15360, K=2048, group=128, zeros=False),
        # one live window (25 segments x 22 channels) through the output projection of MVPFormer-S
        dict(name="int4_window", kind="matmul4", dtype="bf16", M=550, N=768, K=2496, group=64, zeros=True),
        # four live windows at once through the fused projection of the generative model
        dict(name="int4_windows", kind="matmul4", dtype="bf16", M=2200, N=15360, K=2048, group=128, zeros=False),
        # one new segment of a 22-channel patient through the gate of the generative model
        dict(name="gate4_segment", kind="gate4", dtype="bf16", M=22, N=5632, K=2048, group=128, zeros=False),
        # an fp32 model of odd sizes, its weights from another quantiser
        dict(name="gate4_odd", kind="gate4", dtype="fp32", M=133, N=1001, K=1027, group=32, zeros=True),
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], spread over its logarithm; odd values come as they fall."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["gated", "gated", "quantize", "matmul4", "matmul4", "gate4"])
    if kind == "gated":
        E, I = rng.choice([(768, 1728), (2048, 5632), (8 * _log(rng, 1, 256), 8 * _log(rng, 1, 704))])
        return dict(kind=kind, M=_log(rng, 1, min(65536, 16384 * 2048 * 5632 // (E * I))), E=E, I=I, train=rng.random() < 0.6)
    dtype, group, zeros = rng.choice(["bf16", "bf16", "fp32"]), rng.choice([32, 64, 128, 128]), rng.random() < 0.4
    if kind == "quantize":
        N, K = rng.choice([(4736, 768), (768, 2496), (15360, 2048), (2048, 7680), (_log(rng, 1, 8192), _log(rng, 1, 8192))])
        return dict(kind=kind, dtype=dtype, N=N, K=K, group=group, zeros=zeros)
    if kind == "matmul4":
        N, K = rng.choice([(4736, 768), (768, 2496), (15360, 2048), (2048, 7680), (_log(rng, 16, 8192), _log(rng, 16, 8192))])
        return dict(kind=kind, dtype=dtype, M=_log(rng, 1, 2200), N=N, K=K, group=group, zeros=zeros)
    N, K = rng.choice([(1728, 768), (5632, 2048), (_log(rng, 16, 5632), _log(rng, 16, 4096))])
    return dict(kind=kind, dtype=dtype, M=_log(rng, 1, 2200), N=N, K=K, group=group, zeros=zeros)


# ---- the plain forms: elementary torch operations in 32 bits (the rounding to 4 bits in 64: values lie next to its borders) ----

def _quantize(w, group, zeros):
    """(q, scales[, zeros]) of a matrix: q packed, scales in its type, zeros uint8."""
    N, K = w.shape
    y = torch.nn.functional.pad(w.double(), (0, -K % group)).view(N, -1, group)
    if zeros:
        lo, hi = y.amin(2).clamp(max=0), y.amax(2).clamp(min=0)
        scales = ((hi - lo) / 15).to(w.dtype)
    else:
        scales = (y.abs().amax(2) / 7).to(w.dtype)
    s = scales.double()
    some = s > 0
    steps = torch.round(y / torch.where(some, s, 1.0)[..., None]) * some[..., None]
    if zeros:
        z = torch.round(-lo / torch.where(some, s, 1.0)).clamp(0, 15) * some
        q = (steps + z[..., None]).clamp(0, 15)
    else:
        q = steps.clamp(-8, 7) + 8
    q = q.to(torch.uint8).view(N, -1)[:, :K]
    q = torch.nn.functional.pad(q, (0, K % 2))
    packed = torch.zeros((N, (q.shape[1] // 2 + 15) // 16 * 16), dtype=torch.uint8, device=w.device)[:, :q.shape[1] // 2]
    packed.copy_(q[:, 0::2] | (q[:, 1::2] << 4))
    return (packed, scales, z.to(torch.uint8)) if zeros else (packed, scales)


def _stands_for(pair, K, group):
    """The matrix that a pair (or a triple) stands for, in fp32."""
    q = torch.stack((pair[0] & 15, pair[0] >> 4), dim=2).view(pair[0].shape[0], -1)[:, :K].float()
    wide = lambda t: t.float().repeat_interleave(group, dim=1)[:, :K]
    return (q - (wide(pair[2]) if len(pair) == 3 else 8.0)) * wide(pair[1])


def _silu(g):
    return g / (1.0 + torch.exp(-g))


def _plain(state):
    case = state["case"]
    kind = case["kind"]
    if kind == "quantize":
        w = state["w"]
        pair = _quantize(w, case["group"], case["zeros"])
        return (_stands_for(pair, case["K"], case["group"]).to(w.dtype), *pair[1:])
    x = state["x"].float()
    if kind == "matmul4":
        return (x @ _stands_for(state["w"], case["K"], case["group"]).t()).to(state["x"].dtype)
    if kind == "gate4":
        g, u = (x @ _stands_for(state[n], case["K"], case["group"]).t() for n in ("w_gate", "w_up"))
        return (_silu(g) * u).to(state["x"].dtype)
    wg, wu = state["w_gate"].detach().float(), state["w_up"].detach().float()
    x = x.detach()
    g, u = x @ wg.t(), x @ wu.t()
    h = (_silu(g) * u).to(torch.bfloat16)
    if not case["train"]:
        return h
    dh, s = state["dh"].float(), 1.0 / (1.0 + torch.exp(-g))
    dg, du = dh * u * (s * (1.0 + g * (1.0 - s))), dh * (g * s)
    return h, (dg @ wg + du @ wu).to(torch.bfloat16), (dg.t() @ x).to(torch.bfloat16), (du.t() @ x).to(torch.bfloat16)


# ---- inputs ----

def prepare(case, seed):
    device = torch.device("cuda")
    gen = torch.Generator(device=device)
    gen.manual_seed(int(seed))
    randn = lambda rows, width: torch.randn((rows, width), generator=gen, device=device)
    kind = case["kind"]
    if kind == "gated":
        # the norm's output: rows of unit size with channels that stand out; weights whose products have the size of real gates
        M, E, I = case["M"], case["E"], case["I"]
        x = (randn(M, E) * torch.exp(0.5 * randn(1, E))).to(torch.bfloat16)
        wg, wu = ((randn(I, E) * E ** -0.5).to(torch.bfloat16) for _ in range(2))
        state = {"case": case, "x": x, "w_gate": wg, "w_up": wu}
        if case["train"]:
            state["dh"] = (randn(M, I) * 0.1).to(torch.bfloat16)
            for name in ("x", "w_gate", "w_up"):
                state[name].requires_grad_()
        return state
    dtype, group, N, K = TYPES[case["dtype"]], case["group"], case["N"], case["K"]
    weight = lambda: (randn(N, K) * torch.exp(0.3 * randn(N, 1)) * K ** -0.5).to(dtype)
    if kind == "quantize":
        return {"case": case, "w": weight()}
    x = (randn(case["M"], K) * torch.exp(0.5 * randn(case["M"], 1)) * torch.exp(0.5 * randn(1, K))).to(dtype)
    if kind == "matmul4":
        return {"case": case, "x": x, "w": _quantize(weight(), group, case["zeros"])}
    return {"case": case, "x": x, "w_gate": _quantize(weight(), group, case["zeros"]), "w_up": _quantize(weight(), group, case["zeros"])}


# ---- a pass ----

def _ops():
    import importlib
    import os
    import sys
    package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "multi-variate-parallel-transformer_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    return importlib.import_module("mvpa_ops")


_loaded = None


def run(state):
    global _loaded
    if not own:
        return _plain(state)
    if _loaded is None:
        _loaded = _ops()
    case = state["case"]
    kind = case["kind"]
    if kind == "gated":
        x, wg, wu = state["x"], state["w_gate"], state["w_up"]
        h = _loaded.gated_linear(x, wg, wu)
        return (h.detach(), *torch.autograd.grad(h, (x, wg, wu), state["dh"])) if case["train"] else h
    if kind == "quantize":
        w = state["w"]
        pair = _loaded.quantize_int4(w, group=case["group"], zeros=case["zeros"])
        return (_loaded.dequantize_int4(*pair, width=case["K"], group=case["group"]), *pair[1:])
    if kind == "matmul4":
        return _loaded.matmul_int4(state["x"], *state["w"], group=case["group"])
    return _loaded.gated_linear_int4(state["x"], state["w_gate"], state["w_up"], group=case["group"])


def work(case):
    kind = case["kind"]
    if kind == "gated":
        M, E, I = case["M"], case["E"], case["I"]
        once = {"bytes": 2 * (M * E + 2 * I * E + M * I), "flops": 4 * M * E * I}
        if not case["train"]:
            return once
        return {"bytes": once["bytes"] + 2 * (M * I + M * E + 2 * I * E), "flops": 3 * once["flops"]}
    size, N, K = 2 if case["dtype"] == "bf16" else 4, case["N"], case["K"]
    groups = N * -(-K // case["group"])
    packed = N * -(-K // 2) + groups * (size + case["zeros"])
    if kind == "quantize":
        return {"bytes": 2 * size * N * K + packed, "flops": 4 * N * K}
    M = case["M"]
    if kind == "matmul4":
        return {"bytes": packed + size * M * (K + N), "flops": 2 * M * N * K}
    return {"bytes": 2 * packed + size * M * (K + N), "flops": 4 * M * N * K}


# ---- the definition in 64 bits, on its own ----

def _exact_weight(pair, K, group):
    q, scales = pair[0].to(torch.int64), pair[1].double()
    column = torch.arange(K, device=q.device)
    value = (q[:, column // 2] >> (4 * (column % 2))) & 15
    zero = pair[2].to(torch.int64)[:, column // group] if len(pair) == 3 else 8
    return (value - zero).double() * scales[:, column // group]


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "quantize":
        w, group, N, K = s["w"].double(), case["group"], case["N"], case["K"]
        groups = -(-K // group)
        values = torch.empty_like(w)
        scales = torch.empty((N, groups), dtype=torch.float64, device=w.device)
        z = torch.empty((N, groups), dtype=torch.uint8, device=w.device)
        for j in range(groups):
            part = w[:, j * group:(j + 1) * group]
            low, high = part.min(1).values, part.max(1).values
            if case["zeros"]:
                low, high = torch.minimum(low, torch.zeros_like(low)), torch.maximum(high, torch.zeros_like(high))
                scale = ((high - low) / 15).to(s["w"].dtype).double()
            else:
                scale = (torch.maximum(-low, high) / 7).to(s["w"].dtype).double()
            scales[:, j] = scale
            safe = torch.where(scale == 0, torch.ones_like(scale), scale)
            steps = torch.round(part / safe[:, None])
            if case["zeros"]:
                zero = torch.clamp(torch.round(-low / safe), 0, 15)
                z[:, j] = torch.where(scale == 0, torch.zeros_like(zero), zero).to(torch.uint8)
                steps = torch.clamp(steps + zero[:, None], 0, 15) - zero[:, None]
            else:
                steps = torch.clamp(steps, -8, 7)
            values[:, j * group:(j + 1) * group] = steps * scale[:, None]
        return (values, scales, z) if case["zeros"] else (values, scales)
    x = s["x"].detach().double()
    if kind == "matmul4":
        return torch.matmul(x, _exact_weight(s["w"], case["K"], case["group"]).t())
    if kind == "gate4":
        g, u = (torch.matmul(x, _exact_weight(s[n], case["K"], case["group"]).t()) for n in ("w_gate", "w_up"))
        return g * torch.sigmoid(g) * u
    wg, wu = s["w_gate"].detach().double(), s["w_up"].detach().double()
    g, u = torch.matmul(x, wg.t()), torch.matmul(x, wu.t())
    sig = torch.sigmoid(g)
    h = g * sig * u
    if not case["train"]:
        return h
    dh = s["dh"].double()
    du = dh * g * sig
    dg = dh * u * sig * (1 + g - g * sig)
    return h, torch.matmul(dg, wg) + torch.matmul(du, wu), torch.matmul(dg.t(), x), torch.matmul(du.t(), x)
