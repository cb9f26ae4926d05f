"""The 8-bit operators of the inference block as measurable cases: what turns rows and weights into e4m3 with a scale for each
block of 128 (quantisation, the norm with the residual's addition, the SwiGLU gate) and the matrix product that reads them.

A row in 8 bits is a pair (q, scales): q e4m3, one scale for each block of 128 neighbours in the row, the last block as long
as the row leaves it; a weight has one for each block of 128 x 128.  The operators' own scales are powers of two held as their
exponents (e8m0): for a block of values y

    scale = the smallest 2^e, e >= -126, with max|y| <= 448 * 2^e,    q = e4m3(y / scale),    the pair stands for q * scale,

so that the division is exact and nothing but the step to e4m3 rounds.  The matrix product takes fp32 scales as well.

Sizes come from the shipped architectures (MVPFormer-S: width 768, 4 kv heads of 64, gate 1728; the generative model: width
2048, 8 kv heads of 128, gate 5632), whose fused projections are N x K = 4736 x 768 and 768 x 2496, 15360 x 2048 and
2048 x 7680, and from the token counts of one live window up to several long recordings.
"""
from __future__ import annotations

import math

import torch

own = False

BLOCK = 128
TOP = 448.0                  # largest e4m3 value
LOWEST = -126                # exponent of the smallest scale, the smallest normal fp32
EPS = 1e-5
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # the attention output of a six-segment window of a 22-channel patient, before the output projection
        dict(name="rows_window", kind="quantize", dtype="bf16", rows=132, width=768, block_rows=1),
        # the attention output of 16384 tokens of the generative model
        dict(name="rows_16k", kind="quantize", dtype="bf16", rows=16384, width=2048, block_rows=1),
        # the fused projection weight of a generative block, quantised when a checkpoint is loaded
        dict(name="weight_load", kind="quantize", dtype="fp32", rows=15360, width=2048, block_rows=128),
        # the first block of one segment of a 22-channel patient: no residual branch yet
        dict(name="norm_segment", kind="norm", dtype="bf16", rows=22, width=768, add=False),
        # a batch of long recordings through MVPFormer-S, residual added on the way
        dict(name="norm_batch", kind="norm", dtype="bf16", rows=65536, width=768, add=True),
        # an fp32 residual stream of odd width (the wavelet row of a segment of 1000 samples)
        dict(name="norm_odd", kind="norm", dtype="fp32", rows=2500, width=1027, add=True),
        # the gate of MVPFormer-S over the loader's window of a batch: rows of thirteen and a half blocks
        dict(name="gate_s", kind="gate", dtype="bf16", rows=6400, width=1728),
        # the gate of the generative model over two long samples
        dict(name="gate_generative", kind="gate", dtype="bf16", rows=32768, width=5632),
        # one token through the fused projection of the generative model: bound by the weight's bytes
        dict(name="matmul_token", kind="matmul", out="bf16", M=1, N=15360, K=2048, given=False),
        # one live window (25 segments x 22 channels) through the output projection of MVPFormer-S: a ragged last block
        dict(name="matmul_window", kind="matmul", out="bf16", M=550, N=768, K=2496, given=False),
        # 16384 tokens through the fused projection of the generative model
        dict(name="matmul_in", kind="matmul", out="bf16", M=16384, N=15360, K=2048, given=False),
        # two long samples through its output projection, with fp32 scales that another quantiser made
        dict(name="matmul_out", kind="matmul", out="bf16", M=32768, N=2048, K=7680, given=True),
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], spread over its logarithm; odd values come as they fall."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["quantize", "norm", "gate", "matmul", "matmul", "matmul"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
    if kind == "quantize":
        width = rng.choice([768, 2048, _log(rng, 16, 8192)])
        if rng.random() < 0.3:
            return dict(kind=kind, dtype=dtype, rows=_log(rng, 64, 15360), width=width, block_rows=128)
        return dict(kind=kind, dtype=dtype, rows=_log(rng, 1, 65536 * 768 // width), width=width, block_rows=1)
    if kind == "norm":
        width = rng.choice([768, 2048, _log(rng, 16, 2048)])
        return dict(kind=kind, dtype=dtype, rows=_log(rng, 1, 65536 * 768 // width), width=width, add=rng.random() < 0.7)
    if kind == "gate":
        width = rng.choice([1728, 5632, _log(rng, 16, 8192)])
        return dict(kind=kind, dtype=dtype, rows=_log(rng, 1, min(65536, 32768 * 2816 // width)), width=width)
    N, K = rng.choice([(4736, 768), (768, 2496), (15360, 2048), (2048, 7680), (_log(rng, 16, 8192), _log(rng, 16, 8192)),
                       (_log(rng, 16, 8192), _log(rng, 16, 8192))])
    return dict(kind=kind, out=rng.choice(["bf16", "bf16", "bf16", "fp32"]), M=_log(rng, 1, min(65536, 16384 * 15360 * 2048 // (N * K))),
                N=N, K=K, given=rng.random() < 0.5)


# ---- the plain forms: elementary torch operations in 32 bits ----

def _in_blocks(y, block_rows):
    """(rows, width) -> (row blocks, block_rows, column blocks, BLOCK), zeros where the last blocks have nothing."""
    rows, width = y.shape
    y = torch.nn.functional.pad(y, (0, -width % BLOCK, 0, -rows % block_rows))
    return y.view(-1, block_rows, y.shape[1] // BLOCK, BLOCK)


def _quantize(y, block_rows):
    """(q, scales) of a matrix in fp32; q keeps the matrix' shape."""
    rows, width = y.shape
    blocks = _in_blocks(y, block_rows)
    mantissa, exponent = torch.frexp(blocks.abs().amax(dim=(1, 3)))       # largest = mantissa * 2^exponent, mantissa in [0.5, 1)
    exponent = (exponent - 9 + (mantissa > 0.875)).clamp(min=LOWEST)      # 448 = 0.875 * 2^9
    scales = torch.ldexp(torch.ones_like(mantissa), exponent)
    q = (blocks / scales[:, None, :, None]).to(torch.float8_e4m3fn)
    return q.view(blocks.shape[0] * block_rows, -1)[:rows, :width].contiguous(), scales.to(torch.float8_e8m0fnu)


def _stands_for(q, scales, block_rows):
    """The matrix that a pair stands for, in fp32."""
    wide = scales.float().repeat_interleave(BLOCK, dim=1)[:, :q.shape[1]]
    return q.float() * wide.repeat_interleave(block_rows, dim=0)[:q.shape[0]]


def _plain(state):
    case = state["case"]
    kind = case["kind"]
    if kind == "quantize":
        return _quantize(state["x"].float(), case["block_rows"])
    if kind == "norm":
        h = state["x"] if state["add"] is None else (state["x"].float() + state["add"].float()).to(state["x"].dtype)
        hf = h.float()
        rstd = torch.rsqrt((hf * hf).mean(dim=1, keepdim=True) + EPS)
        q, scales = _quantize(hf * rstd * state["weight"].float(), 1)
        return (q, scales) if state["add"] is None else (q, scales, h)
    if kind == "gate":
        g, u = state["gate"].float(), state["up"].float()
        return _quantize(g / (1.0 + torch.exp(-g)) * u, 1)
    a = _stands_for(state["a"], state["a_scales"], 1)
    b = _stands_for(state["b"], state["b_scales"], BLOCK)
    return (a @ b.t()).to(TYPES[case["out"]])


# ---- inputs ----

def _randn(gen, rows, width, device):
    return torch.randn((rows, width), generator=gen, device=device)


def _padded(q):
    """The same e4m3 matrix with rows that start on 16-byte boundaries, as the operators write them."""
    rows, width = q.shape
    wide = torch.zeros((rows, (width + 15) // 16 * 16), dtype=q.dtype, device=q.device)
    wide[:, :width] = q
    return wide[:, :width]


def prepare(case, seed):
    device = torch.device("cuda")
    gen = torch.Generator(device=device)
    gen.manual_seed(int(seed))
    kind = case["kind"]
    if kind == "matmul":
        M, N, K = case["M"], case["N"], case["K"]
        # activations: rows of different sizes and a few channels that stand out; weights as they are initialised
        x = _randn(gen, M, K, device) * torch.exp(0.5 * _randn(gen, M, 1, device))
        x *= torch.where(torch.rand((1, K), generator=gen, device=device) < 0.01, 20.0, 1.0)
        w = _randn(gen, N, K, device) * 0.02
        (a, sa), (b, sb) = _quantize(x, 1), _quantize(w, BLOCK)
        if case["given"]:      # scales from elsewhere: any numbers in fp32, up to twice what a block needs
            sa = sa.float() * (1.0 + torch.rand(sa.shape, generator=gen, device=device))
            sb = sb.float() * (1.0 + torch.rand(sb.shape, generator=gen, device=device))
            a = (x / sa.repeat_interleave(BLOCK, dim=1)[:, :K]).to(torch.float8_e4m3fn)
            b = (w / sb.repeat_interleave(BLOCK, dim=1)[:, :K].repeat_interleave(BLOCK, dim=0)[:N]).to(torch.float8_e4m3fn)
        return {"case": case, "a": _padded(a), "a_scales": sa, "b": _padded(b), "b_scales": sb}
    dtype, rows, width = TYPES[case["dtype"]], case["rows"], case["width"]
    if kind == "quantize":
        spread = 0.02 if case["block_rows"] == BLOCK else 1.0
        return {"case": case, "x": (_randn(gen, rows, width, device) * spread).to(dtype)}
    if kind == "norm":
        # a residual stream with channels that stand out, and the branch sum of the block before
        x = _randn(gen, rows, width, device) * torch.exp(0.7 * _randn(gen, 1, width, device))
        add = (0.3 * _randn(gen, rows, width, device)).to(dtype) if case["add"] else None
        weight = (1.0 + 0.1 * _randn(gen, 1, width, device))[0].to(dtype)
        x = x.to(dtype)
        return {"case": case, "x": x, "add": add, "weight": weight, "h": torch.empty_like(x) if case["add"] else None}
    # gate and up are neighbouring column blocks of one projection's output
    both = torch.empty((rows, 2 * width), dtype=dtype, device=device)
    both[:, :width] = _randn(gen, rows, width, device) * 1.5
    both[:, width:] = _randn(gen, rows, width, device)
    return {"case": case, "gate": both[:, :width], "up": both[:, width:]}


def run(state):
    if not own:
        return _plain(state)
    ops = _operators()
    case = state["case"]
    if case["kind"] == "quantize":
        return ops.quantize_fp8(state["x"], block_rows=case["block_rows"])
    if case["kind"] == "norm":
        q, scales = ops.rmsnorm_fp8(state["x"], state["weight"], EPS, add=state["add"], sum_out=state["h"])
        return (q, scales) if state["add"] is None else (q, scales, state["h"])
    if case["kind"] == "gate":
        return ops.silu_mul_fp8(state["gate"], state["up"])
    return ops.matmul_fp8(state["a"], state["a_scales"], state["b"], state["b_scales"], dtype=TYPES[case["out"]])


_ops = None


def _operators():
    """The framework's operators, as a user imports them."""
    global _ops
    if _ops is None:
        import importlib
        importlib.import_module("multi-variate-parallel-transformer_b200")   # puts the package's folders on sys.path
        _ops = importlib.import_module("mvpa_ops")
    return _ops


def work(case):
    kind = case["kind"]
    if kind == "matmul":
        M, N, K = case["M"], case["N"], case["K"]
        kb = -(-K // BLOCK)
        return {"bytes": (M + N) * K + (4 if case["given"] else 1) * kb * (M + -(-N // BLOCK)) + (2 if case["out"] == "bf16" else 4) * M * N,
                "flops": 2.0 * M * N * K}
    es, rows, width = (2 if case["dtype"] == "bf16" else 4), case["rows"], case["width"]
    n, blocks = rows * width, -(-width // BLOCK) * -(-rows // case.get("block_rows", 1))
    out = n + blocks
    if kind == "quantize":
        return {"bytes": es * n + out, "flops": 3.0 * n}
    if kind == "norm":
        return {"bytes": es * (n * (3 if case["add"] else 1) + width) + out, "flops": (8.0 if case["add"] else 7.0) * n}
    return {"bytes": 2 * es * n + out, "flops": 7.0 * n}


# ---- the definitions in 64 bits ----

def _e4m3(v):
    """Nearest e4m3 value, ties to even: three mantissa bits down to 2^-6, steps of 2^-9 below."""
    _, exponent = torch.frexp(v)                              # |v| in [2^(exponent - 1), 2^exponent)
    step = torch.ldexp(torch.ones_like(v), (exponent - 1).clamp(min=-6) - 3)
    return (torch.round(v / step) * step).clamp(-TOP, TOP)


def _exact_pair(y, tall):
    rows, width = y.shape
    q = torch.empty_like(y)
    down, across = -(-rows // tall), -(-width // BLOCK)
    scales = torch.empty((down, across), dtype=y.dtype, device=y.device)
    for c in range(across):
        part = y[:, c * BLOCK:(c + 1) * BLOCK]
        top = part.abs().max(dim=1).values
        top = torch.cat([top, top.new_zeros(down * tall - rows)]).view(down, tall).max(dim=1).values
        scales[:, c] = torch.exp2(torch.ceil(torch.log2(top / TOP)).clamp(min=LOWEST))
        q[:, c * BLOCK:(c + 1) * BLOCK] = _e4m3(part / scales[:, c].repeat_interleave(tall)[:rows, None])
    return q, scales


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "quantize":
        return _exact_pair(s["x"].double(), case["block_rows"])
    if kind == "norm":
        h = s["x"].double()
        if s["add"] is not None:
            h = (h + s["add"].double()).to(s["x"].dtype).double()      # the residual stream is held in its own type
        y = h / torch.sqrt(h.square().sum(dim=1, keepdim=True) / case["width"] + EPS) * s["weight"].double()
        pair = _exact_pair(y, 1)
        return pair if s["add"] is None else (*pair, h)
    if kind == "gate":
        g = s["gate"].double()
        return _exact_pair(g * torch.sigmoid(g) * s["up"].double(), 1)
    K = case["K"]
    a = s["a"].double() * s["a_scales"].double()[:, torch.arange(K, device="cuda") // BLOCK]
    b = s["b"].double() * s["b_scales"].double()[torch.arange(case["N"], device="cuda") // BLOCK][:, torch.arange(K, device="cuda") // BLOCK]
    return torch.matmul(a, b.t())
