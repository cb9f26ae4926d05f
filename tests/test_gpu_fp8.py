"""GPU: the 8-bit operators (quantisation, norm, gate, matrix product) against their definitions in 64 bits, at the sizes,
layouts and values where they can go wrong, and what they refuse."""
import pytest
import torch

import fp8_oracle as ref
import mvpa_ops as ops

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
EPS = 1e-5


def _gen(*key):
    return torch.Generator().manual_seed(hash(key) % (1 << 30))


def _randn(g, *shape, dtype=F32):
    return torch.randn(*shape, generator=g).to(dtype).cuda()


# ---- quantisation: no arithmetic before the step to e4m3, so it is the definition's, bit for bit ----

@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("block", [1, 128])
@pytest.mark.parametrize("rows,width", [(1, 1), (1, 16), (3, 127), (2, 128), (5, 129), (7, 768), (130, 1000), (128, 2496), (257, 2049)])
def test_quantize(cuda, dtype, block, rows, width):
    g = _gen(rows, width, block)
    x = (_randn(g, rows, width) * torch.exp(2 * _randn(g, rows, 1))).to(dtype)
    q, s = ops.quantize_fp8(x, block_rows=block)
    q64, s64 = ref.pair(x, block)
    assert torch.equal(s.double(), s64) and torch.equal(q.double(), q64)
    assert q.stride(0) % 16 == 0 or rows == 1


@pytest.mark.parametrize("block", [1, 128])
def test_quantize_borders(cuda, block):
    """Largest values on both sides of 448 * 2^e, ties, the smallest and largest numbers, a block of zeros."""
    top = [448.0, 448.00003, 447.99997, 1.75, 1.7500001, 3.4e38, 2.0 ** -126, 1e-40, 0.0, 1.4e-45, 2.0 ** -119 * 1.75, 1.0]
    x = torch.zeros(len(top) * (1 if block == 1 else 128), 256)
    step = 1 if block == 1 else 128
    for i, t in enumerate(top):
        x[i * step, 0] = t
        x[i * step, 1:100] = torch.linspace(-1, 1, 99) * t
        x[i * step, 100:120] = -t * torch.tensor([17 / 448 * (k + 0.5) for k in range(20)])     # halves between two steps among them
        x[i * step, 128] = -t
    x = x.cuda()
    q, s = ops.quantize_fp8(x, block_rows=block)
    q64, s64 = ref.pair(x, block)
    assert torch.equal(s.double(), s64) and torch.equal(q.double(), q64)


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("block", [1, 128])
def test_quantize_not_finite(cuda, bad, dtype, block):
    x = _randn(_gen(1), 140, 300, dtype=dtype)
    x[2, 130] = bad
    q, s = ops.quantize_fp8(x, block_rows=block)
    hit = torch.zeros(140, 300, dtype=torch.bool, device="cuda")
    hit[2 if block == 1 else slice(0, 128), 128:256] = True
    assert bool(q.float().isnan().eq(hit).all())
    assert int(s.float().isnan().sum()) == 1 and bool(s.float()[2 if block == 1 else 0, 1].isnan())
    good, _ = ops.quantize_fp8(torch.where(hit, torch.zeros_like(x), x), block_rows=block)
    assert torch.equal(q.float()[~hit], good.float()[~hit])


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("offset,ld", [(0, 300), (1, 301), (3, 304), (8, 320)])
def test_quantize_strided_in_and_out(cuda, dtype, offset, ld):
    """Rows at any alignment in; a column block of wider buffers out, whose other bytes stay as they were."""
    rows, width = 37, 200
    buf = _randn(_gen(offset, ld), rows, ld, dtype=dtype)
    x = buf[:, offset:offset + width]
    q_all = torch.full((rows + 2, 512), 7, dtype=torch.uint8, device="cuda")
    s_all = torch.full((rows + 2, 9), 9, dtype=torch.uint8, device="cuda")
    q, s = q_all[1:rows + 1, 128:128 + width].view(torch.float8_e4m3fn), s_all[1:rows + 1, 3:5].view(torch.float8_e8m0fnu)
    ops.quantize_fp8(x, out=(q, s))
    q64, s64 = ref.pair(x)
    assert torch.equal(q.double(), q64) and torch.equal(s.double(), s64)
    q_all[1:rows + 1, 128:128 + width] = 7
    s_all[1:rows + 1, 3:5] = 9
    assert bool((q_all == 7).all()) and bool((s_all == 9).all())


# ---- norm ----

def _norm64(h, w):
    h = h.double()
    return h * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS) * w.double()


@pytest.mark.parametrize("add", [None, "out", "in_place"])
@pytest.mark.parametrize("dtype,rows,width", [(BF16, 1, 8), (BF16, 1, 1), (BF16, 9, 768), (BF16, 300, 770), (BF16, 33, 4096), (BF16, 5, 512),
                                              (BF16, 6, 513), (BF16, 1000, 2048), (F32, 7, 4), (F32, 250, 1027), (F32, 40, 2048), (F32, 3, 129)])
def test_norm(cuda, dtype, rows, width, add):
    g = _gen(rows, width, (None, "out", "in_place").index(add))
    x, a = _randn(g, rows, width, dtype=dtype) * 3, _randn(g, rows, width, dtype=dtype)
    w = (1 + 0.1 * _randn(g, width)).to(dtype)
    if add is None:
        h = x
        q, s = ops.rmsnorm_fp8(x, w, EPS)
    else:
        h = (x.double() + a.double()).to(dtype)
        x, before = x.clone(), x
        out = x if add == "in_place" else torch.empty_like(x)
        q, s = ops.rmsnorm_fp8(x, w, EPS, add=a, sum_out=out)
        # the sum of two numbers in fp32 and then in `dtype`: the nearest one, but for double roundings
        assert torch.equal(out, (before.float() + a.float()).to(dtype))
        h = out
    # a chain of width / 32 squares a lane, rounded up to sixteens, and five more sums (halved by the root), rsqrtf within
    # two units (2^-22), the mean's division, two products
    eps = ((width / 32 + 16 + 5) / 2 + 4 + 3) * 2.0 ** -24
    ref.check_pair(q, s, _norm64(h, w), eps)


def test_norm_leading_dimensions_and_empty(cuda):
    x, w = _randn(_gen(3), 2, 3, 5, 64), _randn(_gen(4), 64)
    q, s = ops.rmsnorm_fp8(x, w, EPS)
    q2, s2 = ops.rmsnorm_fp8(x.view(30, 64), w, EPS)
    assert q.shape == (30, 64) and torch.equal(q.float(), q2.float()) and torch.equal(s.float(), s2.float())
    q, s = ops.rmsnorm_fp8(x[:0], w, EPS)
    assert q.shape == (0, 64) and s.shape == (0, 1)
    q, s = ops.quantize_fp8(x.view(30, 64)[:, :0])
    assert q.shape == (30, 0) and s.shape == (30, 0)
    q, s = ops.silu_mul_fp8(x.view(30, 64)[:0], x.view(30, 64)[:0])
    assert q.shape == (0, 64)


def test_norm_rows_that_are_zero_or_not_finite(cuda):
    x = _randn(_gen(5), 40, 200)
    x[3], x[4, 7], x[5, 199] = 0, float("inf"), float("nan")
    q, s = ops.rmsnorm_fp8(x, torch.ones(200, device="cuda"), EPS)
    bad = q.float().isnan() | s.float().isnan().repeat_interleave(128, 1)[:, :200]
    assert bool(bad[5].all()) and bool(bad[4, :128].all())
    assert bool((q.float()[3] == 0).all()) and not bool(s.float()[3].isnan().any())
    rest = [i for i in range(40) if i not in (3, 4, 5)]
    assert not bool(bad[rest].any())
    ref.check_pair(q[rest], s[rest], _norm64(x[rest], torch.ones(200, device="cuda")), 40 * 2.0 ** -24)


# ---- gate ----

def _gate64(g, u):
    g = g.double()
    return g * torch.sigmoid(g) * u.double()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,width,ld", [(1, 16, 32), (1, 7, 14), (5, 128, 256), (33, 1728, 4736), (100, 1001, 2002), (7, 5632, 11264)])
def test_gate(cuda, dtype, rows, width, ld):
    buf = _randn(_gen(rows, width), rows, ld, dtype=dtype) * 2
    gate, up = buf[:, ld - 2 * width:ld - width], buf[:, ld - width:]
    q, s = ops.silu_mul_fp8(gate, up)
    # expf within two units (2^-22), then a sum, a quotient and a product of half a unit (2^-24) each: 7 * 2^-24
    ref.check_pair(q, s, _gate64(gate, up), 8 * 2.0 ** -24)


def test_gate_of_large_arguments(cuda):
    g = torch.tensor([[-1e4, -200.0, -80.0, -30.0, -1e-30, 0.0, 1e-30, 30.0, 80.0, 200.0, 1e4]] * 2, device="cuda")
    u = torch.ones_like(g)
    q, s = ops.silu_mul_fp8(g, u)
    assert not bool(q.float().isnan().any())
    ref.check_pair(q, s, _gate64(g, u), 8 * 2.0 ** -24)


# ---- matrix product ----

def _operands(g, M, N, K, scales=None, padded=True):
    """Pairs with every value of e4m3 among them, scales powers of two or any."""
    def matrix(rows):
        q = torch.randint(0, 254, (rows, K), generator=g, dtype=torch.uint8)
        q[(q & 127) == 127] = 3                                          # (no NaN)
        wide = torch.full((rows, (K + 15) // 16 * 16), 0x7f, dtype=torch.uint8)   # NaN behind the rows: never read
        wide[:, :K] = q
        return wide.cuda().view(torch.float8_e4m3fn)[:, :K]
    kb = -(-K // 128)
    a, b = matrix(M), matrix(N)
    if scales == "fp32":
        sa, sb = (torch.rand(n, kb, generator=g).cuda() + 0.1 for n in (M, -(-N // 128)))
    else:
        sa, sb = (torch.exp2(torch.randint(-12, 4, (n, kb), generator=g).float()).cuda().to(torch.float8_e8m0fnu) for n in (M, -(-N // 128)))
    return a, sa, b, sb


def _check(out, a, sa, b, sb):
    av, bv = ref.value(a, sa), ref.value(b, sb, 128)
    want, size = av @ bv.t(), av.abs() @ bv.abs().t()
    kb = sa.shape[1]
    # a block's 128 products, each added with at most a step of 2^-23 of the sum of magnitudes; a product of scales, a product
    # with it and a sum of half a step a block, and up to three sums more where the blocks are split over CTAs; the result's
    # rounding
    bound = size * (128 * 2.0 ** -23 + (kb + 5) * 2.0 ** -24) + want.abs() * (torch.finfo(out.dtype).eps / 2)
    err = (out.double() - want).abs()
    assert bool((err <= bound).all()), (float((err / bound.clamp(min=1e-300)).max()), int((err > bound).sum()))
    # ... which a wrong term of average size would pass: the whole is held to the roundings' usual size too
    rel = 2.0 ** -8 if out.dtype == BF16 else 2e-6
    assert float(err.norm()) <= rel * float(want.norm()), (float(err.norm()), float(want.norm()))


SIZES = [(1, 128, 128), (1, 1, 1), (1, 15360, 2048), (2, 100, 16), (3, 7, 2000), (16, 128, 256), (17, 129, 129), (33, 768, 2496), (64, 127, 100),
         (65, 4736, 768), (127, 256, 384), (128, 128, 1), (129, 300, 1000), (255, 2048, 640), (257, 257, 257), (550, 768, 2496),
         (1000, 1000, 1000), (2049, 513, 768), (4096, 768, 2496), (5000, 4736, 768)]


@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("dtype,scales", [(BF16, None), (F32, "fp32")])
def test_matmul(cuda, M, N, K, dtype, scales):
    a, sa, b, sb = _operands(_gen(M, N, K), M, N, K, scales)
    out = ops.matmul_fp8(a, sa, b, sb, dtype=dtype)
    assert out.dtype == dtype and out.shape == (M, N)
    _check(out, a, sa, b, sb)


@pytest.mark.parametrize("M,N,K", [(1, 40, 300), (40, 200, 1024), (300, 140, 2500), (1030, 520, 700), (2100, 1300, 1024)])
def test_matmul_of_whole_numbers_is_exact(cuda, M, N, K):
    """Small whole numbers and scales: every sum is exact in fp32, so each element has to be right to the last bit."""
    g = _gen(M, N, K, 1)
    a, b = (torch.randint(-8, 9, (r, (K + 15) // 16 * 16), generator=g).float().cuda().to(torch.float8_e4m3fn)[:, :K] for r in (M, N))
    kb = -(-K // 128)
    sa, sb = (torch.exp2(torch.randint(0, 3, (n, kb), generator=g).float()).cuda().to(torch.float8_e8m0fnu) for n in (M, -(-N // 128)))
    out = ops.matmul_fp8(a, sa, b, sb, dtype=F32)
    assert torch.equal(out.double(), ref.value(a, sa) @ ref.value(b, sb, 128).t())


@pytest.mark.parametrize("M,N,K", [(1, 100, 256), (5, 130, 300), (70, 200, 256), (300, 333, 256), (1100, 600, 520)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_matmul_into_a_column_block(cuda, M, N, K, dtype):
    """The result in a wider buffer at any alignment, and scales with other strides; nothing around it changes."""
    a, sa, b, sb = _operands(_gen(M, N), M, N, K)
    for offset, ld in ((0, N + 1), (1, N + 8), (8, N + 24)):
        whole = torch.full((M + 2, ld + offset), 5.0, dtype=dtype, device="cuda")
        out = whole[1:M + 1, offset:offset + N]
        sa_t = sa.view(torch.uint8).t().contiguous().t().view(torch.float8_e8m0fnu)
        assert ops.matmul_fp8(a, sa_t, b, sb, out=out) is out
        _check(out, a, sa, b, sb)
        out.fill_(5.0)
        assert bool((whole == 5).all())


def test_matmul_of_nothing(cuda):
    a, sa, b, sb = _operands(_gen(9), 4, 6, 128)
    assert ops.matmul_fp8(a[:0], sa[:0], b, sb).shape == (0, 6)
    assert ops.matmul_fp8(a, sa, b[:0], sb[:0]).shape == (4, 0)
    whole = torch.full((6, 10), 5.0, device="cuda")
    ops.matmul_fp8(a[:, :0], sa[:, :0], b[:, :0], sb[:, :0], out=whole[1:5, 2:8])
    assert bool((whole[1:5, 2:8] == 0).all()) and float(whole.sum()) == 5 * (60 - 24)


@pytest.mark.parametrize("M", [3, 200, 1500])
def test_matmul_passes_nan_on(cuda, M):
    """A NaN scale or value shows in its row (its columns, for a weight's block) and nowhere else."""
    a, sa, b, sb = _operands(_gen(10), M, 300, 400)
    sa = sa.clone()
    sa[1, 2] = float("nan")
    out = ops.matmul_fp8(a, sa, b, sb)
    assert bool(out[1].isnan().all()) and int(out.isnan().sum()) == 300
    sb, sa = sb.clone(), _operands(_gen(10), M, 300, 400)[1]
    sb[1, 0] = float("nan")
    out = ops.matmul_fp8(a, sa, b, sb)
    assert bool(out[:, 128:256].isnan().all()) and int(out.isnan().sum()) == 128 * M
    b = b.clone(memory_format=torch.preserve_format)
    b.view(torch.uint8)[7, 399] = 0x7f
    out = ops.matmul_fp8(a, sa, b, _operands(_gen(10), M, 300, 400)[3]) if b.stride(0) % 16 == 0 else None
    if out is not None:
        assert bool(out[:, 7].isnan().all()) and int(out.isnan().sum()) == M


def test_matmul_same_bits_again_and_alone(cuda):
    """The order of the sums goes by the sizes alone."""
    a, sa, b, sb = _operands(_gen(11), 700, 900, 2000)
    first = ops.matmul_fp8(a, sa, b, sb, dtype=F32)
    for _ in range(3):
        assert torch.equal(ops.matmul_fp8(a, sa, b, sb, dtype=F32), first)


def test_streams_and_graph(cuda):
    """Norm, product, gate, product as the block runs them, on a side stream and as a replayed graph over new inputs."""
    E, I, M = 256, 320, 75
    g = _gen(12)
    w = torch.ones(E, device="cuda", dtype=BF16)
    w1, w2 = (ops.quantize_fp8(_randn(g, n, k, dtype=BF16) * 0.05, block_rows=128) for n, k in ((2 * I, E), (E, I)))

    def chain(x):
        both = ops.matmul_fp8(*ops.rmsnorm_fp8(x, w, EPS), *w1)
        return ops.matmul_fp8(*ops.silu_mul_fp8(both[:, :I], both[:, I:]), *w2)

    xs = [_randn(g, M, E, dtype=BF16) for _ in range(3)]
    want = [chain(x) for x in xs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = chain(xs[0])
    side.synchronize()
    assert torch.equal(got, want[0])
    from attentions import attn
    check, attn._CHECK_STATUS = attn._CHECK_STATUS, False        # (reading the status word back synchronises: not under capture)
    try:
        static = xs[0].clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = chain(static)
        for x, y in zip(xs, want):
            static.copy_(x)
            graph.replay()
            assert torch.equal(out, y)
    finally:
        attn._CHECK_STATUS = check


# ---- refusals ----

def test_refusals(cuda):
    x = torch.randn(4, 256, device="cuda")
    q, s = ops.quantize_fp8(x)
    wq, ws = ops.quantize_fp8(x, block_rows=128)
    grad = x.clone().requires_grad_()
    for call in (lambda: ops.quantize_fp8(grad), lambda: ops.rmsnorm_fp8(grad, x[0], EPS), lambda: ops.silu_mul_fp8(x, grad)):
        with pytest.raises(RuntimeError, match="no gradient"):
            call()
    with torch.no_grad():
        ops.quantize_fp8(grad)
    for call, words in [
        (lambda: ops.quantize_fp8(x.half()), "not supported"),
        (lambda: ops.quantize_fp8(x, block_rows=64), "block_rows"),
        (lambda: ops.quantize_fp8(x.t()), "unit inner stride"),
        (lambda: ops.quantize_fp8(x[:1].expand(4, 256)), "overlap"),
        (lambda: ops.quantize_fp8(x, out=(q[:3], s)), "out must be"),
        (lambda: ops.rmsnorm_fp8(x, x[0, :255].contiguous(), EPS), "shapes"),
        (lambda: ops.rmsnorm_fp8(x, x[0].bfloat16(), EPS), "one type"),
        (lambda: ops.rmsnorm_fp8(x, x[0], EPS, add=x[:2]), "shapes"),
        (lambda: ops.rmsnorm_fp8(torch.randn(2, 4104, device="cuda"), torch.randn(4104, device="cuda"), EPS), "2048"),
        (lambda: ops.silu_mul_fp8(x, x[:, :128]), "one shape"),
        (lambda: ops.matmul_fp8(q, s, wq[:, :128], ws[:, :1]), "shapes"),
        (lambda: ops.matmul_fp8(q, s[:, :1], wq, ws), "shapes"),
        (lambda: ops.matmul_fp8(q, s, wq, ws.float()), "scales"),
        (lambda: ops.matmul_fp8(x, s, wq, ws), "float8_e4m3fn"),
        (lambda: ops.matmul_fp8(q[:, 8:136], s[:, :1], wq[:, :128], ws[:, :1]), "16-byte"),
        (lambda: ops.matmul_fp8(q, s, wq, ws, dtype=torch.float16), "not supported"),
        (lambda: ops.matmul_fp8(q, s, wq, ws, out=torch.empty(4, 5, device="cuda")), "out must be"),
        (lambda: ops.matmul_fp8(q, s.cpu(), wq, ws), "CUDA device"),
    ]:
        with pytest.raises(RuntimeError, match=words):
            call()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("width,shift", [(128, 0), (300, 0), (300, 3), (1001, 1)])
def test_gate_between_its_smallest_values(cuda, dtype, width, shift):
    """Gates between -300 and -60, whose e^g leaves fp32's normal numbers, beside factors that bring the product back: blocks of
    such values alone and blocks with ordinary ones among them, at any alignment."""
    g = _gen(width, shift)
    rows = 24
    gate = -60.0 - 240.0 * torch.rand(rows, width + shift, generator=g)
    gate[:4] = -87.0 - torch.linspace(-1.0, 2.0, width + shift)                     # both sides of -87
    gate[4:8].mul_(0.5)
    gate[8:12, ::3] = torch.randn(4, len(range(0, width + shift, 3)), generator=g) * 20
    gate = gate.to(dtype).cuda()[:, shift:]
    # |silu(gate) u| between 1e-30 and 1 where fp32 has such a u, and u at fp32's (bf16's) largest below
    size = 10.0 ** (-30.0 * torch.rand(rows, width, generator=g).double().cuda())
    up = (size / (gate.double() * torch.sigmoid(gate.double())).abs().clamp(min=1e-300)).clamp(max=3e38)
    up = (up * torch.randint(0, 2, (rows, width), generator=g).cuda().mul(2).sub(1)).to(dtype)
    wide = torch.zeros(rows, width + shift, dtype=dtype, device="cuda")
    up = wide[:, shift:].copy_(up)
    q, s = ops.silu_mul_fp8(gate, up)
    # e^(g / 4) four times, each within a unit (2^-23), and four products of half a unit (2^-24) each: 12 * 2^-24.  Values and
    # products of them below 2^-126 are off by up to 2^-150 each time: blocks whose largest value is above 2^-100 do not see that.
    y = _gate64(gate, up)
    seen = (ref.tops(y) > 2.0 ** -100).repeat_interleave(128, 1)[:, :width]
    assert bool(seen[:12].all())
    ref.check_pair(q, s, y, 16 * 2.0 ** -24)


def test_gate_of_infinite_and_missing_numbers(cuda):
    """-inf, NaN and infinite factors in the places that e^g makes zero: as the formula has them."""
    inf, nan = float("inf"), float("nan")
    g = torch.tensor([[-inf, 1.0], [nan, -100.0], [-100.0, 1.0], [-1e30, 2.0], [-100.0, nan], [-300.0, 3.0]], device="cuda")
    u = torch.tensor([[1.0, 1.0], [1.0, 1.0], [inf, 1.0], [1e30, 1.0], [1.0, 1.0], [0.0, 1.0]], device="cuda")
    q, s = ops.silu_mul_fp8(g, u)
    assert s.float().isnan().flatten().tolist() == [True, True, True, False, True, False]
    assert bool(q[[0, 1, 2, 4]].float().isnan().all()) and not bool(q[[3, 5]].float().isnan().any())
    assert q[[3, 5], 0].float().tolist() == [0.0, 0.0]
