"""GPU: weights in 4 bits - quantisation, reading back, products for one token and many, the gate - against their definitions in 64
bits, at the sizes, layouts and values where they can go wrong, and what they refuse."""
import threading

import pytest
import torch

import int4_oracle as ref
import mvpa_native as nat
import mvpa_ops as ops

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def _gen(*key):
    return torch.Generator().manual_seed(sum((i + 1) * 7919 * int(k) for i, k in enumerate(key)) % (1 << 30))


def _randn(g, *shape, dtype=F32):
    return torch.randn(*shape, generator=g).to(dtype).cuda()


def _weight(g, N, K, group, zeros, dtype):
    w = ops.quantize_int4(_randn(g, N, K, dtype=dtype) * K ** -0.5, group, zeros)
    return w if zeros else (*w, None)


# ---- quantisation: every whole number and every scale is the definition's ----

@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("N,K", [(1, 1), (1, 32), (2, 31), (3, 33), (2, 127), (5, 128), (5, 129), (130, 1000), (7, 2496), (33, 2049)])
def test_quantize(cuda, dtype, group, zeros, N, K):
    g = _gen(N, K, group, zeros)
    w = (_randn(g, N, K) * torch.exp(2 * _randn(g, N, 1))).to(dtype)
    got = ops.quantize_int4(w, group, zeros)
    q, s, z = ref.quantize(w, group, zeros)
    assert torch.equal(ref.unpack(got[0], K), q) and torch.equal(got[1], s) and len(got) == 2 + zeros
    assert not zeros or torch.equal(got[2].long(), z)
    assert got[0].stride(0) % 16 == 0 or N == 1
    if K % 2:
        assert not bool((got[0][:, -1] >> 4).any())
    for out in (BF16, F32):
        back = ops.dequantize_int4(*got, width=K, group=group, dtype=out)
        assert torch.equal(back, ref.values(got[0], got[1], got[2] if zeros else None, K, group).float().to(out))
    assert ops.dequantize_int4(*got, width=K, group=group).dtype == dtype


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("zeros", [False, True])
def test_quantize_borders(cuda, dtype, zeros):
    """Quotients on halves and next to them, the smallest and largest numbers, groups of zeros, of one sign, of one value."""
    rows = []
    for top in (7.0, 3.5, 1.0, 3e38, 1e-30, 2.0 ** -126, 3e-39, 1e-44, 0.0, 448.0, 7.0000005):
        step = top / 7
        row = [top] + [step * (k + 0.5) for k in range(-7, 7)] + [step * k for k in range(-7, 8)] + [-0.0, step * 0.49999997]
        rows.append(row)
        rows.append([abs(v) for v in row])
        rows.append([-abs(v) for v in row])
        rows.append([top] * 32)
    w = torch.tensor(rows).to(dtype).cuda()
    got = ops.quantize_int4(w, 32, zeros)
    q, s, z = ref.quantize(w, 32, zeros)
    assert torch.equal(got[1], s) and torch.equal(ref.unpack(got[0], 32), q)
    assert not zeros or torch.equal(got[2].long(), z)


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_quantize_not_finite(cuda, bad, zeros, dtype):
    w = _randn(_gen(1), 40, 300, dtype=dtype)
    w[2, 70] = bad
    got = ops.quantize_int4(w, 64, zeros)
    back = ops.dequantize_int4(*got, width=300, group=64)
    hit = torch.zeros(40, 300, dtype=torch.bool, device="cuda")
    hit[2, 64:128] = True
    assert torch.equal(back.isnan(), hit) and int(got[1].isnan().sum()) == 1
    good = ops.quantize_int4(torch.where(hit, torch.zeros_like(w), w), 64, zeros)
    assert torch.equal(back[~hit], ops.dequantize_int4(*good, width=300, group=64)[~hit])


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("offset,ld", [(0, 300), (1, 301), (3, 304), (8, 320)])
def test_quantize_strided(cuda, dtype, offset, ld):
    buf = _randn(_gen(offset, ld), 37, ld, dtype=dtype)
    w = buf[:, offset:offset + 200]
    q, s = ops.quantize_int4(w, 64)
    q64, s64, _ = ref.quantize(w, 64, False)
    assert torch.equal(ref.unpack(q, 200), q64) and torch.equal(s, s64)


# ---- products ----

SIZES = [(1, 1), (16, 128), (17, 31), (130, 1027), (300, 512), (257, 1000), (768, 2496), (129, 129)]


@pytest.mark.parametrize("M", [1, 2, 8, 9, 16, 17, 32, 33, 64, 65, 128, 129, 300])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
def test_products(cuda, M, dtype, group, zeros):
    half = torch.finfo(dtype).eps / 2
    for i, (N, K) in enumerate(SIZES):
        g = _gen(M, group, zeros, i)
        scales = dtype if i % 2 else (BF16 if dtype == F32 else F32)          # scales of either type beside x of either
        w, up = (_weight(g, N, K, group, zeros, scales) for _ in range(2))
        x = _randn(g, M, K, dtype=dtype)
        y = ops.matmul_int4(x, *w, group=group)
        exact, bound, _ = ref.product(x, w, K, group, half)
        assert y.shape == (M, N) and y.dtype == dtype
        assert ((y.double() - exact).abs() <= bound).all(), (N, K)
        h = ops.gated_linear_int4(x, w if zeros else w[:2], up if zeros else up[:2], group=group)
        exact, bound = ref.gated(x, w, up, K, group, half)
        assert ((h.double() - exact).abs() <= bound).all(), (N, K)


@pytest.mark.parametrize("M,N,K", [(1, 15360, 2048), (5, 2048, 7680), (22, 5632, 2048), (550, 768, 2496), (2200, 4736, 768), (40, 96, 20000), (700, 70, 260)])
def test_models_sizes(cuda, M, N, K):
    g = _gen(M, N, K)
    w, x = _weight(g, N, K, 128, False, BF16), _randn(g, M, K, dtype=BF16)
    y = ops.matmul_int4(x, *w)
    exact, bound, _ = ref.product(x, w, K, 128, 2.0 ** -8)
    assert ((y.double() - exact).abs() <= bound).all()
    for _ in range(3):
        assert torch.equal(y, ops.matmul_int4(x, *w))


@pytest.mark.parametrize("M,N,K,group", [(5000, 3000, 2176, 128), (3000, 4000, 900, 64), (2600, 20000, 384, 32)])
@pytest.mark.parametrize("gate", [False, True])
def test_many_tiles_a_cta(cuda, M, N, K, group, gate):
    """Resident CTAs with several tiles each, odd numbers of chunks among them: rings that do not come out even with a tile's chunks."""
    g = _gen(M, N, K)
    w, up, x = _weight(g, N, K, group, True, BF16), _weight(g, N, K, group, True, BF16), _randn(g, M, K, dtype=BF16)
    run = lambda: ops.gated_linear_int4(x, w, up, group=group) if gate else ops.matmul_int4(x, *w, group=group)
    y = run()
    exact, bound = ref.gated(x, w, up, K, group, 2.0 ** -8) if gate else ref.product(x, w, K, group, 2.0 ** -8)[:2]
    assert ((y.double() - exact).abs() <= bound).all()
    for _ in range(5):
        assert torch.equal(y, run())


@pytest.mark.parametrize("M,dtype", [(17, BF16), (32, BF16), (32, F32), (50, BF16)])
@pytest.mark.parametrize("K", [100, 128, 300, 640])
@pytest.mark.parametrize("gate", [False, True])
def test_many_small_tiles_a_cta(cuda, M, dtype, K, gate):
    """The smallest tiles, several a resident CTA, of one, three and five chunks in groups of 32 with zeros: at each tile's border one set of
    unpacking warps is at the new row's zeros while the other has its next chunk, and the stages go round under both."""
    N, group = 128 * 400 + 40, 32
    g = _gen(M, K, gate)
    w, up = (_weight(g, N, K, group, True, dtype) for _ in range(2))
    x = _randn(g, M, K, dtype=dtype)
    run = lambda: ops.gated_linear_int4(x, w, up, group=group) if gate else ops.matmul_int4(x, *w, group=group)
    y, half = run(), torch.finfo(dtype).eps / 2
    exact, bound = ref.gated(x, w, up, K, group, half) if gate else ref.product(x, w, K, group, half)[:2]
    assert ((y.double() - exact).abs() <= bound).all()
    for _ in range(5):
        assert torch.equal(y, run())


@pytest.mark.parametrize("M", [1, 8, 20, 60, 200])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_strides_and_places(cuda, M, dtype):
    """x at any alignment and as column blocks, turned x, leading dimensions, results into column blocks of wider buffers, scales, zeros and
    packed rows of wider ones; nothing else is written."""
    N, K, group = 150, 200, 64
    g = _gen(M, 5)
    w = _weight(g, N, K, group, True, dtype)
    x = _randn(g, M, K, dtype=dtype)
    want = ops.matmul_int4(x, *w, group=group)
    for offset, ld in ((1, 203), (4, 208), (8, 216)):
        wide = _randn(g, M, ld, dtype=dtype)
        wide[:, offset:offset + K] = x
        assert torch.equal(ops.matmul_int4(wide[:, offset:offset + K], *w, group=group), want)
    assert torch.equal(ops.matmul_int4(x.t().contiguous().t(), *w, group=group), want)
    assert torch.equal(ops.matmul_int4(x.view(1, M, K), *w, group=group), want.view(1, M, N))
    for offset, ld in ((0, N), (3, 161), (8, 168)):
        buf = torch.full((M + 2, ld), 7.0, dtype=dtype, device="cuda")
        got = ops.matmul_int4(x, *w, group=group, out=buf[1:M + 1, offset:offset + N])
        assert torch.equal(got, want)
        buf[1:M + 1, offset:offset + N] = 7
        assert bool((buf == 7).all())
    q = torch.full((N, 160), 0xab, dtype=torch.uint8, device="cuda")
    q[:, 16:116] = w[0]
    s, z = (torch.full((N, 9), 3, dtype=t.dtype, device="cuda") for t in w[1:])
    s[:, 2:6], z[:, 1:5] = w[1], w[2]
    assert torch.equal(ops.matmul_int4(x, q[:, 16:116], s[:, 2:6], z[:, 1:5], group=group), want)
    assert torch.equal(ops.dequantize_int4(q[:, 16:116], s[:, 2:6], z[:, 1:5], group=group), ops.dequantize_int4(*w, group=group))


@pytest.mark.parametrize("M", [1, 8, 9, 40, 100])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_values_at_their_ends(cuda, M, dtype):
    """Infinities and NaN in x stay in their rows and are what the definition makes of them; the largest and smallest fp32 numbers;
    whole numbers past a row's end count for nothing."""
    N, K, group = 40, 70, 32
    g = _gen(M, 9)
    w = _weight(g, N, K, group, True, dtype)
    x = _randn(g, M, K, dtype=dtype)
    want = ops.matmul_int4(x, *w, group=group)
    for bad in (float("inf"), float("-inf"), float("nan")):
        y = x.clone()
        y[M - 1, 33] = bad
        got = ops.matmul_int4(y, *w, group=group)
        assert torch.equal(got[:M - 1], want[:M - 1])
        exact = y[M - 1:].double() @ ref.values(*w, K, group).t()
        assert torch.equal(got[M - 1:].isnan(), exact.isnan()) and torch.equal(got[M - 1:].isinf(), exact.isinf())
        assert torch.equal(got[M - 1:][exact.isinf()].double(), exact[exact.isinf()])
    q, s = torch.full((1, 16), 0x99, dtype=torch.uint8, device="cuda"), torch.ones(1, 1, dtype=dtype, device="cuda")     # ones
    for v in (3.3e38, 1e-30, 1.1754944e-38, 1.2345678):
        y = torch.zeros(M, 32, dtype=dtype, device="cuda")
        y[:, 7] = v
        assert torch.equal(ops.matmul_int4(y, q, s, group=32)[:, 0], y[:, 7])
    # bytes past a row: another matrix' values
    wide = torch.full((N, 64), 0xff, dtype=torch.uint8, device="cuda")
    wide[:, :35] = w[0]
    assert torch.equal(ops.matmul_int4(x, wide[:, :35], w[1], w[2], group=group), want)
    odd = ops.matmul_int4(x[:, :69].contiguous(), wide[:, :35], w[1], w[2], group=group)
    exact, bound, _ = ref.product(x[:, :69], w, 69, group, torch.finfo(dtype).eps / 2)
    assert ((odd.double() - exact).abs() <= bound).all()


@pytest.mark.parametrize("M", [1, 12, 40, 100])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_gate_next_to_the_largest_number(cuda, M, dtype):
    """gate times up past fp32's largest number, silu(gate) times up not."""
    gate, up = (torch.full((1, 16), 0x88, dtype=torch.uint8, device="cuda") for _ in range(2))
    gate[0, 0], up[0, 0] = 0x89, 0x98                   # columns 0 and 1
    s = torch.ones(1, 1, dtype=dtype, device="cuda")
    x = torch.zeros(M, 32, dtype=dtype, device="cuda")
    x[:, 0] = torch.linspace(0.25, 1.25, M).to(dtype)
    x[:, 1] = 3e38
    got = ops.gated_linear_int4(x, (gate, s), (up, s), group=32)[:, 0].double()
    want = x[:, 0].double() * torch.sigmoid(x[:, 0].double()) * x[:, 1].double()
    assert bool(((got - want).abs() <= (2.0 ** -8 + 2.0 ** -18 if dtype == BF16 else 2.0 ** -20) * want.abs()).all())


@pytest.mark.parametrize("M", [1, 9, 40, 100, 300])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("K", [32, 128, 2048])
def test_groups_next_to_the_largest_number(cuda, M, dtype, K):
    """Sums of x (q - zero) past fp32's largest number, whose scale takes them back; scales and results of any size; and small ones, which
    lose no more than fp32's own sums do: an x whose last bits lie above 2^-133, results above 2^-110."""
    N, group = 150, min(K, 128)
    g = _gen(M, K, 3)
    q, zeros = ops.quantize_int4(_randn(g, N, K, dtype=dtype), group, True)[::2]
    for x_size, scale in ((2e37, 1e-3), (3e35, 0.01), (1e36, 1e-30), (1e-30, 1e35), (1e-9, 4e36), (1e-31, 2e-2), (1.0, 1e-32)):
        s = (torch.full((N, -(-K // group)), scale) * torch.exp(0.1 * torch.randn(N, -(-K // group), generator=g))).to(dtype).cuda()
        x = (torch.randn(M, K, generator=g).sign() * (1 + torch.rand(M, K, generator=g)) * x_size).to(dtype).cuda()
        w = (q, s, zeros)
        exact, bound, _ = ref.product(x, w, K, group, torch.finfo(dtype).eps / 2)
        assert exact.abs().max() < 3e38
        assert ((ops.matmul_int4(x, *w, group=group).double() - exact).abs() <= bound).all(), (x_size, scale)


def test_last_row_ends_with_its_bytes(cuda):
    """A packed matrix whose last row ends with the memory it lies in."""
    N, K = 20, 70
    w = _weight(_gen(4), N, K, 32, False, BF16)
    flat = torch.zeros((N - 1) * 48 + 35, dtype=torch.uint8, device="cuda")
    tight = flat.as_strided((N, 35), (48, 1))
    tight.copy_(w[0])
    for M in (3, 30):
        x = _randn(_gen(M), M, K, dtype=BF16)
        assert torch.equal(ops.matmul_int4(x, tight, w[1], group=32), ops.matmul_int4(x, *w, group=32))


def test_nothing_to_do(cuda):
    w = _weight(_gen(2), 6, 64, 64, False, BF16)
    assert ops.matmul_int4(torch.zeros(0, 64, dtype=BF16, device="cuda"), *w, group=64).shape == (0, 6)
    empty = torch.zeros(6, 0, dtype=torch.uint8, device="cuda"), torch.zeros(6, 0, dtype=BF16, device="cuda")
    assert torch.equal(ops.matmul_int4(torch.zeros(3, 0, dtype=BF16, device="cuda"), *empty), torch.zeros(3, 6, dtype=BF16, device="cuda"))
    assert ops.quantize_int4(torch.zeros(0, 64, device="cuda"))[0].shape == (0, 32)
    assert ops.quantize_int4(torch.zeros(4, 0, device="cuda"))[1].shape == (4, 0)


def test_refusals(cuda):
    w = _weight(_gen(2), 6, 64, 64, True, BF16)
    x = torch.zeros(3, 64, dtype=BF16, device="cuda")
    wrong = [lambda: ops.matmul_int4(x, *w, group=48), lambda: ops.matmul_int4(x, *w, group=32), lambda: ops.matmul_int4(x[:, :60], *w, group=64),
             lambda: ops.matmul_int4(x.half(), *w, group=64), lambda: ops.matmul_int4(x, w[0].int(), w[1], w[2], group=64),
             lambda: ops.matmul_int4(x, w[0], w[1].half(), w[2], group=64), lambda: ops.matmul_int4(x, w[0], w[1], w[2].int(), group=64),
             lambda: ops.matmul_int4(x, w[0].cpu(), *w[1:], group=64), lambda: ops.matmul_int4(x.clone().requires_grad_(), *w, group=64),
             lambda: ops.matmul_int4(x, w[0].t(), *w[1:], group=64), lambda: ops.matmul_int4(x, *w, group=64, out=torch.empty(3, 5, dtype=BF16, device="cuda")),
             lambda: ops.matmul_int4(x, *w, group=64, out=torch.empty(3, 6, device="cuda")), lambda: ops.matmul_int4(x, w[0][:, 1:], *w[1:], group=64),
             lambda: ops.gated_linear_int4(x, w, (w[0][:5], w[1][:5]), group=64), lambda: ops.gated_linear_int4(x, w, (w[0], w[1].float()), group=64),
             lambda: ops.quantize_int4(x, 16), lambda: ops.quantize_int4(x.half()), lambda: ops.quantize_int4(x[0]), lambda: ops.dequantize_int4(*w, width=66, group=64),
             lambda: ops.dequantize_int4(*w, group=64, dtype=torch.float16), lambda: ops.matmul_int4(x, torch.empty(6, 40, dtype=torch.uint8, device="cuda")[:, :32], *w[1:], group=64)]
    for i, call in enumerate(wrong):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail(f"call {i} was not refused")


# ---- ways of calling ----

def test_graphs_share_nothing(cuda):
    """Two captured graphs with workspaces of their own (x laid out again), replayed in turn and on two streams at once."""
    cases = []
    check, ops._attn._CHECK_STATUS = ops._attn._CHECK_STATUS, False
    try:
        for i, (M, dtype) in enumerate(((50, F32), (60, F32))):
            w = _weight(_gen(i), 200, 300, 64, False, dtype)
            x = _randn(_gen(i, 1), M, 300, dtype=dtype)
            want = ops.matmul_int4(x, *w, group=64)
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                ops.matmul_int4(x, *w, group=64)
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=side):
                    out = ops.matmul_int4(x, *w, group=64)
            cases.append((graph, out, want, side, w, x))
    finally:
        ops._attn._CHECK_STATUS = check
    torch.cuda.synchronize()
    for _ in range(10):
        for graph, out, _, side, *_ in cases:
            out.zero_()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(c[1], c[2]) for c in cases)


def test_threads_on_their_streams(cuda):
    cases = []
    for i, M in enumerate((1, 20, 100, 300)):
        w, x = _weight(_gen(i), 500, 600, 64, i % 2 == 1, BF16), _randn(_gen(i, 2), M, 600, dtype=BF16)
        cases.append((x, w, ops.matmul_int4(x, *w, group=64)))
    torch.cuda.synchronize()
    bad = []

    def work(i):
        x, w, want = cases[i]
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(30):
                got = ops.matmul_int4(x, *w, group=64)
                torch.cuda.current_stream().synchronize()
                if not torch.equal(got, want):
                    bad.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not bad


def test_python_path_is_the_same(cuda, monkeypatch):
    """Without the extension: the same kernels and results."""
    w = _weight(_gen(1), 100, 130, 64, True, F32)
    xs = [_randn(_gen(M), M, 130, dtype=F32) for M in (2, 30)]
    src = _randn(_gen(5), 40, 100)
    run = lambda: [*(ops.matmul_int4(x, *w, group=64) for x in xs), *(ops.gated_linear_int4(x, w, w, group=64) for x in xs),
                   *ops.quantize_int4(src, 32, True), ops.dequantize_int4(*w, group=64, width=130)]
    native = run()
    monkeypatch.setattr(ops._host, "usable", lambda t: False)
    assert all(torch.equal(a, b) for a, b in zip(native, run()))


def test_offsets_past_32_bits(cuda):
    """More than 2^31 values in the weight, in x and in the result, by rows that are looked at alone."""
    N, K = 1_100_000, 2048                                      # 2.25e9 values
    w = torch.zeros(N, K, dtype=BF16, device="cuda")
    w[-200:] = _randn(_gen(1), 200, K, dtype=BF16)
    q, s = ops.quantize_int4(w)
    last = ops.quantize_int4(w[-200:])
    assert torch.equal(q[-200:], last[0]) and torch.equal(s[-200:], last[1])
    back = ops.dequantize_int4(q, s)
    assert torch.equal(back[-200:], ops.dequantize_int4(*last))
    del back, w
    # (products against the definition: other sizes are summed in another order)
    for M in (2, 20, 40):
        x = _randn(_gen(M), M, K, dtype=BF16)
        exact, bound, _ = ref.product(x, (*last, None), K, 128, 2.0 ** -8)
        assert ((ops.matmul_int4(x, q, s)[:, -200:].double() - exact).abs() <= bound).all()
    x = torch.zeros(N, K, dtype=BF16, device="cuda")
    x[-300:] = _randn(_gen(7), 300, K, dtype=BF16)
    few = ops.quantize_int4(_randn(_gen(8), 2000, K, dtype=BF16))
    exact, bound, _ = ref.product(x[-300:], (*few, None), K, 128, 2.0 ** -8)
    assert ((ops.matmul_int4(x, *few)[-300:].double() - exact).abs() <= bound).all()
