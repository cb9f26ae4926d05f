"""GPU: the 8-bit operators where their callers go less often: offsets past 32 bits, scales at odd places and of extreme sizes,
calls at once from several threads and streams, graphs that share nothing, a padded batch, a norm that only copies."""
import threading

import pytest
import torch

import fp8_oracle as ref
import mvpa_ops as ops
from attentions import attn

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def _pairs(M, N, K, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    a = ops.quantize_fp8(torch.randn(M, K, generator=g, device="cuda"))
    return (*a, *ops.quantize_fp8(torch.randn(N, K, generator=g, device="cuda") * 0.1, block_rows=128))


def _want(a, sa, b, sb):
    return ref.value(a, sa) @ ref.value(b, sb, 128).t()


def test_offsets_past_32_bits(cuda):
    rows, width = 70001, 32768                                         # 2.3e9 values
    x = torch.zeros(rows, width, dtype=BF16, device="cuda")
    tail = torch.randn(3, width, device="cuda", dtype=BF16)
    x[-3:] = tail
    for block in (1, 128):
        q, s = ops.quantize_fp8(x, block_rows=block)
        q3, s3 = q[-3:], s[-3:] if block == 1 else s[-1:]
        full = tail if block == 1 else x[rows - rows % 128:]
        q64, s64 = ref.pair(full, block)
        assert torch.equal(q3.double(), q64[-3:]) and torch.equal(s3.double(), s64[-s3.shape[0]:])
        del q, s
    gate = x.view(-1, 16384)                                           # rows of 16384, half of a projection's
    q, s = ops.silu_mul_fp8(gate[:, :8192], gate[:, 8192:])
    y = torch.nn.functional.silu(gate[-4:, :8192].double()) * gate[-4:, 8192:].double()
    ref.check_pair(q[-4:], s[-4:], y, 8 * 2.0 ** -24)
    del q, s, gate
    h = x.view(-1, 4096)
    q, s = ops.rmsnorm_fp8(h, torch.ones(4096, dtype=BF16, device="cuda"), 1e-5)
    y = h[-9:].double()
    ref.check_pair(q[-9:], s[-9:], y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-5), ((4096 / 32 + 21) / 2 + 7) * 2.0 ** -24)


@pytest.mark.parametrize("fp32_scales", [False, True])
def test_product_with_offsets_past_32_bits(cuda, fp32_scales):
    M, N, K = 66000, 33000, 128                                        # 2.2e9 results
    a, sa, b, sb = _pairs(M, N, K)
    out = ops.matmul_fp8(a, sa.float() if fp32_scales else sa, b, sb.float() if fp32_scales else sb)
    for rows in (slice(0, 5), slice(M - 300, M)):
        want = _want(a[rows], sa[rows], b, sb)
        assert float((out[rows].double() - want).norm() / want.norm()) <= 2.0 ** -8


@pytest.mark.parametrize("M", [5, 40, 700])
def test_scales_at_odd_places(cuda, M):
    """Scales in a wider buffer (rows that start at any byte), one row of scales for all tokens, columns first."""
    N, K = 300, 1100
    a, sa, b, sb = _pairs(M, N, K)
    want = ops.matmul_fp8(a, sa, b, sb, dtype=F32)
    kb = sa.shape[1]
    for offset, width in ((1, 12), (4, 16), (3, 11 + kb)):
        wide = torch.zeros(M, offset + width, dtype=torch.uint8, device="cuda")
        view = wide[:, offset:offset + kb].view(torch.float8_e8m0fnu)
        view.copy_(sa)
        narrow = torch.zeros(kb, sb.shape[0] + 1, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu).t()[1:]
        narrow.copy_(sb)
        assert torch.equal(ops.matmul_fp8(a, view, b, narrow, dtype=F32), want)
    one = sa[:1].expand(M, kb)
    assert torch.equal(ops.matmul_fp8(a, one, b, sb, dtype=F32), ops.matmul_fp8(a, one.contiguous(), b, sb, dtype=F32))


@pytest.mark.parametrize("M", [7, 100])
def test_scales_of_extreme_sizes(cuda, M):
    """The smallest and largest exponents, whose products are ordinary numbers."""
    a, sa, b, sb = _pairs(M, 200, 300)
    lo, hi = (torch.full_like(s.view(torch.uint8), v).view(torch.float8_e8m0fnu) for s, v in ((sa, 0), (sb, 254)))
    got = ops.matmul_fp8(a, lo, b, hi, dtype=F32)
    want = a.double() @ b.double().t()                                  # 2^-127 * 2^127
    assert float((got.double() - want).norm() / want.norm()) <= 2e-6


def test_calls_at_once(cuda):
    """Threads with streams of their own, small and large products among them: everyone's results are those of a call alone."""
    sizes = [(1, 2048, 1024), (30, 700, 2000), (300, 1000, 700), (2000, 1500, 512), (2000, 1500, 513), (5000, 768, 384)]
    work = [_pairs(*s, seed=i) for i, s in enumerate(sizes)]
    want = [ops.matmul_fp8(*w) for w in work]
    torch.cuda.synchronize()
    bad = []

    def run(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for k in range(20):
                j = (i + k) % len(work)
                x = torch.randn(50, 640, device="cuda", generator=torch.Generator(device="cuda").manual_seed(k))
                pair = ops.rmsnorm_fp8(x, torch.ones(640, device="cuda"), 1e-5)
                got = ops.matmul_fp8(*work[j])
                stream.synchronize()
                if not torch.equal(got, want[j]) or bool(pair[0].float().isnan().any()):
                    bad.append((i, k, j))

    threads = [threading.Thread(target=run, args=(i,)) for i in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not bad


def test_two_graphs_on_two_streams(cuda):
    check, attn._CHECK_STATUS = attn._CHECK_STATUS, False
    try:
        work = [_pairs(600, 900, 1024, seed=1), _pairs(20, 4000, 2048, seed=2)]
        want = [ops.matmul_fp8(*w) for w in work]
        graphs, outs = [], []
        for w in work:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                outs.append([ops.matmul_fp8(*w) for _ in range(3)])
            graphs.append(g)
        streams = [torch.cuda.Stream() for _ in graphs]
        for _ in range(10):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for out, w in zip(outs, want) for o in out)
    finally:
        attn._CHECK_STATUS = check


def test_padded_batch(cuda):
    """Rows of zeros behind the last token stay zeros, and change nothing before them; the rows behind an output view stay as
    they were."""
    x = torch.randn(300, 512, device="cuda", dtype=BF16)
    padded = torch.zeros(512, 512, device="cuda", dtype=BF16)
    padded[:300] = x
    w = ops.quantize_fp8(torch.randn(384, 512, device="cuda"), block_rows=128)
    norm = torch.ones(512, device="cuda", dtype=BF16)
    out = torch.full((600, 384), 3.0, device="cuda", dtype=BF16)
    ops.matmul_fp8(*ops.rmsnorm_fp8(padded, norm, 1e-5), *w, out=out[:512])
    alone = ops.matmul_fp8(*ops.rmsnorm_fp8(x, norm, 1e-5), *w)
    assert torch.equal(out[:300], alone) and bool((out[300:512] == 0).all()) and bool((out[512:] == 3).all())


@pytest.mark.parametrize("dtype,width", [(BF16, 768), (BF16, 770), (F32, 1000), (F32, 1001)])
def test_norm_that_copies(cuda, dtype, width):
    """`sum_out` without `add` is a copy of x; `add` may be x itself."""
    x, w = torch.randn(100, width, device="cuda").to(dtype), torch.ones(width, device="cuda", dtype=dtype)
    h = torch.empty_like(x)
    q, s = ops.rmsnorm_fp8(x, w, 1e-5, sum_out=h)
    assert torch.equal(h, x)
    q2, s2 = ops.rmsnorm_fp8(x, w, 1e-5)
    assert torch.equal(q.float(), q2.float()) and torch.equal(s.float(), s2.float())
    ops.rmsnorm_fp8(x, w, 1e-5, add=x, sum_out=h)
    assert torch.equal(h, (x.float() * 2).to(dtype))


def test_default_device_and_inference_mode(cuda):
    x = torch.randn(40, 256, device="cuda")
    want = ops.quantize_fp8(x)
    torch.set_default_device("cuda")
    try:
        got = ops.quantize_fp8(x)
    finally:
        torch.set_default_device(None)
    with torch.inference_mode():
        again = ops.quantize_fp8(x.clone())
    for p in (got, again):
        assert torch.equal(p[0].float(), want[0].float()) and torch.equal(p[1].float(), want[1].float())


def test_outputs_that_require_a_gradient_are_refused(cuda):
    a, sa, b, sb = _pairs(3, 64, 128)
    leaf = torch.zeros(3, 64, device="cuda", requires_grad=True)
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.matmul_fp8(a, sa, b, sb, out=leaf)
    x = torch.randn(3, 64, device="cuda")
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.rmsnorm_fp8(x, torch.ones(64, device="cuda"), 1e-5, sum_out=leaf)
    with torch.no_grad():
        ops.matmul_fp8(a, sa, b, sb, out=leaf)
    assert bool(leaf.detach().ne(0).any())


@pytest.mark.parametrize("M,N,K", [(33, 500, 4096), (100, 300, 4097), (257, 193, 5000), (600, 700, 6200), (1000, 1500, 6200), (200, 2100, 8191),
                                   (300, 64, 7680), (3000, 700, 6145)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_long_sums_of_whole_numbers(cuda, M, N, K, dtype):
    """Long K with few tiles, where several pairs of CTAs share a tile's blocks: small whole numbers, whose sums (below 2^24) are
    exact in fp32, into aligned and odd column blocks; the same bits again."""
    g = torch.Generator().manual_seed(M + N + K)
    a, b = (torch.randint(-8, 9, (r, (K + 15) // 16 * 16), generator=g).float().cuda().to(torch.float8_e4m3fn)[:, :K] for r in (M, N))
    kb = -(-K // 128)
    sa, sb = (torch.exp2(torch.randint(0, 3, (n, kb), generator=g).float()).cuda().to(torch.float8_e8m0fnu) for n in (M, -(-N // 128)))
    want = (ref.value(a, sa) @ ref.value(b, sb, 128).t()).to(dtype)
    for offset, ld in ((0, (N + 7) // 8 * 8), (3, N + 9)):
        whole = torch.full((M + 1, offset + ld), 5.0, dtype=dtype, device="cuda")
        out = whole[:M, offset:offset + N]
        for _ in range(2):
            ops.matmul_fp8(a, sa, b, sb, out=out)
            assert torch.equal(out, want)
        out.fill_(5.0)
        assert bool((whole == 5).all())
    sa[M // 2, kb - 1] = float("nan")
    out = ops.matmul_fp8(a, sa, b, sb, dtype=dtype)
    assert bool(out[M // 2].isnan().all()) and int(out.isnan().sum()) == N


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("fp32_scales", [False, True])
@pytest.mark.parametrize("M,N", [(1, 5), (20, 131), (40, 3), (200, 100), (300, 700), (2500, 1030), (2500, 1033)])
def test_rows_that_end_inside_sixteen_bytes(cuda, M, N, dtype, fp32_scales):
    """Results whose rows start on 16-byte boundaries and end anywhere: what stands behind them stays."""
    a, sa, b, sb = _pairs(M, N, 256, seed=3)
    if fp32_scales:
        sa, sb = sa.float() * 1.25, sb.float() * 0.75
    ld = (N + 7) // 8 * 8 + 8
    whole = torch.full((M + 1, ld), 5.0, dtype=dtype, device="cuda")
    out = whole[:M, :N]
    ops.matmul_fp8(a, sa, b, sb, out=out)
    assert torch.equal(out, ops.matmul_fp8(a, sa, b, sb, dtype=dtype))
    out.fill_(5.0)
    assert bool((whole == 5).all())


@pytest.mark.parametrize("M,N,K", [(33, 500, 2048), (100, 300, 2049), (300, 259, 5000), (600, 700, 6200), (1000, 1500, 6200), (200, 2100, 3200)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_long_sums_with_other_scales(cuda, M, N, K, dtype):
    """The same with fp32 scales, small whole numbers that are no powers of two."""
    g = torch.Generator().manual_seed(M + N + K)
    a, b = (torch.randint(-4, 5, (r, (K + 15) // 16 * 16), generator=g).float().cuda().to(torch.float8_e4m3fn)[:, :K] for r in (M, N))
    kb = -(-K // 128)
    sa, sb = (torch.randint(1, 6, (n, kb), generator=g).float().cuda() for n in (M, -(-N // 128)))
    want = (ref.value(a, sa) @ ref.value(b, sb, 128).t()).to(dtype)      # below 2^24
    for offset, ld in ((0, (N + 7) // 8 * 8), (3, N + 9)):
        whole = torch.full((M + 1, offset + ld), 5.0, dtype=dtype, device="cuda")
        out = whole[:M, offset:offset + N]
        for _ in range(2):
            ops.matmul_fp8(a, sa, b, sb, out=out)
            assert torch.equal(out, want)
        out.fill_(5.0)
        assert bool((whole == 5).all())
    sa[M // 2, kb - 1] = float("nan")
    out = ops.matmul_fp8(a, sa, b, sb, dtype=dtype)
    assert bool(out[M // 2].isnan().all()) and int(out.isnan().sum()) == N


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("fp32_scales", [False, True])
@pytest.mark.parametrize("M,N", [(8192, 1100), (8192, 1033), (20000, 1030)])
@pytest.mark.parametrize("K", [128, 768])
def test_row_ends_of_many_tiles(cuda, M, N, K, dtype, fp32_scales):
    """Rows on 16-byte boundaries that end inside one, with several tiles to a pair of CTAs: a row's last columns, which are stored
    one by one, and the tiles before and after, which the TMA stores, leave through the same shared memory.  Whole numbers, whose sums
    (at most 768 * 16 * 25 < 2^24) are exact in fp32."""
    g = torch.Generator().manual_seed(M + N + K)
    a, b = (torch.randint(-4, 5, (r, K), generator=g).float().cuda().to(torch.float8_e4m3fn) for r in (M, N))
    shapes = (M, K // 128), (-(-N // 128), K // 128)
    if fp32_scales:
        sa, sb = (torch.randint(1, 6, n, generator=g).float().cuda() for n in shapes)
    else:
        sa, sb = (torch.exp2(torch.randint(0, 3, n, generator=g).float()).cuda().to(torch.float8_e8m0fnu) for n in shapes)
    want = (ref.value(a, sa) @ ref.value(b, sb, 128).t()).to(dtype)
    whole = torch.full((M + 1, (N + 7) // 8 * 8), 5.0, dtype=dtype, device="cuda")
    out = whole[:M, :N]
    for _ in range(8):
        out.fill_(7.0)
        ops.matmul_fp8(a, sa, b, sb, out=out)
        assert torch.equal(out, want)
    out.fill_(5.0)
    assert bool((whole == 5).all())


@pytest.mark.parametrize("M,N,K", [(17, 15360, 2048), (22, 2048, 7680), (32, 600, 6144), (31, 129, 641), (1, 2048, 7680), (16, 9500, 1024)])
@pytest.mark.parametrize("fp32_scales", [False, True])
def test_few_rows_of_whole_numbers(cuda, M, N, K, fp32_scales):
    """Up to 32 rows, alone and split along K, more blocks than stages: whole numbers whose sums (below 7680 * 16 * 25 < 2^24) are
    exact in fp32, and the same bits again."""
    g = torch.Generator().manual_seed(M + N + K)
    a, b = (torch.randint(-4, 5, (r, (K + 15) // 16 * 16), generator=g).float().cuda().to(torch.float8_e4m3fn)[:, :K] for r in (M, N))
    kb = -(-K // 128)
    if fp32_scales:
        sa, sb = (torch.randint(1, 6, (n, kb), generator=g).float().cuda() for n in (M, -(-N // 128)))
    else:
        sa, sb = (torch.exp2(torch.randint(0, 3, (n, kb), generator=g).float()).cuda().to(torch.float8_e8m0fnu) for n in (M, -(-N // 128)))
    want = (ref.value(a, sa) @ ref.value(b, sb, 128).t()).float()
    for _ in range(3):
        assert torch.equal(ops.matmul_fp8(a, sa, b, sb, dtype=F32), want)
