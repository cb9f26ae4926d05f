"""GPU: the gated projection and its gradients against their definition in 64 bits, at the sizes, layouts and values where they can
go wrong."""
import threading

import pytest
import torch

import gated_oracle as ref
import mvpa_native as nat
import mvpa_ops as ops

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def _inputs(M, E, I, seed=0, spread=1.0):
    g = torch.Generator().manual_seed(seed + 1000 * M + E + 7 * I)
    rand = lambda *s: torch.randn(*s, generator=g)
    x = (rand(M, E) * spread).to(BF16).cuda()
    wg, wu = ((rand(I, E) * E ** -0.5).to(BF16).cuda() for _ in range(2))
    return x, wg, wu, (rand(M, I) * 0.1).to(BF16).cuda()


def _check(got, x, wg, wu, dh):
    ins = [t.double() for t in (x, wg, wu, dh)]
    want = (ref.forward(*ins[:3]), *ref.gradients(*ins))
    for name, a, b, bound in zip(("h", "dx", "dwg", "dwu"), got, want, ref.bounds(*ins)):
        worst = ((a.double() - b).abs() - bound).max().item()
        assert worst <= 1e-38, (name, worst)


def _all(x, wg, wu, dh):
    leaves = [t.detach().requires_grad_() for t in (x, wg, wu)]
    h = ops.gated_linear(*leaves)
    return (h.detach(), *torch.autograd.grad(h, leaves, dh))


# one of everything; tiles, blocks and boxes that end on their borders, one before and one after; a model's sizes
@pytest.mark.parametrize("M,E,I", [(1, 8, 8), (1, 768, 1728), (22, 768, 1728), (255, 64, 128), (256, 64, 136), (257, 72, 120), (64, 248, 256),
                                   (65, 256, 264), (512, 520, 1024), (700, 1000, 1368), (1500, 2048, 776), (40, 64, 20000), (20000, 16, 24),
                                   (3, 2048, 5632)])
def test_against_64_bits(cuda, M, E, I):
    ins = _inputs(M, E, I)
    launched = nat.lib().mvpa_launch_count()
    got = _all(*ins)
    assert nat.lib().mvpa_launch_count() - launched in (4, 5, 6)        # the kernels (a gradient may be joined), not torch's operations
    _check(got, *ins)
    with torch.no_grad():
        assert torch.equal(ops.gated_linear(*ins[:3]), got[0])  # what is kept for the backward changes no bit


def test_same_bits_from_run_to_run(cuda):
    ins = _inputs(3000, 768, 1728)
    first = _all(*ins)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, _all(*ins)))


@pytest.mark.parametrize("need", [(True, False, False), (False, True, False), (False, False, True), (True, False, True), (False, True, True)])
def test_gradients_of_some(cuda, need):
    ins = _inputs(300, 264, 200)
    whole = _all(*ins)
    leaves = [t.detach().requires_grad_(n) for t, n in zip(ins, need)]
    h = ops.gated_linear(*leaves)
    wanted = [t for t, n in zip(leaves, need) if n]
    got = iter(torch.autograd.grad(h, wanted, ins[3]))
    for n, grad in zip(need, whole[1:]):
        assert not n or torch.equal(next(got), grad)


def test_leading_dimensions_and_strides(cuda):
    x, wg, wu, dh = _inputs(120, 64, 72)
    whole = _all(x, wg, wu, dh)
    got = _all(x.view(2, 3, 20, 64), wg, wu, dh.view(2, 3, 20, 72))
    assert got[0].shape == (2, 3, 20, 72) and got[1].shape == (2, 3, 20, 64)
    assert all(torch.equal(a.view(b.shape), b) for a, b in zip(got, whole))
    wide = torch.zeros(120, 200, dtype=BF16, device="cuda")
    wide[:, 8:72] = x
    again = _all(wide[:, 8:72], wg, wu, dh)
    assert all(torch.equal(a, b) for a, b in zip(again, whole))
    # an incoming gradient of another layout, and one that is broadcast
    leaves = [t.detach().requires_grad_() for t in (x, wg, wu)]
    turned = dh.t().contiguous().t()
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(ops.gated_linear(*leaves), leaves, turned), whole[1:]))
    ones = _all(x, wg, wu, torch.ones_like(dh))
    ops.gated_linear(*leaves).sum().backward()
    assert all(torch.equal(t.grad, b) for t, b in zip(leaves, ones[1:]))


@pytest.mark.parametrize("M,E,I,dtype", [(5, 9, 16, BF16), (5, 16, 9, BF16), (6, 16, 24, torch.float32), (0, 16, 24, BF16), (4, 16, 8, torch.float16)])
def test_other_sizes_and_types_by_torch(cuda, M, E, I, dtype):
    ins = [t.to(dtype) for t in _inputs(M, E, I)]
    got = _all(*ins)
    leaves = [t.detach().requires_grad_() for t in ins[:3]]
    h = torch.nn.functional.silu(leaves[0] @ leaves[1].t()) * (leaves[0] @ leaves[2].t())
    want = (h.detach(), *torch.autograd.grad(h, leaves, ins[3]))
    for a, b in zip(got, want):
        assert a.dtype == dtype and a.shape == b.shape
        torch.testing.assert_close(a, b, rtol=2 * torch.finfo(dtype).eps, atol=4 * torch.finfo(dtype).eps)


def test_unaligned_rows_by_torch(cuda):
    x, wg, wu, dh = _inputs(9, 64, 72)
    flat = torch.zeros(9 * 64 + 1, dtype=BF16, device="cuda")
    moved = flat[1:].view(9, 64)
    moved.copy_(x)
    _check(_all(x, wg, wu, dh), x, wg, wu, dh)
    torch.testing.assert_close(ops.gated_linear(moved, wg, wu), ops.gated_linear(x, wg, wu), rtol=2 ** -6, atol=2 ** -6)


def test_python_path_is_the_same(cuda, monkeypatch):
    """Without the extension: the same kernels and results, forward and backward."""
    ins = _inputs(300, 264, 200)
    native = _all(*ins)
    monkeypatch.setattr(ops._host, "usable", lambda t: False)
    assert all(torch.equal(a, b) for a, b in zip(native, _all(*ins)))


def test_into_a_column_block(cuda):
    x, wg, wu, _ = _inputs(150, 64, 72)
    with torch.no_grad():
        want = ops.gated_linear(x, wg, wu)
    wide = torch.full((152, 200), 3.0, dtype=BF16, device="cuda")
    got = ops.gated_linear_into(wide[1:151, 64:136], x, wg, wu)
    assert torch.equal(got, want)
    wide[1:151, 64:136] = 3
    assert bool((wide == 3).all())
    out = torch.empty_like(want)
    wrong = [lambda: ops.gated_linear_into(out, x.float(), wg, wu), lambda: ops.gated_linear_into(out[:, :64], x, wg, wu),
             lambda: ops.gated_linear_into(out, x, wg, wu[:64]), lambda: ops.gated_linear_into(out, x.t().contiguous().t(), wg, wu),
             lambda: ops.gated_linear_into(out.cpu(), x, wg, wu), lambda: ops.gated_linear_into(out, x.clone().requires_grad_(), wg, wu),
             lambda: ops.gated_linear_into(wide[1:151, 63:135], x, wg, wu), lambda: ops.gated_linear_into(out, x[:, :60].contiguous(), wg[:, :60].contiguous(), wu[:, :60].contiguous())]
    for i, call in enumerate(wrong):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail(f"call {i} was not refused")


def test_saved_tensors_may_move(cuda):
    """What the forward keeps goes to the host and back (a saved-tensor hook) without changing a bit."""
    ins = _inputs(130, 64, 72)
    want = _all(*ins)
    with torch.autograd.graph.save_on_cpu():
        got = _all(*ins)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def _gates(values, ups, dhs):
    """Gates and ups that are exactly these numbers: x holds them beside ones and zeros."""
    n = len(values)
    x = torch.zeros(n, 8)
    x[:, 0], x[:, 1] = torch.tensor(values), torch.tensor(ups)
    wg, wu = torch.zeros(8, 8), torch.zeros(8, 8)
    wg[:, 0] = 1
    wu[:, 1] = 1
    return [t.to(BF16).cuda() for t in (x, wg, wu, torch.tensor(dhs)[:, None].expand(n, 8))]


def test_gates_of_any_size(cuda):
    """Factors far below the smallest number beside a large up, gates that saturate, the largest numbers."""
    gates = [-1e4, -190.0, -180.0, -120.0, -100.0, -90.0, -87.5, -86.0, -40.0, -1.0, -1e-30, 0.0, 1e-30, 1.0, 20.0, 88.0, 90.0, 200.0, 3e38, -3e38]
    for up in (1.0, -3e38, 1e-20):
        x, wg, wu, dh = _gates(gates, [up] * len(gates), [1e-3] * len(gates))
        leaves = [t.detach().requires_grad_() for t in (x, wg, wu)]
        h = ops.gated_linear(*leaves)
        dx = torch.autograd.grad(h, leaves[0], dh)[0]
        g64, u64 = x.double()[:, :1], x.double()[:, 1:2]
        s = torch.sigmoid(g64)
        want = (g64 * s * u64).expand(-1, 8)
        small = 2.0 ** -133                                      # half of bf16's smallest step
        over = want.abs() > 3.39e38
        assert bool(h.double()[over].isinf().all()) and bool((h.double()[over].sign() == want[over].sign()).all())
        assert bool(((h.double() - want).abs() <= (ref.HALF + ref.GATE) * want.abs() + small)[~over].all()), up
        du = (8 * dh.double()[:, :1] * g64 * s)[:, 0]            # the second column of dx: the sum of eight equal du
        off = (dx.double()[:, 1] - du).abs()
        assert bool((off <= 2.1 * (ref.HALF + ref.GATE) * du.abs() + 16 * small).all()), up


def test_products_next_to_the_largest_number(cuda):
    """Results that fp32 can hold beside products of some of their factors that it cannot: gate times up, dh times up, dh times gate, dh
    times the derivative, which is 1.1 at most and passes through zero near -1.28."""
    cases = [(1.203125, 3e38, 1e-3), (0.5, -3.3e38, 2.0), (2.0, 3.3e38, 1e-20), (1.203125, 1.0, 3e38), (0.01, 1.0, -3.3e38), (-1.25, 3e38, 8.0),
             (-1.28125, -3e38, 30.0), (2.40625, 0.5, 3.3e38), (2.40625, -1e-30, 3.3e38), (-0.5, 3.3e38, 3.0), (3e38, 1.1, 0.5), (3e38, 1.0, 1.1),
             (20.0, 3e38, 1.0), (-20.0, 3e38, 1e6)]
    g, u, d = (torch.tensor(c, dtype=torch.float64) for c in zip(*cases))
    x, wg, wu, dh = (torch.zeros(s, dtype=BF16, device="cuda") for s in ((len(cases), 8), (8, 8), (8, 8), (len(cases), 8)))
    x[:, 0], x[:, 1], dh[:, 0], wg[0, 0], wu[0, 1] = g.to(BF16), u.to(BF16), d.to(BF16), 1, 1       # one feature
    h, dx, _, _ = _all(x, wg, wu, dh)
    g, u, d = x[:, 0].double(), x[:, 1].double(), dh[:, 0].double()
    s = torch.sigmoid(g)
    f = 1 + g * (1 - s)
    lose = 1 + (1 + g.abs() * (1 - s)) / f.abs()         # what the derivative's difference makes of its terms' errors
    most = 3.39e38
    off = lambda got, want, err: (got.double() - want).abs() - err * want.abs() - 2.0 ** -133
    want = g * s * u
    assert bool((off(h[:, 0], want, ref.HALF + ref.GATE)[want.abs() <= most] <= 0).all())
    assert bool(h[:, 0][want.abs() > most].isinf().all()) and int((want.abs() > most).sum()) == 2
    dg, du = d * u * s * f, d * g * s
    fits = (dg.abs() <= most) & (du.abs() <= most)        # (where one is infinite, the other's column of dx is infinity times zero beside it)
    assert int(fits.sum()) == 11 and not bool(dx[~fits].isfinite().all(1).any())
    assert bool((off(dx[:, 0], dg, ref.HALF + ref.GATE * lose)[fits] <= 0).all())
    assert bool((off(dx[:, 1], du, ref.HALF + ref.GATE)[fits] <= 0).all())
    # dg where du alone is infinite: by the gate's weights
    x, dh = torch.zeros(1, 8, dtype=BF16, device="cuda"), torch.zeros(1, 8, dtype=BF16, device="cuda")
    x[0, 0], x[0, 1], x[0, 3], dh[0, 0] = 2.40625, 0.5, 2.0 ** -10, 3.3e38
    got = _all(x, wg, wu, dh)[2][0, 3].double()
    s = 1 / (1 + torch.exp(torch.tensor(-2.40625, dtype=torch.float64)))
    want = dh[0, 0].double() * 0.5 * s * (1 + 2.40625 * (1 - s)) * 2.0 ** -10
    assert abs(got - want) <= (2 * ref.HALF + 3 * ref.GATE + 2.0 ** -16) * want


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_not_finite(cuda, bad):
    """A row that holds an infinity or a NaN concerns itself alone in h and dx, and every weight's gradient that it touches."""
    x, wg, wu, dh = _inputs(300, 64, 40)
    whole = _all(x, wg, wu, dh)
    y = x.clone()
    y[131, 5] = bad
    h, dx, dwg, _ = _all(y, wg, wu, dh)
    others = torch.arange(300, device="cuda") != 131
    assert torch.equal(h[others], whole[0][others]) and torch.equal(dx[others], whole[1][others])
    assert not bool(h[131].isfinite().all()) and not bool(dwg[:, 5].isfinite().all())


@pytest.mark.parametrize("M", [1, 7, 8, 9, 31, 33, 120, 121, 127, 128, 129])
def test_few_rows(cuda, M):
    """Up to 128 rows are loaded alone: what larger calls left in shared memory, here NaN, reaches no result."""
    ins = _inputs(M, 264, 1368)
    big = [torch.full_like(t, float("nan")) for t in _inputs(40000, 264, 1368)]
    _all(*big)
    got = _all(*ins)
    _check(got, *ins)
    assert all(bool(t.isfinite().all()) for t in got)


# long axes over few tiles: in pieces, whose sums are joined; pieces of a different length, one and several tiles, ends inside a block
@pytest.mark.parametrize("M,E,I", [(65536, 8, 8), (9973, 64, 72), (3000, 128, 264), (30000, 520, 8), (5, 136, 20000), (300, 8, 5632), (129, 2048, 5632)])
def test_split_sums(cuda, M, E, I, monkeypatch):
    ins = _inputs(M, E, I)
    assert nat.lib().mvpa_gated_linear_bwd_workspace_bytes(M, E, I) > 0
    got = _all(*ins)
    _check(got, *ins)
    for _ in range(2):
        assert all(torch.equal(a, b) for a, b in zip(got, _all(*ins)))
    monkeypatch.setattr(ops._host, "usable", lambda t: False)
    assert all(torch.equal(a, b) for a, b in zip(got, _all(*ins)))


def test_workspace_is_looked_at(cuda):
    """Without a workspace nothing is split, and one that is too short or lies off a 16-byte boundary is refused."""
    M, E, I = 9973, 64, 72
    x, wg, wu, dh = _inputs(M, E, I)
    lib, need = nat.lib(), nat.lib().mvpa_gated_linear_bwd_workspace_bytes(M, E, I)
    h, saved = ops._gated_kernel(x, wg, wu, True)
    ws, dgate, dup, dx = torch.empty(need, dtype=torch.uint8, device="cuda"), torch.empty_like(dh), torch.empty_like(dh), torch.empty_like(x)
    dwg, dwu = torch.empty_like(wg), torch.empty_like(wu)
    call = lambda at, size: lib.mvpa_gated_linear_bwd(dh.data_ptr(), I, saved.data_ptr(), x.data_ptr(), E, wg.data_ptr(), wu.data_ptr(), dgate.data_ptr(),
                                                      dup.data_ptr(), dx.data_ptr(), dwg.data_ptr(), dwu.data_ptr(), M, E, I, at, size, None,
                                                      torch.cuda.current_stream().cuda_stream)
    for at, size in ((ws.data_ptr(), need - 1), (ws.data_ptr() + 8, need)):
        assert call(at, size) != 0 and "workspace" in nat.last_error()
    assert call(None, 0) == 0
    _check((h, dx, dwg, dwu), x, wg, wu, dh)


def test_second_derivative(cuda):
    x, wg, wu, dh = _inputs(6, 16, 24)
    leaves = [t.detach().requires_grad_() for t in (x, wg, wu)]
    dx = torch.autograd.grad(ops.gated_linear(*leaves), leaves[0], dh, create_graph=True)[0]
    got = torch.autograd.grad(dx.float().square().sum(), leaves)
    deep = [t.detach().double().requires_grad_() for t in leaves]
    dx64 = torch.autograd.grad(ref.forward(*deep), deep[0], dh.double(), create_graph=True)[0]
    want = torch.autograd.grad(dx64.square().sum(), deep)
    for a, b in zip(got, want):     # a chain of some ten steps in bf16, relative to the largest
        assert (a.double() - b).abs().max() <= 16 * ref.HALF * b.abs().max()


@pytest.mark.parametrize("M,E,I", [(6, 16, 24), (300, 264, 200)])
@pytest.mark.parametrize("autocast", [None, BF16, torch.float16])
def test_gradients_that_have_a_graph(cuda, M, E, I, autocast):
    """As near to 64 bits as those without (fp32 throughout, one rounding at the end: within the bounds of the kernels' sums alone), also where
    the backward runs inside an autocast region that the forward was outside of."""
    x, wg, wu, dh = _inputs(M, E, I, spread=3.0)
    leaves = [t.detach().requires_grad_() for t in (x, wg, wu)]
    h = ops.gated_linear(*leaves)
    with torch.autocast("cuda", dtype=autocast or BF16, enabled=autocast is not None):
        got = torch.autograd.grad(h, leaves, dh * 64, create_graph=True)
    assert all(t.dtype == BF16 and t.requires_grad for t in got)
    ins = [t.double() for t in (x, wg, wu, dh * 64)]
    small = [t.abs() for t in ins]                 # the sums of magnitudes: fp32 additions and some twenty roundings of 2^-24 on the way
    g, u = small[0] @ small[1].t(), small[0] @ small[2].t()
    s = small[3] * 1.5 * (1 + u) * (1 + g)
    sums = (s @ small[1] + s @ small[2], s.t() @ small[0], s.t() @ small[0])
    for a, b, size in zip(got, ref.gradients(*ins), sums):
        assert bool(((a.double() - b).abs() <= ref.HALF * b.abs() + (M + E + 2 * I + 20) * ref.CUT * size).all())


def test_graph_capture_of_a_step(cuda):
    """Forward and backward in one captured graph, replayed on new inputs."""
    x, wg, wu, dh = _inputs(500, 264, 136)
    leaves = [t.detach().clone().requires_grad_() for t in (x, wg, wu)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    step = lambda: (lambda h: (h.detach(), *torch.autograd.grad(h, leaves, dh)))(ops.gated_linear(*leaves))
    check, ops._attn._CHECK_STATUS = ops._attn._CHECK_STATUS, False
    try:
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
    finally:
        ops._attn._CHECK_STATUS = check
    x2 = _inputs(500, 264, 136, seed=5)[0]
    with torch.no_grad():
        leaves[0].copy_(x2)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, _all(x2, wg, wu, dh)))


def test_streams_and_threads(cuda):
    """Four threads on streams of their own, many calls each, with results that no other call changes."""
    cases = [_inputs(200 + 100 * i, 256, 136, seed=i) for i in range(4)]
    alone = [_all(*c) for c in cases]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got = _all(*cases[i])
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, alone[i])):
                    bad.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not bad


def test_offsets_past_32_bits(cuda):
    M, E, I = 420000, 16, 5632                                   # M I > 2^31 elements
    x, wg, wu, _ = _inputs(64, E, I)
    x = x.repeat(M // 64 + 1, 1)[:M].contiguous()
    dh = torch.zeros(M, I, dtype=BF16, device="cuda")
    dh[-64:] = 0.1
    h, dx, dwg, dwu = _all(x, wg, wu, dh)
    last = x[-64:].contiguous()
    small = _all(last, wg, wu, dh[-64:].contiguous())
    assert torch.equal(h[-64:], small[0])                        # (the sums of dx are split by the number of rows)
    _check((h[-64:], dx[-64:], *small[2:]), last, wg, wu, dh[-64:].contiguous())
    assert not bool(dx[:-64].any())
    _check((h[-64:], dx[-64:], dwg, dwu), last, wg, wu, dh[-64:])
