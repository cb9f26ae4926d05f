"""GPU: the block and the model with the fused gate (`enable_fused_gate`) and with weights in 4 bits (`enable_int4`), in training and
inference, native and through Python, in graphs, after their weights change, copied and refused."""
import copy

import pytest
import torch
import torch.nn.functional as F

import models
import mvpa_native as nat
import mvpa_ops as ops

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def _model(dtype, width=256, heads=4, kv=2, inner=352, layers=2, seed=0, **rates):
    torch.manual_seed(seed)
    cfg = models.MVPFormerConfig(n_positions=16, n_channels=16, n_embd=width, n_layer=layers, n_head=heads, n_head_kv=kv, n_inner=inner,
                                 **{**dict(resid_pdrop=0.0, embd_pdrop=0.0, attn_pdrop=0.0, initializer_range=0.05), **rates})
    return models.MVPFormerModel(cfg).to("cuda", dtype).eval()


def _embeds(dtype, B=2, T=7, C=9, width=256, seed=1):
    return torch.randn(B, T, C, width, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def _rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


@torch.no_grad()
def _run(m, x):
    return m(inputs_embeds=x).last_hidden_state


@torch.no_grad()
def _weights_that_stand_for(m, group, zeros):
    """The model with every projection of its blocks as what its 4 bits stand for (in fp32; concatenated as the blocks do it)."""
    wide = copy.deepcopy(m).float()
    for block, src in zip(wide.h, m.h):
        a, mlp = block.attn, block.mlp
        back = lambda w: ops.dequantize_int4(*ops.quantize_int4(w, group, zeros), width=w.shape[1], group=group, dtype=F32)
        qkv = back(torch.cat([src.attn.q_attn.weight, src.attn.c_attn.weight]))
        out = back(torch.cat([src.attn.c_proj.weight, src.mlp.down_proj.weight], 1))
        n, E = a.q_attn.weight.shape
        a.q_attn.weight.copy_(qkv[:n])
        a.c_attn.weight.copy_(qkv[n:])
        mlp.gate_proj.weight.copy_(back(src.mlp.gate_proj.weight))
        mlp.up_proj.weight.copy_(back(src.mlp.up_proj.weight))
        a.c_proj.weight.copy_(out[:, :n])
        mlp.down_proj.weight.copy_(out[:, n:])
    return wide


# ---- 4 bits ----

@pytest.mark.parametrize("group,zeros", [(128, False), (64, True), (32, False)])
@pytest.mark.parametrize("inner", [352, 200])
@pytest.mark.parametrize("shape", [(1, 1, 3), (2, 7, 9), (3, 16, 16)])
def test_int4_is_the_model_of_the_weights_it_stands_for(cuda, group, zeros, inner, shape):
    """fp32: few rows, some, many.  No weight is rounded in the products, so the two models differ by fp32 roundings alone: some 400
    products to a sum, two blocks and the attention's exponentials, far below 2^-13 of the hidden state."""
    m = _model(F32, inner=inner).enable_int4(group=group, zeros=zeros)
    x = _embeds(F32, *shape)
    assert _rel(_run(m, x), _run(_weights_that_stand_for(m, group, zeros), x)) < 2.0 ** -13


@pytest.mark.parametrize("inner", [352, 200])
def test_int4_in_bf16(cuda, inner):
    """Against the fp32 model of the same weights: a block rounds to bf16 at some ten places, 2^-8 relative each at most."""
    m = _model(BF16, inner=inner).enable_int4()
    x = _embeds(BF16)
    assert _rel(_run(m, x), _run(_weights_that_stand_for(m, 128, False), x.float())) < 20 * 2.0 ** -8


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("inner", [352, 200, 201])
@pytest.mark.parametrize("zeros", [False, True])
def test_int4_native_and_python_paths_agree(cuda, dtype, inner, zeros, monkeypatch):
    m = _model(dtype, inner=inner).enable_int4(group=64, zeros=zeros)
    x = _embeds(dtype)
    native = _run(m, x)
    monkeypatch.setattr(models.mvpformer.mvpa_host, "usable", lambda t: False)
    assert torch.equal(native, _run(m, x))


def test_int4_runs_its_kernels(cuda):
    """A block is the norm, two products, the gate, and the attention: five launches and the attention's own, and the last norm."""
    m, x = _model(BF16, layers=3), _embeds(BF16, 1, 2, 5)
    _run(m, x)
    m.enable_int4()
    _run(m, x)
    before = nat.lib().mvpa_launch_count()
    _run(m, x)
    per_block = (nat.lib().mvpa_launch_count() - before - 1) / 3
    assert per_block in (5, 6)


def test_int4_graph_and_changed_weights(cuda, monkeypatch):
    monkeypatch.setattr(models.mvpformer.attn_mod, "_CHECK_STATUS", False)
    m = _model(BF16).enable_int4()
    x, y = _embeds(BF16), _embeds(BF16, seed=5)
    want = _run(m, x), _run(m, y)
    m.enable_cuda_graph()
    assert torch.equal(_run(m, x), want[0]) and torch.equal(_run(m, y), want[1])
    assert len(m._graphs) == 1
    m.enable_cuda_graph(False)
    with torch.no_grad():
        m.h[0].mlp.gate_proj.weight.mul_(1.5)
    changed = _run(m, x)
    assert not torch.equal(changed, want[0])
    assert torch.equal(changed, _run(copy.deepcopy(m), x))
    other = _run(m.enable_int4(group=32), x)
    assert not torch.equal(other, changed)
    assert torch.equal(_run(m.enable_int4(), x), changed)
    m.enable_int4(False)
    plain = copy.deepcopy(m)
    plain._int4 = None
    assert torch.equal(_run(m, x), _run(plain, x))


def test_int4_and_fp8_take_turns(cuda):
    m, x = _model(BF16), _embeds(BF16)
    plain = _run(m, x)
    in8 = _run(m.enable_fp8(), x)
    in4 = _run(m.enable_int4(), x)
    assert m._fp8 is False and not torch.equal(in4, in8)
    assert torch.equal(_run(m.enable_fp8(), x), in8) and m._int4 is None
    assert torch.equal(_run(m.enable_fp8(False), x), plain)
    # a training pass knows neither
    m.enable_int4()
    h = m(inputs_embeds=x).last_hidden_state
    m.enable_int4(False)
    assert torch.equal(h, m(inputs_embeds=x).last_hidden_state)


def test_int4_refusals(cuda):
    m = _model(BF16)
    with pytest.raises(ValueError):
        m.enable_int4(group=16)
    with pytest.raises(NotImplementedError):
        m.enable_int4().forward_time_sharded(_embeds(BF16).view(-1, 256), 7, 9)


# ---- the fused gate ----

def _grads(m, x, weight):
    leaf = x.detach().clone().requires_grad_()
    h = m(inputs_embeds=leaf).last_hidden_state
    params = [p for n, p in m.named_parameters() if "ln_2" not in n]
    return h.detach(), *torch.autograd.grad(h, [leaf, *params], weight)


@pytest.mark.parametrize("hook", [False, True])
def test_fused_gate_trains(cuda, hook):
    """One function per block, and (a hook) through the modules: hidden state and every gradient against the fp32 model's; some ten
    roundings of a block to bf16 on the way there and as many back, 2^-8 each at most, and no larger than without the flag but for as much."""
    m = _model(BF16).train().enable_fused_gate()
    if hook:
        for block in m.h:
            block.ln_1.register_forward_hook(lambda *_: None)
    x, weight = _embeds(BF16), _embeds(BF16, seed=9)
    wide = copy.deepcopy(m).float().enable_fused_gate(False)
    want = _grads(wide, x.float(), weight.float())
    launched = nat.lib().mvpa_launch_count()
    got = _grads(m, x, weight)
    fused = nat.lib().mvpa_launch_count() - launched
    plain = _grads(m.enable_fused_gate(False), x, weight)
    assert fused != nat.lib().mvpa_launch_count() - launched - fused          # (other kernels ran)
    for a, b, c in zip(got, plain, want):
        assert _rel(a, c) < 40 * 2.0 ** -8 and _rel(a, c) < _rel(b, c) + 4 * 2.0 ** -8


def test_fused_gate_same_bits_through_modules_and_function(cuda):
    """The block as one function and as modules form the gate's projection with the same kernels."""
    m = _model(BF16, layers=1).train().enable_fused_gate()
    block, x = m.h[0], _embeds(BF16)
    act = block.mlp.down_proj
    xn = ops.rmsnorm_train(x, block.ln_1.weight, block.ln_1.eps)
    mlp = block.mlp(xn)
    assert torch.equal(mlp, F.linear(ops.gated_linear(xn, block.mlp.gate_proj.weight, block.mlp.up_proj.weight), act.weight))


def test_fused_gate_second_derivative(cuda):
    """Of one block (the model's own last norm would make a sum of squares a constant, whose derivatives are roundings alone)."""
    m = _model(BF16, layers=1).train().enable_fused_gate()
    wide = copy.deepcopy(m).float().enable_fused_gate(False)
    x, weight = _embeds(BF16, 1, 3, 4), _embeds(BF16, 1, 3, 4, seed=7)
    second = []
    for model, dtype in ((m, BF16), (wide, F32)):
        leaf = x.detach().to(dtype).requires_grad_()
        pos, chan = model.positional_embedding.weight[None, :3], model.channel_embedding.weight[None, :4]
        h = model.h[0](leaf, pos, chan)[0]
        g = torch.autograd.grad((h.float() * weight.float()).sum(), leaf, create_graph=True)[0]
        second.append(torch.autograd.grad((g.float() * weight.float()).square().sum(), leaf)[0])
    assert _rel(*second) < 100 * 2.0 ** -8      # (a chain of some fifty roundings, 2^-8 each at most, and their carries)


@pytest.mark.parametrize("inner", [352, 200, 201])
def test_fused_gate_inference(cuda, inner, monkeypatch):
    """Native and through Python alike; graphs; what the kernel does not take (an odd width) is as without the flag."""
    monkeypatch.setattr(models.mvpformer.attn_mod, "_CHECK_STATUS", False)
    m, x = _model(BF16, inner=inner), _embeds(BF16)
    plain = _run(m, x) if inner != 201 else None
    if inner == 201:
        monkeypatch.setattr(models.mvpformer.mvpa_host, "usable", lambda t: False)
        with pytest.raises(RuntimeError):
            _run(m, x)                                # (16-byte rows of the gate, as before)
        return
    native = _run(m.enable_fused_gate(), x)
    wide = _run(copy.deepcopy(m).float(), x.float())
    assert _rel(native, wide) < _rel(plain, wide) + 4 * 2.0 ** -8 and not torch.equal(native, plain)
    m.enable_cuda_graph()
    assert torch.equal(_run(m, x), native)
    m.enable_cuda_graph(False)
    monkeypatch.setattr(models.mvpformer.mvpa_host, "usable", lambda t: False)
    assert torch.equal(_run(m, x), native)


def test_fused_gate_other_types_and_autocast(cuda):
    m, x = _model(F32), _embeds(F32)
    plain = _run(m, x)
    assert torch.equal(_run(m.enable_fused_gate(), x), plain)
    with torch.autocast("cuda", dtype=BF16):          # (through the modules)
        auto = m(inputs_embeds=x).last_hidden_state
        assert torch.equal(auto, m.enable_fused_gate(False)(inputs_embeds=x).last_hidden_state)


@pytest.mark.parametrize("dtype,inner,autocast", [(F32, 352, False), (F32, 352, True), (torch.float16, 352, False), (BF16, 204, False)])
def test_fused_gate_changes_nothing_else(cuda, dtype, inner, autocast):
    """Other types, autocast and widths that the kernel does not take, through the modules: the bits and the launches of a model without the flag."""
    m = _model(dtype, inner=inner).train()
    m.h[0].ln_1.register_forward_hook(lambda *_: None)
    mlp, x = m.h[0].mlp, _embeds(dtype).requires_grad_()
    got = []
    for flag in (False, True):
        m.enable_fused_gate(flag)
        launched = nat.lib().mvpa_launch_count()
        with torch.autocast("cuda", dtype=BF16, enabled=autocast):
            y = mlp(x)
        grads = torch.autograd.grad(y.float().square().sum(), [x, *mlp.parameters()])
        got.append((nat.lib().mvpa_launch_count() - launched, y, *grads))
    assert got[0][0] == got[1][0] and all(torch.equal(a, b) for a, b in zip(got[0][1:], got[1][1:]))


def _sharded_worker(rank, port, path):
    import os
    import torch.distributed as dist
    os.environ["MASTER_ADDR"], os.environ["MASTER_PORT"] = "127.0.0.1", str(port)
    dist.init_process_group("nccl", rank=0, world_size=1, device_id=torch.device("cuda:0"))
    try:
        m, x = _model(BF16), _embeds(BF16, B=1)
        same = []
        for flag in (True, False):
            m.enable_fused_gate(flag)
            same.append(torch.equal(m.forward_time_sharded(x.view(-1, 256), 7, 9, transport="nccl"), _run(m, x).view(-1, 256)))
        torch.save(same, path)
    finally:
        dist.destroy_process_group()


def test_time_sharded_forward_with_the_fused_gate(cuda, tmp_path):
    """One rank that holds the whole sample: the same kernels on the same rows, hence the plain forward's bits, with the flag and without."""
    import os
    import torch.multiprocessing as mp
    path = str(tmp_path / "same")
    mp.spawn(_sharded_worker, args=(29500 + os.getpid() % 2000, path), nprocs=1, join=True)
    assert torch.load(path) == [True, True]


def test_training_step_in_a_graph(cuda, monkeypatch):
    """Forward, loss and gradients of a fused-gate model captured once and replayed on another batch."""
    monkeypatch.setattr(models.mvpformer.attn_mod, "_CHECK_STATUS", False)
    m = _model(BF16).train().enable_fused_gate()
    x, weight = _embeds(BF16), _embeds(BF16, seed=9)
    params = [p for n, p in m.named_parameters() if "ln_2" not in n]
    static = x.clone()

    def step():
        h = m(inputs_embeds=static).last_hidden_state
        return (h.detach(), *torch.autograd.grad(h, params, weight))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    static.copy_(_embeds(BF16, seed=3))
    graph.replay()
    torch.cuda.synchronize()
    kept = [t.clone() for t in out]
    assert all(torch.equal(a, b) for a, b in zip(kept, step()))


def test_copies_and_pickles(cuda):
    import io
    m, x = _model(BF16).enable_int4().enable_fused_gate(), _embeds(BF16)
    want = _run(m, x)
    buf = io.BytesIO()
    torch.save(m, buf)
    buf.seek(0)
    again = torch.load(buf, weights_only=False)
    assert again.h[0]._fused_int4 is None and torch.equal(_run(again, x), want)
