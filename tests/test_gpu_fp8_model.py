"""GPU: the inference block and model with their projections in 8 bits (`MVPFormerModel.enable_fp8`): one block against the same
chain of definitions in 64 bits, the model against itself in bf16, graphs, changed weights and refusals."""
import pytest
import torch

import fp8_oracle as ref
import models
import mvpa_ops as ops
from attentions import attn, flash_mvpa

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def _model(dtype, width=256, heads=4, kv=2, inner=352, layers=2, seed=0):
    torch.manual_seed(seed)
    cfg = models.MVPFormerConfig(n_positions=16, n_channels=16, n_embd=width, n_layer=layers, n_head=heads, n_head_kv=kv, n_inner=inner,
                                 resid_pdrop=0.0, embd_pdrop=0.0, attn_pdrop=0.0, initializer_range=0.05)
    return models.MVPFormerModel(cfg).to("cuda", dtype).eval()


def _embeds(dtype, B=2, T=7, C=9, width=256, seed=1):
    return torch.randn(B, T, C, width, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("inner", [352, 200])
def test_block_against_the_definitions(cuda, dtype, inner):
    """The chain norm, product, attention, quantisation | gate, product, with every rounding to `dtype` where the block rounds and
    the attention by the operator itself."""
    B, T, C, E, H, Hkv, D = 2, 7, 9, 256, 4, 2, 64
    m = _model(dtype, inner=inner)
    block, N, KV, I = m.h[0], T * C, Hkv * D, inner
    h = _embeds(dtype).view(-1, E)
    rt, rc = (torch.randn(Hkv, n, D, generator=torch.Generator().manual_seed(n)).to(dtype).cuda() * 0.3 for n in (T, C))
    with torch.no_grad():
        pair = ops.rmsnorm_fp8(h, block.ln_1.weight, 1e-5)
        got = block.fused_branches_fp8(pair, rt, rc, B, T, C, dtype)
        a, mlp = block.attn, block.mlp
        w_in = torch.cat([a.q_attn.weight, a.c_attn.weight, mlp.gate_proj.weight, mlp.up_proj.weight])
        w_out = torch.cat([a.c_proj.weight, mlp.down_proj.weight], 1)
        big = (ref.value(*pair) @ ref.value(*ref.pair(w_in, 128), 128).t()).to(dtype)
        head = lambda c, n: big[:, c:c + n * D].view(B, N, n, D).permute(0, 2, 1, 3)
        u, vt, z = (b.view(1, Hkv, 1, D).to(dtype) for b in a.attn_bias.split(KV))
        att = flash_mvpa(head(0, H), u, vt, z, head(E, Hkv), rt[None], rc[None], head(E + KV, Hkv), True, D ** -0.5, 10)
        att = att.permute(0, 2, 1, 3).reshape(B * N, E)
        g, up = big[:, E + 2 * KV:E + 2 * KV + I].double(), big[:, E + 2 * KV + I:].double()
        (qa, sa), (qg, sg) = ref.pair(att), ref.pair(g * torch.sigmoid(g) * up)
        mixed = torch.cat([ref.value(qa, sa), ref.value(qg, sg)], 1)
        want = mixed @ ref.value(*ref.pair(w_out, 128), 128).t()
    # Where the first product's sums (fp32 against fp64) fall on two sides of a rounding border to bf16 - some 1e-3 of them - a value
    # moves by 2^-8, and one in twenty of those to another e4m3 value, by a tenth: 7e-4 of the result's norm at most; in fp32 the
    # values themselves move by some 1e-6 and one in 1e5 to another e4m3 value.  The result's own rounding in bf16: 2^-8 at most.
    rel = float((got.double() - want).norm() / want.norm())
    assert rel <= (2.0 ** -8 + 7e-4 if dtype == BF16 else 7e-4), rel


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("inner", [352, 200, 201])
def test_native_call_and_python_path_agree(cuda, dtype, inner, monkeypatch):
    import mvpa_host
    m, x = _model(dtype, inner=inner).enable_fp8(), _embeds(dtype)
    with torch.no_grad():
        native = m(inputs_embeds=x).last_hidden_state.clone()
        monkeypatch.setattr(mvpa_host, "usable", lambda t: False)
        assert torch.equal(m(inputs_embeds=x).last_hidden_state, native)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_model_near_itself_in_16_bits(cuda, dtype):
    m, x = _model(dtype), _embeds(dtype)
    with torch.no_grad():
        plain = m(inputs_embeds=x).last_hidden_state
        assert m.enable_fp8() is m
        eight = m(inputs_embeds=x).last_hidden_state
        assert torch.equal(m.enable_fp8(False)(inputs_embeds=x).last_hidden_state, plain)
    # Operands in e4m3 have a relative error of 2^-4 / sqrt(3) = 3.6 % in the mean at most, both operands of a product 5.1 %; two
    # products after one another, where the gate at most doubles the first one's, 15 % of the branches, which are added to the
    # residual stream: less than that of the sum's norm
    rel = float((eight.double() - plain.double()).norm() / plain.double().norm())
    assert 1e-4 < rel <= 0.15, rel


def test_graph_weights_and_training(cuda):
    m = _model(BF16).enable_fp8()
    xs = [_embeds(BF16, seed=s) for s in (1, 2)]
    with torch.no_grad():
        want = [m(inputs_embeds=x).last_hidden_state.clone() for x in xs]
        m.enable_cuda_graph()
        for x, y in zip(xs, want):
            assert torch.equal(m(inputs_embeds=x).last_hidden_state, y)
        m.enable_cuda_graph(False)
        m.h[0].mlp.down_proj.weight.mul_(2.0)                            # a changed weight is quantised again
        changed = m(inputs_embeds=xs[0]).last_hidden_state
        assert not torch.equal(changed, want[0])
        m.h[0].mlp.down_proj.weight.mul_(0.5)
        assert torch.equal(m(inputs_embeds=xs[0]).last_hidden_state, want[0])
    # with gradients the blocks run as ever
    x = xs[0].clone().requires_grad_()
    out = m(inputs_embeds=x).last_hidden_state
    out.float().square().sum().backward()
    again = _model(BF16)
    x2 = xs[0].clone().requires_grad_()
    out2 = again(inputs_embeds=x2).last_hidden_state
    out2.float().square().sum().backward()
    assert torch.equal(out, out2) and torch.equal(x.grad, x2.grad)


def test_model_refusals(cuda):
    with pytest.raises(ValueError, match="multiple of 128"):
        _model(BF16, width=64, heads=1, kv=1).enable_fp8()
    m = _model(BF16).enable_fp8()
    with pytest.raises(NotImplementedError, match="8 bits"):
        m.forward_time_sharded(torch.zeros(4, 256, device="cuda", dtype=BF16), 2, 2)


@pytest.mark.parametrize("fp8", [False, True])
def test_weights_prepared_on_one_stream_are_read_on_another(cuda, fp8):
    """The first call makes the concatenated (and quantised) weights on its stream, behind other work; a call on another stream right
    after it finds them finished."""
    m, x = _model(BF16).enable_fp8(fp8), _embeds(BF16)
    with torch.no_grad():
        want = _model(BF16).enable_fp8(fp8)(inputs_embeds=x).last_hidden_state
        torch.cuda.synchronize()
        one, two = torch.cuda.Stream(), torch.cuda.Stream()
        got = []
        for stream in (one, two, one):
            with torch.cuda.stream(stream):
                if not got:
                    torch.cuda._sleep(20_000_000)                        # some 10 ms
                got.append(m(inputs_embeds=x).last_hidden_state)
        torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


@pytest.mark.parametrize("fp8", [False, True])
def test_a_capture_without_a_call_before_it_keeps_nothing(cuda, fp8, monkeypatch):
    """Weights that a capture makes exist only after a replay: calls outside the graph make their own."""
    monkeypatch.setattr(attn, "_CHECK_STATUS", False)                    # (reading a status word back is not for captures)
    m, x = _model(BF16).enable_fp8(fp8), _embeds(BF16)
    with torch.no_grad():
        want = _model(BF16).enable_fp8(fp8)(inputs_embeds=x).last_hidden_state
        torch.cuda.synchronize()
        graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(graph, stream=side):
            captured = m(inputs_embeds=x).last_hidden_state
        assert torch.equal(m(inputs_embeds=x).last_hidden_state, want)
        graph.replay()
        assert torch.equal(captured, want)


@pytest.mark.parametrize("fp8", [False, True])
def test_a_graph_keeps_the_weights_that_it_reads(cuda, fp8):
    """Graphs are for frozen weights; one that is replayed after some have changed all the same reads those that were prepared for
    it, also when another shape's capture has prepared them anew and their old memory could have gone to something else."""
    m, x, y = _model(BF16).enable_fp8(fp8), _embeds(BF16), _embeds(BF16, T=5)
    with torch.no_grad():
        m.enable_cuda_graph()
        want = m(inputs_embeds=x).last_hidden_state.clone()
        kept = [t.data_ptr() for entry in m._kept() for t in entry[1]]
        for block in m.h:
            block.mlp.down_proj.weight.mul_(2.0)
            block.attn.position_net.weight.mul_(2.0)
        other = m(inputs_embeds=y).last_hidden_state.clone()
        others = torch.full((1 << 20,), 0x7f, dtype=torch.uint8, device="cuda"), [torch.full((n,), 3e38, device="cuda") for n in range(1000, 200000, 1999)]
        assert not set(kept) & {t.data_ptr() for entry in m._kept() for t in entry[1]}
        assert torch.equal(m(inputs_embeds=x).last_hidden_state, want)
        fresh = m.enable_cuda_graph(False)(inputs_embeds=y).last_hidden_state
    del others
    assert torch.equal(fresh, other)
