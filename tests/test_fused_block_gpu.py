"""The fused operators as a model runs them: a feed-forward block of two packed
layers and a norm against its 64-bit form, transformers' BERT and Llama with
fused epilogues against the same models without."""
import pytest
import torch

import packr_b200 as packr
from fused_reference import act64, weights64

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def rel(a, b):
    return float((a.detach().double() - b.double()).norm() / b.double().norm())


@pytest.mark.parametrize("M", [1, 3, 40, 300])
@pytest.mark.parametrize("prenorm", [False, True])
def test_feed_forward_block(cuda, M, prenorm):
    """h = down(gelu(up(x))); post-norm: norm(h + x); pre-norm: norm first, then
    h + x in the down projection's epilogue.  bf16 throughout.

    Every stored bf16 tensor on the way costs at most 2^-8 / sqrt(3) = 2.3e-3 of
    its 2-norm; the longest path (forward to the upstream gradient's way back:
    up, down, norm, dz twice, dx twice) has eight, and a factor 2 covers the
    norm's and the activation's slopes: 2 * sqrt(8) * 2.3e-3 = 1.3e-2."""
    K, H = 192, 512
    up = packr.PackRLinear.synthetic(K, H, seed=1, lut_std=0.05, wf_std=0.005)
    down = packr.PackRLinear.synthetic(H, K, seed=2, lut_std=0.05, wf_std=0.005)
    for lin in (up, down):
        lin.out_dtype = BF16
        lin.lut.requires_grad_(False)
        torch.nn.init.normal_(lin.bias_f, std=0.2)
    up.activation = "gelu"
    norm = packr.PackRLayerNorm(K, dtype=BF16, device="cuda")
    torch.nn.init.normal_(norm.weight, 1.0, 0.1)
    torch.nn.init.normal_(norm.bias, 0.0, 0.1)
    g = torch.Generator(device="cuda").manual_seed(M)
    x = torch.randn(M, K, generator=g, device="cuda").bfloat16().requires_grad_(True)
    dy = torch.randn(M, K, generator=g, device="cuda").bfloat16()
    params = [up.W_f, up.bias_f, down.W_f, down.bias_f, norm.weight, norm.bias]
    y = down(up(norm(x)), residual=x) if prenorm else norm(down(up(x)), residual=x)
    got = torch.autograd.grad(y, [x] + params, dy)

    d = lambda t: t.detach().double().requires_grad_(True)  # noqa: E731
    x64, b1, b2, nw, nb = d(x), d(up.bias_f), d(down.bias_f), d(norm.weight), d(norm.bias)
    w1 = weights64(up.W_p, up.W_f, up.lut).requires_grad_(True)
    w2 = weights64(down.W_p, down.W_f, down.lut).requires_grad_(True)

    def ln(s):
        c = s - s.mean(1, keepdim=True)
        return c / torch.sqrt((c * c).mean(1, keepdim=True) + 1e-5) * nw + nb

    ffn = lambda t: act64(t @ w1 + b1, "gelu") @ w2 + b2  # noqa: E731
    ref = ffn(ln(x64)) + x64 if prenorm else ln(ffn(x64) + x64)
    want = torch.autograd.grad(ref, [x64, w1, b1, w2, b2, nw, nb], dy.double())
    assert rel(y, ref.detach()) < 1.3e-2
    for name, a, b in zip(("x", "W_f up", "bias up", "W_f down", "bias down", "norm weight", "norm bias"), got, want):
        assert rel(a, b) < 1.3e-2, name


def test_bert_with_fused_epilogues(cuda):
    """Same logits and gradients as the unfused model up to rounding: f32
    activations, bf16 operands in both (a rounding that falls the other way
    moves an operand by 2^-8 of itself)."""
    from packr_b200 import workloads as wl
    models = [wl.bert_classifier(cuda, layers=2, seed=0, fused=f).eval() for f in (False, True)]
    assert sum(isinstance(m, packr.PackRAddNorm) for m in models[1].modules()) == 4
    models[1].load_state_dict(models[0].state_dict())
    ids, labels = wl.bert_batch(cuda, batch=4, seq=32)
    outs = []
    for m in models:
        out = m(input_ids=ids, labels=labels)
        out.loss.backward()
        outs.append(out)
    assert rel(outs[1].logits, outs[0].logits.detach()) < 2e-2
    grads = [dict(m.named_parameters()) for m in models]
    for name, p in grads[0].items():
        if p.grad is not None and float(p.grad.norm()) > 1e-6:
            assert rel(grads[1][name].grad, p.grad) < 5e-2, name
    models[1].train()  # dropout between the layer and the norm
    models[1](input_ids=ids, labels=labels).loss.backward()


def test_llama_with_fused_epilogues(cuda):
    from packr_b200 import workloads as wl
    sizes = dict(hidden_size=256, intermediate_size=512, num_attention_heads=4, num_key_value_heads=2, vocab_size=1024)
    models = [wl.llama_decoder("cuda", layers=2, seed=0, fused=f, **sizes).eval() for f in (False, True)]
    gates = [m for n, m in models[1].named_modules() if n.endswith("gate_proj")]
    assert gates and all(g.activation == "silu" and g.out_dtype == BF16 for g in gates)
    ids = wl.llama_batch("cuda", seq=64, vocab=1024)
    outs = [m(input_ids=ids, labels=ids) for m in models]
    for o in outs:
        o.loss.backward()
    assert rel(outs[1].logits, outs[0].logits.detach()) < 2e-2
    for (n, p), (_, q) in zip(models[0].named_parameters(), ((n.replace(".inner", ""), p) for n, p in models[1].named_parameters())):
        if p.grad is not None and float(p.grad.float().norm()) > 1e-6:
            assert rel(q.grad, p.grad) < 6e-2, n


def test_training_step_with_the_8_bit_optimizer(cuda):
    """The gradients of fused layers reach CUDA8BitAdam as the plain ones do."""
    from packr_b200.cuda_adam import CUDA8BitAdam
    up = packr.PackRLinear.synthetic(128, 256, seed=1)
    up.activation = "silu"
    norm = packr.PackRLayerNorm(256, device="cuda")
    params = [p for m in (up, norm) for p in m.parameters() if p.requires_grad]
    opt = CUDA8BitAdam(params, lr=1e-3)
    x = torch.randn(64, 128, device="cuda")
    before = [p.detach().clone() for p in params]
    norm(up(x)).square().mul(torch.randn(64, 256, device="cuda")).sum().backward()
    opt.step()
    assert all(torch.isfinite(p).all() and not torch.equal(p, b) for p, b in zip(params, before))


def test_layer_attributes_change_the_route_only(cuda):
    lin = packr.PackRLinear.synthetic(96, 160, seed=3)
    x = torch.randn(2, 9, 96, device="cuda").bfloat16()
    plain = lin(x)
    assert plain.dtype == F32 and plain.shape == (2, 9, 160)
    r = torch.randn(2, 9, 160, device="cuda")
    assert torch.allclose(lin(x, residual=r), plain + r, rtol=1e-5, atol=1e-5)
    lin.activation = "relu"
    assert torch.allclose(lin(x), plain.clamp_min(0), rtol=1e-5, atol=1e-5)
    lin.activation, lin.out_dtype = None, BF16
    assert torch.allclose(lin(x).float(), plain, rtol=2.0 ** -8, atol=1e-5)
    assert torch.equal(lin(x.half()), lin(x.half().float()))


@pytest.mark.parametrize("dense,given", [(BF16, F32), (F32, BF16), (torch.float16, F32), (torch.float16, torch.float16)])
def test_add_norm_of_mixed_types(cuda, dense, given):
    """The sum is taken in the wider type: a residual stream of f32 is not rounded
    to a bf16 projection's type.  f32 sums of 64 terms: 1e-5 covers them."""
    from packr_b200.layer_patcher import PackRAddNorm
    lin = torch.nn.Linear(64, 64, device="cuda", dtype=dense)
    norm = torch.nn.LayerNorm(64, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(5, 64, generator=g, device="cuda").to(dense)
    r = torch.randn(5, 64, generator=g, device="cuda").to(given)
    got = PackRAddNorm(lin, norm)(x, r)
    want = norm(lin(x).float() + r.float())
    assert got.dtype == F32 and torch.allclose(got, want, rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("M", [1, 2, 8, 40, 200])
def test_chain_of_overlapped_launches(cuda, M):
    """Eight pre-norm blocks in a row, each kernel reading what the one before it
    wrote: in a stream, in a graph and with a synchronisation after every call the
    results are the same bits, also right after the input and a weight were
    overwritten in place."""
    K, H = 512, 2048
    ups = [packr.PackRLinear.synthetic(K, H, seed=i, lut_std=0.05, wf_std=0.005) for i in range(8)]
    downs = [packr.PackRLinear.synthetic(H, K, seed=50 + i, lut_std=0.02, wf_std=0.005) for i in range(8)]
    for lin in ups + downs:
        lin.out_dtype = BF16
    for lin in ups:
        lin.activation = "silu"
    norms = [packr.PackRLayerNorm(K, dtype=BF16, device="cuda") for _ in range(8)]
    g = torch.Generator(device="cuda").manual_seed(M)
    xs = [torch.randn(M, K, generator=g, device="cuda").bfloat16() for _ in range(3)]
    x = xs[0].clone()

    @torch.no_grad()
    def chain(each=lambda: None):
        h = x
        for norm, up, down in zip(norms, ups, downs):
            n = norm(h)
            each()
            a = up(n)
            each()
            h = down(a, residual=h)
            each()
        return h

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        chain()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = chain()
    for new in xs:
        with torch.no_grad():
            norms[0].weight.mul_(1.25)
            ups[3].W_f.mul_(1.5)
        x.copy_(new)
        got = [chain() for _ in range(3)]
        graph.replay()
        got.append(out.clone())
        torch.cuda.synchronize()
        want = chain(torch.cuda.synchronize)
        for y in got:
            assert torch.equal(y, want)


@pytest.mark.parametrize("M", [1, 8, 40])
def test_overlapped_launches_after_a_copy_and_on_two_streams(cuda, M):
    """The kernel in front is a copy, a fill or another stream's; the one behind
    overwrites the inputs."""
    lin = packr.PackRLinear.synthetic(2048, 4096, seed=1, lut_std=0.05, wf_std=0.005)
    lin.out_dtype = BF16
    norm = packr.PackRLayerNorm(4096, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(M)
    host = [torch.randn(M, 2048, generator=g, device="cuda").bfloat16().cpu().pin_memory() for _ in range(4)]

    @torch.no_grad()
    def f(x):
        return norm(lin(x))

    want = [f(h.cuda()) for h in host]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    bufs = [torch.empty(M, 2048, dtype=BF16, device="cuda") for _ in streams]
    got = []
    for rep in range(8):
        for s, x in zip(streams, bufs):
            with torch.cuda.stream(s):
                x.copy_(host[rep % 4], non_blocking=True)
                got.append(f(x))
                x.zero_()
    torch.cuda.synchronize()
    for i, y in enumerate(got):
        assert torch.equal(y, want[i // 2 % 4])


@pytest.mark.parametrize("lut,bias", [(BF16, BF16), (torch.float16, torch.float16), (torch.float64, torch.float64)])
def test_layer_with_converted_parameters(cuda, lut, bias):
    """model.to(dtype) converts the lut and the bias; the fused layer takes what the
    plain one takes, and its gradients come back in the parameters' types.  18 rows:
    both routes decode W alike (f32 sums of 96 terms: 1e-5)."""
    lin = packr.PackRLinear.synthetic(96, 160, seed=3, lut_std=0.05)
    torch.nn.init.normal_(lin.bias_f, std=0.2)
    lin.lut.data = lin.lut.data.to(lut)
    lin.bias_f.data = lin.bias_f.data.to(bias)
    x = torch.randn(18, 96, device="cuda").bfloat16()
    plain = lin(x)
    want = torch.autograd.grad(plain.clamp_min(0).sum(), [lin.lut, lin.bias_f])
    lin.activation = "relu"
    got = lin(x)
    assert got.dtype == F32 and torch.allclose(got, plain.clamp_min(0), rtol=1e-5, atol=1e-5)
    for a, b in zip(torch.autograd.grad(got.sum(), [lin.lut, lin.bias_f]), want):
        assert a.dtype == b.dtype and rel(a, b) < 2e-2
    lin.activation = None
    assert torch.allclose(lin(x, residual=torch.ones_like(plain)), plain + 1, rtol=1e-5, atol=1e-5)


def test_whole_layer_converted_to_bf16(cuda):
    lin = packr.PackRLinear.synthetic(96, 160, seed=3)
    lin.activation, lin.out_dtype = "gelu", BF16
    lin.to(BF16)
    assert lin.lut.dtype == BF16 and lin.W_p.dtype == torch.uint8
    for M in (1, 8, 40, 200):
        y = lin(torch.randn(M, 96, device="cuda").bfloat16())
        y.sum().backward()
        assert y.shape == (M, 160) and lin.lut.grad.dtype == BF16
        lin.zero_grad()


@pytest.mark.parametrize("M", [1, 2, 3, 4, 5, 18, 200])
@pytest.mark.parametrize("xt", [F32, BF16])
def test_attributes_move_a_result_by_its_operands_rounding_only(cuda, M, xt):
    """The plain layer's few-row kernel takes f32 x and W = W_f + f16(lut[W_p]) as they
    are; the fused operator rounds x and W to bf16 at every row count, as both do from
    many rows on.  Half a step of each operand apart (2^-8 of |x| |W| twice, 2^-8 + 2^-11
    of |x| |lut| for the two roundings of lut), and f32 sums of 256 terms."""
    lin = packr.PackRLinear.synthetic(256, 160, seed=3, lut_std=0.05, wf_std=0.01)
    torch.nn.init.normal_(lin.bias_f, std=0.2)
    g = torch.Generator(device="cuda").manual_seed(M)
    x = torch.randn(M, 256, generator=g, device="cuda").to(xt)
    lut = lin.lut.detach()[lin.W_p.long()].double().abs()
    W = lin.W_f.detach().double().abs() + lut
    xa = x.double().abs()
    bound = (2 * 2.0 ** -8 + 2 * 258 * 2.0 ** -23) * (xa @ W) + (2.0 ** -8 + 2.0 ** -11) * (xa @ lut) + 1e-6
    with torch.no_grad():
        plain = lin(x).double()
        fused = lin(x, residual=torch.zeros(M, 160, device="cuda")).double()
        assert ((fused - plain).abs() <= bound).all()
        lin.activation = "relu"
        assert ((lin(x).double() - plain.clamp_min(0)).abs() <= bound).all()
        # the definition at every row count: rounded operands, f32 sums
        w = weights64(lin.W_p, lin.W_f, lin.lut)
        z = x.bfloat16().double() @ w + lin.bias_f.double()
        zb = 258 * 2.0 ** -23 * (xa @ W + lin.bias_f.double().abs()) * (1 + 2.0 ** -7)
        assert ((fused - z).abs() <= zb).all()
