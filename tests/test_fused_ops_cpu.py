"""What the fused feed-forward operators refuse, without a GPU, and their
64-bit reference forms against torch's own functions."""
import copy
import ctypes
import pickle

import pytest
import torch

import packr_b200 as packr
from packr_b200 import _lib
from packr_b200.autograd import grad_sink
from fused_reference import ACTS, act64, linear64, norm64, slope64, weights64


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 8)
    with pytest.raises(RuntimeError, match="CUDA"):
        packr.packr_layer_norm(x)
    with pytest.raises(RuntimeError, match="CUDA"):
        packr.packr_linear_act(x, torch.zeros(8, 4, dtype=torch.uint8), torch.zeros(8, 4, dtype=torch.bfloat16),
                               torch.zeros(256))


def _fake(n=64):
    """An address that no refused call reads."""
    return ctypes.c_void_p(0x7F0000000000 + n)


def test_linear_act_c_entry_refuses_bad_arguments():
    lib = _lib.load()
    a = _fake()

    def fwd(x=a, xd=1, wp=a, wf=a, lut=a, bias=None, bd=0, act=0, res=None, out=a, z=None, od=1, M=4, K=8, N=8):
        return lib.packr_linear_act_forward(x, xd, wp, wf, lut, bias, bd, act, res, out, z, od, M, K, N, None, 0, None)

    assert fwd(M=-1) == 2 and fwd(K=0) == 2 and fwd(N=0) == 2 and fwd(N=1 << 31) == 2
    assert fwd(xd=2) == 1 and fwd(od=2) == 1 and fwd(od=-1) == 1 and fwd(act=5) == 1 and fwd(act=-1) == 1
    assert fwd(bias=a, bd=2) == 1
    for name in ("x", "wp", "wf", "lut", "out"):
        assert fwd(**{name: None}) == 1, name
    odd = _fake(1)
    for name in ("wf", "lut", "out", "res", "z", "x"):
        assert fwd(**{name: odd}) == 3, name
    assert fwd(od=0, out=_fake(2)) == 3 and fwd(bias=_fake(2), bd=0) == 3

    def bwd(dout=a, z=a, od=1, act=2, x=a, xd=1, M=4, K=8, N=8, flags=0, db=None, dbd=0, dw=a):
        return lib.packr_linear_act_backward(dout, z, od, act, x, xd, a, a, a, None, a, dw, None, db, dbd, M, K, N,
                                             flags, None, 0, None)

    assert bwd(M=-1) == 2 and bwd(act=9) == 1 and bwd(flags=2) == 1 and bwd(dout=None) == 1
    assert bwd(z=None) == 1  # an activation's backward needs z
    assert bwd(db=a, dbd=2) == 1 and bwd(dout=odd) == 3 and bwd(dw=odd) == 3 and bwd(db=_fake(2), dbd=0) == 3


@pytest.mark.parametrize("dim", ["M", "K", "N"])
def test_linear_act_c_entry_refuses_dimensions_next_to_2_31(dim):
    """A tile or a slab that starts inside them would end past an int's range."""
    lib, a = _lib.load(), _fake()
    d = {"M": 4, "K": 8, "N": 8, dim: 0x7FFFFFFF}
    assert lib.packr_linear_act_forward(a, 1, a, a, a, None, 0, 0, None, a, None, 1, d["M"], d["K"], d["N"], None, 0,
                                        None) == 2
    assert lib.packr_linear_act_backward(a, a, 1, 2, a, 1, a, a, a, None, a, a, None, None, 0, d["M"], d["K"], d["N"], 0,
                                         None, 0, None) == 2


def test_layer_norm_c_entry_refuses_bad_arguments():
    lib = _lib.load()
    a, odd = _fake(), _fake(1)

    def fwd(x=a, res=None, xd=1, w=a, b=a, wd=1, eps=1e-5, y=a, mean=None, M=4, N=8):
        return lib.packr_layer_norm_forward(x, res, xd, w, b, wd, eps, y, mean, None, M, N, None)

    assert fwd(M=-1) == 2 and fwd(N=0) == 2 and fwd(M=1 << 31) == 2 and fwd(N=1 << 31) == 2
    assert fwd(xd=2) == 1 and fwd(wd=3) == 1 and fwd(eps=-1.0) == 1 and fwd(eps=float("nan")) == 1
    assert fwd(x=None) == 1 and fwd(y=None) == 1
    for name in ("x", "res", "y", "w", "b", "mean"):
        assert fwd(**{name: odd}) == 3, name

    def bwd(dy=a, x=a, xd=1, wd=1, mean=a, rstd=a, dx=a, M=4, N=8):
        return lib.packr_layer_norm_backward(dy, x, None, xd, a, wd, mean, rstd, dx, a, a, M, N, None, 0, None)

    assert bwd(M=-1) == 2 and bwd(N=0) == 2 and bwd(xd=2) == 1 and bwd(wd=2) == 1
    for name in ("dy", "x", "mean", "rstd"):
        assert bwd(**{name: None}) == 1, name
    assert bwd(dx=odd) == 3 and bwd(mean=_fake(2)) == 3


def test_workspace_queries_of_empty_problems():
    lib = _lib.load()
    assert lib.packr_layer_norm_backward_workspace_bytes(0, 8) == 0
    assert lib.packr_layer_norm_backward_workspace_bytes(-3, 8) == 0
    assert lib.packr_linear_act_workspace_bytes(0, 8, 8, 1, 1, None, None) == 0
    assert lib.packr_linear_act_backward_workspace_bytes(4, 0, 8, 1, 0, None, None) == 0


def test_activation_names():
    assert _lib.ACTIVATIONS == {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}


def test_module_takes_one_dimension():
    with pytest.raises(ValueError):
        packr.PackRLayerNorm((4, 8))
    with pytest.raises(ValueError):
        packr.PackRLayerNorm.from_layer_norm(torch.nn.LayerNorm((4, 8)))
    with pytest.raises(TypeError):
        packr.PackRLayerNorm.from_layer_norm(torch.nn.Linear(4, 4))


@pytest.mark.parametrize("act", ACTS)
def test_reference_forms_follow_torch(act):
    f = {"none": lambda z: z, "relu": torch.relu, "gelu": torch.nn.functional.gelu, "silu": torch.nn.functional.silu,
         "gelu_tanh": lambda z: torch.nn.functional.gelu(z, approximate="tanh")}[act]
    z = torch.linspace(-8, 8, 801, dtype=torch.float64).requires_grad_(True)
    assert torch.allclose(act64(z, act), f(z), rtol=1e-12, atol=1e-14)
    want = torch.autograd.grad(f(z).sum(), z)[0]
    assert torch.allclose(slope64(z, act), want, rtol=1e-9, atol=1e-11)
    # the Lipschitz bounds that the tolerances use
    s = slope64(z, act)
    assert s.abs().max() <= 1.13
    if act != "relu":
        assert (s.diff() / z.detach().diff()).abs().max() <= 0.8


def test_reference_norm_and_linear_follow_torch():
    g = torch.Generator().manual_seed(0)
    x, r, dy = (torch.randn(5, 24, generator=g) for _ in range(3))
    w, b = torch.randn(24, generator=g), torch.randn(24, generator=g)
    s = (x.double() + r.double()).requires_grad_(True)
    wd, bd = w.double().requires_grad_(True), b.double().requires_grad_(True)
    y = torch.nn.functional.layer_norm(s, (24,), wd, bd, 1e-5)
    dx, dw, db = torch.autograd.grad(y, [s, wd, bd], dy.double())
    got = norm64(x, r, w, b, 1e-5, dy)
    for k, v in (("y", y), ("dx", dx), ("dweight", dw), ("dbias", db)):
        assert torch.allclose(got[k][0], v, rtol=1e-10, atol=1e-12), k
    W_p = torch.randint(0, 256, (24, 16), generator=g, dtype=torch.uint8)
    W_f, lut = torch.randn(24, 16, generator=g).bfloat16(), torch.randn(256, generator=g)
    W = weights64(W_p, W_f, lut)
    assert torch.equal(W.bfloat16(), W_f + lut[W_p.long()].bfloat16())  # the layer's decode (a bf16 sum)
    W = W.requires_grad_(True)
    xb = x.bfloat16()
    xd, bias, dout = xb.double().requires_grad_(True), torch.randn(16, generator=g), torch.randn(5, 16, generator=g)
    out = torch.nn.functional.gelu(xd @ W + bias.double())
    dx, dw = torch.autograd.grad(out, [xd, W], dout.double())
    got = linear64(xb, W_p, W_f, lut, bias, "gelu", None, torch.float32, dout)
    for k, v in (("out", out), ("dx", dx), ("dW_f", dw)):
        assert torch.allclose(got[k][0], v, rtol=1e-10, atol=1e-12), k


def _bert_block():
    from transformers import BertConfig
    from transformers.models.bert.modeling_bert import BertLayer
    cfg = BertConfig(hidden_size=32, num_attention_heads=2, intermediate_size=64, hidden_act="gelu")
    cfg._attn_implementation = "eager"
    block = torch.nn.ModuleDict({"layer": BertLayer(cfg)})
    layer = block["layer"]
    for parent, name in ((layer.intermediate, "dense"), (layer.output, "dense")):
        lin = getattr(parent, name)
        setattr(parent, name, packr.PackRLinear(lin.in_features, lin.out_features))
    return block


def test_fuse_epilogues_rewires_a_bert_layer():
    block = _bert_block().eval()
    keys = list(block.state_dict())
    norms = {n: p for n, p in block.named_parameters()}
    assert packr.fuse_epilogues(block) is block
    layer = block["layer"]
    assert layer.intermediate.dense.activation == "gelu"
    assert isinstance(layer.intermediate.intermediate_act_fn, torch.nn.Identity)
    for m in (layer.output, layer.attention.output):
        assert isinstance(m, packr.PackRAddNorm) and isinstance(m.LayerNorm, packr.PackRLayerNorm) and not m.training
    assert list(block.state_dict()) == keys
    assert all(p is norms[n] for n, p in block.named_parameters())
    packr.fuse_epilogues(block)  # a second run changes nothing
    assert layer.intermediate.dense.activation == "gelu"


@pytest.mark.parametrize("fn,name", [
    (torch.nn.GELU(), "gelu"), (torch.nn.GELU(approximate="tanh"), "gelu_tanh"), (torch.nn.ReLU(), "relu"),
    (torch.nn.SiLU(), "silu"), (torch.nn.functional.gelu, "gelu"), (torch.relu, "relu"), (torch.nn.Tanh(), None),
    (torch.nn.ReLU6(), None), (lambda z: z, None), (None, None)])
def test_which_activations_are_fused(fn, name):
    class Block(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.gate_proj = packr.PackRLinear(8, 16, bias=False)
            self.act_fn = fn

    b = Block()
    packr.fuse_epilogues(b)
    assert b.gate_proj.activation == name
    assert isinstance(b.act_fn, torch.nn.Identity) == (name is not None)


def test_plain_linears_keep_their_activation():
    class Block(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.fc1 = torch.nn.Linear(8, 16)
            self.activation_fn = torch.nn.ReLU()

    b = Block()
    packr.fuse_epilogues(b)
    assert isinstance(b.activation_fn, torch.nn.ReLU)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_norms_of_other_types_stay(dtype):
    class BertOutput(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.dense = torch.nn.Linear(8, 8)
            self.LayerNorm = torch.nn.LayerNorm(8, dtype=dtype)
            self.dropout = torch.nn.Dropout(0.0)

    model = torch.nn.Sequential(BertOutput())
    packr.fuse_epilogues(model)
    assert (type(model[0]).__name__ == "PackRAddNorm") == (dtype != torch.float16)


def test_layer_takes_known_activations():
    assert packr.PackRLinear(4, 8).activation is None
    assert packr.PackRLinear(4, 8, activation="silu", out_dtype=torch.bfloat16).extra_repr().endswith(
        "activation=silu, out_dtype=torch.bfloat16")
    with pytest.raises(ValueError):
        packr.PackRLinear(4, 8, activation="tanh")
    assert packr.PackRConfig().fuse_epilogues is False


class _Scale(torch.autograd.Function):
    """x * w whose backward writes w's gradient into the buffer it is lent."""

    @staticmethod
    def forward(ctx, x, w):
        ctx.save_for_backward(x)
        ctx.w = w
        return x * w

    @staticmethod
    def backward(ctx, g):
        x, = ctx.saved_tensors
        out = grad_sink(ctx.w)
        return None, g * x if out is None else torch.mul(g, x, out=out)


def _parameter_with_sink():
    w = torch.nn.Parameter(torch.ones(4))
    w._packr_grad_sink = (torch.zeros(6), 2)
    return w, w._packr_grad_sink[0][2:].data_ptr()


def test_gradients_of_a_parameter_used_twice_are_summed():
    w, at = _parameter_with_sink()
    x = torch.arange(4.0)
    for _ in range(2):
        (_Scale.apply(x, w).sum() + _Scale.apply(5 * x, w).sum()).backward()
        assert torch.equal(w.grad, 6 * x)
        w.grad = None
    for k in range(3):  # used once, the buffer itself becomes the gradient
        _Scale.apply(k * x, w).sum().backward()
        assert torch.equal(w.grad, k * x) and w.grad.data_ptr() == at
        w.grad = None


def test_a_gradient_in_hand_is_not_overwritten():
    w, _ = _parameter_with_sink()
    x = torch.arange(4.0)
    a, = torch.autograd.grad(_Scale.apply(x, w).sum(), w)
    b, = torch.autograd.grad(_Scale.apply(3 * x, w).sum(), w)
    assert torch.equal(a, x) and torch.equal(b, 3 * x)


def test_a_parameter_with_a_buffer_can_be_copied():
    w, _ = _parameter_with_sink()
    _Scale.apply(torch.ones(4), w).sum().backward()
    assert torch.equal(copy.deepcopy(w), w)
    assert torch.equal(pickle.loads(pickle.dumps(w)), w)


def test_a_parameter_with_a_buffer_can_be_saved_and_loaded(tmp_path):
    """With torch.load's default, which takes tensors and plain values only."""
    w, _ = _parameter_with_sink()
    _Scale.apply(torch.ones(4), w).sum().backward()
    torch.save({"w": w}, tmp_path / "w.pt")
    assert torch.equal(torch.load(tmp_path / "w.pt")["w"], w)


def test_a_copied_parameter_has_a_loan_of_its_own():
    w, _ = _parameter_with_sink()
    c = pickle.loads(pickle.dumps(w))
    x = torch.arange(4.0)
    g, = torch.autograd.grad(_Scale.apply(x, w).sum(), w)  # w's buffer is lent
    _Scale.apply(x, c).sum().backward()
    assert c.grad.data_ptr() == c._packr_grad_sink[0][2:].data_ptr() and torch.equal(g, x)


@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_derivatives_are_refused(grad):
    """No input requires a gradient, so the operators call their kernels past
    autograd; a tangent must not be dropped there.  Refused before the device is
    looked at."""
    from torch.autograd import forward_ad
    x, w = torch.ones(2, 8), torch.ones(8)
    W_p, W_f = torch.zeros(8, 4, dtype=torch.uint8), torch.zeros(8, 4, dtype=torch.bfloat16)
    lut, bias, res = torch.zeros(256), torch.zeros(4), torch.zeros(2, 4)
    norm = dict(x=x, weight=w, bias=w, residual=x)
    lin = dict(x=x, W_p=W_p, W_f=W_f, lut=lut, bias=bias, residual=res)
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        for f, args in ((packr.packr_layer_norm, norm), (packr.packr_linear_act, lin)):
            with pytest.raises(RuntimeError, match="CUDA"):  # nothing dual: the usual checks
                f(**args)
            for name, t in args.items():
                if t.is_floating_point():
                    with pytest.raises(NotImplementedError, match="forward-mode"):
                        f(**{**args, name: forward_ad.make_dual(t, torch.ones_like(t))})
        with pytest.raises(NotImplementedError, match="forward-mode"):
            packr.PackRLayerNorm(8)(forward_ad.make_dual(x, x))


def test_norm_module_follows_autocast(monkeypatch):
    """What reaches the operator: nn.LayerNorm's types, f32 under autocast."""
    from packr_b200 import norm
    seen = []

    def plain(x, weight=None, bias=None, eps=1e-5, residual=None):
        seen.append((x.dtype, None if residual is None else residual.dtype))
        s = x if residual is None else x + residual
        return torch.nn.functional.layer_norm(s, s.shape[-1:], None, None, eps)

    monkeypatch.setattr(norm, "packr_layer_norm", plain)
    m, ref = packr.PackRLayerNorm(8), torch.nn.LayerNorm(8)
    bf, f16, f32 = torch.bfloat16, torch.float16, torch.float32
    x = torch.randn(2, 8)
    for dtype in (bf, f16, f32):
        with torch.autocast("cpu", dtype=bf):
            assert m(x.to(dtype), residual=x.to(bf)).dtype == f32 and seen[-1] == (f32, f32)
            assert m(x.to(dtype)).dtype == f32 and seen[-1] == (f32, None)
    with torch.autocast("cpu", dtype=bf, enabled=False):
        assert m(x.to(bf), residual=x.to(bf)).dtype == bf and seen[-1] == (bf, bf)
    with torch.autocast("cuda", dtype=bf):  # another device type's
        m(x.to(bf))
        assert seen[-1] == (bf, None)
    assert ref(x).dtype == f32


def test_decoded_linear_act_c_entries_refuse_bad_arguments():
    lib, a, odd = _lib.load(), _fake(), _fake(8)

    def fwd(x=a, xd=1, wd=a, out=a, od=1, act=0, M=4, K=8, N=8):
        return lib.packr_linear_act_forward_decoded(x, xd, wd, None, 0, act, None, out, None, od, M, K, N, None, 0, None)

    assert fwd(M=-1) == 2 and fwd(K=0) == 2 and fwd(N=0) == 2 and fwd(N=12) == 2 and fwd(N=0x7FFFFFF8) == 2
    assert fwd(wd=None) == 1 and fwd(x=None) == 1 and fwd(out=None) == 1 and fwd(xd=2) == 1 and fwd(act=7) == 1
    assert fwd(wd=odd) == 3 and fwd(x=_fake(1)) == 3

    def bwd(wd=a, M=4, K=8, N=8, z=a):
        return lib.packr_linear_act_backward_decoded(a, z, 1, 2, a, 1, a, a, a, wd, None, a, a, None, None, 0, M, K, N, 0,
                                                     None, 0, None)

    assert bwd(wd=None) == 1 and bwd(wd=odd) == 3 and bwd(N=12) == 2 and bwd(M=-1) == 2 and bwd(z=None) == 1
    assert lib.packr_linear_act_forward_decoded_workspace_bytes(0, 8, 8, 1, 1) == 0
    assert lib.packr_linear_act_backward_decoded_workspace_bytes(4, 8, 0, 1, 0, None, None) == 0
