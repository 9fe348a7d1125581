"""fuse_epilogues takes a block only where its forward is seen to apply the
activation to the packed layer's output and to nothing else."""
import pytest
import torch
import torch.nn as nn

import packr_b200 as packr


class Mlp(nn.Module):
    def __init__(self, act=None):
        super().__init__()
        self.fc1 = packr.PackRLinear(8, 16)
        self.activation_fn = nn.GELU() if act is None else act
        self.fc2 = nn.Linear(16, 8)
        self.norm = nn.LayerNorm(16)

    def forward(self, x):
        return self.fc2(self.activation_fn(self.fc1(x)))


class Named(Mlp):
    def forward(self, hidden_states):
        h = self.fc1(hidden_states)
        h = self.activation_fn(h)
        h = nn.functional.dropout(h, 0.1, training=self.training)
        return self.fc2(h) + hidden_states


class ShapeTest(Mlp):
    def forward(self, x):
        if x.shape[0] > 4:
            x = x.clone()
        return self.fc2(self.activation_fn(self.fc1(x)))


class Gated(Mlp):
    def forward(self, x):
        h, gate = self.fc1(x).chunk(2, dim=-1)
        return self.fc2(self.activation_fn(gate) * h)


class TwiceUsed(Mlp):
    def forward(self, x):
        return self.activation_fn(self.fc2(self.activation_fn(self.fc1(x))))


class NormBetween(Mlp):
    def forward(self, x):
        return self.fc2(self.activation_fn(self.norm(self.fc1(x))))


class ResidualOfThePreactivation(Mlp):
    def forward(self, x):
        h = self.fc1(x)
        return self.fc2(self.activation_fn(h) + h)


class OnlyOnSomeShapes(Mlp):
    def forward(self, x):
        h = self.fc1(x)
        if x.shape[0] > 4:
            h = self.norm(h)
        return self.fc2(self.activation_fn(h))


class OnlyWhenNotTraining(Mlp):
    def forward(self, x):
        h = self.fc1(x)
        return self.fc2(self.activation_fn(h) if self.training else h)


class ActivationOfSomethingElse(Mlp):
    def forward(self, x):
        return self.fc2(self.activation_fn(self.fc1(x)) + self.activation_fn(x[..., :1]))


class ReadsTheWeights(Mlp):
    def forward(self, x):
        return self.fc2(self.activation_fn(x @ self.fc1.W_f.to(x.dtype)))


class OptionalArgument(Mlp):
    def forward(self, x, scale=None):
        h = self.fc1(x)
        if scale is None:
            return self.fc2(self.activation_fn(h))
        return self.fc2(self.activation_fn(h * scale))


class TypeTest(Mlp):
    def forward(self, x):
        h = self.fc1(x)
        if isinstance(x, torch.Tensor):
            h = self.norm(h)
        return self.fc2(self.activation_fn(h))


class NotCalledHere(Mlp):
    def forward(self, x):
        return self.fc2(x)


class ScaledActivation(nn.Module):
    """Calls its activation with a second argument's help."""

    def __init__(self):
        super().__init__()
        self.dense = packr.PackRLinear(8, 16)
        self.intermediate_act_fn = torch.nn.functional.gelu

    def forward(self, x):
        return self.intermediate_act_fn(self.dense(x), approximate="tanh")


def fused(block, layer="fc1", act="activation_fn"):
    model = nn.Sequential(block)
    before = getattr(block, act)
    keys = list(model.state_dict())
    assert packr.fuse_epilogues(model) is model
    lin, now = getattr(block, layer), getattr(block, act)
    assert list(model.state_dict()) == keys
    if lin.activation is None:  # left as it was
        assert now is before
        return False
    assert isinstance(now, nn.Identity)
    return True


@pytest.mark.parametrize("cls", [Mlp, Named, ShapeTest])
@pytest.mark.parametrize("act", [None, torch.nn.functional.gelu])
def test_plain_blocks_are_fused(cls, act):
    block = cls(act)
    block.eval()
    assert fused(block) and not block.training and block.fc1.activation == "gelu"


@pytest.mark.parametrize("cls", [Gated, TwiceUsed, NormBetween, ResidualOfThePreactivation, OnlyOnSomeShapes,
                                 OnlyWhenNotTraining, ActivationOfSomethingElse, ReadsTheWeights, OptionalArgument,
                                 TypeTest, NotCalledHere])
def test_blocks_that_do_something_else_are_left_alone(cls):
    for act in (None, torch.nn.functional.gelu):
        assert not fused(cls(act))


def test_activation_called_with_more_than_the_layers_output():
    assert not fused(ScaledActivation(), "dense", "intermediate_act_fn")


def test_containers_are_left_alone():
    d = nn.ModuleDict({"fc1": packr.PackRLinear(8, 16), "activation_fn": nn.ReLU()})
    packr.fuse_epilogues(d)
    assert d["fc1"].activation is None and isinstance(d["activation_fn"], nn.ReLU)

    class Inner(nn.Module):  # no forward: whoever holds it applies its parts
        def __init__(self):
            super().__init__()
            self.fc1, self.activation_fn = packr.PackRLinear(8, 16), nn.ReLU()

    assert not fused(Inner())


def test_tracing_leaves_no_mark():
    class Counts(Mlp):
        def __init__(self):
            super().__init__()
            self.calls = 0
            self.register_buffer("steps", torch.zeros(1))

        def forward(self, x):
            self.calls += 1
            self.steps += 1
            return self.fc2(self.activation_fn(self.fc1(x)))

    b = Counts()
    assert fused(b) and b.calls == 0 and not b.steps.any() and b.training
    assert b.fc2(b.norm(torch.zeros(2, 16))).shape == (2, 8)


def test_gated_and_reused_activations_of_transformers():
    from transformers import MoonshineConfig
    from transformers.models.llama4.configuration_llama4 import Llama4VisionConfig
    from transformers.models.llama4.modeling_llama4 import Llama4VisionMLP2
    from transformers.models.moonshine.modeling_moonshine import MoonshineDecoderMLP
    c = MoonshineConfig(hidden_size=8, intermediate_size=16)
    for block in (MoonshineDecoderMLP(c, "silu"), Llama4VisionMLP2(Llama4VisionConfig(
            hidden_size=8, intermediate_size=16, projector_input_dim=16, projector_output_dim=16))):
        block.fc1 = packr.PackRLinear(8, 16)
        assert not fused(block)


def test_gated_mlps_of_transformers_are_fused():
    from transformers import GPTNeoXConfig, LlamaConfig
    from transformers.models.gpt_neox.modeling_gpt_neox import GPTNeoXMLP
    from transformers.models.llama.modeling_llama import LlamaMLP
    b = LlamaMLP(LlamaConfig(hidden_size=8, intermediate_size=16, num_attention_heads=2))
    b.gate_proj = packr.PackRLinear(8, 16, bias=False)
    assert fused(b, "gate_proj", "act_fn") and b.gate_proj.activation == "silu"
    b = GPTNeoXMLP(GPTNeoXConfig(hidden_size=8, intermediate_size=16, num_attention_heads=2))
    b.dense_h_to_4h = packr.PackRLinear(8, 16)
    assert fused(b, "dense_h_to_4h", "act") and b.dense_h_to_4h.activation == "gelu"


def add_norm(forward):
    def init(self):
        nn.Module.__init__(self)
        self.dense, self.LayerNorm, self.dropout = nn.Linear(8, 8), nn.LayerNorm(8), nn.Dropout(0.1)

    return type("BertOutput", (nn.Module,), {"__init__": init, "forward": forward})


@pytest.mark.parametrize("forward,taken", [
    (lambda self, h, x: self.LayerNorm(self.dropout(self.dense(h)) + x), True),
    (lambda self, h, x: self.LayerNorm(x + self.dropout(self.dense(h))), True),
    (lambda self, h, x: self.LayerNorm(torch.add(self.dropout(self.dense(h)), x)), True),
    (lambda self, h, x: self.LayerNorm(self.dropout(self.dense(h))) + x, False),
    (lambda self, h, x: self.LayerNorm(self.dense(self.dropout(h)) + x), False),
    (lambda self, h, x: self.LayerNorm(self.dropout(self.dense(h)) + h), False),
    (lambda self, h, x: self.LayerNorm(torch.add(self.dropout(self.dense(h)), x, alpha=2)), False),
    (lambda self, h, x: self.LayerNorm(self.dropout(self.dense(h)) + x) * 2, False),
    (lambda self, h, x=None: self.LayerNorm(self.dropout(self.dense(h)) + x), False),
])
def test_which_add_norm_blocks_are_replaced(forward, taken):
    model = nn.Sequential(add_norm(forward)())
    packr.fuse_epilogues(model)
    assert isinstance(model[0], packr.PackRAddNorm) == taken


def test_a_layer_that_two_blocks_hold_is_left_alone():
    """Its activation would be applied by the layer and again by the other block."""
    a, b = Mlp(), Mlp()
    b.fc1 = a.fc1
    for model in (nn.Sequential(a, b), nn.Sequential(a, a.fc1)):
        packr.fuse_epilogues(model)
        assert a.fc1.activation is None and isinstance(a.activation_fn, nn.GELU) and isinstance(b.activation_fn, nn.GELU)
    # the same block in two places is one holder
    assert packr.fuse_epilogues(nn.Sequential(a, a))[0].fc1.activation == "gelu"


HOOKS = ["register_forward_hook", "register_forward_pre_hook", "register_full_backward_hook",
         "register_full_backward_pre_hook", "forward"]


def watch(module, how):
    if how == "forward":
        module.forward = type(module).forward.__get__(module)
    else:
        getattr(module, how)(lambda *a: None)


@pytest.mark.parametrize("how", HOOKS)
def test_watched_modules_are_left_alone(how):
    for part in ("fc1", "activation_fn"):
        b = Mlp()
        watch(getattr(b, part), how)
        assert not fused(b), part
    b = Mlp()
    watch(b.fc2, how)  # a part that stays as it is
    assert fused(b)
    for part in (None, "LayerNorm"):
        model = nn.Sequential(add_norm(lambda self, h, x: self.LayerNorm(self.dropout(self.dense(h)) + x))())
        watch(model[0] if part is None else model[0].LayerNorm, how)
        before = model[0]
        packr.fuse_epilogues(model)
        assert model[0] is before, part
    model = nn.Sequential(add_norm(lambda self, h, x: self.LayerNorm(self.dropout(self.dense(h)) + x))())
    watch(model[0].dense, how)
    dense = model[0].dense
    packr.fuse_epilogues(model)
    assert isinstance(model[0], packr.PackRAddNorm) and model[0].dense is dense


def test_add_norm_broadcasts_its_sum(monkeypatch):
    """As h + input_tensor does; the norm is handed two tensors of one shape."""
    from packr_b200 import norm
    seen = []

    def plain(x, weight, bias, eps, residual):
        seen.append((x.shape, residual.shape))
        return nn.functional.layer_norm(x + residual, x.shape[-1:], weight, bias, eps)

    monkeypatch.setattr(norm, "packr_layer_norm", plain)
    dense, ln = nn.Linear(8, 8), nn.LayerNorm(8)
    block = packr.PackRAddNorm(dense, ln)
    h = torch.randn(2, 3, 8, requires_grad=True)
    for shape in ((2, 3, 8), (1, 3, 8), (3, 8), (8,), (4, 2, 3, 8)):
        r = torch.randn(shape, requires_grad=True)
        got, want = block(h, r), ln(dense(h) + r)
        assert torch.allclose(got, want, rtol=1e-6, atol=1e-6) and seen[-1][0] == seen[-1][1]
        for a, b in zip(torch.autograd.grad(got.square().sum(), [h, r]), torch.autograd.grad(want.square().sum(), [h, r])):
            assert a.shape == b.shape and torch.allclose(a, b, rtol=1e-5, atol=1e-5)


def test_forwards_that_cannot_be_followed_are_left_alone():
    class Own(nn.Module):  # a forward set on the instance of a class without one
        def __init__(self):
            super().__init__()
            self.fc1, self.activation_fn = packr.PackRLinear(8, 16), nn.ReLU()
            self.forward = lambda x: self.activation_fn(self.fc1(x).flip(-1))

    class NoCopy(Mlp):
        def __copy__(self):
            raise RuntimeError("not copied")

    class Scripted(Mlp):
        forward = torch.no_grad()  # callable, but nothing to read arguments from

    class Loop(Mlp):
        def forward(self, x):
            h = self.fc1(x)
            while h.sum() > 1:
                h = h / 2
            return self.activation_fn(h)

    own = Own()
    packr.fuse_epilogues(own)  # the model itself
    assert own.fc1.activation is None
    for block in (Own(), NoCopy(), Scripted(), Loop()):
        assert not fused(block), type(block).__name__
