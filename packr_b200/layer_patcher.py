"""compress_model — replace nn.Linear layers by PackRLinear
(reference packr/layer_patcher.py:9-130, same name-based scope rules) — and
fuse_epilogues, which moves what a model computes around its packed layers
(activation, residual sum, layer norm) into their kernels."""
from __future__ import annotations

import collections
import copy
import inspect
import operator
import warnings

import torch
import torch.fx
import torch.nn as nn
import torch.nn.functional as F

from .config import PackRConfig
from .layer import PackRLinear
from .norm import PackRLayerNorm


def compress_model(model: nn.Module, config: PackRConfig = None):
    """Replace nn.Linear layers of `model` with PackRLinear.  Returns the model."""
    if config is None:
        config = PackRConfig()
    if config.mode == "zpackr":
        raise NotImplementedError("mode='zpackr' is not available: its modules are absent from the reference tree")
    packr_layers = []
    for name, module in list(model.named_modules()):
        if not isinstance(module, nn.Linear):
            continue
        if not _matches_scope(name, config.layer_scope):
            continue
        packr = PackRLinear.from_linear(module)
        packr.lut.requires_grad_(config.learnable_lut)
        if name == "":  # the model itself is the Linear
            model = packr
        else:
            _replace_module(model, name, packr)
        packr_layers.append((name, packr))
    if config.fuse_epilogues:
        fuse_epilogues(model)
    if config.gradient_checkpointing:
        _enable_gradient_checkpointing(model)
    if config.offload and packr_layers:
        warnings.warn("PackRConfig.offload is ignored: this build keeps W_p and the optimizer state in HBM",
                      stacklevel=2)
    return model


def _replace_module(model, name, new_module):
    parent = model
    parts = name.split(".")
    for part in parts[:-1]:
        parent = getattr(parent, part)
    setattr(parent, parts[-1], new_module)


def _matches_scope(name: str, scope: str) -> bool:
    if scope == "all":
        return True
    if scope == "ffn":
        return _is_ffn(name)
    if scope == "attention":
        return _is_attention(name) and not _is_ffn(name)
    return False


def _is_ffn(name: str) -> bool:
    ffn_intermediate = ["intermediate", "fc1", "mlp.up", "ffn.up", "dense_h_to_4h"]
    ffn_output = ["output.dense", "fc2", "mlp.down", "ffn.down", "dense_4h_to_h"]
    n = name.lower()
    if any(m in n for m in ffn_intermediate):
        return True
    if any(m in n for m in ffn_output) and "attention" not in n:
        return True
    return False


def _is_attention(name: str) -> bool:
    attn = ["query", "key", "value", "q_proj", "k_proj", "v_proj", "o_proj", "out_proj"]
    n = name.lower()
    return any(m in n for m in attn)


def _enable_gradient_checkpointing(model: nn.Module):
    try:
        model.gradient_checkpointing_enable()
    except AttributeError:
        pass


# (layer, activation) attribute pairs of transformer feed-forward blocks, fused
# where the block's forward applies the activation to the layer's output and to
# nothing else (_only_activates)
_ACTIVATED = [("dense", "intermediate_act_fn"), ("gate_proj", "act_fn"), ("fc1", "activation_fn"),
              ("dense_h_to_4h", "act")]
_ACTIVATION_CLASSES = {"ReLU": "relu", "SiLU": "silu", "SiLUActivation": "silu", "GELUActivation": "gelu",
                       "NewGELUActivation": "gelu_tanh", "GELUTanh": "gelu_tanh", "PytorchGELUTanh": "gelu_tanh"}
_ACTIVATION_FUNCTIONS = {F.relu: "relu", torch.relu: "relu", F.gelu: "gelu", F.silu: "silu"}


# blocks fused where their forward is LayerNorm(dropout(dense(hidden_states)) +
# input_tensor) (_only_adds_and_normalises)
_ADD_NORM_CLASSES = {a + b for a in ("Bert", "Roberta", "Electra") for b in ("Output", "SelfOutput")}


def _activation_name(fn):
    """packr_linear_act's name of an activation module or function, or None."""
    if isinstance(fn, nn.GELU):
        return {"none": "gelu", "tanh": "gelu_tanh"}.get(fn.approximate)
    if isinstance(fn, nn.Module):
        return _ACTIVATION_CLASSES.get(type(fn).__name__)
    try:
        return _ACTIVATION_FUNCTIONS.get(fn)
    except TypeError:  # not hashable
        return None


class _Marker(nn.Identity):
    """Stands for a submodule while a forward is traced."""


class _Tracer(torch.fx.Tracer):
    """Traces one path through a forward: submodules are opaque, and the n-th test
    of a traced value comes out as `decisions` says, then False."""

    MOST_TESTS = 6

    def __init__(self, decisions):
        super().__init__()
        self.decisions, self.asked = decisions, 0

    def is_leaf_module(self, m, qualname):
        return True

    def to_bool(self, obj):
        self.asked += 1
        if self.asked > self.MOST_TESTS:
            raise torch.fx.proxy.TraceError("too many tests of traced values")
        return self.asked <= len(self.decisions) and self.decisions[self.asked - 1]


def _hooked(module):
    """Whether somebody watches or replaces what `module` computes."""
    return isinstance(module, nn.Module) and bool(
        "forward" in module.__dict__ or module._forward_hooks or module._forward_pre_hooks or module._backward_hooks
        or module._backward_pre_hooks)


def _own_forward(module):
    """Whether the module computes something of its own when called."""
    return type(module).forward is not nn.Module.forward or "forward" in module.__dict__


def _paths(module, parameters, **markers):
    """The fx graphs of every path through module.forward, training and not, for
    each outcome of its tests of traced values, with `markers` in the place of the
    attributes that they name; None where it cannot be followed.  Only forwards of
    exactly `parameters` arguments without defaults are, as a test for None or for
    a type cannot be seen in a trace."""
    forward = type(module).forward
    if "forward" in module.__dict__ or not inspect.isfunction(forward):
        return None
    ps = list(inspect.signature(forward).parameters.values())[1:]
    if len(ps) != parameters or any(p.default is not p.empty or p.kind is not p.POSITIONAL_OR_KEYWORD for p in ps):
        return None
    code = getattr(inspect.unwrap(forward), "__code__", None)
    if code is None or {"isinstance", "type"} & set(code.co_names):
        return None
    graphs = []
    for training in (True, False):
        todo = [()]
        while todo:
            decisions = todo.pop()
            tracer = _Tracer(decisions)
            try:
                # a copy of its own, so that neither the markers nor the trace touch the module
                probe = copy.copy(module)
                probe.__dict__.update({k: dict(v) if isinstance(v, dict) else v for k, v in module.__dict__.items()})
                probe._buffers = {k: None if b is None else b.clone() for k, b in module._buffers.items()}
                probe.training = training
                for name, marker in markers.items():
                    probe.__dict__.pop(name, None)
                    probe._modules[name] = marker
                graphs.append(tracer.trace(probe))
            except Exception:  # a module that is not copied, a value that a forward cannot read
                return None
            todo += [decisions + (False,) * (k - len(decisions)) + (True,) for k in range(len(decisions), tracer.asked)]
    return graphs


def _only_activates(module, layer, act):
    """Whether every path through the block's forward gives each output of
    `layer` to `act`, and to nothing else, and gives `act` nothing but that."""
    graphs = _paths(module, 1, **{layer: _Marker(), act: _Marker()})
    if graphs is None:
        return False
    found = False
    for graph in graphs:
        for node in graph.nodes:
            if node.op == "get_attr" and node.target.split(".")[0] in (layer, act):
                return False
            if node.op != "call_module":
                continue
            if node.target == layer:
                users = list(node.users)
                if len(users) != 1 or users[0].op != "call_module" or users[0].target != act:
                    return False
                found = True
            elif node.target == act:
                given = node.args[0] if len(node.args) == 1 and not node.kwargs else None
                if not (isinstance(given, torch.fx.Node) and given.op == "call_module" and given.target == layer):
                    return False
    return found


def _only_adds_and_normalises(module):
    """Whether the block's forward is LayerNorm(dropout(dense(a)) + b)."""
    graphs = _paths(module, 2, dense=_Marker(), dropout=_Marker(), LayerNorm=_Marker())
    if graphs is None:
        return False
    for graph in graphs:
        nodes = list(graph.nodes)
        if [n.op for n in nodes[:2]] != ["placeholder"] * 2 or len(nodes) != 7:
            return False
        a, b, dense, drop, add, norm, out = nodes
        ok = (dense.op == drop.op == norm.op == "call_module" and not (dense.kwargs or drop.kwargs or norm.kwargs)
              and dense.target == "dense" and dense.args == (a,)
              and drop.target == "dropout" and drop.args == (dense,)
              and add.op == "call_function" and add.target in (operator.add, torch.add) and not add.kwargs
              and add.args in ((drop, b), (b, drop))
              and norm.target == "LayerNorm" and norm.args == (add,) and out.op == "output" and out.args == (norm,))
        if not ok:
            return False
    return True


class PackRAddNorm(nn.Module):
    """LayerNorm(dropout(dense(x)) + residual), the close of a post-norm block,
    with the sum taken inside the norm's kernel.  Takes over the submodules of
    the block it replaces under their names, so state dicts keep their keys."""

    def __init__(self, dense, LayerNorm, dropout=None):
        super().__init__()
        self.dense = dense
        self.LayerNorm = PackRLayerNorm.from_layer_norm(LayerNorm)
        self.dropout = dropout if dropout is not None else nn.Identity()

    def forward(self, hidden_states, input_tensor):
        h = self.dropout(self.dense(hidden_states))
        # the sum's type is the wider one's, as h + input_tensor's; fp16 is
        # widened (the norm takes f32 and bf16)
        t = torch.promote_types(h.dtype, input_tensor.dtype)
        t = torch.float32 if t == torch.float16 else t
        if h.shape != input_tensor.shape:  # the sum's shape, as h + input_tensor's
            h, input_tensor = torch.broadcast_tensors(h, input_tensor)
        return self.LayerNorm(h.to(t), residual=input_tensor.to(t))


def fuse_epilogues(model: nn.Module):
    """Fuses what surrounds the packed layers of `model`, in place:

    * an activation that follows a PackRLinear (BERT's dense +
      intermediate_act_fn, a gated MLP's gate_proj + act_fn, fc1 +
      activation_fn, dense_h_to_4h + act) becomes the layer's `activation`;
    * blocks that add their input before a layer norm (BERT's BertOutput and
      BertSelfOutput, and their Roberta and Electra twins) become PackRAddNorm.

    A block is taken only where its forward, followed by torch.fx over all of its
    paths, is seen to do just that: one that gates, normalises or splits the
    layer's output first, uses the activation a second time, takes optional
    arguments (decoder layers that hold fc1 themselves) or cannot be followed
    stays as it is, and so does a layer that more than one block holds.  A block
    without a forward of its own is taken when it is the model itself.  Where the
    layer, the activation, the norm or a block that would be replaced carries hooks
    (or a forward set on the instance), they would see other values or none at all,
    so it stays too.

    Activations other than relu, gelu (either form) and silu stay as they are,
    and so do norms whose weights are neither f32 nor bf16.
    Parameters, their names and the model's results (up to rounding) do not
    change.  Returns the model."""
    holders = collections.Counter(id(m) for parent in model.modules() for m in parent._modules.values())
    for name, module in list(model.named_modules()):
        for layer, act in _ACTIVATED:
            lin = getattr(module, layer, None)
            known = _activation_name(getattr(module, act, None))
            if (isinstance(lin, PackRLinear) and lin.activation is None and known is not None
                    and holders[id(lin)] == 1 and not _hooked(lin) and not _hooked(getattr(module, act))):
                if not (_only_activates(module, layer, act) if _own_forward(module)
                        else name == "" and not isinstance(module, nn.ModuleDict)):
                    continue
                lin.activation = known
                if act in module._modules:
                    module._modules[act] = nn.Identity()
                else:
                    setattr(module, act, nn.Identity())
        if type(module).__name__ in _ADD_NORM_CLASSES and name:
            norm = getattr(module, "LayerNorm", None)
            # a block without a forward of its own: its submodules keep what they do
            if (type(norm) is nn.LayerNorm and len(norm.normalized_shape) == 1
                    and (norm.weight is None or norm.weight.dtype in (torch.float32, torch.bfloat16))
                    and not _hooked(module) and not _hooked(norm)
                    and (not _own_forward(module) or _only_adds_and_normalises(module))):
                fused = PackRAddNorm(module.dense, norm, module.dropout)
                fused.train(module.training)
                _replace_module(model, name, fused)
    return model
