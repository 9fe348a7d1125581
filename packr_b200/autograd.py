"""Autograd for the PackR linear map on B200.

PackRLinearFunction: out = x @ (W_f + lut[W_p]) + bias, with the bias fused
into the forward GEMM's epilogue and its gradient produced by the backward
launch sequence.  Backward semantics follow reference packr/autograd.py:56-88:
  grad_x    = bf16(bf16(dY) @ W_bf16^T), returned in x's dtype
  grad_W_f  = bf16(x^T @ dY)                  (fp32 accumulate)
  grad_lut  = scatter_add(x^T @ dY by W_p) / (bincount(W_p) + 1e-8)
  grad_bias = bf16(dY.sum(0))                 (autograd of layer.py:97)
W_p is frozen and gets no gradient.

PackRMatmulFunction keeps the reference's signature
(x, W_p, W_f, lut, evict_cb=None, layer_name=None, offload_mgr=None) and
bias-free output (reference autograd.py:17-53).  Host offload is not part of
this build (W_p stays in HBM), so layer_name / offload_mgr are accepted and
ignored; evict_cb still fires at the end of backward.
"""
from __future__ import annotations

import os
import weakref

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from . import kernel as _k

# Off by default: between forward and backward a layer holds only its packed
# weights (3 bytes per weight), as PackR promises.  PACKR_KEEP_DECODED_W=1
# trades 2 more bytes per weight, held from forward to backward on the
# many-row route, for the second decode of W in the backward.
KEEP_DECODED_W = os.environ.get("PACKR_KEEP_DECODED_W", "0") == "1"


def grad_sink(param: torch.Tensor) -> torch.Tensor | None:
    """A fresh view of the gradient buffer an optimizer registered for
    `param` (param._packr_grad_sink = (flat_buffer, element_offset)), or None.
    Only offered while param.grad is None: the backward then writes the
    gradient straight into the buffer and autograd adopts the view as
    param.grad without a copy; with a gradient already present, autograd
    accumulates into it as usual.  Not offered either while a view lent before
    is still held: by autograd, when the parameter is used more than once and
    its gradients are yet to be summed, or by a caller of torch.autograd.grad."""
    spec = getattr(param, "_packr_grad_sink", None)
    if spec is None or param.grad is not None:
        return None
    buf, off = spec
    n = param.numel()
    if buf.dtype != param.dtype or buf.device != param.device or off + n > buf.numel():
        return None
    key = id(param)
    lent = _lent.get(key)
    if lent is not None and lent[0]() is param:
        if lent[1]() is not None:
            return None
        owner = lent[0]
    else:
        owner = weakref.ref(param, lambda _: _lent.pop(key, None))
    view = buf[off:off + n].view(param.shape)
    _lent[key] = owner, weakref.ref(view)
    return view


# id of a parameter -> (the parameter, the last view of its gradient buffer that
# was given out), both weak.  Not an attribute of the parameter, which would have
# to be saved and loaded with it.
_lent: dict = {}


def _forward_keep_w(ctx, x, W_p, W_f, lut, bias):
    """The forward; on the route where it decodes all of W first (many rows)
    and dX will be needed, the decoded W is kept on ctx for the backward's
    dX GEMM (2 bytes per weight held until the backward), so W is decoded
    once per step instead of twice."""
    ctx.wd = None
    x2 = x.reshape(-1, x.shape[-1]) if x.dim() != 2 else x
    M, K = x2.shape
    N = W_p.shape[1]
    if KEEP_DECODED_W and ctx.needs_input_grad[0] and _k.predecode_route(M, K, N, W_p, W_f):
        ctx.wd = _k.predecode_bf16(W_p, W_f, lut)
        return _k.forward_decoded(x, ctx.wd, bias)
    return _k.forward(x, W_p, W_f, lut, bias)


class PackRLinearFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, W_p, W_f, lut, bias=None, counts=None, evict_cb=None):
        if not x.is_cuda:
            raise RuntimeError("PackRLinear runs on CUDA tensors only (no CPU path in the B200 build)")
        ctx.save_for_backward(x, W_p, W_f, lut, counts)
        ctx.has_bias = bias is not None
        ctx.evict_cb = evict_cb
        ctx.wf_param = W_f
        return _forward_keep_w(ctx, x, W_p, W_f, lut, bias)

    @staticmethod
    def backward(ctx, grad_out):
        x, W_p, W_f, lut, counts = ctx.saved_tensors
        nx, _, nwf, nlut, nb = ctx.needs_input_grad[:5]
        dX, dW, dlut, dbias = _k.backward(grad_out, x, W_p, W_f, lut, counts, need_dx=nx, need_dw=nwf,
                                          need_dlut=nlut, need_dbias=ctx.has_bias and nb,
                                          dW_out=grad_sink(ctx.wf_param) if nwf else None,
                                          Wd=ctx.wd if nx else None)
        ctx.wd = None
        if ctx.evict_cb is not None:
            ctx.evict_cb()
        if dX is not None and dX.dtype != x.dtype:
            dX = dX.to(x.dtype)
        return dX, None, dW, dlut, dbias, None, None


class PackRMatmulFunction(torch.autograd.Function):
    """Custom autograd for out = x @ (W_f + lut[W_p]) (bias handled outside),
    reference packr/autograd.py:17-88."""

    @staticmethod
    def forward(ctx, x, W_p, W_f, lut, evict_cb=None, layer_name=None, offload_mgr=None):
        ctx.save_for_backward(x, W_p, W_f, lut)
        ctx._evict_cb = evict_cb
        ctx.wf_param = W_f
        return _k.packr_matmul(x, W_p, W_f, lut)

    @staticmethod
    def backward(ctx, grad_out):
        x, W_p, W_f, lut = ctx.saved_tensors
        nx, _, nwf, nlut = ctx.needs_input_grad[:4]
        dX, dW, dlut, _ = _k.backward(grad_out, x, W_p, W_f, lut, None, need_dx=nx, need_dw=nwf, need_dlut=nlut,
                                      need_dbias=False, dW_out=grad_sink(ctx.wf_param) if nwf else None)
        if ctx._evict_cb is not None:
            ctx._evict_cb()
        if dX is not None and dX.dtype != x.dtype:
            dX = dX.to(x.dtype)
        return dX, None, dW, dlut, None, None, None


def _linear_act_backward(ctx, grad_out):
    x, W_p, W_f, lut, z, counts = ctx.saved_tensors
    nx, _, nwf, nlut, nb, nr = ctx.needs_input_grad[:6]
    g = grad_out if grad_out.dtype == ctx.out_dtype else grad_out.to(ctx.out_dtype)
    g = _k.aligned16(g.contiguous())
    dX, dW, dlut, dbias = _k.linear_act_backward(g, z, ctx.activation, x, W_p, W_f, lut, counts, nx, nwf, nlut,
                                                 ctx.bias_dtype if nb else None,
                                                 dW_out=grad_sink(ctx.wf_param) if nwf else None, Wd=ctx.wd)
    ctx.wd = None
    return dX, None, dW, dlut, dbias, grad_out if nr else None, None, None, None


_linear_act_backward_once = once_differentiable(_linear_act_backward)


class PackRLinearActFunction(torch.autograd.Function):
    """out = act(x @ W + bias) + residual on contiguous 2-D operands; keeps x
    and, for an activation, z = x @ W + bias in out's dtype, and with
    KEEP_DECODED_W the decoded W (see there)."""

    @staticmethod
    def forward(ctx, x, W_p, W_f, lut, bias, residual, activation, out_dtype, counts):
        ctx.wd = None
        if KEEP_DECODED_W and ctx.needs_input_grad[0] and _k.predecode_route(x.shape[0], *W_p.shape, W_p, W_f):
            ctx.wd = _k.predecode_bf16(W_p, W_f, lut)
        out, z = _k.linear_act_forward(x, W_p, W_f, lut, bias, activation, residual, out_dtype,
                                       keep_z=activation != _NO_ACTIVATION, Wd=ctx.wd)
        ctx.save_for_backward(x, W_p, W_f, lut, z, counts)
        ctx.activation, ctx.out_dtype = activation, out_dtype
        ctx.bias_dtype = None if bias is None else bias.dtype
        ctx.wf_param = W_f
        return out

    @staticmethod
    def backward(ctx, grad_out):
        # a backward that records (create_graph) must refuse a second derivative
        return (_linear_act_backward_once if torch.is_grad_enabled() else _linear_act_backward)(ctx, grad_out)


_NO_ACTIVATION = _lib.ACTIVATIONS["none"]
_FLOATS = (torch.bfloat16, torch.float32)


def packr_linear_act(x, W_p, W_f, lut, bias=None, activation=None, residual=None, out_dtype=torch.float32, counts=None):
    """act(x @ (W_f + lut[W_p]) + bias) + residual, in one pass over the output,
    differentiable in x, W_f, lut, bias and residual.

    Args:
        x:          [..., K] f32 or bf16 (CUDA); f32 is rounded to bf16, the tensor cores' operand
        W_p:        [K, N] uint8 byte indices (contiguous)
        W_f:        [K, N] bf16 residual weights
        lut:        [256] f32 lookup table
        bias:       [N] bf16 or f32, or None
        activation: None or "none", "relu", "gelu" (error function), "gelu_tanh", "silu"
        residual:   [..., N] of out_dtype, or None
        out_dtype:  torch.float32 (the packed layers' output type) or torch.bfloat16; the
                    pre-activation kept for the backward has it too
        counts:     int32 [256] bincount of W_p (PackRLinear.lut_counts), used by the lut
                    gradient; counted there when None

    W = bf16(W_f + bf16(lut[W_p])) and x rounded to bf16 at every row count, also
    at the few rows (1 to 4, up to 16 for some widths) where packr_matmul takes f32
    x and the unrounded sum: there the two differ by those roundings.
    Gradients: the kept pre-activation has out_dtype (bf16: its slope is off by up
    to half a step of it).  dX is taken from the pre-activation's gradient rounded
    to bf16 and is itself rounded to bf16, for f32 x too, as PackRLinear's is.
    With bf16 x that gradient enters the weight and lut gradients rounded
    to bf16, as in PackRLinear; with f32 x as bf16 hi + lo parts
    (PACKR_DW_PRECISION).  The f32 lut gradient is short by about 1e-9 of itself
    per token (the tensor cores truncate the sums it is taken from), and its sums
    over CTAs are added in any order.
    Backward mode, once: second and forward-mode derivatives are refused."""
    _k.refuse_tangents("packr_linear_act", x, W_f, lut, bias, residual)
    if not x.is_cuda:
        raise RuntimeError("packr_linear_act runs on CUDA tensors only (no CPU path in the B200 build)")
    act = _lib.ACTIVATIONS.get("none" if activation is None else activation)
    if act is None:
        raise ValueError(f"packr_linear_act: activation must be one of {sorted(_lib.ACTIVATIONS)}, not {activation!r}")
    if x.dtype not in _FLOATS:
        raise TypeError(f"packr_linear_act: unsupported dtype {x.dtype}")
    if out_dtype not in _FLOATS:
        raise TypeError(f"packr_linear_act: out_dtype must be float32 or bfloat16, not {out_dtype}")
    if W_p.dtype != torch.uint8 or W_f.dtype != torch.bfloat16 or lut.dtype != torch.float32:
        raise TypeError("packr_linear_act: W_p must be uint8, W_f bfloat16 and lut float32")
    if W_p.dim() != 2 or W_p.shape != W_f.shape or lut.shape != _LUT_SHAPE or W_p.numel() == 0:
        raise ValueError("packr_linear_act: W_p and W_f must be [K, N] (K, N >= 1) and lut [256]")
    K, N = W_p.shape
    if x.dim() < 1 or x.shape[-1] != K:
        raise ValueError(f"packr_linear_act: x's last dimension must be {K}, got {tuple(x.shape)}")
    if not W_p.is_contiguous():
        raise ValueError("packr_linear_act: W_p must be contiguous")
    dev = x.device
    if W_p.device != dev or W_f.device != dev or lut.device != dev:
        raise ValueError("packr_linear_act: every tensor must be on x's device")
    grad = x.requires_grad or W_f.requires_grad or lut.requires_grad
    flat = x.dim() == 2
    x2 = _k.aligned16((x if flat else x.reshape(-1, K)).contiguous())
    W_f, lut = W_f.contiguous(), lut.contiguous()
    if bias is not None:
        if bias.dim() != 1 or bias.shape[0] != N or bias.dtype not in _FLOATS:
            raise ValueError(f"packr_linear_act: bias must be bf16 or f32 [{N}]")
        if bias.device != dev:
            raise ValueError("packr_linear_act: every tensor must be on x's device")
        grad = grad or bias.requires_grad
        bias = bias.contiguous()
    if residual is not None:
        if residual.shape != x.shape[:-1] + (N,) or residual.dtype != out_dtype:
            raise ValueError(f"packr_linear_act: residual must be {tuple(x.shape[:-1]) + (N,)} of {out_dtype}")
        if residual.device != dev:
            raise ValueError("packr_linear_act: every tensor must be on x's device")
        grad = grad or residual.requires_grad
        residual = (residual if flat else residual.reshape(-1, N)).contiguous()
    if counts is not None:
        if counts.dtype != torch.int32 or counts.shape != _LUT_SHAPE or not counts.is_contiguous():
            raise ValueError("packr_linear_act: counts must be contiguous int32 [256]")
        if counts.device != dev:
            raise ValueError("packr_linear_act: every tensor must be on x's device")
    if grad and torch.is_grad_enabled():
        out = PackRLinearActFunction.apply(x2, W_p, W_f, lut, bias, residual, act, out_dtype, counts)
    else:
        out = _k.linear_act_forward(x2, W_p, W_f, lut, bias, act, residual, out_dtype)[0]
    return out if flat else out.reshape(x.shape[:-1] + (N,))


_LUT_SHAPE = torch.Size([256])


# Legacy alias (reference packr/__init__.py:32)
PHRMatmulFunction = PackRMatmulFunction
