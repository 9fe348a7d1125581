"""Layer norm on B200: packr_layer_norm (functional, differentiable) and the
PackRLayerNorm module, over packr_layer_norm_forward / _backward of
libpackr_b200.so.

    s = x + residual                                   (f32, not rounded)
    y = (s - mean(s)) / sqrt(var(s) + eps) * weight + bias

over the last dimension.  x, residual and y share one dtype (bf16 or f32);
weight and bias another.  The backward recomputes s from x and residual, keeps
mean and rstd (f32, 8 bytes per row) and returns one gradient for both x and
residual.  The reference has no norm of its own: its models run torch's
LayerNorm between the packed layers.  No CPU path: CPU tensors raise.
"""
from __future__ import annotations

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import _lib
from .kernel import _addr, _on_device, _raw_stream, aligned16, refuse_tangents

_F32, _BF16 = torch.float32, torch.bfloat16
# A tensor that starts off the 16-byte grid is copied first where its rows are ones
# that the kernels hold in registers and there are _COPY_FROM elements or more: the
# kernels' path for any alignment has scalar loads and one CTA per row.  Measured
# (bf16, calls in a row, us that way / with the copy): forward 2800 x 768 21 / 25,
# 5600 x 768 39 / 25, 512 x 4096 16 / 25, 1024 x 4096 25 / 25, 16384 x 4096 404 / 142;
# backward 1400 x 768 34 / 34, 5600 x 768 95 / 34, 512 x 4096 28 / 34, 16384 x 4096
# 848 / 172.
_MAX_REGISTER_ROW = 16384
_COPY_FROM = 1 << 21
_CODE = {_F32: _lib.PACKR_DTYPE_F32, _BF16: _lib.PACKR_DTYPE_BF16}


def layer_norm_forward(x, weight, bias, eps, residual=None, stats=False):
    """(y, s) of a contiguous [..., N] x; with `stats` s is f32 [2, M], the rows'
    means and reciprocal standard deviations, else None.  Arguments as
    packr_layer_norm checks them."""
    lib = _lib.load()
    n = x.shape[-1]
    m = x.numel() // n
    y = torch.empty_like(x)
    s = torch.empty((2, m), dtype=_F32, device=x.device) if stats else None
    mean = _addr(s)
    w = weight if weight is not None else bias
    with _on_device(x.device):
        code = lib.packr_layer_norm_forward(
            x.data_ptr(), _addr(residual), _CODE[x.dtype], _addr(weight), _addr(bias),
            _CODE[w.dtype] if w is not None else 0, eps, y.data_ptr(), mean, None if s is None else mean + 4 * m, m, n,
            _raw_stream(x.device))
    _lib.check("packr_layer_norm_forward", code)
    return y, s


def layer_norm_backward(dy, x, weight, stats, residual=None, w_dtype=_F32, need_dx=True, need_dweight=True,
                        need_dbias=True):
    """(dx, dweight, dbias); entries not requested are None.  dx is also the
    residual's gradient."""
    lib = _lib.load()
    n = x.shape[-1]
    m = x.numel() // n
    dev = x.device
    dx = torch.empty_like(x) if need_dx else None
    dw = torch.empty(n, dtype=w_dtype, device=dev) if need_dweight else None
    db = torch.empty(n, dtype=w_dtype, device=dev) if need_dbias else None
    with _on_device(dev):
        nbytes = lib.packr_layer_norm_backward_workspace_bytes(m, n) if need_dweight or need_dbias else 0
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
        code = lib.packr_layer_norm_backward(
            dy.data_ptr(), x.data_ptr(), _addr(residual), _CODE[x.dtype], _addr(weight), _CODE[w_dtype],
            stats.data_ptr(), stats.data_ptr() + 4 * m, _addr(dx), _addr(dw), _addr(db), m, n, _addr(ws), nbytes,
            _raw_stream(dev))
    _lib.check("packr_layer_norm_backward", code)
    return dx, dw, db


def _norm_backward(ctx, dy):
    x, weight, residual, stats = ctx.saved_tensors
    nx, nw, nb, _, nr = ctx.needs_input_grad
    if dy.dtype != x.dtype:
        dy = dy.to(x.dtype)
    dx, dw, db = layer_norm_backward(_operand(dy), x, weight, stats, residual, ctx.w_dtype, nx or nr, nw, nb)
    return dx if nx else None, dw, db, None, dx if nr else None


_norm_backward_once = once_differentiable(_norm_backward)


class PackRLayerNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, residual):
        y, stats = layer_norm_forward(x, weight, bias, eps, residual, stats=True)
        ctx.save_for_backward(x, weight, residual, stats)
        w = weight if weight is not None else bias
        ctx.w_dtype = _F32 if w is None else w.dtype
        return y

    @staticmethod
    def backward(ctx, dy):
        # a backward that records (create_graph) must refuse a second derivative
        return _norm_backward_once(ctx, dy) if torch.is_grad_enabled() else _norm_backward(ctx, dy)


def packr_layer_norm(x, weight=None, bias=None, eps=1e-5, residual=None):
    """Layer norm of x (+ residual) over its last dimension, differentiable in
    x, residual, weight and bias.

    Args:
        x:        [..., N] f32 or bf16 (CUDA)
        weight:   [N] f32 or bf16, or None
        bias:     [N] of weight's dtype, or None
        eps:      added to the variance
        residual: tensor of x's shape and dtype added to x first, or None

    Backward mode, once: second and forward-mode derivatives are refused."""
    refuse_tangents("packr_layer_norm", x, weight, bias, residual)
    if not x.is_cuda:
        raise RuntimeError("packr_layer_norm runs on CUDA tensors only (no CPU path in the B200 build)")
    if x.dtype not in _CODE:
        raise TypeError(f"packr_layer_norm: unsupported dtype {x.dtype}")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("packr_layer_norm: x needs a last dimension of at least 1")
    grad = x.requires_grad
    x = _operand(x)
    if weight is not None:
        _check_vector("weight", weight, x)
        grad = grad or weight.requires_grad
        weight = weight.contiguous()
    if bias is not None:
        _check_vector("bias", bias, x)
        if weight is not None and weight.dtype != bias.dtype:
            raise TypeError("packr_layer_norm: weight and bias must have one dtype")
        grad = grad or bias.requires_grad
        bias = bias.contiguous()
    if residual is not None:
        if residual.shape != x.shape or residual.dtype != x.dtype or residual.device != x.device:
            raise ValueError("packr_layer_norm: residual must have x's shape, dtype and device")
        grad = grad or residual.requires_grad
        residual = _operand(residual)
    eps = float(eps)
    if not eps >= 0.0:
        raise ValueError(f"packr_layer_norm: eps must be >= 0, got {eps}")
    if grad and torch.is_grad_enabled():
        return PackRLayerNormFunction.apply(x, weight, bias, eps, residual)
    return layer_norm_forward(x, weight, bias, eps, residual)[0]


def _operand(t):
    t = t.contiguous()
    return aligned16(t) if t.shape[-1] <= _MAX_REGISTER_ROW and t.numel() >= _COPY_FROM else t


def _check_vector(name, t, x):
    if t.dim() != 1 or t.shape[0] != x.shape[-1] or t.dtype not in _CODE or t.device != x.device:
        raise ValueError(f"packr_layer_norm: {name} must be f32 or bf16 [{x.shape[-1]}] on x's device")


class PackRLayerNorm(nn.LayerNorm):
    """nn.LayerNorm over one dimension, run by packr_layer_norm; forward takes
    an optional residual that is added to the input first (post-norm blocks:
    norm(dense(x), residual=x)).  Under autocast it is computed and returned in
    f32, as nn.LayerNorm is."""

    def __init__(self, normalized_shape, eps=1e-5, elementwise_affine=True, bias=True, device=None, dtype=None):
        super().__init__(normalized_shape, eps=eps, elementwise_affine=elementwise_affine, bias=bias, device=device,
                         dtype=dtype)
        if len(self.normalized_shape) != 1:
            raise ValueError("PackRLayerNorm normalises the last dimension only")

    def forward(self, x, residual=None):
        if x.shape[-1:] != torch.Size(self.normalized_shape):
            raise ValueError(f"PackRLayerNorm: last dimension {tuple(x.shape[-1:])} != {tuple(self.normalized_shape)}")
        if torch.is_autocast_enabled(x.device.type):
            # f64 stays (and is refused), as autocast leaves it
            x = x.float() if x.dtype != torch.float64 else x
            residual = residual.float() if residual is not None and residual.dtype != torch.float64 else residual
        return packr_layer_norm(x, self.weight, self.bias, self.eps, residual)

    @classmethod
    def from_layer_norm(cls, module: nn.LayerNorm):
        """Takes over an nn.LayerNorm's parameters (the same objects)."""
        if not isinstance(module, nn.LayerNorm):
            raise TypeError(f"Expected nn.LayerNorm, got {type(module)}")
        if len(module.normalized_shape) != 1:
            raise ValueError("PackRLayerNorm normalises the last dimension only")
        m = cls.__new__(cls)
        nn.Module.__init__(m)
        m.normalized_shape, m.eps = tuple(module.normalized_shape), module.eps
        m.elementwise_affine = module.elementwise_affine
        m.weight, m.bias = module.weight, module.bias
        m.training = module.training
        return m
