"""Plain 64-bit forms of the fused feed-forward operators, with elementwise
bounds on what the kernels may differ from them.  Runs on any device.

Bounds count roundings: U[t] is half a step of type t relative to the value
(bf16 2^-8, f32 2^-24).  An f32 sum of n products kept by the tensor cores or
by f32 additions is off by at most n * 2^-23 times the sum of the products'
magnitudes (each addition loses at most one unit of the running sum, which
that sum bounds).  The activations are 1.13-Lipschitz at most, their slopes
0.8-Lipschitz (relu's apart), and their f32 evaluation is off by at most
4e-7 * (1 + |z|) (erfc approximated within 1.5e-7, a few roundings)."""
import math

import torch

U = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
LIP, LIP2, EVAL = 1.13, 0.8, 4e-7
ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]


def act64(z, a):
    if a == "relu":
        return z.clamp_min(0)
    if a == "gelu":
        return z * 0.5 * torch.special.erfc(-z / math.sqrt(2))
    if a == "gelu_tanh":
        return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
    if a == "silu":
        return z * torch.sigmoid(z)
    return z


def slope64(z, a):
    if a == "none":
        return torch.ones_like(z)
    if a == "relu":
        return (z > 0).double()
    z = z.detach().requires_grad_(True)
    with torch.enable_grad():
        return torch.autograd.grad(act64(z, a).sum(), z)[0]


def weights64(W_p, W_f, lut):
    """W = bf16(W_f + bf16(lut[W_p])): the sum of two bf16 values is exact in 64 bits."""
    return (W_f.detach().double() + lut.detach().bfloat16().double()[W_p.long()]).bfloat16().double()


def linear64(x, W_p, W_f, lut, bias, activation, residual, out_dtype, dout=None, x_split=False):
    """{name: (value, bound)} of out and, with dout, dx, dW_f, dbias, dlut.
    x_split: f32 x, whose dW takes hi + lo parts."""
    W = weights64(W_p, W_f, lut)
    K, N = W.shape
    x64 = x.detach().double()
    xh = x.detach().bfloat16().double()
    b = torch.zeros(N, dtype=torch.float64, device=x.device) if bias is None else bias.detach().double()
    z = xh @ W + b
    zerr = (K + 2) * 2.0 ** -23 * (xh.abs() @ W.abs() + b.abs()) + 1e-30
    y = act64(z, activation)
    r = torch.zeros_like(y) if residual is None else residual.detach().double()
    out = y + r
    u = U[out_dtype]
    oerr = LIP * zerr + (EVAL * (1 + z.abs()) if activation != "none" else 0) + 2.0 ** -23 * (y.abs() + r.abs())
    got = {"out": (out, oerr + u * (out.abs() + oerr))}
    if dout is None:
        return got
    g = dout.detach().double()
    M = x.shape[0]
    s = slope64(z, activation)
    dz = g * s
    if activation == "none":
        f32err = torch.zeros_like(dz)
    else:  # z stored with a rounding; the slope's evaluation
        f32err = g.abs() * (LIP2 * (zerr + u * z.abs()) + EVAL * (1 + z.abs()) + 2.0 ** -22)
        if activation == "relu":  # z within its error of zero may fall on either side
            f32err = g.abs() * (z.abs() <= zerr).double() + 2.0 ** -23 * dz.abs()
    operand = 0.0 if activation == "none" and out_dtype == torch.bfloat16 else U[torch.bfloat16]
    derr = f32err + operand * (dz.abs() + f32err)  # as the bf16 operand of a GEMM
    uh = U[torch.bfloat16]
    dx = dz @ W.t()
    dxerr = derr @ W.abs().t() + (N + 2) * 2.0 ** -23 * (dz.abs() @ W.abs().t())
    got["dx"] = (dx, dxerr + uh * (dx.abs() + dxerr))
    if x_split:  # hi + lo parts of both: 2^-16 relative, the lo * lo term dropped
        xa, werr = x64, f32err + 2.0 ** -16 * dz.abs()
        dw = xa.t() @ dz
        dwerr = xa.abs().t() @ werr + 3 * 2.0 ** -16 * (xa.abs().t() @ dz.abs())
    else:
        xa, werr = xh, derr
        dw = xa.t() @ dz
        dwerr = xa.abs().t() @ werr
    dwerr = dwerr + 3 * (M + 2) * 2.0 ** -23 * (xa.abs().t() @ dz.abs())
    got["dW_f"] = (dw, dwerr + uh * (dw.abs() + dwerr))
    db = dz.sum(0)
    dberr = f32err.sum(0) + (M + 2) * 2.0 ** -23 * dz.abs().sum(0)
    ub = uh if bias is None else U[bias.dtype]
    got["dbias"] = (db, dberr + ub * (db.abs() + dberr))
    idx = W_p.reshape(-1).long()
    n = torch.bincount(idx, minlength=256).double()
    zero = torch.zeros(256, dtype=torch.float64, device=x.device)
    dlut = zero.index_add(0, idx, dw.reshape(-1)) / (n + 1e-8)
    # the fixed-point bins add 2^-21 of the tile's largest value per element
    lerr = zero.index_add(0, idx, dwerr.reshape(-1)) / (n + 1e-8) + 2.0 ** -21 * dw.abs().max() + 2.0 ** -14 * zero.index_add(
        0, idx, dw.abs().reshape(-1)) / (n + 1e-8)
    got["dlut"] = (dlut, lerr)
    return got


def norm64(x, residual, weight, bias, eps, dy=None):
    """{name: (value, bound)} of y and, with dy, dx, dweight, dbias.

    f32 arithmetic on s = x + residual: mean and the two backward means are
    sums over N kept in E elements a thread, then log2 steps, so 64 roundings
    bound them; h is then off by herr."""
    s = x.detach().double() + (0 if residual is None else residual.detach().double())
    M, N = s.shape
    f = 2.0 ** -23
    mean = s.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(((s - mean) ** 2).mean(1, keepdim=True) + eps)
    h = (s - mean) * rstd
    depth = 64 + (N / 256 if N > 16384 else 0)
    merr = depth * f * s.abs().mean(1, keepdim=True)
    herr = (f * s.abs() + merr) * rstd + h.abs() * (depth * f + merr * rstd)
    w = torch.ones(N, dtype=torch.float64, device=x.device) if weight is None else weight.detach().double()
    b = torch.zeros(N, dtype=torch.float64, device=x.device) if bias is None else bias.detach().double()
    y = h * w + b
    yerr = herr * w.abs() + 2 * f * (h.abs() * w.abs() + b.abs())
    u = U[x.dtype]
    got = {"y": (y, yerr + u * (y.abs() + yerr))}
    if dy is None:
        return got
    d = dy.detach().double()
    g = d * w
    m1, m2 = g.mean(1, keepdim=True), (g * h).mean(1, keepdim=True)
    dx = rstd * (g - m1 - h * m2)
    gerr = 2 * f * g.abs()
    m1err = depth * f * g.abs().mean(1, keepdim=True)
    m2err = depth * f * (g * h).abs().mean(1, keepdim=True) + (g.abs() * herr).mean(1, keepdim=True)
    dxerr = rstd * (gerr + m1err + h.abs() * m2err + herr * m2.abs()) + 4 * f * rstd * (
        g.abs() + m1.abs() + (h * m2).abs()) + dx.abs() * (depth * f + merr * rstd)
    got["dx"] = (dx, dxerr + u * (dx.abs() + dxerr))
    uw = U[torch.float32 if weight is None and bias is None else (weight if weight is not None else bias).dtype]
    dw, db = (d * h).sum(0), d.sum(0)
    dwerr = (d.abs() * herr).sum(0) + (M + 8) * f * (d * h).abs().sum(0)
    dberr = (M + 8) * f * d.abs().sum(0)
    got["dweight"] = (dw, dwerr + uw * (dw.abs() + dwerr))
    got["dbias"] = (db, dberr + uw * (db.abs() + dberr))
    return got


def check(name, got, want, rel=None):
    """Every element within its bound; with `rel`, the 2-norm of the error too."""
    value, bound = want
    got = got.detach().double().reshape(value.shape)
    assert torch.isfinite(got).all(), f"{name}: not finite"
    err = (got - value).abs()
    over = err - bound
    assert (over <= 0).all(), (name, "largest error over its bound", float((err / bound.clamp_min(1e-300)).max()),
                               float(err.flatten()[over.flatten().argmax()]))
    if rel is not None and value.numel():
        off = float(err.norm() / value.norm().clamp_min(1e-300))
        assert off <= rel, (name, "relative error", off)
