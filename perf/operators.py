"""Measured cases of the fused feed-forward operators: the compressed linear layer with bias, activation and residual
in its epilogue, and layer norm with its residual sum, each forward and backward.

`run` computes a case either with the framework's kernels (`own` true) or in its plain form: elementary torch
operations in 32 bits, rounded once at the end.  `exact` restates the definitions in 64 bits.

Definitions (M rows, K input features, N output features):
  linear   W = bf16(W_f + bf16(lut[W_p]));  z = bf16(x) W + bias;  out = act(z) + residual
           dz = dout * act'(z);  dx = dz W^T;  dW_f = x^T dz;  dbias = sum over rows of dz;
           dlut[b] = sum of dW_f over W_p == b, / (count[b] + 1e-8);  dresidual = dout
  norm     s = x + residual;  h = (s - mean(s)) / sqrt(var(s) + eps);  y = h * weight + bias
           g = dy * weight;  dx = dresidual = (g - mean(g) - h mean(g h)) / sqrt(var(s) + eps);
           dweight = sum over rows of dy * h;  dbias = sum over rows of dy
The rounding of W and of an f32 x to bf16 is the layer's own: its weights are stored that way and its operands are bf16.
"""
import math

import torch

own = False

EPS = 1e-5
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
ACTS = ("none", "relu", "gelu", "gelu_tanh", "silu")


def _linear(name, rows, k, n, act, x="bf16", out="bf16", bias=True, residual=False, train=False, lut=False):
    c = {"op": "linear", "rows": rows, "k": k, "n": n, "act": act, "x": x, "out": out, "bias": bias,
         "residual": residual, "train": train, "lut": lut}
    return dict(c, name=name) if name else c


def _norm(name, rows, n, x="bf16", weight="bf16", residual=False, train=False):
    c = {"op": "norm", "rows": rows, "n": n, "x": x, "weight": weight, "residual": residual, "train": train}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one token through a 7B decoder's gate projection
        _linear("linear 1 gate silu", 1, 4096, 11008, "silu", bias=False),
        # sixteen sequences decoding: the down projection added to the residual stream
        _linear("linear 16 down residual", 16, 11008, 4096, "none", residual=True),
        # a short prompt through a layer of odd sizes, f32 activations as in the BERT workload
        _linear("linear 777 odd f32", 777, 1000, 1111, "gelu_tanh", x="f32", out="f32", residual=True),
        # a prompt through a 7B-sized up projection
        _linear("linear 4096 up gelu", 4096, 4096, 11008, "gelu_tanh"),
        # training, the up projection with its activation; the table frozen (learnable_lut=False)
        _linear("linear 4096 up train", 4096, 4096, 11008, "gelu", train=True),
        # training, the down projection added to the residual stream; the table learnt
        _linear("linear 4096 down train", 4096, 11008, 4096, "none", residual=True, train=True, lut=True),
        # a small fine-tuning batch, output features that fit no tile
        _linear("linear 100 odd train", 100, 768, 1001, "relu", train=True),
        # one token's norm in a decoder
        _norm("norm 1 token", 1, 4096, residual=True),
        # a prompt's norm, wide rows
        _norm("norm 2048 prompt", 2048, 8192),
        # BERT-base fine-tuning, batch 32 x seq 128: the norm after each sublayer, in f32
        _norm("norm 4096 bert train", 4096, 768, x="f32", weight="f32", residual=True, train=True),
        # decoder training, 8 sequences of 2048
        _norm("norm 16384 train", 16384, 4096, residual=True, train=True),
        # rows of an odd length, bf16 activations under f32 weights
        _norm("norm 3001 odd train", 3001, 5001, weight="f32", train=True),
    ]


def _log(rng, lo, hi):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return min(hi, max(lo, v))


def draw(rng):
    """Sizes over their logarithms, half of the widths multiples of 64 as models have them and half of any value."""
    if rng.random() < 0.6:
        train = rng.random() < 0.5
        most = 4096 * 4096 * 11008
        while True:
            rows, k, n = _log(rng, 1, 8192), _log(rng, 64, 11008), _log(rng, 64, 14336)
            if rng.random() < 0.5:
                k, n = max(64, k // 64 * 64), max(64, n // 64 * 64)
            if rows * k * n <= most:
                break
        act, lut = rng.choice(ACTS), False
        if train:
            x, out = "bf16", "bf16"
            lut = act == "none"
        else:
            x, out = rng.choice((("bf16", "bf16"), ("bf16", "f32"), ("f32", "f32")))
        return _linear("", rows, k, n, act, x, out, rng.random() < 0.7, rng.random() < 0.5, train, lut)
    while True:
        rows, n = _log(rng, 1, 32768), _log(rng, 64, 16384)
        if rng.random() < 0.5:
            n = n // 64 * 64
        if rows * n <= 16384 * 4096:
            break
    x, weight = rng.choice((("bf16", "bf16"), ("bf16", "f32"), ("f32", "f32")))
    return _norm("", rows, n, x, weight, rng.random() < 0.5, rng.random() < 0.6)


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def prepare(case, seed):
    g, c = _generator(seed), case
    if c["op"] == "linear":
        m, k, n, fan = c["rows"], c["k"], c["n"], math.sqrt(768.0 / c["k"])
        s = {"x": _normal(g, m, k).to(TYPES[c["x"]]),
             "W_p": torch.randint(0, 256, (k, n), generator=g, device="cuda", dtype=torch.uint8),
             "lut": torch.sort(_normal(g, 256) * (0.02 * fan)).values,
             "W_f": (_normal(g, k, n) * (0.002 * fan)).bfloat16(),
             "bias": (_normal(g, n) * 0.1).bfloat16() if c["bias"] else None,
             "residual": _normal(g, m, n).to(TYPES[c["out"]]) if c["residual"] else None}
        # the layer's bin counts: W_p is frozen, so a layer counts it once
        s["counts"] = torch.bincount(s["W_p"].view(-1), minlength=256).int() if c["lut"] else None
        s["dout"] = _normal(g, m, n).to(TYPES[c["out"]]) if c["train"] else None
        wanted = ["x", "W_f"] + ["bias"] * c["bias"] + ["residual"] * c["residual"] + ["lut"] * c["lut"]
    else:
        m, n = c["rows"], c["n"]
        # hidden states: offsets and scales of their own per feature, a few features far larger than the rest
        scale = torch.exp(0.5 * _normal(g, n)) * torch.where(torch.rand(n, generator=g, device="cuda") < 0.004, 20.0, 1.0)
        s = {"x": (_normal(g, m, n) * scale + 0.3 * _normal(g, n)).to(TYPES[c["x"]]),
             "residual": (_normal(g, m, n) * scale).to(TYPES[c["x"]]) if c["residual"] else None,
             "weight": (1.0 + 0.1 * _normal(g, n)).to(TYPES[c["weight"]]),
             "bias": (0.1 * _normal(g, n)).to(TYPES[c["weight"]]),
             "dy": _normal(g, m, n).to(TYPES[c["x"]]) if c["train"] else None}
        wanted = ["x", "weight", "bias"] + ["residual"] * c["residual"]
    if c["train"]:
        for name in wanted:
            s[name].requires_grad_(True)
    s["case"], s["wanted"] = c, wanted
    return s


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return _plain_linear(state) if state["case"]["op"] == "linear" else _plain_norm(state)


def _run_own(s):
    import packr_b200 as packr
    c = s["case"]
    if c["op"] == "linear":
        out = packr.packr_linear_act(s["x"], s["W_p"], s["W_f"], s["lut"], s["bias"], activation=c["act"],
                                     residual=s["residual"], out_dtype=TYPES[c["out"]], counts=s["counts"])
        upstream = s["dout"]
    else:
        out = packr.packr_layer_norm(s["x"], s["weight"], s["bias"], eps=EPS, residual=s["residual"])
        upstream = s["dy"]
    if not c["train"]:
        return {"out": out}
    grads = torch.autograd.grad(out, [s[name] for name in s["wanted"]], upstream)
    return {"out": out.detach(), **dict(zip(("d" + name for name in s["wanted"]), grads))}


# ------------------------------------------------------------------ plain forms, 32 bits

def _act(z, act):
    if act == "relu":
        return z.clamp_min(0)
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _act_slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * math.sqrt(0.5 / math.pi)
    if act == "gelu_tanh":
        r = math.sqrt(2 / math.pi)
        t = torch.tanh(r * (z + 0.044715 * z ** 3))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * r * (1 + 3 * 0.044715 * z * z)
    if act == "silu":
        p = 1 / (1 + torch.exp(-z))
        return p * (1 + z * (1 - p))
    return torch.ones_like(z)


def _plain_linear(s):
    c = s["case"]
    x = s["x"].bfloat16().float()
    idx = s["W_p"].long()
    w = (s["W_f"].float() + s["lut"].bfloat16().float()[idx]).bfloat16().float()
    z = x @ w
    if s["bias"] is not None:
        z = z + s["bias"].float()
    out = _act(z, c["act"])
    if s["residual"] is not None:
        out = out + s["residual"].float()
    got = {"out": out.to(TYPES[c["out"]])}
    if c["train"]:
        dz = s["dout"].float() * _act_slope(z, c["act"])
        dw = x.t() @ dz
        got["dx"] = (dz @ w.t()).to(s["x"].dtype)
        got["dW_f"] = dw.to(s["W_f"].dtype)
        if s["bias"] is not None:
            got["dbias"] = dz.sum(0).to(s["bias"].dtype)
        if s["residual"] is not None:
            got["dresidual"] = s["dout"]
        if c["lut"]:  # long sums: K * N / 256 terms a bin, in 64 bits
            bins = torch.zeros(256, dtype=torch.float64, device="cuda").index_add_(0, idx.view(-1), dw.double().view(-1))
            got["dlut"] = (bins / (s["counts"].double() + 1e-8)).float()
    return got


def _plain_norm(s):
    c = s["case"]
    x = s["x"].float()
    if s["residual"] is not None:
        x = x + s["residual"].float()
    centred = x - x.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt((centred * centred).mean(1, keepdim=True) + EPS)
    h, w = centred * rstd, s["weight"].float()
    got = {"out": (h * w + s["bias"].float()).to(s["x"].dtype)}
    if c["train"]:
        dy = s["dy"].float()
        g = dy * w
        dx = ((g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True)) * rstd).to(s["x"].dtype)
        got["dx"] = dx
        got["dweight"] = (dy * h).sum(0).to(s["weight"].dtype)
        got["dbias"] = dy.sum(0).to(s["bias"].dtype)
        if s["residual"] is not None:
            got["dresidual"] = dx
    return got


# ------------------------------------------------------------------ work and the 64-bit definition

def work(case):
    c, size = case, {"f32": 4, "bf16": 2}
    m, n = c["rows"], c["n"]
    if c["op"] == "linear":
        k, xb, ob = c["k"], size[c["x"]], size[c["out"]]
        read = m * k * xb + 3 * k * n + 1024 + 2 * n * c["bias"] + m * n * ob * c["residual"]
        written, flops = m * n * ob, 2 * m * k * n
        if c["train"]:  # the residual's gradient is the upstream one
            read += m * n * ob
            written += m * k * xb + 2 * k * n + 2 * n * c["bias"] + 1024 * c["lut"]
            flops *= 3
        return {"bytes": read + written, "flops": flops}
    xb, wb = size[c["x"]], size[c["weight"]]
    passes = 2 + c["residual"] + 2 * c["train"]
    return {"bytes": m * n * xb * passes + n * wb * (4 if c["train"] else 2), "flops": m * n * (20 if c["train"] else 8)}


def exact(case, seed):
    """From the definitions, through torch's autograd in 64 bits where gradients are wanted."""
    s = prepare(case, seed)
    d = {k: v.detach().double() for k, v in s.items() if torch.is_tensor(v) and v.is_floating_point()}
    leaf = lambda t: t.requires_grad_(case["train"])  # noqa: E731
    if case["op"] == "norm":
        x = leaf(d["x"] + d["residual"] if case["residual"] else d["x"])
        weight, bias = leaf(d["weight"]), leaf(d["bias"])
        mean = x.sum(1, keepdim=True) / case["n"]
        y = (x - mean) * torch.rsqrt(((x - mean) ** 2).sum(1, keepdim=True) / case["n"] + EPS) * weight + bias
        if not case["train"]:
            return {"out": y}
        dx, dweight, dbias = torch.autograd.grad(y, [x, weight, bias], d["dy"])
        got = {"out": y.detach(), "dx": dx, "dweight": dweight, "dbias": dbias}
        return dict(got, dresidual=dx) if case["residual"] else got
    x = leaf(s["x"].detach().bfloat16().double())
    table = s["lut"].detach().bfloat16().double()
    # a bf16 sum of two bf16 values is exact in 64 bits before its rounding
    w = leaf((d["W_f"] + table.take(s["W_p"].long())).bfloat16().double())
    z = torch.matmul(x, w)
    bias = leaf(d["bias"]) if case["bias"] else None
    z = z if bias is None else z.add(bias)
    a = case["act"]
    y = (torch.where(z > 0, z, 0 * z) if a == "relu"
         else z * (0.5 * torch.special.erfc(-z / 2 ** 0.5)) if a == "gelu"
         else z * torch.sigmoid(2 * (2 / math.pi) ** 0.5 * (z + 0.044715 * z * z * z)) if a == "gelu_tanh"
         else z * torch.sigmoid(z) if a == "silu" else z)
    y = y + d["residual"] if case["residual"] else y
    if not case["train"]:
        return {"out": y}
    wanted = [x, w] + ([bias] if case["bias"] else [])
    grads = torch.autograd.grad(y, wanted, d["dout"])
    got = {"out": y.detach(), "dx": grads[0], "dW_f": grads[1]}
    if case["bias"]:
        got["dbias"] = grads[2]
    if case["residual"]:
        got["dresidual"] = d["dout"]
    if case["lut"]:
        flat = s["W_p"].view(-1)
        order = torch.argsort(flat)
        total = torch.cat([torch.zeros(1, dtype=torch.float64, device="cuda"), grads[1].view(-1)[order].cumsum(0)])
        ends = torch.bincount(flat, minlength=256).cumsum(0)
        per_bin = torch.diff(total[ends], prepend=total[:1])
        got["dlut"] = per_bin / (torch.bincount(flat, minlength=256) + 1e-8)
    return got
