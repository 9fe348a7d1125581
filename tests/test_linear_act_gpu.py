"""packr_linear_act on the GPU against its 64-bit form: every route of the
forward and the backward, types, activations, odd sizes."""
import pytest
import torch

import packr_b200 as packr
from packr_b200.synthetic import linear_case
from fused_reference import ACTS, check, linear64

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
# bf16 results: one rounding, at most 2^-8 / sqrt(3) in the 2-norm; gradients
# through a kept bf16 z and a bf16 operand: two more of the same size
REL_OUT, REL_GRAD = 2.4e-3, 4.2e-3


def case(M, K, N, xt, out, seed=0, bias=BF16, residual=True):
    c = linear_case(M, K, N, x_dtype=xt, bias=True, seed=seed, device="cuda", fanin_scaled=True)
    g = torch.Generator(device="cuda").manual_seed(seed + 1000)
    c["bias"] = None if bias is None else (torch.randn(N, generator=g, device="cuda") * 0.3).to(bias)
    c["residual"] = torch.randn(M, N, generator=g, device="cuda").to(out) if residual else None
    c["dout"] = torch.randn(M, N, generator=g, device="cuda").to(out)
    return c


def call(c, act, out, **kw):
    return packr.packr_linear_act(c["x"], c["W_p"], c["W_f"], c["lut"], c["bias"], activation=act,
                                  residual=c["residual"], out_dtype=out, **kw)


def grads(c, act, out, need=("x", "W_f", "bias", "lut", "residual"), **kw):
    leaves = {k: c[k].detach().requires_grad_(True) for k in need if c[k] is not None}
    y = call({**c, **leaves}, act, out, **kw)
    got = torch.autograd.grad(y, list(leaves.values()), c["dout"])
    return {"out": y, **dict(zip(("d" + k for k in leaves), got))}


def compare(c, got, act, out):
    want = linear64(c["x"], c["W_p"], c["W_f"], c["lut"], c["bias"], act, c["residual"], out,
                    c["dout"] if len(got) > 1 else None, x_split=c["x"].dtype == F32)
    for k, v in got.items():
        if k == "dresidual":
            assert torch.equal(v, c["dout"])
            continue
        rel = REL_OUT if k == "out" and out == BF16 else REL_GRAD if k in ("dx", "dW_f") else None
        check(k, v, want[k], rel if v.numel() > 2000 else None)


# up to 4 rows, 5..128, above; widths that TMA reads and that it does not
SIZES = [(6, 72, 144), (13, 700, 1040), (17, 520, 256), (31, 96, 128), (32, 4104, 144), (1, 64, 64), (1, 1000, 1001), (2, 256, 130), (4, 130, 96), (3, 33, 20), (5, 128, 64), (7, 100, 33),
         (16, 64, 1000), (100, 768, 1001), (128, 200, 256), (129, 64, 512), (200, 1000, 520), (257, 72, 1111),
         (300, 40, 50), (1, 1, 1), (130, 1, 3), (1030, 128, 272)]


@pytest.mark.parametrize("xt,out", [(BF16, BF16), (BF16, F32), (F32, F32), (F32, BF16)])
@pytest.mark.parametrize("M,K,N", SIZES)
def test_forward(cuda, M, K, N, xt, out):
    c = case(M, K, N, xt, out, seed=M + K + N)
    act = ACTS[(M + K + N) % len(ACTS)]
    compare(c, {"out": call(c, act, out)}, act, out)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M", [2, 24, 150])
def test_activations(cuda, act, M):
    for out in (F32, BF16):
        c = case(M, 96, 160, BF16, out, seed=M, bias=F32)
        compare(c, grads(c, act, out), act, out)


@pytest.mark.parametrize("xt,out", [(BF16, BF16), (BF16, F32), (F32, F32)])
@pytest.mark.parametrize("M,K,N", [(1, 64, 64), (3, 130, 33), (100, 768, 1001), (64, 256, 320), (150, 200, 272),
                                   (513, 100, 77), (1100, 264, 528)])
def test_gradients(cuda, M, K, N, xt, out):
    for i, act in enumerate(("none", "gelu", "silu")):
        c = case(M, K, N, xt, out, seed=M + i, residual=i != 1, bias=None if i == 2 else BF16)
        compare(c, grads(c, act, out), act, out)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M", [1, 8, 30, 140])
def test_activations_of_huge_values(cuda, act, M):
    """z = +-1e30, whose square is past the type's range: act and slope are those
    of the limits, 0 and z, 0 and 1."""
    K, N = 64, 96
    z = torch.where(torch.arange(N, device="cuda") % 2 == 0, 1e30, -1e30)
    c = dict(x=torch.zeros(M, K, dtype=BF16, device="cuda"), W_p=torch.zeros(K, N, dtype=torch.uint8, device="cuda"),
             W_f=torch.zeros(K, N, dtype=BF16, device="cuda"), lut=torch.zeros(256, device="cuda"),
             bias=z.clone().requires_grad_(True))
    y = packr.packr_linear_act(**c, activation=act)
    db, = torch.autograd.grad(y, c["bias"], torch.ones_like(y))
    kept = z if act == "none" else z.clamp_min(0.0)
    assert torch.equal(y, kept.expand(M, N))
    assert torch.equal(db, torch.full_like(z, float(M)) if act == "none" else M * (z > 0).float())


@pytest.mark.parametrize("need", [("x",), ("W_f",), ("lut",), ("bias",), ("residual",), ("x", "bias")])
def test_only_the_gradients_asked_for(cuda, need):
    c = case(140, 128, 144, BF16, BF16, seed=2)
    got = grads(c, "gelu", BF16, need=need)
    assert set(got) == {"out"} | {"d" + k for k in need}
    compare(c, got, "gelu", BF16)


def test_counts_given_or_counted(cuda):
    c = case(40, 128, 144, BF16, BF16, seed=2)
    counts = torch.bincount(c["W_p"].view(-1), minlength=256).int()
    a = grads(c, "none", BF16, counts=counts)["dlut"]
    b = grads(c, "none", BF16)["dlut"]
    assert torch.allclose(a, b, rtol=1e-4, atol=1e-6)  # f32 atomics over CTAs: their order may differ


def test_split_weight_gradient_of_f32_inputs(cuda):
    """f32 x and f32 out: z is kept in f32 and dW takes hi + lo parts, so the
    f32 lut gradient is good to 2^-14, not to the bf16 operand's 2^-8."""
    c = case(200, 192, 320, F32, F32, seed=3)
    got = grads(c, "gelu", F32)
    want = linear64(c["x"], c["W_p"], c["W_f"], c["lut"], c["bias"], "gelu", c["residual"], F32, c["dout"], x_split=True)
    v = want["dlut"][0]
    assert float((got["dlut"].double() - v).norm() / v.norm()) < 2.0 ** -14


def test_wide_range_of_preactivations(cuda):
    """Saturated and tail values of every activation, infinities included,
    through bias alone (x = 0)."""
    z = torch.tensor([0.0, -0.0, 1e-30, -1e-30, 1e-3, -1e-3, 0.5, -0.5, 3.0, -3.0, 5.5, -5.5, 9.0, -9.0, 13.0, -13.0,
                      40.0, -40.0, 1e4, -1e4, 3e18, -3e18], device="cuda")
    N = z.numel()
    for M in (1, 20, 200):
        x = torch.zeros(M, 8, device="cuda")
        W_p, lut = torch.zeros(8, N, dtype=torch.uint8, device="cuda"), torch.zeros(256, device="cuda")
        W_f = torch.zeros(8, N, dtype=BF16, device="cuda")
        for act in ACTS:
            y = packr.packr_linear_act(x, W_p, W_f, lut, z, activation=act)
            want = linear64(x, W_p, W_f, lut, z, act, None, F32)["out"]
            check(act, y, want)
        zi = z.clone()
        zi[0], zi[1] = float("inf"), float("nan")
        for act in ACTS:
            y = packr.packr_linear_act(x, W_p, W_f, lut, zi, activation=act)
            assert y[:, 0].eq(float("inf")).all() and y[:, 1].isnan().all() and not y[:, 2:].isnan().any()


def test_non_finite_rows_stay_in_their_rows(cuda):
    for M in (3, 60, 200):
        c = case(M, 64, 96, BF16, BF16, seed=M)
        clean = call(c, "gelu", BF16)
        c["x"][1, 5] = float("nan")
        got = call(c, "gelu", BF16)
        keep = [i for i in range(M) if i != 1]
        assert got[1].isnan().all() and torch.equal(got[keep], clean[keep])


def test_matches_the_plain_layer(cuda):
    """Without activation and residual the f32 result is PackRLinear's on the
    routes that decode W alike (from 5 rows on), bit for bit on the plain one."""
    c = case(300, 256, 512, BF16, F32, seed=4, residual=False)
    assert torch.equal(call(c, None, F32), packr.packr_matmul(c["x"], c["W_p"], c["W_f"], c["lut"], c["bias"]))


def test_empty_batch_and_leading_dimensions(cuda):
    c = case(0, 64, 96, BF16, BF16, seed=1)
    got = grads(c, "gelu", BF16)
    assert got["out"].shape == (0, 96) and got["dx"].shape == (0, 64)
    assert not got["dW_f"].any() and not got["dbias"].any() and not got["dlut"].any()
    c = case(24, 64, 96, BF16, BF16, seed=1)
    flat = call(c, "silu", BF16)
    cube = call({**c, "x": c["x"].view(2, 3, 4, 64), "residual": c["residual"].view(2, 3, 4, 96)}, "silu", BF16)
    assert torch.equal(cube, flat.view(2, 3, 4, 96))
    one = call({**c, "x": c["x"][0], "residual": c["residual"][0]}, "silu", BF16)
    assert one.shape == (96,)


def test_strided_and_misaligned_inputs(cuda):
    c = case(150, 64, 96, BF16, BF16, seed=6)
    want = call(c, "gelu", BF16)
    wide = torch.zeros(150, 200, dtype=BF16, device="cuda")
    wide[:, 3:67] = c["x"]
    wide[:, 101:197] = c["residual"]
    assert torch.equal(call({**c, "x": wide[:, 3:67], "residual": wide[:, 101:197]}, "gelu", BF16), want)
    flat = torch.empty(150 * 64 + 1, dtype=BF16, device="cuda")
    flat[1:] = c["x"].view(-1)
    assert torch.equal(call({**c, "x": flat[1:].view(150, 64)}, "gelu", BF16), want)
    # a residual and weights that start off a 16-byte boundary
    flat = torch.empty(150 * 96 + 1, dtype=BF16, device="cuda")
    flat[1:] = c["residual"].view(-1)
    assert torch.equal(call({**c, "residual": flat[1:].view(150, 96)}, "gelu", BF16), want)
    wf = torch.empty(64 * 96 + 1, dtype=BF16, device="cuda")
    wf[1:] = c["W_f"].view(-1)
    wp = torch.empty(64 * 96 + 3, dtype=torch.uint8, device="cuda")
    wp[3:] = c["W_p"].view(-1)
    for M in (1, 20, 150):
        d = {**c, "x": c["x"][:M], "residual": c["residual"][:M], "dout": c["dout"][:M],
             "W_f": wf[1:].view(64, 96), "W_p": wp[3:].view(64, 96)}
        compare(d, grads(d, "gelu", BF16), "gelu", BF16)


def test_upstream_gradient_of_any_layout(cuda):
    """A broadcast (stride 0) or transposed upstream gradient."""
    c = case(130, 64, 96, BF16, BF16, seed=6)
    ones = {**c, "dout": torch.ones((), dtype=BF16, device="cuda").expand(130, 96)}
    compare(ones, grads(ones, "gelu", BF16), "gelu", BF16)
    turned = {**c, "dout": c["dout"].t().contiguous().t()}
    compare(turned, grads(turned, "none", BF16), "none", BF16)


def test_weight_gradient_lands_in_the_optimizer_buffer(cuda):
    c = case(40, 64, 96, BF16, BF16, seed=2)
    W_f = torch.nn.Parameter(c["W_f"])
    buf = torch.zeros(64 * 96 + 256, dtype=BF16, device="cuda")
    W_f._packr_grad_sink = (buf, 256)
    out = call({**c, "W_f": W_f}, "gelu", BF16)
    out.backward(c["dout"])
    assert W_f.grad.data_ptr() == buf[256:].data_ptr()
    assert torch.equal(W_f.grad, grads(c, "gelu", BF16, need=("W_f",))["dW_f"])


def test_shared_weights_with_an_optimizer_buffer(cuda):
    """A layer applied twice: the two gradients are summed, not the second one
    written over the first."""
    c = case(40, 96, 96, BF16, BF16, seed=2, residual=False)
    got = []
    for sink in (False, True):
        W_f = torch.nn.Parameter(c["W_f"])
        if sink:
            W_f._packr_grad_sink = (torch.zeros(96 * 96, dtype=BF16, device="cuda"), 0)
        d = {**c, "W_f": W_f}
        call({**d, "x": call(d, "gelu", BF16)}, "gelu", BF16).backward(c["dout"])
        got.append(W_f.grad)
    assert torch.equal(got[0], got[1])


def test_other_stream_and_captured_graph(cuda):
    for M in (2, 8, 40, 200):
        c = case(M, 128, 256, BF16, BF16, seed=M)
        want = call(c, "gelu", BF16)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got = call(c, "gelu", BF16)
        s.synchronize()
        assert torch.equal(got, want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = call(c, "gelu", BF16)
        c2 = case(M, 128, 256, BF16, BF16, seed=M + 50)
        for k in ("x", "residual", "W_p", "W_f", "lut", "bias"):
            c[k].copy_(c2[k])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, call(c2, "gelu", BF16))


def test_gradient_against_differences(cuda):
    """Directional derivatives of sum(out * dout) by central differences of the
    64-bit form; the bf16 operands of the backward cost up to 2^-7 of the
    summed magnitudes' norm."""
    from fused_reference import act64, weights64
    for act in ("gelu", "gelu_tanh", "silu", "none"):
        c = case(33, 64, 80, F32, F32, seed=5)
        c["x"] = c["x"].bfloat16().float()
        got = grads(c, act, F32)
        W = weights64(c["W_p"], c["W_f"], c["lut"])
        base = {"x": c["x"].double(), "W_f": W, "bias": c["bias"].double(), "residual": c["residual"].double()}
        g = torch.Generator(device="cuda").manual_seed(1)
        for k in base:
            v = torch.randn(base[k].shape, generator=g, device="cuda").double()

            def f(t):
                d = {**base, k: base[k] + t * v}
                y = act64(d["x"] @ d["W_f"] + d["bias"], act) + d["residual"]
                return float((y * c["dout"].double()).sum())

            num = (f(1e-5) - f(-1e-5)) / 2e-5
            terms = got["d" + k].double() * v
            assert abs(float(terms.sum()) - num) <= 2.0 ** -7 * float(terms.norm()) * 4 + 1e-5 * (1 + abs(num)), (act, k)


@pytest.mark.parametrize("K,N", [(4096, 4864), (4100, 4720), (4104, 4723)])
@pytest.mark.parametrize("act", ["none", "gelu"])
def test_weight_gradient_of_large_layers(cuda, K, N, act):
    """Enough 512 x 256 tiles and tokens for the held-accumulator dW kernels,
    with the lut gradient (act none) and without; edges inside a tile."""
    c = case(1030, K, N, BF16, BF16, seed=K, residual=False, bias=None)
    need = ("x", "W_f", "lut") if act == "none" else ("W_f",)
    got = grads(c, act, BF16, need=need)
    compare(c, got, act, BF16)
    if act == "none":
        only = grads(c, act, BF16, need=("lut",))["dlut"]
        assert torch.allclose(only, got["dlut"], rtol=1e-4, atol=1e-6 * float(got["dlut"].abs().max()))


def test_weight_gradient_with_non_finite_and_zero_tiles(cuda):
    """The integer histogram's fallbacks: a tile of zeros adds nothing, a tile
    with an infinity adds its values as they are."""
    c = case(1024, 4096, 4864, BF16, BF16, seed=1, residual=False, bias=None)
    c["dout"][:, :256] = 0
    got = grads(c, "none", BF16, need=("W_f", "lut"))
    assert not got["dW_f"][:, :256].any()
    compare(c, got, "none", BF16)
    c["W_p"].fill_(7)
    c["W_p"][5, 300] = 200
    c["x"][3, 5] = float("inf")
    got = grads(c, "none", BF16, need=("W_f", "lut"))
    assert not torch.isfinite(got["dlut"][7]) and not torch.isfinite(got["dlut"][200])
    assert not got["dlut"][:7].any() and not got["dlut"][8:200].any() and not got["dlut"][201:].any()


@pytest.mark.parametrize("need", ["x", "W_f", "lut"])
def test_first_cuda_work_of_a_thread(cuda, need):
    """A backward whose first driver call is a tensor-map encoding, on a host
    thread that has made no runtime call (the autograd engine's threads)."""
    import threading
    from packr_b200 import kernel as K
    c = case(160, 128, 144, BF16, BF16, seed=2, residual=False, bias=None)
    args = (c["dout"], None, 0, c["x"], c["W_p"], c["W_f"], c["lut"], None, need == "x", need == "W_f", need == "lut", None)
    want = [t for t in K.linear_act_backward(*args) if t is not None]
    torch.cuda.synchronize()
    got = []

    def work():
        try:
            got.append(K.linear_act_backward(*args))
        except Exception as e:  # noqa: BLE001
            got.append(e)

    t = threading.Thread(target=work)
    t.start()
    t.join()
    assert not isinstance(got[0], Exception), got[0]
    torch.cuda.synchronize()
    for a, b in zip((t for t in got[0] if t is not None), want):
        assert torch.allclose(a.float(), b.float(), rtol=1e-4, atol=1e-6)


@pytest.mark.parametrize("M,K,N", [(300, 11008, 520), (2100, 9000, 1040), (64, 11008, 272)])
def test_f32_output_of_a_long_reduction(cuda, M, K, N):
    """The tensor cores truncate every accumulation; an f32 output sums at most
    1024 elements in one accumulator (64 accumulations of up to 2^-23 of a sum
    that grows as its square root: 64 * 2^-23 / 2 * 2/3 = 2.6e-6 of the result at
    worst, one way), where 11008 in one gave 1.1e-5."""
    c = case(M, K, N, BF16, F32, seed=1, residual=False)
    want = linear64(c["x"], c["W_p"], c["W_f"], c["lut"], c["bias"], "none", None, F32)["out"][0]
    got = call(c, "none", F32).double()
    assert float((got - want).norm() / want.norm()) < 3e-6


@pytest.mark.parametrize("act", ["none", "gelu"])
@pytest.mark.parametrize("M", [6, 200])
def test_captured_training_step(cuda, M, act):
    """Forward and backward in one graph, replayed on new inputs; a second graph
    of the same tensors beside it."""
    c = case(M, 128, 256, BF16, BF16, seed=M)
    names = ("x", "W_f", "bias", "residual") + (("lut",) if act == "none" else ())
    leaves = {k: c[k].detach().clone().requires_grad_(True) for k in names}
    d = {**c, **leaves, "W_p": c["W_p"].clone(), "lut": leaves.get("lut", c["lut"].clone())}
    dout = c["dout"].clone()

    def step():
        y = call(d, act, BF16)
        return (y, *torch.autograd.grad(y, list(leaves.values()), dout))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step())
        graphs.append(g)
    c2 = case(M, 128, 256, BF16, BF16, seed=M + 90)
    with torch.no_grad():
        for k, v in d.items():
            if k in c2 and k != "dY":
                v.copy_(c2[k]) if k != "dout" else None
        dout.copy_(c2["dout"])
    for g in graphs:
        g.replay()
    torch.cuda.synchronize()
    want = grads(c2, act, BF16, need=names)
    for out in outs:
        for name, a in zip(("out",) + tuple("d" + n for n in names), out):
            if name == "dlut":  # f32 atomics over CTAs
                assert torch.allclose(a, want[name], rtol=1e-3, atol=1e-5)
            else:
                assert torch.equal(a, want[name]), name


@pytest.mark.parametrize("M", [1, 12, 60, 300])
def test_two_streams_at_once(cuda, M):
    cs = [case(M, 520, 1040, BF16, BF16, seed=i) for i in range(2)]
    need = ("x", "W_f", "bias")
    want = [grads(c, "silu", BF16, need=need) for c in cs]
    streams = [torch.cuda.Stream() for _ in cs]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        for c, s in zip(cs, streams):
            with torch.cuda.stream(s):
                got.append(grads(c, "silu", BF16, need=need))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        for k, v in want[i % 2].items():
            assert torch.equal(g[k], v), k


@pytest.mark.parametrize("out", [BF16, F32])
def test_output_beyond_32_bit_offsets(cuda, out):
    M, K, N = 200005, 32, 11008  # 2.2e9 outputs
    assert M * N > 1 << 31
    c = case(5, K, N, BF16, out, seed=3, residual=False)
    x = torch.zeros(M, K, dtype=BF16, device="cuda")
    x[-5:] = c["x"]
    y = packr.packr_linear_act(x, c["W_p"], c["W_f"], c["lut"], c["bias"], activation="gelu", out_dtype=out)
    want = linear64(c["x"], c["W_p"], c["W_f"], c["lut"], c["bias"], "gelu", None, out)["out"]
    check("out", y[-5:], want)
    bias = linear64(torch.zeros_like(c["x"]), c["W_p"], c["W_f"], c["lut"], c["bias"], "gelu", None, out)["out"]
    check("out", y[M // 2:M // 2 + 5], bias)


def test_second_derivative_is_refused(cuda):
    c = case(4, 64, 64, F32, F32, seed=1)
    x = c["x"].requires_grad_(True)
    y = packr.packr_linear_act(x, c["W_p"], c["W_f"], c["lut"], activation="silu")
    g, = torch.autograd.grad(y.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), x)


def test_refused_arguments(cuda):
    c = case(4, 64, 96, BF16, BF16, seed=1)
    ok = dict(x=c["x"], W_p=c["W_p"], W_f=c["W_f"], lut=c["lut"], bias=c["bias"], out_dtype=BF16)
    packr.packr_linear_act(**ok)
    bad_values = [dict(x=c["x"][:, :63]), dict(W_p=c["W_p"][:, :95]), dict(W_p=c["W_p"].t()), dict(lut=c["lut"][:255]),
                  dict(bias=c["bias"][:95]), dict(bias=c["bias"].double()), dict(bias=c["bias"].cpu()),
                  dict(residual=c["residual"][:3]), dict(residual=c["residual"].float()),
                  dict(residual=c["residual"].cpu()), dict(activation="tanh"), dict(W_f=c["W_f"].cpu()),
                  dict(counts=torch.zeros(256, device="cuda")), dict(counts=torch.zeros(256, dtype=torch.int32))]
    for bad in bad_values:
        with pytest.raises(ValueError):
            packr.packr_linear_act(**{**ok, **bad})
    for bad in (dict(x=c["x"].half()), dict(out_dtype=torch.float16), dict(W_f=c["W_f"].float()),
                dict(W_p=c["W_p"].int()), dict(lut=c["lut"].double())):
        with pytest.raises(TypeError):
            packr.packr_linear_act(**{**ok, **bad})


def test_c_entry_refuses_a_small_workspace_and_a_misaligned_x(cuda):
    from packr_b200 import _lib
    lib = _lib.load()
    for M in (8, 64, 200):
        c = case(M, 64, 96, BF16, BF16, seed=1, residual=False)
        out = torch.zeros(M, 96, dtype=BF16, device="cuda")
        wp, wf = c["W_p"].data_ptr(), c["W_f"].data_ptr()
        need = lib.packr_linear_act_workspace_bytes(M, 64, 96, 1, 1, wp, wf)
        ws = torch.zeros(need + 256, dtype=torch.uint8, device="cuda")

        def fwd(x, ws_ptr, nbytes):
            return lib.packr_linear_act_forward(x, 1, wp, wf, c["lut"].data_ptr(), None, 0, 0, None, out.data_ptr(), None,
                                                1, M, 64, 96, ws_ptr, nbytes, None)

        x = c["x"].data_ptr()
        assert need > 0 and fwd(x, ws.data_ptr(), need - 1) == 4 and fwd(x, None, need) == 4
        assert fwd(x, ws.data_ptr() + 16, need) == 4 and fwd(x + 2, ws.data_ptr(), need) == 3
        torch.cuda.synchronize()
        assert not out.any()  # nothing ran


@pytest.mark.parametrize("xt,out", [(BF16, BF16), (F32, F32)])
@pytest.mark.parametrize("M,K,N", [(1, 8192, 272), (2, 8200, 16), (2, 4100, 2064), (1, 9001, 1040), (5, 16400, 144),
                                   (16, 20000, 16)])
def test_few_rows_of_a_long_reduction(cuda, M, K, N, xt, out):
    """One tile's sum is cut into up to one share per SM."""
    c = case(M, K, N, xt, out, seed=M + K)
    for act in ("none", "gelu"):
        compare(c, {"out": call(c, act, out)}, act, out)


@pytest.mark.parametrize("xt,out", [(BF16, BF16), (F32, F32), (BF16, F32)])
@pytest.mark.parametrize("M,K,N", [(129, 72, 144), (300, 256, 512), (1100, 2056, 1040)])
def test_decoded_weight_kept_for_the_backward(cuda, monkeypatch, M, K, N, xt, out):
    """PACKR_KEEP_DECODED_W=1: W decoded in the forward serves the dX GEMM; the same
    bits as with two decodes."""
    from packr_b200 import autograd
    c = case(M, K, N, xt, out, seed=M)
    need = ("x", "W_f", "bias", "residual")
    for act in ("none", "gelu"):
        want = grads(c, act, out, need=need)
        assert not autograd.KEEP_DECODED_W
        leaf = {**c, "x": c["x"].detach().requires_grad_(True)}
        assert call(leaf, act, out).grad_fn.wd is None
        with monkeypatch.context() as m:
            m.setattr(autograd, "KEEP_DECODED_W", True)
            y = call(leaf, act, out)
            node = y.grad_fn
            assert node.wd.shape == (K, N) and node.wd.dtype == BF16
            dx, = torch.autograd.grad(y, leaf["x"], c["dout"], retain_graph=True)
            assert node.wd is None and torch.equal(dx, want["dx"]) and torch.equal(y, want["out"])
            again, = torch.autograd.grad(y, leaf["x"], c["dout"])  # decoded once more
            assert torch.equal(again, dx)
            got = grads(c, act, out, need=need)
            for k, v in want.items():
                assert torch.equal(got[k], v), k
            # not kept where dX is not asked for, few rows, or a width the decode does not take
            assert grads(c, act, out, need=("W_f",))["out"].grad_fn.wd is None
            few = {**leaf, "x": leaf["x"][:20], "residual": c["residual"][:20]}
            assert call(few, act, out).grad_fn.wd is None


def test_decoded_weight_through_the_c_entry(cuda):
    """Every row count reads it, on any stream, with the exact workspace."""
    from packr_b200 import _lib, kernel
    lib = _lib.load()
    for M in (1, 40, 200):
        c = case(M, 72, 144, BF16, BF16, seed=M)
        Wd = kernel.predecode_bf16(c["W_p"], c["W_f"], c["lut"])
        args = (c["x"], c["W_p"], c["W_f"], c["lut"], c["bias"], 2, c["residual"], BF16)
        got = kernel.linear_act_forward(*args, keep_z=True, Wd=Wd)
        compare(c, {"out": got[0]}, "gelu", BF16)
        if M > 128:
            assert all(torch.equal(a, b) for a, b in zip(got, kernel.linear_act_forward(*args, keep_z=True)))
        bwd = (c["dout"], got[1], 2, c["x"], c["W_p"], c["W_f"], c["lut"], None, True, True, True, BF16)
        a, b = kernel.linear_act_backward(*bwd, Wd=Wd), kernel.linear_act_backward(*bwd)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and torch.equal(a[3], b[3])
        need = lib.packr_linear_act_forward_decoded_workspace_bytes(M, 72, 144, 1, 1)
        ws = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
        out = torch.zeros(M, 144, dtype=BF16, device="cuda")

        def fwd(nbytes):
            return lib.packr_linear_act_forward_decoded(c["x"].data_ptr(), 1, Wd.data_ptr(), None, 0, 0, None,
                                                        out.data_ptr(), None, 1, M, 72, 144, ws.data_ptr(), nbytes, None)

        assert need > 0 and fwd(need - 1) == 4
        torch.cuda.synchronize()
        assert not out.any() and fwd(need) == 0
        torch.cuda.synchronize()
        assert torch.equal(out, kernel.linear_act_forward(c["x"], c["W_p"], c["W_f"], c["lut"], None, 0, None, BF16,
                                                          Wd=Wd)[0])
