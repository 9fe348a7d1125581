"""packr_layer_norm on the GPU against its 64-bit form, forward and backward,
at the sizes, types and alignments where its paths differ."""
import pytest
import torch

import packr_b200 as packr
from fused_reference import check, norm64

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
TYPES = [(BF16, BF16), (BF16, F32), (F32, F32), (F32, BF16)]


def case(M, N, xt, wt, seed=0, residual=True, affine="wb", offset=0.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    return {"x": (n(M, N) * 2 + offset).to(xt), "residual": n(M, N).to(xt) if residual else None,
            "weight": (1 + 0.2 * n(N)).to(wt) if "w" in affine else None,
            "bias": (0.3 * n(N)).to(wt) if "b" in affine else None, "dy": n(M, N).to(xt)}


def run(c, eps=1e-5, need=("x", "residual", "weight", "bias")):
    leaves = {k: c[k].detach().requires_grad_(True) for k in need if c[k] is not None}
    args = {**c, **leaves}
    y = packr.packr_layer_norm(args["x"], args["weight"], args["bias"], eps, args["residual"])
    if not leaves:
        return {"y": y}
    grads = torch.autograd.grad(y, list(leaves.values()), c["dy"])
    return {"y": y, **dict(zip(("d" + k for k in leaves), grads))}


def compare(c, got, eps=1e-5):
    # bf16: one rounding of the result, at most 2^-8 / sqrt(3) in the 2-norm
    rel = 2.4e-3 if c["x"].dtype == BF16 else None
    want = norm64(c["x"], c["residual"], c["weight"], c["bias"], eps, c["dy"])
    for k, v in got.items():
        ref = want["dx" if k == "dresidual" else k]
        check(k, v, ref, rel if k in ("y", "dx", "dresidual") and c["x"].shape[1] > 8 else None)


@pytest.mark.parametrize("xt,wt", TYPES)
@pytest.mark.parametrize("M,N", [(1, 1), (3, 2), (5, 7), (1, 64), (2, 255), (33, 256), (7, 257), (64, 768), (9, 1000),
                                 (40, 1001), (17, 4096), (5, 4104), (3, 8192), (2, 8200), (3, 8193), (2, 16384)])
def test_sizes(cuda, M, N, xt, wt):
    c = case(M, N, xt, wt, seed=M * 31 + N)
    compare(c, run(c))


@pytest.mark.parametrize("xt,wt", [(BF16, BF16), (F32, F32)])
@pytest.mark.parametrize("N", [16385, 20000])
def test_rows_wider_than_the_register_path(cuda, N, xt, wt):
    for residual in (True, False):
        c = case(3, N, xt, wt, seed=N, residual=residual)
        compare(c, run(c))


@pytest.mark.parametrize("affine", ["wb", "w", "b", ""])
@pytest.mark.parametrize("residual", [True, False])
@pytest.mark.parametrize("N", [96, 8200])
def test_optional_inputs(cuda, affine, residual, N):
    c = case(21, N, BF16, BF16, seed=3, residual=residual, affine=affine)
    compare(c, run(c))


@pytest.mark.parametrize("M,N", [(5000, 64), (3000, 768), (2001, 1001), (700, 4096)])
def test_many_rows(cuda, M, N):
    """More rows than one wave of CTAs: the column sums of many slabs."""
    c = case(M, N, BF16, F32, seed=9)
    compare(c, run(c))


@pytest.mark.parametrize("need", [("x",), ("weight",), ("bias",), ("residual",), ("weight", "bias"), ()])
def test_only_the_gradients_asked_for(cuda, need):
    c = case(50, 200, F32, F32, seed=5)
    got = run(c, need=need)
    assert set(got) == {"y"} | {"d" + k for k in need}
    compare(c, got)


def test_large_offset_and_constant_rows(cuda):
    """A mean far above the spread loses nothing but the input's own bits, and
    a constant row (variance 0) gives the bias."""
    c = case(8, 512, F32, F32, seed=1, residual=False, offset=300.0)
    compare(c, run(c))
    x = torch.full((4, 96), 7.5, device="cuda")
    b = torch.randn(96, device="cuda")
    assert torch.equal(packr.packr_layer_norm(x, torch.ones(96, device="cuda"), b), b.expand(4, 96))


def test_non_finite_rows_stay_in_their_rows(cuda):
    c = case(6, 300, BF16, BF16, seed=2)
    clean = run(c)
    for bad in (float("inf"), float("nan")):
        c["x"][2, 17] = bad
        got = run(c)
        for k in ("y", "dx"):
            assert torch.isnan(got[k][2]).any()
            keep = [0, 1, 3, 4, 5]
            assert torch.equal(got[k][keep], clean[k][keep])


def test_empty_batch_and_leading_dimensions(cuda):
    w = torch.ones(32, device="cuda", requires_grad=True)
    b = torch.zeros(32, device="cuda", requires_grad=True)
    x = torch.zeros(0, 32, device="cuda", requires_grad=True)
    y = packr.packr_layer_norm(x, w, b)
    gx, gw, gb = torch.autograd.grad(y, [x, w, b], torch.zeros_like(y))
    assert y.shape == (0, 32) and gx.shape == (0, 32) and not gw.any() and not gb.any()
    c = case(12, 32, F32, F32, seed=4)
    flat = packr.packr_layer_norm(c["x"], c["weight"], c["bias"], residual=c["residual"])
    cube = packr.packr_layer_norm(c["x"].view(3, 4, 32), c["weight"], c["bias"], residual=c["residual"].view(3, 4, 32))
    assert torch.equal(cube, flat.view(3, 4, 32))
    assert torch.equal(packr.packr_layer_norm(c["x"][0], c["weight"], c["bias"], residual=c["residual"][0]), flat[0])


def test_strided_and_misaligned_inputs(cuda):
    g = torch.Generator(device="cuda").manual_seed(8)
    wide = torch.randn(40, 300, generator=g, device="cuda").bfloat16()
    x, res = wide[:, 3:131], wide[:, 150:278]
    w = torch.randn(257, generator=g, device="cuda").bfloat16()[1:129]
    got = packr.packr_layer_norm(x, w, residual=res)
    assert torch.equal(got, packr.packr_layer_norm(x.contiguous(), w.clone(), residual=res.contiguous()))
    # contiguous but starting 2 bytes after a 16-byte boundary
    flat = torch.randn(64 * 128 + 1, generator=g, device="cuda").bfloat16()
    odd = flat[1:].view(64, 128)
    want = norm64(odd, None, w, None, 1e-5)
    check("y", packr.packr_layer_norm(odd, w), want["y"], 2.4e-3)


def test_results_do_not_depend_on_timing(cuda):
    c = case(3000, 768, BF16, F32, seed=6)
    a, b = run(c), run(c)
    for k in a:
        assert torch.equal(a[k], b[k]), k


def test_other_stream_and_captured_graph(cuda):
    c = case(100, 640, BF16, BF16, seed=7)
    want = run(c)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = run(c)
    s.synchronize()
    for k in want:
        assert torch.equal(got[k], want[k])
    args = (c["x"], c["weight"], c["bias"], 1e-5, c["residual"])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = packr.packr_layer_norm(*args)
    c2 = case(100, 640, BF16, BF16, seed=17)
    for k in ("x", "residual", "weight", "bias"):
        c[k].copy_(c2[k])
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, run(c2, need=())["y"])


def test_gradient_against_differences(cuda):
    """Directional derivative of sum(y * dy) by central differences of the
    64-bit form, against the kernel's f32 gradients."""
    c = case(7, 129, F32, F32, seed=12)
    got = run(c)
    g = torch.Generator(device="cuda").manual_seed(1)
    for k in ("x", "residual", "weight", "bias"):
        v = torch.randn(c[k].shape, generator=g, device="cuda").double()
        h = 1e-5

        def f(t):
            d = {**{q: c[q].double() for q in ("x", "residual", "weight", "bias")}, k: c[k].double() + t * v}
            s = d["x"] + d["residual"]
            y = (s - s.mean(1, keepdim=True)) / torch.sqrt(s.var(1, unbiased=False, keepdim=True) + 1e-5) * d["weight"] + d["bias"]
            return float((y * c["dy"].double()).sum())

        num = (f(h) - f(-h)) / (2 * h)
        terms = got["d" + k].double() * v
        # f32 gradients: 2^-18 of the summed magnitudes; differences: h^2
        assert abs(float(terms.sum()) - num) <= 2.0 ** -18 * float(terms.abs().sum()) + 1e-6 * (1 + abs(num))


def test_module_follows_torch(cuda):
    ref = torch.nn.LayerNorm(96, eps=1e-12).cuda()
    with torch.no_grad():
        ref.weight.normal_()
        ref.bias.normal_()
    m = packr.PackRLayerNorm.from_layer_norm(ref)
    assert m.weight is ref.weight and m.bias is ref.bias and list(m.state_dict()) == list(ref.state_dict())
    x, r = torch.randn(4, 5, 96, device="cuda"), torch.randn(4, 5, 96, device="cuda")
    want = norm64(x.view(20, 96), r.view(20, 96), m.weight, m.bias, 1e-12)
    check("y", m(x, residual=r), want["y"])
    assert repr(m).startswith("PackRLayerNorm((96,)")


def test_captured_training_step(cuda):
    """Forward and backward in one graph, replayed on new inputs; a second graph
    of the same tensors beside it."""
    c = case(60, 384, BF16, F32, seed=7)
    leaves = {k: c[k].detach().clone().requires_grad_(True) for k in ("x", "residual", "weight", "bias")}
    dy = c["dy"].clone()

    def step():
        y = packr.packr_layer_norm(leaves["x"], leaves["weight"], leaves["bias"], 1e-5, leaves["residual"])
        return (y, *torch.autograd.grad(y, list(leaves.values()), dy))

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
    c2 = case(60, 384, BF16, F32, seed=70)
    with torch.no_grad():
        for k, v in leaves.items():
            v.copy_(c2[k])
        dy.copy_(c2["dy"])
    for g in graphs:
        g.replay()
    torch.cuda.synchronize()
    want = run(c2)
    for out in outs:
        for a, b in zip(out, (want["y"], want["dx"], want["dresidual"], want["dweight"], want["dbias"])):
            assert torch.equal(a, b)


def test_two_streams_at_once(cuda):
    cs = [case(2000, 1001, BF16, F32, seed=i) for i in range(2)]
    want = [run(c) for c in cs]
    streams = [torch.cuda.Stream() for _ in cs]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        for c, s in zip(cs, streams):
            with torch.cuda.stream(s):
                got.append(run(c))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        for k, v in want[i % 2].items():
            assert torch.equal(g[k], v), k


def test_tensors_beyond_32_bit_offsets(cuda):
    M, N = 140001, 16384  # 2.29e9 elements; the last rows start past 2^31
    assert M * N > 1 << 31
    x = torch.zeros(M, N, dtype=BF16, device="cuda")
    tail = case(5, N, BF16, BF16, seed=3, residual=False)
    x[-5:] = tail["x"]
    w, b = tail["weight"].requires_grad_(True), tail["bias"].requires_grad_(True)
    x.requires_grad_(True)
    y = packr.packr_layer_norm(x, w, b)
    dy = torch.zeros_like(y)
    dy[-5:] = tail["dy"]
    dx, dw, db = torch.autograd.grad(y, [x, w, b], dy)
    want = norm64(tail["x"], None, w, b, 1e-5, tail["dy"])
    check("y", y[-5:], want["y"], 2.4e-3)
    check("dx", dx[-5:], want["dx"], 2.4e-3)
    check("dweight", dw, want["dweight"])
    check("dbias", db, want["dbias"])
    assert not dx[:10].any() and torch.equal(y[0], b.detach())


def test_second_derivative_is_refused(cuda):
    c = case(4, 64, F32, F32, seed=1)
    x = c["x"].requires_grad_(True)
    y = packr.packr_layer_norm(x, c["weight"], c["bias"])
    g, = torch.autograd.grad(y.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), x)


def test_refused_arguments(cuda):
    x = torch.zeros(4, 8, device="cuda")
    w = torch.ones(8, device="cuda")
    for bad in (dict(weight=torch.ones(7, device="cuda")), dict(weight=torch.ones(8)), dict(weight=w.half()),
                dict(weight=w, residual=x[:2]), dict(weight=w, residual=x.bfloat16()), dict(weight=w, residual=x.cpu()),
                dict(weight=w, eps=-1.0), dict(weight=w, eps=float("nan"))):
        with pytest.raises(ValueError):
            packr.packr_layer_norm(x, **bad)
    with pytest.raises(TypeError):
        packr.packr_layer_norm(x, w, w.bfloat16())
    with pytest.raises(TypeError):
        packr.packr_layer_norm(x.half(), w)
    with pytest.raises(ValueError):
        packr.packr_layer_norm(torch.zeros(4, 0, device="cuda"))
    with pytest.raises(ValueError):
        packr.PackRLayerNorm(9, device="cuda")(x)


@pytest.mark.parametrize("xt", [BF16, F32])
@pytest.mark.parametrize("M,N", [(13, 1), (3, 1), (11, 2), (9, 3), (7, 5), (1201, 1), (5003, 3), (6001, 7)])
def test_rows_shorter_than_a_chunk_inside_larger_buffers(cuda, xt, M, N):
    """Several rows share the tensor's last 16 bytes; what lies behind it is
    neither read into a result nor written."""
    c = case(M, N, xt, xt, seed=M + N)
    inner = {}
    for k in ("x", "residual", "dy"):
        buf = torch.full((M * N + 64,), float("nan"), dtype=xt, device="cuda")
        inner[k] = buf[:M * N].view(M, N)
        inner[k].copy_(c[k])
    got = run({**c, **inner})
    compare(c, got)
    lib = packr._lib.load()
    for name in ("y", "dx"):
        out = torch.full((M * N + 64,), 7.0, dtype=xt, device="cuda")
        stats = torch.empty(2, M, device="cuda")
        code = 0 if xt == F32 else 1
        s = torch.cuda.current_stream().cuda_stream
        p = lambda t: t.data_ptr()  # noqa: E731
        other = torch.empty_like(c["x"])
        assert lib.packr_layer_norm_forward(p(inner["x"]), p(inner["residual"]), code, p(c["weight"]), p(c["bias"]), code,
                                            1e-5, p(out if name == "y" else other), p(stats), p(stats) + 4 * M, M, N,
                                            s) == 0
        if name == "dx":
            assert lib.packr_layer_norm_backward(p(inner["dy"]), p(inner["x"]), p(inner["residual"]), code, p(c["weight"]),
                                                 code, p(stats), p(stats) + 4 * M, p(out), None, None, M, N, None, 0, s) == 0
        torch.cuda.synchronize()
        assert torch.equal(out[:M * N].view(M, N), got[name]) and bool((out[M * N:] == 7).all())


@pytest.mark.parametrize("M,N,xt,wt", [(1, 4096, BF16, BF16), (300, 768, F32, F32), (2000, 1001, BF16, F32),
                                       (600, 8192, BF16, BF16), (70, 16384, BF16, F32)])
def test_training_chain_of_overlapped_launches(cuda, M, N, xt, wt):
    """Four norms forward, then their backward passes, each kernel set up while the
    one in front of it writes what it reads (statistics directly before the
    backward, sums before their reduction), in buffers that the allocator gives out
    again and with inputs and weights overwritten between the passes: the same bits
    as with a synchronisation after every call."""
    cs = [case(M, N, xt, wt, seed=i) for i in range(3)]
    x = cs[0]["x"].clone().requires_grad_(True)
    ws = [(cs[0]["weight"].clone().requires_grad_(True), cs[0]["bias"].clone().requires_grad_(True)) for _ in range(4)]
    leaves = [x] + [t for w in ws for t in w]

    def step(dy):
        h = x
        for w, b in ws:
            h = packr.packr_layer_norm(h, w, b, residual=x)
        return (h, *torch.autograd.grad(h, leaves, dy))

    def alone(dy):
        """The same, every backward pass by itself."""
        hs, h = [], x
        for w, b in ws:
            i = h.detach().requires_grad_(True)
            r = x.detach().requires_grad_(True)
            o = packr.packr_layer_norm(i, w, b, residual=r)
            torch.cuda.synchronize()
            hs.append((i, r, w, b, o))
            h = o
        out, d, params = h.detach(), dy, []
        for i, r, w, b, o in reversed(hs):
            di, _, dw, db = torch.autograd.grad(o, [i, r, w, b], d)
            torch.cuda.synchronize()
            params = [dw, db] + params
            d = di
        return out, params

    for c in cs:
        with torch.no_grad():
            x.copy_(c["x"])
            for w, b in ws:
                w.copy_(c["weight"]).mul_(1.25)
                b.copy_(c["bias"])
        dy = c["dy"].clone()
        got = [step(dy) for _ in range(4)]
        out, params = alone(dy)
        torch.cuda.synchronize()
        for g in got:
            assert torch.equal(g[0], out)
            for a, b in zip(g[2:], params):
                assert torch.equal(a, b)
        for g in got[1:]:
            assert torch.equal(g[1], got[0][1])


# both sides of the widths where the launch rule changes: 1024, 4096, 8192 and
# 16384 columns, and the ragged rows just below, which cover more than they have
EDGES = [1017, 1023, 1024, 1025, 4089, 4090, 4093, 4094, 4095, 4097, 8185, 8191, 16369, 16375, 16376, 16377]


@pytest.mark.parametrize("residual", [True, False])
@pytest.mark.parametrize("xt,wt", [(BF16, F32), (F32, F32)])
@pytest.mark.parametrize("N", EDGES)
def test_widths_around_the_thresholds(cuda, N, xt, wt, residual):
    c = case(9, N, xt, wt, seed=N, residual=residual)
    compare(c, run(c))
    compare(c, run(c, need=()))


@pytest.mark.parametrize("xt", [BF16, F32])
@pytest.mark.parametrize("N", [16, 64, 512, 2048, 8192, 16384])
def test_gradients_of_huge_constant_rows(cuda, N, xt):
    """mean * rstd past f32's range: h is zero all the same, and what a thread holds
    outside the row adds nothing.  N is a power of two, so the mean is exact;
    dx = rstd * (g - mean(g)), sums of N products: 2^-17 of the largest covers them
    in f32, half a step more in bf16."""
    g = torch.Generator(device="cuda").manual_seed(N)
    x = torch.full((5, N), 2.0 ** 112, device="cuda").to(xt)  # 2^112 * 2^14 columns stays finite
    x[1] = 0.0
    w = torch.randn(N, generator=g, device="cuda")
    dy = torch.randn(5, N, generator=g, device="cuda").to(xt)
    eps = 1e-12
    assert 2.0 ** 112 * eps ** -0.5 > torch.finfo(F32).max
    got = run({"x": x, "residual": None, "weight": w, "bias": torch.zeros_like(w), "dy": dy}, eps=eps)
    assert not got["y"].any() and not got["dweight"].any()
    gw = dy.double() * w.double()
    want = (gw - gw.mean(1, keepdim=True)) * eps ** -0.5
    off = (got["dx"].double() - want).abs()
    assert (off <= 2.0 ** -17 * want.abs().max() + torch.finfo(xt).eps / 2 * want.abs()).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_module_under_autocast(cuda, dtype):
    """f32 arithmetic on the same values in both: 64 roundings
    of values up to 4 are 1.5e-5."""
    ref = torch.nn.LayerNorm(96, device="cuda")
    m = packr.PackRLayerNorm.from_layer_norm(ref)
    x = torch.randn(5, 96, device="cuda").to(dtype).requires_grad_(True)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        a, b = m(x), ref(x)
    assert a.dtype == b.dtype == torch.float32 and torch.allclose(a, b, rtol=1e-5, atol=2e-5)
    ga, = torch.autograd.grad(a.square().sum(), x)
    assert ga.dtype == dtype


@pytest.mark.parametrize("xt,wt", [(BF16, BF16), (F32, F32)])
@pytest.mark.parametrize("M,N", [(33, 64), (5, 8192), (40000, 64), (2100, 1001), (260, 8192), (130, 16375), (130, 16640)])
def test_tensors_off_the_16_byte_grid(cuda, M, N, xt, wt):
    """Slices that start an element after a boundary.  Large ones take the same path
    as aligned ones: the same bits up to 16384 columns, forward and backward."""
    c = case(M, N, xt, wt, seed=N)
    want = run(c)

    def shifted(t):
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
        flat[1:] = t.reshape(-1)
        s = flat[1:].view(t.shape)
        assert s.data_ptr() % 16 != 0
        return s

    for names in (("x",), ("residual",), ("dy",), ("x", "residual", "dy", "weight", "bias")):
        got = run({**c, **{k: shifted(c[k]) for k in names}})
        compare(c, got)
        for k, v in want.items():
            assert N > 16384 or M * N < 1 << 21 or torch.equal(got[k], v), (names, k)
