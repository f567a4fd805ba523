"""Gated feed-forward block, forward and backward, against the formulas in 64 bits.

Bounds, in steps u = 2^-24 of float32, carried from value to value.  A sum of K products on the tensor cores: 16 at a time are added to
the running sum, each time losing at most one unit (2 u) of the sum of magnitudes so far; float32 operands take six such rounds per 16
and start anew after 64, whose sums are added in registers (u each).  What the three pieces of an operand leave out is below u / 2 of a
product.  16-bit types: the hidden features and their gradients are rounded once (half a step), and every result is."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
NAMES = ("x", "w_gate", "w_up", "w_down", "b_gate", "b_up", "b_down")


def step(dtype):
    return torch.finfo(dtype).eps / 2


def floor(dtype):
    """Below the smallest normal number steps do not shrink."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


def sums(K, dtype):
    """Error of a sum of K products, relative to the sum of their magnitudes."""
    return (2 * 24 + K / 64 + 4) * U if dtype == torch.float32 else (K / 8 + 6) * U


def gate(g, act):
    """Value, derivative, and how far the latter can be off where g is off by e (a function of e)."""
    if act == "silu":
        p = torch.sigmoid(g)
        return g * p, p * (1 + g * (1 - p)), lambda e: 0.5 * e + 8 * U
    if act == "gelu":
        p = 0.5 * (1 + torch.erf(g * 0.5 ** 0.5))
        return g * p, p + g * torch.exp(-0.5 * g * g) * 0.3989422804014327, lambda e: 0.8 * e + 8 * U
    return g.clamp(min=0), (g > 0).double(), lambda e: (g.abs() <= e).double()


def reference(x, wg, wu, wd, bg, bu, bd, gy, act):
    """Results in 64 bits by name, and the bounds of their errors before they are stored."""
    dtype = x.dtype
    half = 0.0 if dtype == torch.float32 else step(dtype)
    x, wg, wu, wd, gy = (t.double() for t in (x, wg, wu, wd, gy))
    N, D = x.shape
    F = wg.shape[0]
    bg, bu, bd = (torch.zeros(n, dtype=torch.float64, device="cuda") if b is None else b.double() for b, n in ((bg, F), (bu, F), (bd, D)))
    g, u = x @ wg.t() + bg, x @ wu.t() + bu
    eg, eu = (sums(D, dtype) * (x.abs() @ w.abs().t() + b.abs()) + 2 * U * (v.abs() + b.abs()) for w, b, v in ((wg, bg, g), (wu, bu, u)))
    a, da, slope = gate(g, act)
    ea = 1.13 * eg + 8 * U * g.abs()
    h = a * u
    eh = ea * (u.abs() + eu) + a.abs() * eu + 2 * U * h.abs()
    rounded = lambda e, v: e + half * (v.abs() + e) + (floor(dtype) if half else 0.0)  # noqa: E731
    eh = rounded(eh, h)
    y = h @ wd.t() + bd
    out = dict(y=(y, eh @ wd.abs().t() + sums(F, dtype) * ((h.abs() + eh) @ wd.abs().t() + bd.abs()) + 2 * U * y.abs()))
    dh = gy @ wd
    edh = sums(D, dtype) * (gy.abs() @ wd.abs())
    du, dg = dh * a, dh * u * da
    edu = rounded(edh * (a.abs() + ea) + dh.abs() * ea + 2 * U * du.abs(), du)
    ada, eda = da.abs(), slope(eg)
    edg = rounded((edh * (u.abs() + eu) + dh.abs() * eu) * (ada + eda) + (dh * u).abs() * eda + 4 * U * dg.abs(), dg)
    wide = (dg.abs() + edg) @ wg.abs() + (du.abs() + edu) @ wu.abs()
    out["x"] = dg @ wg + du @ wu, edg @ wg.abs() + edu @ wu.abs() + sums(2 * F, dtype) * wide
    for n, v, e in (("gate", dg, edg), ("up", du, edu)):
        out["w_" + n] = v.t() @ x, e.t() @ x.abs() + sums(N, dtype) * ((v.abs() + e).t() @ x.abs())
        out["b_" + n] = v.sum(0), e.sum(0) + (N / 64 + 80) * U * (v.abs() + e).sum(0)
    out["w_down"] = gy.t() @ h, gy.abs().t() @ eh + sums(N, dtype) * (gy.abs().t() @ (h.abs() + eh))
    out["b_down"] = gy.sum(0), (N / 64 + 80) * U * gy.abs().sum(0)
    return out


def compare(name, got, want, dtype):
    ref, bound = want
    assert got.dtype == dtype and got.shape == ref.shape
    limit = bound + step(dtype) * (ref.abs() + bound) + floor(dtype)
    worst = ((got.double() - ref).abs() / limit).max() if got.numel() else torch.tensor(0.0)
    assert worst <= 1, (name, float(worst))  # (false for what is no number)


def make(N, D, F, dtype, bias=True, seed=0):
    gen = torch.Generator().manual_seed(seed + N + 3 * D + 7 * F)
    rand = lambda *s, std=1.0: (torch.randn(s, generator=gen) * std).to(dtype).cuda()  # noqa: E731
    b = (lambda n: rand(n, std=0.3)) if bias else (lambda n: None)
    return [rand(N, D), rand(F, D, std=D ** -0.5), rand(F, D, std=D ** -0.5), rand(D, F, std=F ** -0.5), b(F), b(F), b(D)], rand(N, D)


def both_ways(tensors, gy, act):
    from crystalformer_b200.feedforward import gated_feed_forward
    leaves = [None if t is None else t.detach().requires_grad_() for t in tensors]
    y = gated_feed_forward(*leaves, activation=act)
    there = [t for t in leaves if t is not None]
    return y.detach(), dict(zip((n for n, t in zip(NAMES, leaves) if t is not None), torch.autograd.grad(y, there, gy)))


CASES = [
    # rows, features, hidden: single rows and few, one of each, the model's layer, tiles and one more or less, rows off 16 bytes, many
    # blocks of the contraction, split contractions
    (1, 128, 512), (1, 1, 1), (2, 40, 24), (3, 129, 65), (4, 256, 512), (8, 64, 200), (9, 128, 512), (127, 128, 512), (128, 64, 64), (129, 200, 136),
    (300, 33, 517), (1000, 128, 512), (257, 512, 1032), (5, 2048, 264), (4100, 128, 512), (640, 7, 3), (70, 1024, 2048), (20000, 16, 24),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("N,D,F", CASES)
def test_output_and_gradients(N, D, F, act, dtype):
    for bias in (True, False):
        tensors, gy = make(N, D, F, dtype, bias)
        y, grads = both_ways(tensors, gy, act)
        want = reference(*tensors, gy, act)
        compare("y", y, want["y"], dtype)
        for n, g in grads.items():
            compare(n, g, want[n], dtype)


def test_float32_accuracy():
    """Errors of float32 products: on average, not only within their bounds."""
    tensors, gy = make(3000, 128, 512, torch.float32)
    y, grads = both_ways(tensors, gy, "silu")
    want = reference(*tensors, gy, "silu")
    # A sum of K terms of random sign, each rounding off by u / 2 on average: sqrt(K) u at most of a result's size.  Two products in a
    # row, pieces and activation: four times that.
    for n, v in dict(grads, y=y).items():
        K = dict(y=512, x=1024).get(n, 3000)
        assert (v.double() - want[n][0]).norm() <= 4 * K ** 0.5 * U * want[n][0].norm(), n


@pytest.mark.parametrize("dtype", TYPES)
def test_strided_rows_and_shapes(dtype):
    from crystalformer_b200.feedforward import gated_feed_forward
    tensors, gy = make(60, 64, 96, dtype)
    rest = tensors[1:]
    wide = torch.randn((60, 200), device="cuda").to(dtype)
    for x in (wide[:, 8:72], wide[:, 3:67], wide[:1, :64].expand(60, 64), wide[:, ::3][:, :64], wide[::2, 64:128], wide.t()[:64, :40].t()):
        y, yc = gated_feed_forward(x, *rest), gated_feed_forward(x.contiguous(), *rest)
        assert torch.equal(y, yc)
    x = tensors[0]
    assert torch.equal(gated_feed_forward(x.view(3, 4, 5, 64), *rest).view(60, 64), gated_feed_forward(x, *rest))
    assert gated_feed_forward(x[0], *rest).shape == (64,)
    # weights as views of a joint matrix, off 16 bytes and transposed
    joint = torch.cat((rest[0].reshape(-1), rest[1].reshape(-1).new_zeros(3), rest[1].reshape(-1)))
    up = joint[96 * 64 + 3:].view(96, 64)
    assert torch.equal(gated_feed_forward(x, joint[:96 * 64].view(96, 64), up, *rest[2:]), gated_feed_forward(x, *rest))
    assert torch.equal(gated_feed_forward(x, rest[0], rest[1], rest[2].t().contiguous().t(), *rest[3:]), gated_feed_forward(x, *rest))
    # an incoming gradient with strides
    a = both_ways(tensors, gy, "silu")[1]
    b = both_ways(tensors, torch.cat((gy, gy), 1)[:, 64:], "silu")[1]
    c = both_ways([t.clone() for t in tensors], gy.t().contiguous().t(), "silu")[1]
    assert all(torch.equal(a[n], b[n]) and torch.equal(a[n], c[n]) for n in a)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [5, 200])
def test_gradients_that_are_not_wanted(rows, dtype):
    from crystalformer_b200 import ops
    tensors, gy = make(rows, 72, 40, dtype)
    every = ops.gated_ffn_bwd(*tensors, "silu", gy)
    for i in range(7):
        wanted = [j == i for j in range(7)]
        some = ops.gated_ffn_bwd(*tensors, "silu", gy, wanted)
        assert all((s is None) == (not w) for s, w in zip(some, wanted)) and torch.equal(some[i], every[i])


def test_gradients_against_differences():
    tensors, gy = make(12, 6, 5, torch.float32)
    _, grads = both_ways(tensors, gy, "gelu")
    base, w = [t.double() for t in tensors], gy.double()
    value = lambda t: float((((gate(t[0] @ t[1].t() + t[4], "gelu")[0] * (t[0] @ t[2].t() + t[5])) @ t[3].t() + t[6]) * w).sum())  # noqa: E731
    h = 1e-6
    for i, n in enumerate(NAMES):
        for at in range(base[i].numel()):
            moved = []
            for sign in (1, -1):
                t = [b.clone() for b in base]
                t[i].view(-1)[at] += sign * h
                moved.append(value(t))
            slope = (moved[0] - moved[1]) / (2 * h)
            # (h^2 times third derivatives, 64-bit differences of sums of some hundred, 1e-14 / h; float32 sums of some tens of terms)
            assert abs(float(grads[n].view(-1)[at]) - slope) <= 1e-5 * (abs(slope) + 10)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [3, 150])
def test_rows_stay_apart(rows, dtype):
    """What is no number in one row does not reach another; memory behind the outputs is left as it was."""
    from crystalformer_b200 import ops
    tensors, gy = make(rows, 40, 72, dtype)
    x = tensors[0]
    x[1, 3] = float("nan")
    y = ops.gated_ffn_fwd(*tensors)
    keep = torch.arange(rows, device="cuda") != 1
    assert torch.isfinite(y[keep]).all() and torch.isnan(y[1]).all()
    gx = ops.gated_ffn_bwd(*tensors, "silu", gy, [True] + [False] * 6)[0]
    assert torch.isfinite(gx[keep]).all() and torch.isnan(gx[1]).all()


def test_outputs_end_where_they_end():
    """No kernel writes behind an output: outputs inside larger buffers, their surroundings marked."""
    import ctypes

    from crystalformer_b200 import _lib
    for dtype in TYPES:
        for N, D, F in ((3, 33, 17), (130, 33, 17), (130, 72, 136), (2000, 40, 24)):
            tensors, gy = make(N, D, F, dtype)
            args = _lib.GatedFFN(TYPES.index(dtype), 0, N, D, F, tensors[0].data_ptr(), D, *[t.data_ptr() for t in tensors[1:]])
            stream = torch.cuda.current_stream().cuda_stream
            shapes = [(N, D)] + [tuple(t.shape) for t in tensors]
            room = [torch.full((torch.Size(s).numel() + 64,), 7.0, dtype=dtype, device="cuda") for s in shapes]
            outs = [r[32:32 + torch.Size(s).numel()] for r, s in zip(room, shapes)]
            for back in (False, True):
                nbytes = _lib.load().cf_gated_ffn_workspace_bytes(ctypes.byref(args), gy.data_ptr(), int(back))
                work = torch.full((nbytes + 512,), 77, dtype=torch.uint8, device="cuda")
                assert work.data_ptr() % 256 == 0
                if back:
                    grads = _lib.GatedFFNGrads(gy.data_ptr(), *[o.data_ptr() for o in outs[1:]])
                    _lib.call("cf_gated_ffn_bwd", ctypes.byref(args), ctypes.byref(grads), work.data_ptr(), stream)
                else:
                    _lib.call("cf_gated_ffn_fwd", ctypes.byref(args), outs[0].data_ptr(), work.data_ptr(), stream)
                torch.cuda.synchronize()
                assert (work[nbytes:] == 77).all()
            assert all((r[:32] == 7).all() and (r[32 + o.numel():] == 7).all() for r, o in zip(room, outs))
            y, grads = both_ways(tensors, gy, "silu")
            assert torch.equal(outs[0].view(N, D), y) and all(torch.equal(o.view(g.shape), g) for o, g in zip(outs[1:], grads.values()))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_repeated_captured_and_on_a_stream(dtype):
    from crystalformer_b200 import ops
    for rows in (4, 700):
        tensors, gy = make(rows, 128, 512, dtype)
        run = lambda: (ops.gated_ffn_fwd(*tensors), *ops.gated_ffn_bwd(*tensors, "silu", gy))  # noqa: E731
        first = run()
        for _ in range(3):
            assert all(torch.equal(a, b) for a, b in zip(first, run()))
        streams = [torch.cuda.Stream() for _ in range(2)]
        others = []
        for s in streams:  # two at a time
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                others.append(run())
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for o in others for a, b in zip(first, o))
        graphs = []
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                captured = run()
            graphs.append((graph, captured))
        tensors[0].copy_(tensors[0].flip(0))
        expected = run()
        for graph, _ in (*graphs, *graphs[::-1]):
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for _, captured in graphs for a, b in zip(expected, captured))
    ops.check_waits()


def test_no_rows():
    tensors, gy = make(0, 16, 24, torch.float32)
    y, grads = both_ways(tensors, gy, "silu")
    assert y.shape == (0, 16) and all((g == 0).all() for g in grads.values())


def test_module():
    from crystalformer_b200.feedforward import GatedFeedForward
    block = GatedFeedForward(32, 48, "gelu", device="cuda")
    x = torch.randn((2, 9, 32), device="cuda", requires_grad=True)
    y = block(x)
    y.sum().backward()
    plain = block.down(torch.nn.functional.gelu(block.gate(x.detach().double().float())) * block.up(x.detach()))
    assert torch.allclose(y, plain, rtol=1e-4, atol=1e-5) and all(p.grad is not None for p in block.parameters()) and x.grad.shape == x.shape


def test_refusals():
    from crystalformer_b200.feedforward import GatedFeedForward, gated_feed_forward
    t, _ = make(10, 16, 24, torch.float32)
    change = lambda i, v: [v if j == i else u for j, u in enumerate(t)]  # noqa: E731
    bad = [change(0, t[0].cpu()), change(1, t[1].cpu()), change(0, t[0].double()), change(2, t[2].half()), change(1, t[1][:-1]), change(2, t[2].t()),
           change(3, t[3].t()), change(4, t[4][:-1]), change(6, t[4]), change(0, t[0][:, :8]), change(1, t[1][0])]
    for args in bad:
        with pytest.raises((RuntimeError, TypeError, ValueError)):
            gated_feed_forward(*args)
    with pytest.raises(ValueError):
        gated_feed_forward(*t, activation="tanh")
    with pytest.raises(ValueError):
        GatedFeedForward(8, 8, "tanh")
    x = t[0].requires_grad_()
    (gx,) = torch.autograd.grad(gated_feed_forward(*t), x, torch.ones_like(x, requires_grad=True), create_graph=True)
    with pytest.raises(RuntimeError):  # (once differentiable)
        gx.sum().backward()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [5, 12])
def test_offsets_beyond_32_bits(rows, dtype):
    """Rows of x 2^28 values apart."""
    from crystalformer_b200 import ops
    tensors, gy = make(rows, 64, 96, dtype)
    far = torch.zeros((rows - 1) * 2 ** 28 + 64, dtype=dtype, device="cuda")
    x = far.as_strided((rows, 64), (2 ** 28, 1))
    x.copy_(tensors[0])
    assert torch.equal(ops.gated_ffn_fwd(x, *tensors[1:]), ops.gated_ffn_fwd(*tensors))
    for a, b in zip(ops.gated_ffn_bwd(x, *tensors[1:], "silu", gy), ops.gated_ffn_bwd(*tensors, "silu", gy)):
        assert torch.equal(a, b)
