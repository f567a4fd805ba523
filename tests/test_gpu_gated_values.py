"""Gated feed-forward block: values at the ends of their types, long contractions, many short launches in a row."""
import pytest
import torch
from test_gpu_gated import TYPES, compare, make, reference, step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
def test_short_launches_in_a_row(dtype):
    """Blocks follow one another on an SM at once: every call's results are those of the first."""
    from crystalformer_b200 import ops
    for N, D, F in ((1000, 128, 512), (700, 256, 264)):
        tensors, gy = make(N, D, F, dtype)
        run = lambda: (ops.gated_ffn_fwd(*tensors), *ops.gated_ffn_bwd(*tensors, "silu", gy))  # noqa: E731
        first, rest = run(), [run() for _ in range(40)]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for r in rest for a, b in zip(first, r))
    ops.check_waits()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("on_16_bytes", [True, False])
@pytest.mark.parametrize("rows", [4, 8, 9])
def test_hidden_units_at_the_end_of_the_range(rows, on_16_bytes, dtype):
    """One hidden unit of a value near float16's largest and beyond it (and, in both types, an ordinary one and a small one): nothing but an
    overflow gives an infinity, and nothing gives what is no number."""
    from crystalformer_b200.feedforward import gated_feed_forward
    D, F = (8, 16) if on_16_bytes else (9, 17)
    zeros = lambda *s: torch.zeros(s, dtype=dtype, device="cuda")  # noqa: E731
    x, w_gate, w_up, w_down, b_gate = zeros(rows, D), zeros(F, D), zeros(F, D), zeros(D, F), zeros(F) + 1
    x[:, 0], x[:, 1] = 2, 1
    w_down[:] = 0.25
    values = [(0, 1e-5), (0, 0.3), (2.5, 0.125)]
    if dtype == torch.float16:
        values += [(32752, 15), (32752, 16), (32752, 17), (-32752, -17), (32752, 4496), (-32752, -4496), (65504, -8), (65504, 30000), (float("inf"), 0)]
    for pair in values:
        w_up[3, 0], w_up[3, 1] = pair
        h = 2 * float(w_up[3, 0]) + float(w_up[3, 1])  # (a product and a sum that are exact in float32)
        y = gated_feed_forward(x, w_gate, w_up, w_down, b_gate, activation="relu").double()
        largest = torch.finfo(dtype).max * (1 + 2.0 ** -12)  # (from here on, half a step behind the largest, values round to an infinity)
        limit = float("inf") if not on_16_bytes and rows <= 8 else 2 * largest - 32 if rows <= 8 else largest
        if abs(h) >= limit:
            assert (y == float("inf") * (1 if h > 0 else -1)).all(), (pair, y[0, 0])
            continue
        # h in one value of the type, two, or one of float32; then the result.  (What is left of h beyond the largest value, 16 off at
        # most, is 2^-12 of it.)
        held = step(dtype) if rows > 8 else 2.0 ** -12 if abs(h) > 65504 else step(dtype) ** 2
        small = torch.finfo(dtype).smallest_normal * step(dtype) * 2
        bound = 0.25 * (held * abs(h) + small) + 2 * step(dtype) * abs(0.25 * h) * 0.5 + small
        assert ((y - 0.25 * h).abs() <= bound * (1 + step(dtype))).all(), (pair, y[0, 0])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [5, 40, 5000])
@pytest.mark.parametrize("D", [16, 33])
def test_infinite_gradients_of_biases(D, rows, dtype):
    """Sums of columns with infinities of one sign, of both, and with what is no number; the other columns stay as they are."""
    from crystalformer_b200 import ops
    tensors, gy = make(rows, D, 24, dtype)
    bias_of = lambda: ops.gated_ffn_bwd(*tensors, "silu", gy, [False] * 6 + [True])[6]  # noqa: E731
    before = bias_of()
    inf = float("inf")
    gy[rows // 2, 1], gy[0, 3], gy[rows - 1, 3] = inf, -inf, -inf
    gy[0, 5], gy[rows - 1, 5], gy[1, 8] = inf, -inf, float("nan")
    gb = bias_of()
    keep = torch.ones(D, dtype=torch.bool, device="cuda")
    keep[[1, 3, 5, 8]] = False
    assert gb[1] == inf and gb[3] == -inf and gb[5].isnan() and gb[8].isnan() and torch.equal(gb[keep], before[keep])
    # dg and du with an infinity: positive inputs and weights, so that nothing cancels (float32: see the values at the ends of its range)
    positive, one = [t.abs() + 0.1 for t in tensors], torch.ones_like(gy)
    one[2] = inf
    gb_gate, gb_up = ops.gated_ffn_bwd(*positive, "relu", one, [False] * 4 + [True, True, False])[4:6]
    if dtype != torch.float32:
        assert (gb_gate == inf).all() and (gb_up == inf).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_infinite_weights_and_few_rows(dtype):
    """Rows whose hidden units are handed on in two values: what was left of a unit does not meet an infinite weight."""
    from crystalformer_b200 import ops
    tensors, _ = make(3, 16, 24, dtype)
    tensors = [t.abs() + 0.1 for t in tensors]
    for value in (float("inf"), -float("inf")):
        tensors[3][3, 7] = value
        y = ops.gated_ffn_fwd(*tensors, activation="relu")
        assert (y[:, 3] == value).all() and y[:, :3].isfinite().all() and y[:, 4:].isfinite().all()


def plain(x, w_gate, w_up, w_down, b_gate, b_up, b_down):
    """With a ReLU, which has a value and a slope at infinity."""
    linear = torch.nn.functional.linear
    return linear(torch.relu(linear(x, w_gate, b_gate)) * linear(x, w_up, b_up), w_down, b_down)


@pytest.mark.parametrize("rows", [3, 12, 300])
def test_largest_floats(rows):
    """Finite values that round to an infinity in bfloat16, as a mask's lowest value is: the same bounds as of any others."""
    from crystalformer_b200 import ops
    for sign in (1, -1):
        tensors, _ = make(rows, 16, 24, torch.float32)
        x, w_gate, w_up, w_down = tensors[:4]
        w_gate[:, 0], w_up[:, 0] = 2.0 ** -10 * (1 + torch.linspace(0, 1, 24, device="cuda")), 0.0
        x[1, 0] = sign * torch.finfo(torch.float32).max
        want = reference(*tensors, torch.zeros_like(x), "relu")["y"]
        compare("y", ops.gated_ffn_fwd(*tensors, activation="relu"), want, torch.float32)
        assert (want[0][1].abs().max() > 1e34) == (sign > 0)
        # ... and among the weights
        w_down[3, 5] = sign * torch.finfo(torch.float32).max
        x[1, 0] = 0.0
        x *= 0.1
        want = reference(*tensors, torch.zeros_like(x), "relu")["y"]
        assert want[0].abs().max() < torch.finfo(torch.float32).max
        compare("y", ops.gated_ffn_fwd(*tensors, activation="relu"), want, torch.float32)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [3, 12, 300])
def test_infinities(rows, dtype):
    """An infinity among the inputs, the weights and the incoming gradient: infinities and what is no number where the formulas have them."""
    from crystalformer_b200 import ops
    inf = float("inf")
    tensors, gy = make(rows, 16, 24, dtype)
    positive = [t.abs() + 0.1 for t in tensors]  # (so that nothing is inf - inf by itself)
    for i, at, value in ((0, (1, 0), inf), (0, (1, 0), -inf), (1, (5, 2), inf), (2, (5, 2), -inf), (3, (3, 7), -inf), (0, (2, 4), float("nan"))):
        t = [v.clone() for v in positive]
        t[i][at] = value
        y, want = ops.gated_ffn_fwd(*t, activation="relu"), plain(*(v.double() for v in t))
        assert torch.equal(y.isnan(), want.isnan()) and torch.equal(y.isinf(), want.isinf()) and torch.equal(y[want.isinf()].double(), want[want.isinf()]), (i, value)
        assert not want.isfinite().all()
    one = gy.abs() + 0.1
    one[2, 3] = inf
    leaves = [v.double().requires_grad_() for v in positive]
    want = torch.autograd.grad(plain(*leaves), leaves, one.double())
    for n, a, b in zip(range(7), ops.gated_ffn_bwd(*positive, "relu", one), want):
        assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.isinf(), b.isinf()) and b.isinf().any(), n


def test_smallest_floats():
    """Three pieces of bfloat16 end at 2^-133: from there on digits are lost, half of that number of a value at most."""
    from crystalformer_b200 import ops
    N, D, F = 12, 16, 24
    tensors, _ = make(N, D, F, torch.float32, bias=False)
    for scale in (1e-30, 1e-33, 1e-36, 1e-38):
        x, w_gate, w_up, w_down = tensors[0] * scale, torch.zeros_like(tensors[1]), tensors[2], tensors[3]
        t = [x, w_gate, w_up, w_down, torch.ones(F, device="cuda"), None, None]
        y = ops.gated_ffn_fwd(*t, activation="relu")
        h = x.double() @ w_up.double().t()
        ref = h @ w_down.double().t()
        lost = 2.0 ** -134 * (w_up.double().abs().sum(1)[None] + 1) + 2.0 ** -148  # of h: of the values of x, then of itself; of float32 sums
        bound = reference(*t, torch.zeros_like(x), "relu")["y"][1] + (lost * 2) @ w_down.double().abs().t() + 2.0 ** -148 * F
        assert ((y.double() - ref).abs() <= bound).all(), scale


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_sums_over_many_rows(dtype):
    """Sums of one sign over 2^19 rows do not drift.  Every instruction adds 16 products to a running sum and cuts what lies below its last
    bits: three units of 2^-23 of it at the most that was seen, of 1,024 instructions in a row 1.8e-4 of their sum."""
    from crystalformer_b200 import ops
    N, D, F = 2 ** 19, 1024, 2048
    gen = torch.Generator(device="cuda").manual_seed(1)
    zeros = lambda *s: torch.zeros(s, dtype=dtype, device="cuda")  # noqa: E731
    hidden = ((torch.rand(F, generator=gen, device="cuda") + 0.5) * 2.0 ** -5).to(dtype)  # h, by the biases alone: in every row the same
    gy = torch.rand((N, D), generator=gen, device="cuda").mul_(2.0 ** -6).to(dtype)
    got = ops.gated_ffn_bwd(zeros(1, D).expand(N, D), zeros(F, D), zeros(F, D), zeros(D, F), zeros(F) + 1, hidden, None, "relu", gy,
                            [False] * 3 + [True] + [False] * 3)[3].double()
    want = sum(g.double().sum(0) for g in gy.split(2 ** 16))[:, None] * hidden.double()
    off = got / want - 1
    assert off.abs().max() <= step(dtype) * (1 + 1.8e-4) + 1.8e-4
    assert off.mean().abs() <= 1.8e-4  # (roundings of the result cancel)
    del got, want, off
    torch.cuda.empty_cache()
