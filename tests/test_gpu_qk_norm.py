"""Norms of query and key heads with the rotation by positions, against the formulas in 64 bits.

Bounds, in steps u = 2^-24 of float32: a mean of D squares is off by (D + 2) u of itself, its inverse root by half of that and two
more; products and the rotation add a step each; an angle, of whose turns 2^-24 is lost before and 2^-25 in the multiplication, is
off by 2 pi (2^-24 + 2^-25) = 9.5 u, times the pair's other entry, and the sines by two more each.  Storage adds half a step."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def store(dtype, ref):
    return torch.finfo(dtype).eps / 2 * ref.abs() + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


def turns(x, pos, waves, interleaved, back=False):
    """x (N,H,D) with its pairs turned, and the magnitudes that its rounding errors go by."""
    x, size = x.clone(), x.abs().clone()
    if waves is None or waves.shape[1] == 0:
        return x, size
    P = waves.shape[1]
    theta = 2 * math.pi * torch.einsum("nc,hpc->nhp", pos.double(), waves.double())
    theta = theta.repeat_interleave(x.shape[1] // theta.shape[1], dim=1) * (-1 if back else 1)
    i, j = (slice(0, 2 * P, 2), slice(1, 2 * P, 2)) if interleaved else (slice(0, P), slice(P, 2 * P))
    a, b = x[..., i].clone(), x[..., j].clone()
    x[..., i], x[..., j] = a * theta.cos() - b * theta.sin(), b * theta.cos() + a * theta.sin()
    size[..., i] = size[..., j] = a.abs() + b.abs()
    return x, size


def reference(x, w, g, pos, waves, interleaved, eps):
    """(y, gx, gw) and the bounds of their errors in float32."""
    D = x.shape[-1]
    x, w = x.double(), (torch.ones(D, dtype=torch.float64, device="cuda") if w is None else w.double())
    r = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    y, size = turns(x * r * w, pos, waves, interleaved)
    ebound = (D / 2 + 20) * U * size
    g, gsize = turns(g.double(), pos, waves, interleaved, back=True)
    n = x * r
    wg = w * g
    m, msize = (wg * n).mean(-1, keepdim=True), (w.abs() * gsize * n.abs()).mean(-1, keepdim=True)
    gx = r * (wg - n * m)
    gbound = r * (2.5 * D + 60) * U * (w.abs() * gsize + n.abs() * msize)
    over = (0,) if w.dim() == 2 else (0, 1)
    gw, wsize = (g * n).sum(over), (gsize * n.abs()).sum(over)
    wbound = (x.shape[0] * x.shape[1] + D / 2 + 30) * U * wsize
    return (y, ebound), (gx, gbound), (gw, wbound)


def compare(got, want, dtype):
    ref, bound = want
    assert got.dtype == dtype and got.shape == ref.shape
    assert ((got.double() - ref).abs() <= bound + store(dtype, ref)).all(), float(((got.double() - ref).abs() / (bound + store(dtype, ref))).max())


def make(N, Hq, Hk, D, P, C, wave_heads, weights, dtype, seed, reach=1.0):
    gen = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(s, generator=gen).to(dtype).cuda()  # noqa: E731
    q, k, gq, gk = rand(N, Hq, D), rand(N, Hk, D), rand(N, Hq, D), rand(N, Hk, D)
    wq, wk = (None if weights == "none" else rand(H, D) if weights == "each" else rand(D) for H in (Hq, Hk))
    pos = waves = None
    if C:
        pos = (torch.rand((N, C), generator=gen) * reach).cuda()
        waves = (torch.randint(-4, 5, (wave_heads, P, C), generator=gen).float() if reach == 1.0
                 else torch.rand((wave_heads, P, C), generator=gen)).cuda()
    return q, k, wq, wk, pos, waves, gq, gk


def both_ways(q, k, wq, wk, pos, waves, gq, gk, interleaved, eps=1e-6):
    from crystalformer_b200.qk_norm import normalize_rotate
    leaves = [None if t is None else t.detach().requires_grad_() for t in (q, k, wq, wk)]
    outs = normalize_rotate(*leaves, pos, waves, eps, interleaved)
    grads = iter(torch.autograd.grad(outs, [t for t in leaves if t is not None], (gq, gk)))
    return outs, [None if t is None else next(grads) for t in leaves]


CASES = [
    # N, Hq, Hk, D, P, C, wave_heads, weights: no rows to share, the model's heads, shared key heads, odd sizes, part of a head turned,
    # norms alone, heads of one entry and of 512
    (1, 1, 1, 2, 1, 1, 1, "shared"), (37, 8, 8, 16, 8, 3, 8, "each"), (300, 8, 8, 16, 8, 3, 1, "shared"), (33, 8, 2, 128, 64, 1, 1, "shared"),
    (29, 6, 3, 64, 16, 2, 3, "each"), (41, 12, 4, 80, 20, 3, 1, "each"), (50, 3, 1, 33, 7, 2, 1, "each"), (65, 4, 4, 7, 3, 3, 4, "none"),
    (17, 2, 2, 24, 0, 0, 1, "shared"), (19, 5, 5, 1, 0, 0, 1, "each"), (9, 2, 1, 512, 256, 1, 1, "each"), (5, 3, 3, 511, 100, 2, 3, "shared"),
    (1000, 16, 16, 16, 8, 3, 16, "each"), (700, 24, 8, 48, 24, 1, 8, "shared"), (260, 40, 8, 32, 16, 1, 1, "each"), (77, 2, 2, 256, 128, 1, 2, "none"),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("case", CASES)
def test_outputs_and_gradients(case, interleaved, dtype):
    data = make(*case, dtype, sum(case[:6]))
    q, k, wq, wk, pos, waves, gq, gk = data
    outs, grads = both_ways(*data, interleaved)
    for i, (x, w, g) in enumerate(((q, wq, gq), (k, wk, gk))):
        y, gx, gw = reference(x, w, g, pos, waves, interleaved, 1e-6)
        compare(outs[i], y, dtype)
        compare(grads[i], gx, dtype)
        if w is not None:
            compare(grads[2 + i], gw, dtype)


@pytest.mark.parametrize("reach", [1e3, 1e6, 2.0 ** 24])
def test_far_positions(reach):
    data = make(200, 4, 4, 32, 16, 2, 1, "shared", torch.float32, 3, reach)
    outs, grads = both_ways(*data, False)
    q, k, wq, wk, pos, waves, gq, gk = data
    y, gx, _ = reference(q, wq, gq, pos, waves, False, 1e-6)
    compare(outs[0], y, torch.float32)
    compare(grads[0], gx, torch.float32)


def test_lattice_translations_do_not_matter():
    """Whole-numbered waves on fractional coordinates with few digits: shifted by whole cells, the outputs are the same bits."""
    from crystalformer_b200.qk_norm import normalize_rotate
    q, k, wq, wk, pos, waves, *_ = make(100, 8, 8, 16, 8, 3, 8, "each", torch.float32, 4)
    pos = (pos * 4096).floor() / 4096
    shift = torch.tensor([[5.0, -3.0, 11.0]], device="cuda")
    for a, b in zip(normalize_rotate(q, k, wq, wk, pos, waves), normalize_rotate(q, k, wq, wk, pos + shift, waves)):
        assert torch.equal(a, b)


def test_products_depend_on_differences():
    """q_i . k_j of turned heads depends on the difference of the positions alone."""
    from crystalformer_b200.qk_norm import normalize_rotate
    q, k, wq, wk, pos, waves, *_ = make(20, 4, 4, 16, 8, 3, 4, "each", torch.float32, 4)
    logits = []
    for shift in (0.0, 0.37):
        a, b = normalize_rotate(q, k, wq, wk, pos + shift, waves)
        logits.append(torch.einsum("ihd,jhd->hij", a.double(), b.double()))
    # (shifted positions are rounded: half a step of 2 in each of three axes, waves of up to 4, on heads of norm below 4 x 3)
    assert (logits[0] - logits[1]).abs().max() < 2 * math.pi * 3 * 4 * 2 * U * 2 * float(logits[0].abs().max() + 64)


@pytest.mark.parametrize("dtype", TYPES)
def test_views_of_a_joint_projection(dtype):
    """Strided q and k, on and off 16 bytes, give what their copies give."""
    from crystalformer_b200.qk_norm import normalize_rotate
    *_, wq, wk, pos, waves, gq, gk = make(50, 8, 2, 16, 8, 3, 2, "each", dtype, 9)
    for lead in (0, 1, 8):
        joint = torch.randn((50, lead + 12 * 16 + 3), device="cuda").to(dtype)
        q, k = joint[:, lead:lead + 128].unflatten(1, (8, 16)), joint[:, lead + 128:lead + 160].unflatten(1, (2, 16))
        # (other vector widths add a head's squares in another order: the bounds of the reference again)
        outs, grads = both_ways(q, k, wq, wk, pos, waves, gq, gk, False)
        for i, (x, w, g) in enumerate(((q, wq, gq), (k, wk, gk))):
            y, gx, gw = reference(x, w, g, pos, waves, False, 1e-6)
            compare(outs[i], y, dtype)
            compare(grads[i], gx, dtype)
            compare(grads[2 + i], gw, dtype)
    q = torch.randn((50, 1, 16), device="cuda").to(dtype).expand(50, 8, 16)  # one head for all, transposed rows
    k = torch.randn((2, 50, 16), device="cuda").to(dtype).transpose(0, 1)
    for a, b in zip(normalize_rotate(q, k, wq, wk, pos, waves), normalize_rotate(q.contiguous(), k.contiguous(), wq, wk, pos, waves)):
        assert torch.equal(a, b)


def test_gradients_against_differences():
    q, k, wq, wk, pos, waves, gq, gk = (t.double() if t is not None else t for t in make(3, 2, 2, 8, 4, 3, 2, "each", torch.float32, 2))
    f32 = [t.float() for t in (q, k, wq, wk, pos, waves, gq, gk)]
    _, grads = both_ways(*f32, False)

    def value(*leaves):
        return sum((turns(x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w, pos, waves, False)[0] * g).sum()
                   for x, w, g in ((leaves[0], leaves[2], gq), (leaves[1], leaves[3], gk)))
    h = 1e-6
    leaves = [q, k, wq, wk]
    for i, t in enumerate(leaves):
        for at in range(t.numel()):
            moved = []
            for sign in (1, -1):
                u = t.clone().view(-1)
                u[at] += sign * h
                moved.append(value(*leaves[:i], u.view_as(t), *leaves[i + 1:]))
            slope = float(moved[0] - moved[1]) / (2 * h)
            # (differences: h^2 times a third derivative, 1e-12 x some hundred; float32 sums of some ten terms of size ten)
            assert abs(float(grads[i].view(-1)[at]) - slope) < 1e-4 + 1e-5 * abs(slope)


def test_zero_rows_empty_batches_and_eps():
    from crystalformer_b200.qk_norm import normalize_rotate
    q, k, wq, wk, pos, waves, gq, gk = make(6, 2, 2, 16, 8, 1, 1, "shared", torch.float32, 2)
    q[2] = 0.0
    outs, grads = both_ways(q, k, wq, wk, pos, waves, gq, gk, False, 1e-6)
    assert (outs[0][2] == 0).all() and torch.isfinite(grads[0]).all()
    q[3, 1, 5] = float("nan")
    k[4, 0, 0] = float("inf")
    outs, grads = both_ways(q, k, wq, wk, pos, waves, gq, gk, False)
    keep = torch.ones((6, 2), dtype=torch.bool, device="cuda")
    keep[3, 1] = False
    assert torch.isfinite(outs[0][keep]).all() and torch.isfinite(grads[0][keep]).all() and torch.isnan(outs[0][3, 1]).all()
    keep[:] = True
    keep[4, 0] = False
    assert torch.isfinite(outs[1][keep]).all() and torch.isfinite(grads[1][keep]).all()
    outs, grads = both_ways(q[:0], k[:0], wq, wk, pos[:0], waves, gq[:0], gk[:0], False)
    assert outs[0].shape == (0, 2, 16) and (grads[2] == 0).all() and (grads[3] == 0).all()


def test_one_output_alone():
    from crystalformer_b200.qk_norm import normalize_rotate
    q, k, wq, wk, pos, waves, gq, gk = make(40, 4, 2, 16, 8, 1, 1, "each", torch.float32, 2)
    q, k, wq = q.requires_grad_(), k.requires_grad_(), wq.requires_grad_()
    normalize_rotate(q, k, wq, wk, pos, waves)[0].backward(gq)
    assert (k.grad == 0).all() and wk.grad is None
    _, (gx, gxb), _ = reference(q.detach(), wq.detach(), gq, pos, waves, False, 1e-6)
    compare(q.grad, (gx, gxb), torch.float32)


def test_repeated_captured_and_on_a_stream():
    from crystalformer_b200 import ops
    data = make(5000, 8, 8, 16, 8, 3, 8, "each", torch.float32, 7)
    q, k, wq, wk, pos, waves, gq, gk = data
    run = lambda: (*ops.qk_norm_fwd(q, k, wq, wk, pos, waves), *ops.qk_norm_bwd(q, k, wq, wk, pos, waves, 1e-6, False, gq, gk))  # noqa: E731
    first = run()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, run()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = run()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run()
    q.copy_(q.flip(0))
    expected = run()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(expected, captured))


def test_module_of_another_type():
    """Made on the device or moved there, made in a type or converted to it: the same module."""
    from crystalformer_b200.qk_norm import QKNorm
    q, k, _, _, pos, *_ = make(30, 4, 4, 16, 8, 3, 4, "none", torch.bfloat16, 5)
    outs = [m(q, k, pos) for m in (QKNorm(4, 16, 8, device="cuda", dtype=torch.bfloat16), QKNorm(4, 16, 8).cuda().bfloat16())]
    assert all(torch.equal(a, b) for a, b in zip(*outs)) and outs[0][0].dtype == torch.bfloat16


def test_refusals():
    from crystalformer_b200 import _lib
    from crystalformer_b200.qk_norm import QKNorm, normalize_rotate
    q, k, wq, wk, pos, waves, *_ = make(10, 4, 2, 16, 8, 3, 1, "each", torch.float32, 1)
    bad = [
        (q.cpu(), k, wq, wk, pos, waves), (q.double(), k.double()), (q, k.half()), (q[0], k), (q, k[:-1]), (q, k[..., :8]), (q, k, wq[:2], wk),
        (q, k, wq, wk[:, :8]), (q, k, wq.half(), wk), (q, k, wq, wk, pos[:-1], waves), (q, k, wq, wk, pos, waves[0]), (q, k, wq, wk, pos, None),
        (q, k, wq, wk, None, waves), (q, k, wq, wk, pos.double(), waves), (q, k, wq, wk, pos[:, :2], waves), (q, k, wq.cpu(), wk),
        (q, k, wq, wk, pos, waves.expand(3, 8, 3)), (q, k, wq, wk, pos, waves.repeat(1, 2, 1)), (q[:, :3], k),
        (q, k, wq, wk, torch.cat((pos, pos), 1), torch.cat((waves, waves), 2)), (q.repeat(1, 1, 40), k.repeat(1, 1, 40)),
    ]
    for args in bad:
        with pytest.raises((RuntimeError, TypeError, ValueError)):
            normalize_rotate(*args)
    assert issubclass(_lib.CrystalformerB200Error, RuntimeError)
    with pytest.raises(ValueError):
        QKNorm(8, 16, 9)
    with pytest.raises(ValueError):
        QKNorm(4, 16, 8).cuda()(q, k.repeat(1, 2, 1))


def test_offsets_beyond_32_bits():
    """Rows 2^28 values apart."""
    from crystalformer_b200 import ops
    far = torch.zeros(9 * 2 ** 28 + 128, dtype=torch.bfloat16, device="cuda")
    q, k = far.as_strided((10, 4, 16), (2 ** 28, 16, 1)), far[64:].as_strided((10, 2, 16), (2 ** 28, 16, 1))
    *_, wq, wk, pos, waves, gq, gk = make(10, 4, 2, 16, 8, 3, 2, "each", torch.bfloat16, 3)
    q.copy_(torch.randn(q.shape, device="cuda"))
    k.copy_(torch.randn(k.shape, device="cuda"))
    for a, b in zip(ops.qk_norm_fwd(q, k, wq, wk, pos, waves), ops.qk_norm_fwd(q.contiguous(), k.contiguous(), wq, wk, pos, waves)):
        assert torch.equal(a, b)
    back = lambda q, k: ops.qk_norm_bwd(q, k, wq, wk, pos, waves, 1e-6, False, gq, gk)  # noqa: E731
    assert all(torch.equal(a, b) for a, b in zip(back(q, k), back(q.contiguous(), k.contiguous())))
