"""Embedding lookup by id and the gradient of its table from sorted ids, against 64-bit sums of the same values.

Bounds: a value is scaled in float32 and stored in its type (half a step each); a sum of m rows in float32 is off by at most
m 2^-24 of the sum of magnitudes, whatever its order, before it is scaled and stored."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def make(N, V, D, dtype, seed, layout="table", skew=True, padding=False):
    gen = torch.Generator().manual_seed(seed)
    table = torch.randn((V, D) if layout == "table" else (D, V), generator=gen).to(dtype).cuda()
    ids = (torch.rand(N, generator=gen) ** (3 if skew else 1) * V).long().clamp_(max=V - 1)
    if padding and N:
        ids[torch.rand(N, generator=gen) < 0.3] = -1
        ids[0] = V  # (outside on the other side)
    gout = torch.randn((N, D), generator=gen).to(dtype).cuda()
    return (table if layout == "table" else table.t()), ids.cuda(), gout


def check(table, ids, gout, out, grad, scale):
    dtype, (V, D) = table.dtype, table.shape
    valid = (ids >= 0) & (ids < V)
    ref = torch.zeros((*ids.shape, D), dtype=torch.float64, device="cuda")
    ref[valid] = table.double()[ids[valid]] * scale
    assert ((out.double() - ref).abs() <= (half_step(dtype) + 2.0 ** -23) * ref.abs() + tiny(dtype)).all()
    assert (out[~valid] == 0).all()
    if grad is None:
        return
    g = gout.reshape(-1, D).double()[valid.reshape(-1)]
    at = ids[valid]
    total = torch.zeros((V, D), dtype=torch.float64, device="cuda").index_add_(0, at, g) * scale
    size = torch.zeros((V, D), dtype=torch.float64, device="cuda").index_add_(0, at, g.abs()) * abs(scale)
    count = torch.bincount(at, minlength=V).double()[:, None]
    assert ((grad.double() - total).abs() <= (count + 2) * 2.0 ** -24 * size + half_step(dtype) * total.abs() + tiny(dtype)).all()
    assert (grad[torch.bincount(at, minlength=V) == 0] == 0).all()


def tiny(dtype):
    """Half a step of the smallest numbers: below them steps do not shrink."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


CASES = [
    # N, V, D: one row; one id; odd widths; more digits than one; ids of three bytes; exact tiles and one more or less
    (1, 1, 1), (1, 98, 128), (7, 3, 5), (31, 98, 128), (32, 98, 128), (33, 98, 128), (2047, 98, 24), (2048, 1, 128), (2049, 255, 40),
    (3000, 256, 33), (5000, 257, 64), (4097, 65536, 8), (3001, 70001, 130), (20000, 98, 128), (1000, 98, 1024), (500, 10, 1023),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,V,D", CASES)
def test_lookup_and_gradient(N, V, D, dtype):
    from crystalformer_b200.embedding import embed_species
    for layout in ("table", "linear"):
        for padding in (False, True):
            table, ids, gout = make(N, V, D, dtype, N + V + D, layout, padding=padding)
            table.requires_grad_()
            out = embed_species(ids, table, 0.25)
            (grad,) = torch.autograd.grad(out, table, gout)
            assert out.dtype == grad.dtype == dtype and grad.shape == table.shape
            check(table.detach(), ids, gout, out.detach(), grad, 0.25)


@pytest.mark.parametrize("N,V,D", [(262145, 70001, 8), (600001, 98, 16), (1000003, 300, 3)])
def test_many_rows(N, V, D):
    """More blocks of rows than the sort's passes read the counts of themselves."""
    from crystalformer_b200 import ops
    table, ids, gout = make(N, V, D, torch.float32, 4, padding=True)
    check(table, ids, gout, ops.embed_fwd(ids, table, 0.5), ops.embed_bwd(ids, gout, V, 0.5), 0.5)


def test_layout_of_the_gradient():
    """The gradient reaches the weight of a Linear contiguous."""
    from crystalformer_b200.embedding import embed_species
    linear = torch.nn.Linear(98, 128, bias=False, device="cuda")
    ids = torch.arange(300, device="cuda") % 98
    embed_species(ids, linear.weight.t()).sum().backward()
    assert linear.weight.grad.is_contiguous() and linear.weight.grad.shape == (128, 98)
    onehot = torch.nn.functional.one_hot(ids, 98).float()
    (expected,) = torch.autograd.grad(onehot.double() @ linear.weight.double().t(), linear.weight, torch.ones((300, 128), device="cuda").double())
    assert torch.equal(linear.weight.grad, expected)  # (whole numbers)


@pytest.mark.parametrize("dtype", TYPES)
def test_shapes_strides_and_emptiness(dtype):
    from crystalformer_b200 import ops
    from crystalformer_b200.embedding import embed_species
    table, ids, gout = make(60, 11, 16, dtype, 3)
    # ids of several dimensions and of other whole types, and strided
    out = embed_species(ids.view(3, 4, 5).to(torch.int32), table, 2.0)
    assert out.shape == (3, 4, 5, 16) and torch.equal(out.view(60, 16), embed_species(ids, table, 2.0))
    assert torch.equal(embed_species(ids.view(4, 15).t(), table), embed_species(ids, table).view(4, 15, 16).transpose(0, 1))
    # a table inside a larger one, off 16 bytes, and one row for all ids
    large = torch.randn((11, 40), device="cuda").to(dtype)
    for part in (large[:, 3:19], large[:, 8:24], large[:, ::2][:, :16], large[4:5, :16].expand(11, 16)):
        check(part, ids, gout, embed_species(ids, part, 3.0), None, 3.0)
    # strided and repeated gradients
    wide = torch.randn((60, 50), device="cuda").to(dtype)
    for g in (wide[:, 1:17], wide[:, 16:32], wide[:1, :16].expand(60, 16), wide[:, ::3][:, :16]):
        assert torch.equal(ops.embed_bwd(ids, g, 11, 0.5), ops.embed_bwd(ids, g.contiguous(), 11, 0.5))
    # no rows
    none = torch.empty(0, dtype=torch.int64, device="cuda")
    assert embed_species(none, table).shape == (0, 16)
    assert (ops.embed_bwd(none, gout[:0], 11) == 0).all()
    # all rows padded
    pad = torch.full((60,), -1, device="cuda")
    assert (embed_species(pad, table) == 0).all() and (ops.embed_bwd(pad, gout, 11) == 0).all()


def test_values_that_are_no_numbers_stay_in_their_rows():
    from crystalformer_b200 import ops
    table, ids, gout = make(400, 9, 32, torch.float32, 8)
    table[4] = float("nan")
    ids[17] = -1
    gout[17] = float("inf")  # of a padded row: no part in the gradient
    out, grad = ops.embed_fwd(ids, table), ops.embed_bwd(ids, gout, 9)
    assert torch.isnan(out[ids == 4]).all() and torch.isfinite(out[ids != 4]).all() and torch.isfinite(grad).all()
    gout[ids == 2] = float("nan")
    grad = ops.embed_bwd(ids, gout, 9)
    assert torch.isnan(grad[2]).all() and torch.isfinite(grad[[0, 1, 3, 4, 5, 6, 7, 8]]).all()


def test_the_same_bits_every_time():
    from crystalformer_b200 import ops
    table, ids, gout = make(50000, 98, 128, torch.float32, 5)
    first = ops.embed_bwd(ids, gout, 98)
    for _ in range(5):
        assert torch.equal(first, ops.embed_bwd(ids, gout, 98))


def test_on_a_stream_and_captured():
    from crystalformer_b200 import ops
    table, ids, gout = make(3000, 300, 64, torch.float32, 6, padding=True)
    out, grad = ops.embed_fwd(ids, table, 0.5), ops.embed_bwd(ids, gout, 300, 0.5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out2, grad2 = ops.embed_fwd(ids, table, 0.5), ops.embed_bwd(ids, gout, 300, 0.5)
    side.synchronize()
    assert torch.equal(out, out2) and torch.equal(grad, grad2)
    graphs = []
    for _ in range(2):  # two graphs that run one after the other in any order
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = ops.embed_fwd(ids, table, 0.5), ops.embed_bwd(ids, gout, 300, 0.5)
        graphs.append((g, outs))
    ids.copy_(ids.flip(0))
    expected = ops.embed_fwd(ids, table, 0.5), ops.embed_bwd(ids, gout, 300, 0.5)
    for order in ((0, 1), (1, 0)):
        for i in order:
            graphs[i][0].replay()
        torch.cuda.synchronize()
        for _, outs in graphs:
            assert torch.equal(outs[0], expected[0]) and torch.equal(outs[1], expected[1])


def test_refusals():
    from crystalformer_b200 import _lib
    from crystalformer_b200.embedding import embed_species
    table, ids, gout = make(10, 5, 8, torch.float32, 1)
    for bad in ((ids.cpu(), table), (ids, table.double()), (ids.float(), table), (ids, table[0]), (ids, table.cpu())):
        with pytest.raises((RuntimeError, TypeError, ValueError)):
            embed_species(*bad)
    from crystalformer_b200 import ops
    with pytest.raises(ValueError):
        ops.embed_bwd(ids, gout[:-1], 5)
    with pytest.raises(_lib.CrystalformerB200Error):
        ops.embed_bwd(ids, gout, 0)
    table.requires_grad_()
    out = embed_species(ids, table)
    (grad,) = torch.autograd.grad(out, table, gout.requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError):  # (once differentiable)
        grad.sum().backward()


def test_offsets_beyond_32_bits():
    from crystalformer_b200 import ops
    # rows of a table and of a gradient 2^28 values apart
    far = torch.zeros(8 * 2 ** 28 + 64, dtype=torch.bfloat16, device="cuda")
    view = far.as_strided((9, 64), (2 ** 28, 1))
    view.copy_(torch.randn((9, 64), device="cuda"))
    ids = torch.tensor([8, 0, 3, 8, -1, 7], device="cuda")
    assert torch.equal(ops.embed_fwd(ids, view), ops.embed_fwd(ids, view.contiguous()))
    nine = torch.arange(9, device="cuda") % 4
    assert torch.equal(ops.embed_bwd(nine, view, 5), ops.embed_bwd(nine, view.contiguous(), 5))
    del far, view
    # an output of more than 2^31 values, and its gradient's rows
    N, D = 2 ** 24 + 77, 128
    table = torch.randn((98, D), device="cuda").bfloat16()
    ids = torch.randint(0, 98, (N,), device="cuda")
    out = ops.embed_fwd(ids, table)
    for part in (slice(0, 1000), slice(2 ** 24 - 500, 2 ** 24 + 77)):
        assert torch.equal(out[part], table[ids[part]])
    out[:-50] = 0
    grad = ops.embed_bwd(ids, out, 98)  # (the last fifty rows alone are not zero)
    expected = torch.zeros((98, D), device="cuda").index_add_(0, ids[-50:], out[-50:].float())
    assert (grad.float() - expected).abs().max() <= (2.0 ** -9 + 50 * 2.0 ** -24) * 2 * expected.abs().max()


def test_from_several_threads():
    """Calls of several host threads at once, each on its own stream."""
    import threading

    from crystalformer_b200 import ops
    from crystalformer_b200.feedforward import gated_feed_forward
    data = [make(3000 + 100 * i, 98, 64, torch.float32, i) for i in range(4)]
    w = [torch.randn(s, device="cuda") * 0.1 for s in ((96, 64), (96, 64), (64, 96))]
    alone = [(ops.embed_bwd(ids, gout, 98), gated_feed_forward(gout, *w)) for _, ids, gout in data]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        _, ids, gout = data[i]
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                a, b = ops.embed_bwd(ids, gout, 98), gated_feed_forward(gout, *w)
                torch.cuda.current_stream().synchronize()
                if not (torch.equal(a, alone[i][0]) and torch.equal(b, alone[i][1])):
                    wrong.append(i)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
