"""The model with species ids, norms and rotation of queries and keys, and gated feed-forward blocks: the operators as the layers use them,
together, against the same layers of plain torch operations."""
import copy
import math
import types

import numpy as np
import pytest
import torch
import torch.nn.functional as F

from crystalformer_b200.synthetic import make_crystals, uniform_atoms

pytestmark = pytest.mark.gpu


def batch(seed=5, crystals=9, hi=20):
    cb = make_crystals(seed, crystals, uniform_atoms(1, hi), length_range=(4.0, 9.0))
    t = lambda x: torch.as_tensor(x).cuda()  # noqa: E731
    data = dict(pos=t(cb.pos), trans_vec=t(cb.trans_vec), sizes=t(cb.sizes))
    return types.SimpleNamespace(x=t(cb.x), **data), types.SimpleNamespace(z=t(cb.x).argmax(1), **data)


def make_model(**options):
    from crystalformer_b200.model import Latticeformer, default_params
    torch.manual_seed(3)
    model = Latticeformer(default_params(num_layers=2, **options)).cuda()
    if options.get("qk_norm"):
        for layer in model.encoder.layers:
            for w in (layer.self_attn.qk_norm.q_weight, layer.self_attn.qk_norm.k_weight):
                torch.nn.init.normal_(w, 1.0, 0.2)
    model.train()(batch()[0])  # sets the width statistics
    return model


def plain_ff(layer, x):
    act = dict(silu=F.silu, gelu=F.gelu, relu=F.relu)[layer.gate]
    return layer.linear2(act(layer.linear_gate(x)) * layer.linear1(x))


def plain_norm(norm, q, k, pos=None):
    outs = []
    for x, w in ((q, norm.q_weight), (k, norm.k_weight)):
        y = x * (x.square().mean(-1, keepdim=True) + norm.eps).rsqrt() * w
        if norm.waves is not None:
            theta = 2 * math.pi * torch.einsum("nc,hpc->nhp", pos.double(), norm.waves.double())
            c, s, P = theta.cos().float(), theta.sin().float(), theta.shape[2]
            a, b = y[..., :P], y[..., P:2 * P]
            y = torch.cat((a * c - b * s, b * c + a * s, y[..., 2 * P:]), -1)
        outs.append(y.to(x.dtype))
    return outs


def plain_copy(model):
    """The same parameters with plain torch in the place of the operators."""
    plain = copy.deepcopy(model)
    for layer in plain.encoder.layers:
        if layer.gate is not None:
            layer._ff_block = types.MethodType(plain_ff, layer)
        if layer.self_attn.qk_norm is not None:
            layer.self_attn.qk_norm.forward = types.MethodType(plain_norm, layer.self_attn.qk_norm)
    return plain


OPTIONS = [
    dict(t_activation="swiglu"), dict(t_activation="geglu", ff_dim=200), dict(t_activation="reglu"), dict(qk_norm=True),
    dict(qk_norm=True, qk_rotation=8), dict(qk_norm=True, qk_rotation=3, domain="multihead"), dict(t_activation="swiglu", qk_norm=True, qk_rotation=8),
]


@pytest.mark.parametrize("options", OPTIONS, ids=lambda o: "-".join(map(str, o.values())))
def test_training_and_inference(options):
    model = make_model(**options)
    plain = plain_copy(model)
    onehot, ids = batch()
    weight = torch.randn((9, 1), device="cuda")
    grads = []
    for m, data in ((model, onehot), (model, ids), (plain, onehot)):
        m.zero_grad()
        y = m.train()(data)
        (y * weight).sum().backward()
        grads.append((y.detach(), {n: p.grad.clone() for n, p in m.named_parameters() if p.grad is not None}))
    assert set(grads[0][1]) == set(grads[1][1]) == set(grads[2][1])
    # Two layers of float32 operations whose roundings (2^-24) differ and grow through them: some hundred roundings of the largest value
    for y, g in grads[:2]:
        assert (y - grads[2][0]).abs().max() <= 512 * 2.0 ** -24 * grads[2][0].abs().max()
        for n, v in g.items():
            ref = grads[2][1][n]
            assert (v - ref).norm() <= 2048 * 2.0 ** -24 * max(float(ref.norm()), 1e-3 * max(float(t.norm()) for t in grads[2][1].values())), n
    with torch.no_grad():
        for data in (onehot, ids):
            y = model.eval()(data)
            assert (y - grads[2][0]).abs().max() <= 512 * 2.0 ** -24 * grads[2][0].abs().max()


def test_species_ids_of_the_ordinary_model():
    """The same model on ids and on one-hot rows, with padding ids as rows of zeros."""
    model = make_model()
    onehot, ids = batch()
    with torch.no_grad():
        a, b = model.eval()(onehot), model(ids)
        assert (a - b).abs().max() <= 512 * 2.0 ** -24 * a.abs().max()
        onehot.x[2], ids.z[2] = 0.0, -1
        a, b = model(onehot), model(ids)
        assert (a - b).abs().max() <= 512 * 2.0 ** -24 * a.abs().max()
    with pytest.raises((ValueError, RuntimeError)):
        model(types.SimpleNamespace(z=ids.z[:-1], pos=ids.pos, trans_vec=ids.trans_vec, sizes=ids.sizes))
    with pytest.raises((ValueError, RuntimeError)):
        model(types.SimpleNamespace(z=ids.z.cpu(), pos=ids.pos, trans_vec=ids.trans_vec, sizes=ids.sizes))


def test_rotation_does_not_see_lattice_translations():
    """Atoms moved by lattice vectors, and the origin of the cells moved: the same products of turned queries and keys.  (The model's
    output changes by more: the lattice sums are cut off at boxes that are not centred on the moved atoms.)"""
    from crystalformer_b200.encoder import BatchGeometry
    model = make_model(qk_norm=True, qk_rotation=8).eval()
    norm = model.encoder.layers[0].self_attn.qk_norm
    onehot, _ = batch()
    gen = torch.Generator().manual_seed(1)
    crystal = torch.repeat_interleave(torch.arange(9, device="cuda"), onehot.sizes)
    n = torch.randint(-1, 2, (onehot.pos.shape[0], 3), generator=gen).float().cuda()
    moved = onehot.pos + torch.einsum("ni,nij->nj", n, onehot.trans_vec[crystal]) + torch.tensor([0.3, -0.2, 0.7], device="cuda")
    q, k = torch.randn((2, onehot.pos.shape[0], 8, 16), generator=gen).cuda().unbind(0)
    logits, same = [], crystal[:, None] == crystal[None]
    with torch.no_grad():
        for pos in (onehot.pos, moved):
            g = BatchGeometry(pos, onehot.trans_vec, onehot.sizes)
            assert ((g.fractional >= 0) & (g.fractional <= 1)).all()
            a, b = norm(q, k, g.fractional)
            logits.append(torch.einsum("ihd,jhd->hij", a.double(), b.double()))
    # A moved position is rounded three times (the products, the sum, the shift), by half a step of its largest value each time; a
    # fractional coordinate changes by that times the rows of the inverse cell, an angle by 2 pi times the wave's entries times that,
    # a product of two heads by the angles of both times their lengths.  The coordinates' own storage adds half a step of 1.
    off = 3 * 2.0 ** -24 * 2 * float(moved.abs().max()) * float(torch.linalg.inv(onehot.trans_vec.double()).abs().sum(1).max()) + 2.0 ** -24
    bound = 2 * (2 * math.pi * float(norm.waves.abs().sum(-1).max()) * off) * float(a.norm(dim=-1).max() * b.norm(dim=-1).max()) + 1e-4
    assert bound < 0.1 and (logits[0] - logits[1])[:, same].abs().max() <= bound


def test_serving_ids_to_a_gated_model():
    from crystalformer_b200.serving import PipelinedPredictor
    model = make_model(t_activation="swiglu").eval()
    onehot, ids = batch()
    with torch.no_grad():
        expected = model(ids).cpu()
    host = types.SimpleNamespace(**{n: v.cpu().pin_memory() for n, v in vars(ids).items()})
    runner = PipelinedPredictor(model, depth=2)
    for _ in range(3):
        assert torch.equal(runner.result(runner.submit(host)), expected)
    host = types.SimpleNamespace(**{n: v.cpu().pin_memory() for n, v in vars(onehot).items()})
    y = runner.result(runner.submit(host))
    assert (y - expected).abs().max() <= 512 * 2.0 ** -24 * expected.abs().max()


def test_a_captured_step_of_the_operators_together():
    """Embedding, norms, attention products and the gated block, forward and backward, in one graph: the operators as a layer of another
    model would use them, in bfloat16."""
    from crystalformer_b200.embedding import embed_species
    from crystalformer_b200.feedforward import GatedFeedForward
    from crystalformer_b200.qk_norm import QKNorm
    torch.manual_seed(0)
    N, V = 96, 40
    table = torch.randn((V, 64), device="cuda").bfloat16().requires_grad_()
    qkv = torch.nn.Linear(64, 192, device="cuda", dtype=torch.bfloat16)
    norm, block = QKNorm(4, 16, 8, device="cuda", dtype=torch.bfloat16), GatedFeedForward(64, 136, device="cuda", dtype=torch.bfloat16)
    ids, pos = torch.randint(0, V, (N,), device="cuda"), torch.rand((N, 3), device="cuda")
    leaves = [table, *qkv.parameters(), *norm.parameters(), *block.parameters()]

    def step(block_of=None, norm_of=None, embed_of=embed_species):
        x = embed_of(ids, table, 0.5)
        q, k, v = qkv(x).split(64, 1)
        q, k = (norm_of or norm)(q.unflatten(1, (4, 16)), k.unflatten(1, (4, 16)), pos)
        p = torch.softmax(torch.einsum("ihd,jhd->hij", q, k) * 0.25, -1)
        x = x + torch.einsum("hij,jhd->ihd", p, v.unflatten(1, (4, 16))).flatten(1)
        y = x + (block_of or block)(x)
        return (y, *torch.autograd.grad(y.float().square().mean(), leaves))

    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        captured = step()
    ids.copy_(ids.flip(0))
    graph.replay()
    torch.cuda.synchronize()
    eager = step()
    assert all(torch.equal(a, b) for a, b in zip(captured, eager))
    f = F.silu
    plain = step(lambda x: block.down(f(block.gate(x)) * block.up(x)), lambda q, k, p: plain_norm(norm, q, k, p),
                 lambda i, t, s: (t * s)[i])
    for a, b in zip(eager, plain):
        # a dozen bfloat16 roundings in a row (2^-8 half a step) on either side
        assert (a.double() - b.double()).norm() <= 24 * 2.0 ** -9 * 2 * b.double().norm()


FRESH = """
import torch
from crystalformer_b200 import ops
from crystalformer_b200.embedding import embed_species
from crystalformer_b200.feedforward import gated_feed_forward
from crystalformer_b200.qk_norm import normalize_rotate
torch.manual_seed(0)
r = lambda *s: torch.randn(s, device="cuda")
table, ids, pos, waves = r(9, 128), torch.randint(0, 9, (300,), device="cuda"), torch.rand((300, 3), device="cuda"), torch.ones((1, 8, 3), device="cuda")
w = [r(512, 128) * 0.1, r(512, 128) * 0.1, r(128, 512) * 0.1]
leaves = [t.requires_grad_() for t in (table, *w)]
gout = r(300, 128)
def step():
    x = embed_species(ids, table, 0.5)
    q, k = normalize_rotate(x.view(300, 8, 16), x.view(300, 8, 16), None, None, pos, waves)
    y = gated_feed_forward((q + k).reshape(300, 128), *w)
    return (y, *torch.autograd.grad(y, leaves, gout))
graph = torch.cuda.CUDAGraph()
torch.zeros(1, device="cuda").add_(1)  # (a context; none of the library's kernels has run)
torch.cuda.synchronize()
with torch.cuda.graph(graph):
    captured = step()
graph.replay()
torch.cuda.synchronize()
captured = [t.clone() for t in captured]
eager = step()
assert all(torch.equal(a, b) for a, b in zip(captured, eager))
ops.set_chained_launches(False)
assert all(torch.equal(a, b) for a, b in zip(captured, step()))
print("the same")
"""


def test_a_process_that_starts_with_a_capture():
    """The first calls of a process may be captured ones; results do not depend on how the kernels of a call are chained."""
    import subprocess
    import sys
    done = subprocess.run([sys.executable, "-c", FRESH], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "the same" in done.stdout, done.stderr[-2000:]


def test_refusals():
    from crystalformer_b200.model import Latticeformer, default_params
    with pytest.raises(NotImplementedError):
        Latticeformer(default_params(t_activation="swiglu", dropout=0.1))
    with pytest.raises(ValueError):
        Latticeformer(default_params(qk_rotation=4))
    with pytest.raises(ValueError):
        Latticeformer(default_params(qk_norm=True, qk_rotation=9))
    with pytest.raises(RuntimeError):
        Latticeformer(default_params(t_activation="tanhglu"))
