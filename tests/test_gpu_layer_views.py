"""Operators of a layer on views whose negation is still to be done (imaginary parts of conjugated complex tensors)."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def negated(t):
    """-t as a view of t's memory."""
    view = torch.complex(t, t).conj().imag
    assert view.is_neg() and torch.equal(view, -t)
    return view


@pytest.mark.parametrize("view", [negated, torch._neg_view], ids=["strided", "contiguous"])
def test_views_to_be_negated(view):
    from crystalformer_b200 import ops
    r = lambda *s: torch.randn(s, device="cuda")  # noqa: E731
    ids, table, gout = torch.tensor([2, 0, 3], device="cuda"), r(4, 8), r(3, 8)
    heads, gated = [r(3, 2, 4), r(3, 2, 4), r(4), r(2, 4), r(3, 1), r(1, 2, 1)], [r(30, 4), r(5, 4), r(5, 4), r(4, 5), r(5), r(5), r(4)]
    assert torch.equal(ops.embed_fwd(ids, view(table)), ops.embed_fwd(ids, -table))
    assert torch.equal(ops.embed_fwd(torch._neg_view(-ids), table), ops.embed_fwd(ids, table))
    assert torch.equal(ops.embed_bwd(ids, view(gout), 4), ops.embed_bwd(ids, -gout, 4))
    for i in range(6):
        a, b = ([f(t) if j == i else t for j, t in enumerate(heads)] for f in (view, torch.neg))
        assert all(torch.equal(u, v) for u, v in zip(ops.qk_norm_fwd(*a), ops.qk_norm_fwd(*b))), i
        assert all(torch.equal(u, v) for u, v in zip(ops.qk_norm_bwd(*a, 1e-6, False, view(heads[0]), view(heads[1])),
                                                     ops.qk_norm_bwd(*b, 1e-6, False, -heads[0], -heads[1]))), i
    gy = r(30, 4)
    for i in range(7):
        a, b = ([f(t) if j == i else t for j, t in enumerate(gated)] for f in (view, torch.neg))
        assert torch.equal(ops.gated_ffn_fwd(*a), ops.gated_ffn_fwd(*b)), i
        assert all(torch.equal(u, v) for u, v in zip(ops.gated_ffn_bwd(*a, "silu", view(gy)), ops.gated_ffn_bwd(*b, "silu", -gy))), i
