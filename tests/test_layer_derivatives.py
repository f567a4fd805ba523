"""Derivatives that the operators of a layer do not have are refused, before the device is touched."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad


@pytest.fixture(scope="module", autouse=True)
def built():
    from crystalformer_b200 import build
    build.build()


def dual(t):
    return forward_ad.make_dual(t, torch.ones_like(t))


def calls(device):
    """Every operator with one argument after the other as a tangent's carrier: (call, arguments, places of the carriers)."""
    from crystalformer_b200.embedding import embed_species
    from crystalformer_b200.feedforward import gated_feed_forward
    from crystalformer_b200.qk_norm import normalize_rotate
    r = lambda *s: torch.randn(s, device=device)  # noqa: E731
    return [(embed_species, [torch.zeros(3, dtype=torch.int64, device=device), r(4, 8)], [1]),
            (normalize_rotate, [r(3, 2, 4), r(3, 2, 4), r(4), r(2, 4), r(3, 1), r(1, 2, 1)], range(6)),
            (gated_feed_forward, [r(3, 4), r(5, 4), r(5, 4), r(4, 5), r(5), r(5), r(4)], range(7))]


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_forward_mode_is_refused(device):
    """Outputs would have no tangent: a derivative of zero, and nothing would say so."""
    for f, args, carriers in calls(device):
        for i in carriers:
            for requires in (False, True):
                with forward_ad.dual_level():
                    some = [dual(a.clone().requires_grad_(requires)) if j == i else a for j, a in enumerate(args)]
                    for grad in (True, False):  # (forward mode does not go by the gradients' switch)
                        with torch.set_grad_enabled(grad), pytest.raises(NotImplementedError, match="forward-mode"):
                            f(*some)


def test_forward_mode_of_the_plain_functions_is_refused():
    from crystalformer_b200 import ops
    (_, (ids, table), _), (_, heads, _), (_, gated, _) = calls("cpu")
    with forward_ad.dual_level():
        for call in (lambda: ops.embed_fwd(ids, dual(table)), lambda: ops.embed_bwd(ids, dual(torch.zeros(3, 8)), 4),
                     lambda: ops.qk_norm_fwd(dual(heads[0]), *heads[1:]), lambda: ops.gated_ffn_fwd(dual(gated[0]), *gated[1:]),
                     lambda: ops.qk_norm_bwd(dual(heads[0]), *heads[1:], 1e-6, False, heads[0], heads[1]),
                     lambda: ops.gated_ffn_bwd(dual(gated[0]), *gated[1:], "silu", gated[0])):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()


@pytest.mark.gpu
def test_forward_over_reverse_is_refused():
    """A gradient that carries a tangent, into the backward of an ordinary call."""
    for f, args, carriers in calls("cuda"):
        leaf = args[carriers[0]].requires_grad_()
        out = f(*args)
        out = out if isinstance(out, torch.Tensor) else out[0]
        with forward_ad.dual_level(), pytest.raises((NotImplementedError, RuntimeError), match="forward-mode"):
            torch.autograd.grad(out, leaf, dual(torch.ones_like(out)))


@pytest.mark.gpu
def test_functional_transforms_are_refused():
    for f, args, carriers in calls("cuda"):
        i = carriers[0]
        one = lambda t: (lambda y: y if isinstance(y, torch.Tensor) else y[0])(f(*(t if j == i else a for j, a in enumerate(args))))  # noqa: E731
        with pytest.raises(RuntimeError):
            torch.func.vmap(one)(torch.stack([args[i], args[i]]))
        with pytest.raises(RuntimeError):
            torch.func.grad(lambda t: one(t).sum())(args[i])
        with pytest.raises(RuntimeError):
            torch.func.jvp(one, (args[i],), (args[i],))
