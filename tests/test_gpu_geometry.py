"""A batch's geometry belongs to the positions that it was built from, the fractional coordinates too."""
import pytest
import torch
from test_gpu_layer_options import batch, make_model

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model():
    return make_model(qk_norm=True, qk_rotation=8).eval()


@pytest.mark.parametrize("ahead", [None, True])
def test_positions_that_change_behind_a_geometry(model, ahead):
    from crystalformer_b200.encoder import BatchGeometry
    data, _ = batch()
    with torch.no_grad():
        expected = model(data)
        for use_before in (False, True):
            data, _ = batch()
            g = BatchGeometry(data.pos, data.trans_vec, data.sizes, with_fractional=ahead)
            if use_before:
                assert torch.equal(model(data, geometry=g), expected)
            data.pos.add_(0.4 * torch.arange(data.pos.shape[0], device="cuda")[:, None])
            assert torch.equal(model(data, geometry=g), expected)
        assert not torch.equal(model(data), expected)  # (and a new geometry has the new positions)


def test_fractional_coordinates_outlive_a_capture(model):
    """First asked for inside a capture, whose memory holds nothing until the graph has run."""
    from crystalformer_b200.encoder import BatchGeometry
    data, _ = batch()
    want = BatchGeometry(data.pos, data.trans_vec, data.sizes).fractional
    g = BatchGeometry(data.pos, data.trans_vec, data.sizes)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        g.fractional
    assert torch.equal(g.fractional, want)


def test_a_geometry_without_fractional_coordinates(model):
    from crystalformer_b200.encoder import BatchGeometry
    data, _ = batch()
    g = BatchGeometry(data.pos, data.trans_vec, data.sizes, with_fractional=False)
    with torch.no_grad(), pytest.raises(RuntimeError, match="with_fractional"):
        model(data, geometry=g)
    plain = make_model(qk_norm=True).eval()
    with torch.no_grad():
        assert torch.equal(plain(data, geometry=g), plain(data))


def test_positions_that_ask_for_a_gradient(model):
    """The rotation has none to give."""
    from crystalformer_b200.encoder import BatchGeometry
    for name in ("pos", "trans_vec"):
        data, _ = batch()
        with torch.no_grad():
            expected = model(data)
        getattr(data, name).requires_grad_()
        with pytest.raises(ValueError, match="detach"):
            model(data)
        with pytest.raises(ValueError, match="detach"):
            model(data, geometry=BatchGeometry(data.pos, data.trans_vec, data.sizes))
        with torch.no_grad():
            assert torch.equal(model(data), expected)
        plain = make_model(qk_norm=True)
        plain(data).sum().backward()  # (a model that does not turn its heads takes them as before)
