"""Which species a batch may carry: one-hot rows ``x`` of any type, or positions ``z`` of their ones."""
import types

import pytest
import torch


def batch(device="cpu", **species):
    gen = torch.Generator().manual_seed(0)
    sizes = torch.tensor([3, 1, 4])
    data = dict(pos=torch.rand((8, 3), generator=gen) * 5, trans_vec=torch.eye(3).repeat(3, 1, 1) * 5, sizes=sizes, **species)
    return types.SimpleNamespace(**{n: v.to(device) for n, v in data.items()})


Z = torch.tensor([5, 7, 5, 0, 97, 12, 13, 7])
ONEHOT = torch.nn.functional.one_hot(Z, 98)
TYPES = [torch.float32, torch.float64, torch.int64, torch.uint8, torch.bool]


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_any_type_hold_a_batch(dtype):
    from crystalformer_b200.model import check_batch
    check_batch(batch(x=ONEHOT.to(dtype)), 8)
    for bad in (batch(x=ONEHOT.to(dtype)[:7]), batch(x=ONEHOT.to(dtype)[:, 0]), batch(x=ONEHOT.to(dtype)[None])):
        with pytest.raises(ValueError, match="do not hold"):
            check_batch(bad, 8)


def test_positions_hold_a_batch():
    from crystalformer_b200.model import check_batch
    for z in (Z, Z.int()):
        check_batch(batch(z=z), 8)
        for bad in (batch(z=z[:7]), batch(z=z[:, None]), batch(z=ONEHOT)):
            with pytest.raises(ValueError, match="do not hold"):
                check_batch(bad, 8)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_inference_on_rows_of_any_type(dtype):
    """With the sizes known on the host and without: what rows of float32 give."""
    from crystalformer_b200.model import Latticeformer, default_params
    torch.manual_seed(0)
    model = Latticeformer(default_params(num_layers=2)).cuda()
    rows = batch("cuda", x=ONEHOT.float())
    model.train()(rows)  # sets the width statistics
    model.eval()
    with torch.no_grad():
        for counts in (None, (8, 26, 4)):
            assert torch.equal(model(batch("cuda", x=ONEHOT.to(dtype)), counts=counts), model(rows, counts=counts))
            with pytest.raises((ValueError, IndexError)):
                model(batch("cuda", x=Z), counts=counts)
