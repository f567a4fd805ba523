"""Gated feed-forward block: values at the ends of their types, long contractions, many short launches in a row."""
import pytest
import torch
from test_gpu_gated import TYPES, make

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
