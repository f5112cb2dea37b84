"""The end of a block without columns."""
import pytest

import tensorplay_amd as tp
from tests.test_block_ops_gpu import DTYPES, _stream  # noqa: F401

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("gates", [0, 2])
def test_no_columns(gates, dtype):
    """The mean of no squares is NaN, and so are the roots; gradients are as empty as the
    inputs."""
    f = tp.from_torch
    x, w = torch.zeros((2, 3, 0), device="cuda", dtype=dtype), torch.zeros((0,), device="cuda", dtype=dtype)
    g = torch.zeros((gates, 0), device="cuda", dtype=dtype) if gates else None
    more = dict(post_weight=f(w), gate=f(g) if gates else None, p=0.1, seed=3)
    # blocks that the outputs may be given hold numbers
    for _ in range(4):
        f(torch.zeros((6,), device="cuda")).clone()
    out, y, rpost, rpre = tp.gated_residual_norm(f(x), f(x), f(w), **more)
    assert out.shape == [2, 3, 0] and y.shape == [2, 3, 0] and rpost.shape == [2, 3] and rpre.shape == [2, 3]
    assert bool(tp.to_torch(rpost).isnan().all()) and bool(tp.to_torch(rpre).isnan().all())
    grads = tp.gated_residual_norm_backward(f(x), f(x), f(x), out, rpost, rpre, f(w), **more)
    shapes = [None if t is None else t.shape for t in grads]
    assert shapes == [[2, 3, 0], [2, 3, 0], [0], [0], [gates, 0] if gates else None]
    # without a post weight there is one root
    out, y, rpost, rpre = tp.gated_residual_norm(f(x), f(x), f(w))
    assert rpost is None and bool(tp.to_torch(rpre).isnan().all())
    with pytest.raises(ValueError, match="gates must divide"):
        tp.gated_residual_norm(f(x), f(x), f(w), gate=f(torch.zeros((4, 0), device="cuda", dtype=dtype)))
