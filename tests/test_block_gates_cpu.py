"""Gates that the rows of a block cannot have are refused before anything is allocated or
launched, so this needs no GPU."""
import pytest

import tensorplay_amd as tp
from tensorplay_amd import _C


def fake(*shape):
    """A tensor at an address that no refused call follows."""
    strides = [1] * len(shape)
    for i in range(len(shape) - 1, 0, -1):
        strides[i - 1] = strides[i] * max(shape[i], 1)
    return _C._from_device_ptr(256, list(shape), strides, tp.float32, 0, None)


@pytest.mark.parametrize("gate", [(0, 8), (2, 0, 8)])
def test_no_gates_for_some_rows(gate):
    x, w = fake(4, 8), fake(8)
    with pytest.raises(ValueError, match="gates must divide"):
        tp.gated_residual_norm(x, x, w, gate=fake(*gate))
    with pytest.raises(ValueError, match="gates must divide"):
        tp.gated_residual_norm_backward(x, x, x, x, None, fake(4), w, gate=fake(*gate))
