"""Norms around a block of no rows: a gate with a row a sample still has values, and a gradient of zeros."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape", [(4, 0, 6), (4, 6, 0, 3), (4, 6, 3, 0), (0, 5, 6), (0, 6)])
@pytest.mark.parametrize("gate", ["channel", "sample", "value"])
def test_gradients_are_zero(shape, gate):
    import gpu_util as g
    import mytorch_b200.nn.functional as F

    c = shape[1] if len(shape) == 4 else shape[-1]
    gates = {"channel": (c,), "sample": (shape[0], c), "value": shape}[gate]
    dirty = [g.dev(np.full((4, c), 7.0, np.float32)) for _ in range(4)]  # what freed memory holds
    del dirty
    operands = [g.dev(np.ones(s, np.float32), True) for s in (shape, shape, (c,), (c,), gates)]
    new, y = F.add_rms_norm(*operands)
    assert new.shape == y.shape == shape
    loss = (new * y).sum()
    loss.backward()
    for t in operands:
        assert t.grad.shape == t.shape and not g.host(t.grad).any()
