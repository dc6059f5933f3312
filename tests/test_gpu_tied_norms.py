"""One parameter in several roles of the norms around a block, with and without its window of the data-parallel wrapper's flat buffer."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.mark.parametrize("window", [False, True])
@pytest.mark.parametrize("rows,c", [(50, 24), (300, 96), (70, 1000), (9, 9001)])
def test_gradients_of_all_roles_are_added(rows, c, window):
    import gpu_util as g
    import mytorch_b200.nn.functional as F
    from mytorch_b200.backends.cuda.env import CudaMemory, CudaMemoryView

    rng = np.random.default_rng(c)
    x, b = (rng.standard_normal((rows, c)).astype(np.float32) for _ in range(2))
    value = rng.standard_normal(c).astype(np.float32)

    def gradients(*weights):
        new, y = F.add_rms_norm(g.dev(x), g.dev(b), *weights)
        (new * y).sum().backward()

    apart = [g.dev(value, True) for _ in range(3)]
    gradients(*apart)
    parts = [g.host(t.grad).astype(np.float64) for t in apart]

    tied = g.dev(value, True)
    if window:
        flat = CudaMemory(tied.device.index, 4 * (c + 8))
        tied._grad_slot = CudaMemoryView(flat, 16, 4 * c, flat.device_index)
    gradients(tied, tied, tied)
    # two additions in 32 bits
    off = np.abs(g.host(tied.grad) - sum(parts))
    assert (off <= 2 * U * sum(np.abs(p) for p in parts)).all()
    if window:
        again = [g.dev(value, True) for _ in range(2)]
        again[0]._grad_slot = tied._grad_slot
        gradients(again[0], again[0], again[1])
        assert (np.abs(g.host(again[0].grad) - parts[0] - parts[1]) <= U * (np.abs(parts[0]) + np.abs(parts[1]))).all()
        assert np.array_equal(g.host(again[1].grad), parts[2])
