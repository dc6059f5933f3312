"""Clipping in place where gradients share memory: it is multiplied once, and counts for each of them."""
import numpy as np
import pytest
from test_gpu_clip import U

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("size,windows", [
    (1000, [(0, 600), (400, 600)]),  # (start, elements) of each gradient in a block of `size`
    (1000, [(1, 999), (0, 10), (5, 20), (3, 3)]),
    (100000, [(0, 100000), (37, 20000), (8192, 70000), (37, 5)]),
    (100000, [(50000, 50000), (0, 50001), (99999, 1)]),
    (64, [(32, 32), (0, 32)]),  # side by side
    (64, [(0, 8), (0, 64), (0, 8)])])
def test_windows_of_one_block(size, windows):
    import gpu_util as g
    import mytorch_b200 as mt
    from mytorch_b200.backends.cuda.env import CudaMemory, CudaMemoryView
    from mytorch_b200.optim import clip_grad_norm_

    values = np.random.default_rng(size).standard_normal(size).astype(np.float32)
    block = CudaMemory(0, 4 * size)
    CudaMemoryView(block, 0, 4 * size, 0).write(values)
    params, touched = [], np.zeros(size, bool)
    for start, count in windows:
        p = mt.Tensor(shape=(count,), dtype=mt.float32, device="cuda:0", requires_grad=True)
        p.grad = mt.Tensor._on_device((count,), mt.float32, p.device, CudaMemoryView(block, 4 * start, 4 * count, 0))
        params.append(p)
        touched[start:start + count] = True
    want = float(np.sqrt(sum((values[s:s + n].astype(np.float64) ** 2).sum() for s, n in windows)))
    assert abs(g.host(clip_grad_norm_(params, want / 4))[0] - want) <= 2 * U * want
    factor = np.where(touched, want / 4 / (want + 1e-6), 1.0)
    got = g.host(mt.Tensor._on_device((size,), mt.float32, params[0].device, CudaMemoryView(block, 0, 4 * size, 0)))
    assert (np.abs(got - values * factor) <= 4 * U * np.abs(values)).all()
