"""GroupNorm's sums over very many values, all nearly alike, so that the roundings of one long chain would all go the same way: a chain of n equal
numbers in 32 bits may end n 2^-25 of itself off.  The bounds are those of the other tests, whose count of roundings does not grow with the size."""
import numpy as np
import pytest
from test_gpu_group_norm import STEPS, U, Oracle, _check_backward, _check_forward

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, scope="module")
def blocks_of_these_sizes_go_back_to_the_driver():
    """A later module's test of the memory pool counts on sizes that no earlier one left there."""
    yield
    from mytorch_b200.backends.cuda.env import CudaEnv

    CudaEnv.instance().lib.pool_trim()


@pytest.mark.parametrize("low,high", [(-0.3, 0.3), (0.1, 0.7), (-0.7, 1.7)])
@pytest.mark.parametrize("n,c,h,w", [(1, 1 << 22, 1, 1), (1, 1, 4096, 2048), (1500, 4, 1, 1), (1 << 21, 4, 1, 1), (1, 3, 1500, 1300)])
def test_two_values(n, c, h, w, low, high):
    import gpu_util as g

    shape = (n, c, h, w)
    rng = np.random.default_rng(c + h)
    x = np.where(rng.random(shape) < 0.5, np.float32(low), np.float32(high)).astype(np.float32)
    dy = np.full(shape, 0.3, np.float32)
    gamma, beta = np.full(c, 0.7, np.float32), np.full(c, 0.1, np.float32)
    o = Oracle(x, 1, gamma, beta, 1e-5, None)
    device = (lambda a: g.dev(a.reshape(n, c) if h * w == 1 else a))
    xt, gt, bt = device(x), g.dev(gamma), g.dev(beta)
    y, mean, rstd = g.op("group_norm")(xt, 1, gt, bt, 1e-5, None)
    _check_forward(g.host(y).reshape(shape), o)
    assert (np.abs(g.host(mean) - o.mean) <= STEPS * U).all() and (np.abs(g.host(rstd) - o.rstd) <= STEPS * U * o.rstd).all()
    dx, dgamma, dbeta = g.op("group_norm_backward")(device(dy), mean, rstd, xt, gt, bt, 1, None)
    _check_backward([g.host(dx).reshape(shape), g.host(dgamma), g.host(dbeta)], o, dy, None)
