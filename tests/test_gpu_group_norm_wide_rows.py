"""GroupNorm of rows of millions of channels: what the forward takes, the backward takes too."""
import numpy as np
import pytest
from test_gpu_group_norm import Oracle, _check_backward, _check_forward, _inputs

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, scope="module")
def blocks_of_these_sizes_go_back_to_the_driver():
    """A later module's test of the memory pool counts on sizes that no earlier one left there."""
    yield
    from mytorch_b200.backends.cuda.env import CudaEnv

    CudaEnv.instance().lib.pool_trim()


@pytest.mark.parametrize("n,c,groups", [(1, 32 * 65535, 15), (1, 32 * 65535 + 5, 5), (2, 2500000, 4)])
def test_both_directions(n, c, groups):
    import gpu_util as g
    import mytorch_b200.nn.functional as F

    x, dy, gamma, beta = _inputs((n, c, 1, 1), groups, c % 1000)
    o = Oracle(x, groups, gamma, beta, 1e-5, "silu")
    xt, gt, bt = g.dev(x.reshape(n, c), True), g.dev(gamma, True), g.dev(beta, True)
    y = F.group_norm(xt, groups, gt, bt, activation="silu")
    _check_forward(g.host(y).reshape(x.shape), o)
    (y * g.dev(dy.reshape(n, c))).sum().backward()
    _check_backward([g.host(xt.grad).reshape(x.shape), g.host(gt.grad), g.host(bt.grad)], o, dy, "silu")
