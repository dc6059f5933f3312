"""GroupNorm by clusters whose CTAs have little to do before they write to one another: call after call, so that CTAs of one launch begin
while others of the launch before end."""
import numpy as np
import pytest
from test_gpu_group_norm import Oracle, _check_backward, _check_forward, _inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape,groups", [((2, 64, 8, 8), 1), ((16, 128, 16, 16), 4), ((3, 30, 37, 41), 3), ((64, 64, 32, 32), 32), ((1, 512, 28, 28), 2)])
def test_call_after_call(shape, groups):
    import gpu_util as g

    x, dy, gamma, beta = _inputs(shape, groups, shape[1])
    o = Oracle(x, groups, gamma, beta, 1e-5, "silu")
    xt, dyt, gt, bt = (g.dev(a) for a in (x, dy, gamma, beta))
    calls = []
    for _ in range(60):
        y, mean, rstd = g.op("group_norm")(xt, groups, gt, bt, 1e-5, "silu")
        calls.append((y, *g.op("group_norm_backward")(dyt, mean, rstd, xt, gt, bt, groups, "silu")))
    first = [g.host(t) for t in calls[0]]
    _check_forward(first[0], o)
    _check_backward(first[1:], o, dy, "silu")
    for call in calls[1:]:
        assert all(np.array_equal(g.host(t), want) for t, want in zip(call, first))
