"""A step needs the gradient of every parameter, with clipping as without; where one is missing it says so and changes nothing."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("steps_before", [0, 1])
def test_a_parameter_without_gradient(steps_before):
    import gpu_util as g
    import mytorch_b200.nn as nn
    from mytorch_b200.optim import SGD, clip_grad_norm_

    p, q = nn.Parameter(g.dev(np.ones(8, np.float32))), nn.Parameter(g.dev(np.ones((2, 4), np.float32)))
    opt = SGD([p, q], lr=0.5, momentum=0.9, max_grad_norm=100.0)
    ones = [np.ones(8, np.float32), np.ones((2, 4), np.float32)]
    for _ in range(steps_before):
        p.grad, q.grad = (g.dev(a) for a in ones)
        opt.step()
    before = [g.host(p), g.host(q)]
    p.grad, q.grad = g.dev(ones[0]), None
    with pytest.raises(RuntimeError, match="no gradient"):
        opt.step()
    assert np.array_equal(g.host(p), before[0]) and np.array_equal(g.host(q), before[1]) and len(opt.state) == 2 * steps_before
    assert g.host(clip_grad_norm_([p, q], 100.0))[0] == np.float32(np.sqrt(8))  # a norm of those that there are
    q.grad = g.dev(ones[1])
    opt.step()
    assert (g.host(p) < before[0]).all() and (g.host(q) < before[1]).all()
