"""ReLU behind GroupNorm: the backward passes exactly what the forward left at zero or above, also where one of the two directions holds its slabs on the chip and
the other one takes them through memory, and where a value lies within rounding of zero."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape,groups", [
    ((1, 64, 100, 100), 1),   # forward on the chip, backward through memory
    ((2, 30, 130, 130), 1),   # the same, two channels at a time
    ((1, 64, 40, 40), 8),     # both on the chip
    ((1, 64, 200, 200), 1)])  # both through memory
def test_the_backward_sees_the_forwards_side_of_zero(shape, groups):
    import gpu_util as g

    n, c, h, w = shape
    rng = np.random.default_rng(c + h)
    x = rng.standard_normal(shape).astype(np.float32)
    at = rng.standard_normal(c).astype(np.float32)  # of each channel a value that half of its positions have
    x = np.where(rng.random(shape) < 0.5, at[None, :, None, None], x)
    gamma = rng.uniform(0.5, 1.5, c).astype(np.float32)
    xt, gt = g.dev(x), g.dev(gamma)
    none = g.dev(np.zeros(c, np.float32))
    _, mean, rstd = g.op("group_norm")(xt, groups, gt, none, 1e-5, "relu")
    # beta puts that value at zero but for a rounding or two of the first image
    of = np.arange(c) // (c // groups)
    beta = (-(at.astype(np.float64) - g.host(mean)[0, of]) * g.host(rstd)[0, of] * gamma).astype(np.float32)
    near = 0
    for steps in (-1, 0, 1):
        b = beta
        for _ in range(abs(steps)):
            b = np.nextafter(b, np.float32(steps * np.inf))
        bt = g.dev(b)
        z = g.host(g.op("group_norm")(xt, groups, gt, bt, 1e-5, None)[0])
        y, mean, rstd = g.op("group_norm")(xt, groups, gt, bt, 1e-5, "relu")
        assert np.array_equal(g.host(y), np.maximum(z, 0))
        near += int((np.abs(z) < 1e-6).sum())
        # one position at a time would be slow: dbeta of a channel counts the positions whose gradient passes
        _, dgamma, dbeta = g.op("group_norm_backward")(g.dev(np.ones(shape, np.float32)), mean, rstd, xt, gt, bt, groups, "relu")
        assert np.array_equal(g.host(dbeta), (z >= 0).sum((0, 2, 3)).astype(np.float32))
    assert near > c * h * w // 3
