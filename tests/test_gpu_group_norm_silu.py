"""SiLU behind GroupNorm, value by value: with a weight of zero the activation's input is the bias, bit by bit.

Bound: sigmoid is a power of two (2^-22 of itself by the hardware), times a remainder that a few units of 2^-24 round, plus one, and a reciprocal (2^-23):
under 2^-20 of itself all in all, for every input whose result is a normal number.  Its slope is s + s z (1 - s), in which 1 - s is off by the
roundings of s: 2^-20 of s (1 + |z|)."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

BOUND = 2.0 ** -20
CHANNELS = [4096, 1022, 1021, 4095, 30000]  # four, two and one at a time; on the chip, and through memory in one group


@pytest.mark.parametrize("groups", [1, "channels"])
@pytest.mark.parametrize("channels", CHANNELS)
@pytest.mark.parametrize("low,high", [(-85, -10), (-10, 10), (10, 85), (-1e-3, 1e-3), (-1.3, -1.25)])
def test_every_size_of_input(low, high, channels, groups):
    import gpu_util as g

    groups = channels if groups == "channels" else groups
    rng = np.random.default_rng(channels)
    z = rng.uniform(low, high, channels).astype(np.float32)
    x, dy = rng.standard_normal((2, channels)).astype(np.float32), rng.standard_normal((2, channels)).astype(np.float32)
    xt, gt, bt = g.dev(x), g.dev(np.zeros(channels, np.float32)), g.dev(z)
    y, mean, rstd = g.op("group_norm")(xt, groups, gt, bt, 1e-5, "silu")
    exact = z.astype(np.float64)
    s = 1 / (1 + np.exp(-exact))
    assert (np.abs(g.host(y) - exact * s) <= BOUND * np.abs(exact * s)).all()
    _, _, dbeta = g.op("group_norm_backward")(g.dev(dy), mean, rstd, xt, gt, bt, groups, "silu")
    size = np.abs(dy.astype(np.float64)).sum(0)
    assert (np.abs(g.host(dbeta) - (dy.astype(np.float64) * (s + s * exact * (1 - s))).sum(0)) <= BOUND * s * (1 + np.abs(exact)) * size).all()


@pytest.mark.parametrize("channels", CHANNELS)
def test_inputs_beyond(channels):
    import gpu_util as g

    values = np.array([-3e38, -1e30, -1e7, -1000, -100, -90, 0, 90, 100, 1000, 1e7, 1e30, 3e38, np.inf, np.nan], np.float32)
    z = np.resize(values, channels)
    x = np.random.default_rng(1).standard_normal((1, channels)).astype(np.float32)
    xt, gt, bt = g.dev(x), g.dev(np.zeros(channels, np.float32)), g.dev(z)
    y, mean, rstd = g.op("group_norm")(xt, 1, gt, bt, 1e-5, "silu")
    got = g.host(y)[0]
    assert (np.abs(got[z < 0]) <= 1e-36).all() and np.array_equal(got[z >= 0], z[z >= 0]) and np.isnan(got[np.isnan(z)]).all()
    _, _, dbeta = g.op("group_norm_backward")(g.dev(np.ones_like(x)), mean, rstd, xt, gt, bt, 1, "silu")
    slope = g.host(dbeta)
    finite = np.isfinite(z)
    want = np.where(z < 0, 0, np.where(z > 0, 1, 0.5))
    assert (np.abs(slope - want)[finite] <= 1e-6).all() and np.isnan(slope[np.isnan(z)]).all()
