"""GroupNorm with an activation, forward and backward, against the formulas in 64 bits and against differences.

Bounds: u = 2^-24.  A sum is added up in chains of at most some dozens of terms a thread and a tree over the threads, a value goes through a
handful of roundings: STEPS roundings of the largest number on the way are allowed.  For a value of z that number is
|gamma| (|xh| + r (|mean| + mean |x|)) + |beta|: what is subtracted, multiplied and added; the activations' slopes are at most 1.1."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, scope="module")
def blocks_of_these_sizes_go_back_to_the_driver():
    """A later module's test of the memory pool counts on sizes that no earlier one left there."""
    yield
    from mytorch_b200.backends.cuda.env import CudaEnv

    CudaEnv.instance().lib.pool_trim()


U, STEPS = 2.0 ** -24, 64

SHAPES = [  # n, c, h, w, groups
    (1, 4, 1, 1, 2), (2, 8, 1, 1, 8), (3, 6, 5, 7, 3), (2, 64, 32, 32, 32), (5, 150, 9, 11, 15), (1, 32, 3, 3, 1), (2, 48, 17, 19, 48), (4, 96, 40, 40, 8),
    (1, 512, 2, 2, 32), (2, 7, 23, 29, 7), (1, 64, 160, 160, 8), (300, 16, 4, 4, 4), (1, 1, 1, 7, 1), (2, 1030, 3, 5, 2), (1, 2048, 7, 7, 32), (9, 36, 64, 1, 4),
    (1, 260, 1, 300, 1), (1, 8, 333, 301, 2), (3, 130, 70, 70, 1)]


def _silu(z):
    s = 1 / (1 + np.exp(-z))
    return z * s, s * (1 + z * (1 - s))


def _f(z, act):
    if act == "silu":
        return _silu(z)
    if act == "relu":
        return np.maximum(z, 0), (z >= 0).astype(np.float64)
    return z, np.ones_like(z)


class Oracle:
    """In 64 bits, arrays [n, c, h, w]."""

    def __init__(self, x, groups, gamma, beta, eps, act):
        n, c = x.shape[:2]
        self.grouped = (n, groups, -1)
        x = x.astype(np.float64)
        v = x.reshape(self.grouped)
        self.mean, var = v.mean(2), v.var(2)
        self.rstd = 1 / np.sqrt(var + eps)
        self.m = v.shape[2]
        self.r = self.of_values(self.rstd, x.shape)
        self.xh = (x - self.of_values(self.mean, x.shape)) * self.r
        col = lambda t, one: np.full((1, c, 1, 1), one) if t is None else t.astype(np.float64)[None, :, None, None]
        self.gamma, self.beta = col(gamma, 1.0), col(beta, 0.0)
        self.z = self.xh * self.gamma + self.beta
        self.y, self.slope = _f(self.z, act)
        size = self.of_values(np.abs(v).mean(2) + np.abs(self.mean), x.shape)
        self.unit_xh = np.abs(self.xh) + self.r * size
        self.unit = np.abs(self.gamma) * self.unit_xh + np.abs(self.beta) + np.abs(self.y)

    def of_values(self, t, shape):
        n, groups = t.shape
        return np.broadcast_to(t[:, :, None, None, None], (n, groups, shape[1] // groups, *shape[2:])).reshape(shape)

    def mean_of_group(self, t):
        return self.of_values(t.reshape(self.grouped).mean(2), t.shape)

    def backward(self, dy, act):
        """(dx, dgamma, dbeta) and what a rounding in each may be a part of."""
        dy = dy.astype(np.float64)
        dz = dy * self.slope
        # what xh is off shows in z, and there in the slope (of SiLU, at most half as steep)
        unit_dz = np.abs(dz) + (0.5 * np.abs(dy) * (np.abs(self.gamma) * self.unit_xh + np.abs(self.beta)) if act == "silu" else 0)
        w, unit_w = self.gamma * dz, np.abs(self.gamma) * unit_dz
        a, b = self.mean_of_group(w), self.mean_of_group(w * self.xh)
        dx = self.r * (w - a - self.xh * b)
        unit_b = self.mean_of_group(unit_w * self.unit_xh)
        unit = self.r * (unit_w + self.mean_of_group(unit_w) + self.unit_xh * unit_b)
        total = lambda t: t.sum((0, 2, 3))
        return (dx, total(dz * self.xh), total(dz)), (unit, total(unit_dz * self.unit_xh), total(unit_dz))


def _inputs(shape, groups, seed, act="silu", mean=0.5):
    rng = np.random.default_rng(seed)
    f32 = lambda *s: rng.standard_normal(s).astype(np.float32)
    x = (f32(*shape) * 2 + mean).astype(np.float32)
    gamma, beta = rng.uniform(0.5, 1.5, shape[1]).astype(np.float32), f32(shape[1]) * np.float32(0.3)
    return x, f32(*shape), gamma, beta


def _check_forward(got, o):
    assert (np.abs(got - o.y) <= STEPS * U * 1.1 * o.unit).all(), np.max(np.abs(got - o.y) / o.unit) / U


def _check_backward(got, o, dy, act):
    want, units = o.backward(dy, act)
    for name, g, w, u in zip(("dx", "dgamma", "dbeta"), got, want, units):
        assert (np.abs(g - w) <= 4 * STEPS * U * u).all(), (name, np.max(np.abs(g - w) / u) / U)


@pytest.mark.parametrize("act", [None, "relu", "silu"])
@pytest.mark.parametrize("n,c,h,w,groups", SHAPES)
def test_against_the_formulas(n, c, h, w, groups, act):
    import gpu_util as g
    import mytorch_b200.nn.functional as F

    x, dy, gamma, beta = _inputs((n, c, h, w), groups, n * 1000 + c + w, act)
    o = Oracle(x, groups, gamma, beta, 1e-5, act)
    if act == "relu":  # which side of zero a value is on cannot be told from 64 bits where it is this near
        dy = np.where(np.abs(o.z) > STEPS * U * o.unit, dy, 0).astype(np.float32)
    xt, gt, bt = g.dev(x, True), g.dev(gamma, True), g.dev(beta, True)
    y = F.group_norm(xt, groups, gt, bt, activation=act)
    assert y.requires_grad and y.shape == x.shape
    _check_forward(g.host(y), o)
    (y * g.dev(dy)).sum().backward()
    _check_backward([g.host(t.grad) for t in (xt, gt, bt)], o, dy, act)


@pytest.mark.parametrize("n,c,groups", [(7, 40, 5), (1, 6, 1), (300, 2050, 2), (2, 33, 33)])
def test_rows_without_positions(n, c, groups):
    import gpu_util as g
    import mytorch_b200.nn.functional as F

    x, dy, gamma, beta = _inputs((n, c, 1, 1), groups, c)
    o = Oracle(x, groups, gamma, beta, 1e-5, "silu")
    xt, gt, bt = g.dev(x.reshape(n, c), True), g.dev(gamma, True), g.dev(beta, True)
    y = F.group_norm(xt, groups, gt, bt, activation="silu")
    _check_forward(g.host(y).reshape(x.shape), o)
    (y * g.dev(dy.reshape(n, c))).sum().backward()
    _check_backward([g.host(xt.grad).reshape(x.shape), g.host(gt.grad), g.host(bt.grad)], o, dy, "silu")


@pytest.mark.parametrize("n,c,groups", [(65600, 1028, 1), (70001, 96, 4)])
def test_as_many_rows_as_tokens(n, c, groups):
    """More rows than a grid has blocks in y, of groups too wide for a block's lanes and of others."""
    import gpu_util as g
    import mytorch_b200.nn.functional as F

    x, dy, gamma, beta = _inputs((n, c, 1, 1), groups, c)
    xt, gt, bt = g.dev(x.reshape(n, c), True), g.dev(gamma, True), g.dev(beta, True)
    y = F.group_norm(xt, groups, gt, bt, activation="silu")
    (y * g.dev(dy.reshape(n, c))).sum().backward()
    y, dx = g.host(y).reshape(x.shape), g.host(xt.grad).reshape(x.shape)
    sums = np.zeros((4, c))
    for i in range(0, n, 8192):
        o = Oracle(x[i:i + 8192], groups, gamma, beta, 1e-5, "silu")
        _check_forward(y[i:i + 8192], o)
        want, units = o.backward(dy[i:i + 8192], "silu")
        assert (np.abs(dx[i:i + 8192] - want[0]) <= 4 * STEPS * U * units[0]).all()
        sums += np.stack([*want[1:], *units[1:]])
    for got, want, unit in zip((gt.grad, bt.grad), sums[:2], sums[2:]):
        assert (np.abs(g.host(got) - want) <= 4 * STEPS * U * unit).all()


@pytest.mark.parametrize("which", ["neither", "weight", "bias"])
@pytest.mark.parametrize("shape,groups", [((3, 24, 6, 5), 4), ((2, 15, 12, 12), 5)])
def test_without_weight_or_bias(shape, groups, which):
    import gpu_util as g
    import mytorch_b200.nn.functional as F

    x, dy, gamma, beta = _inputs(shape, groups, 5)
    gamma, beta = gamma if which == "weight" else None, beta if which == "bias" else None
    o = Oracle(x, groups, gamma, beta, 1e-3, "silu")
    xt, gt, bt = (None if a is None else g.dev(a, True) for a in (x, gamma, beta))
    y = F.group_norm(xt, groups, gt, bt, eps=1e-3, activation="silu")
    _check_forward(g.host(y), o)
    (y * g.dev(dy)).sum().backward()
    want, units = o.backward(dy, "silu")
    for t, w, u in zip((xt, gt, bt), want, units):
        if t is not None:
            assert (np.abs(g.host(t.grad) - w) <= 4 * STEPS * U * u).all()


@pytest.mark.parametrize("shape,groups", [((2, 32, 16, 16), 4), ((1, 10, 33, 7), 2), ((2, 64, 80, 80), 8)])
def test_a_mean_far_from_zero(shape, groups):
    """Values around 1000 with a deviation of 2: squares added up without the mean taken off would leave nothing of the variance."""
    import gpu_util as g
    import mytorch_b200.nn.functional as F

    x, _, gamma, beta = _inputs(shape, groups, 3, mean=1000.0)
    o = Oracle(x, groups, gamma, beta, 1e-5, None)
    got = g.host(F.group_norm(g.dev(x), groups, g.dev(gamma), g.dev(beta)))
    _check_forward(got, o)
    # the mean's own error moves all values of a group alike; the spread is right to a few units beside it
    spread = (got - beta[None, :, None, None]) / gamma[None, :, None, None]
    spread = spread.reshape(shape[0], groups, -1).std(2)
    assert np.abs(spread - 1).max() < 1e-3


def test_constant_groups_and_single_values():
    import gpu_util as g
    import mytorch_b200.nn.functional as F

    beta = np.array([0.5, -1.0, 2.0, 0.0], np.float32)
    for x, groups in ((np.full((2, 4, 8, 8), 3.0, np.float32), 2), (np.arange(8, dtype=np.float32).reshape(2, 4, 1, 1), 4)):
        xt = g.dev(x, True)
        y = F.group_norm(xt, groups, g.dev(np.ones(4, np.float32)), g.dev(beta))
        assert np.array_equal(g.host(y), np.broadcast_to(beta[None, :, None, None], x.shape))
        (y * g.dev(np.ones(x.shape, np.float32))).sum().backward()
        assert np.isfinite(g.host(xt.grad)).all() and np.abs(g.host(xt.grad)).max() < 1e-3


@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_a_bad_value_stays_in_its_group(bad):
    import gpu_util as g
    import mytorch_b200.nn.functional as F

    x, _, gamma, beta = _inputs((3, 16, 9, 9), 4, 11)
    clean = g.host(F.group_norm(g.dev(x), 4, g.dev(gamma), g.dev(beta), activation="silu"))
    x[1, 6, 3, 4] = bad
    got = g.host(F.group_norm(g.dev(x), 4, g.dev(gamma), g.dev(beta), activation="silu"))
    assert np.isnan(got[1, 4:8]).all()
    got[1, 4:8] = clean[1, 4:8]
    assert np.array_equal(got, clean)


def test_very_negative_and_positive_values_of_silu():
    import gpu_util as g
    import mytorch_b200.nn.functional as F

    x = np.array([[-1.0, 1.0]], np.float32).reshape(1, 2, 1, 1)
    for factor in (100.0, 1e4, 3e38):
        gamma = np.full(2, factor, np.float32)
        xt = g.dev(x, True)
        y = F.group_norm(xt, 1, g.dev(gamma), None, activation="silu")
        got = g.host(y).reshape(2)
        assert abs(got[0]) < 1e-30 and abs(got[1] / factor - 1) < 1e-4
        (y * g.dev(np.ones(x.shape, np.float32))).sum().backward()
        assert not np.isnan(g.host(xt.grad)).any()


@pytest.mark.parametrize("offsets", [(1, 0), (0, 2), (3, 3)])
@pytest.mark.parametrize("shape,groups", [((2, 32, 9, 9), 4), ((1, 128, 30, 30), 4), ((2, 20, 50, 50), 2)])
def test_windows_at_any_float(shape, groups, offsets):
    import gpu_util as g
    import mytorch_b200 as mt
    from mytorch_b200.backends.cuda.env import CudaMemory, CudaMemoryView

    def window(array, offset):
        view = CudaMemoryView(CudaMemory(0, 4 * (array.size + 4)), 4 * offset, 4 * array.size, 0)
        view.write(np.ascontiguousarray(array.transpose(0, 2, 3, 1)))
        return mt.Tensor._on_device(array.shape, mt.float32, mt.Device("cuda:0"), view)

    x, dy, gamma, beta = _inputs(shape, groups, 21)
    o = Oracle(x, groups, gamma, beta, 1e-5, "silu")
    xt, dyt, gt, bt = window(x, offsets[0]), window(dy, offsets[1]), g.dev(gamma), g.dev(beta)
    y, mean, rstd = g.op("group_norm")(xt, groups, gt, bt, 1e-5, "silu")
    _check_forward(g.host(y), o)
    assert np.allclose(g.host(mean), o.mean, rtol=0, atol=STEPS * U * 3) and np.allclose(g.host(rstd), o.rstd, rtol=STEPS * U)
    _check_backward([g.host(t) for t in g.op("group_norm_backward")(dyt, mean, rstd, xt, gt, bt, groups, "silu")], o, dy, "silu")


@pytest.mark.parametrize("shape,groups", [((2, 32, 9, 9), 4), ((1, 30, 50, 50), 3), ((70, 64, 28, 28), 32), ((2, 64, 200, 200), 2)])
def test_the_same_bits_every_time(shape, groups):
    import gpu_util as g

    x, dy, gamma, beta = _inputs(shape, groups, 2)
    xt, dyt, gt, bt = (g.dev(a) for a in (x, dy, gamma, beta))
    first = None
    for _ in range(3):
        y, mean, rstd = g.op("group_norm")(xt, groups, gt, bt, 1e-5, "silu")
        got = [g.host(t) for t in (y, mean, rstd, *g.op("group_norm_backward")(dyt, mean, rstd, xt, gt, bt, groups, "silu"))]
        first = first or got
        assert all(np.array_equal(a, b) for a, b in zip(first, got))


def test_only_what_is_asked_for():
    import gpu_util as g

    x, dy, gamma, beta = _inputs((4, 64, 12, 12), 8, 9)
    xt, dyt, gt, bt = (g.dev(a) for a in (x, dy, gamma, beta))
    _, mean, rstd = g.op("group_norm")(xt, 8, gt, bt, 1e-5, "silu")
    args = (dyt, mean, rstd, xt, gt, bt, 8, "silu")
    whole = [g.host(t) for t in g.op("group_norm_backward")(*args)]
    for needed in ((True, False, False), (False, True, True), (False, False, True), (False, True, False)):
        part = g.op("group_norm_backward")(*args, needed)
        for want, t, asked in zip(whole, part, needed):
            assert (t is not None) == asked and (t is None or np.array_equal(g.host(t), want))


@pytest.mark.parametrize("n,h,w", [(0, 4, 4), (2, 0, 4), (2, 4, 0)])
def test_nothing(n, h, w):
    import gpu_util as g
    import mytorch_b200 as mt

    x = mt.Tensor(shape=(n, 8, h, w), dtype=mt.float32, device="cuda:0")
    gamma = g.dev(np.ones(8, np.float32))
    y, mean, rstd = g.op("group_norm")(x, 2, gamma, gamma, 1e-5, None)
    dx, dg, db = g.op("group_norm_backward")(x, mean, rstd, x, gamma, gamma, 2, None)
    assert y.shape == dx.shape == x.shape and not g.host(dg).any() and not g.host(db).any()


@pytest.mark.parametrize("act", [None, "silu"])
@pytest.mark.parametrize("shape,groups", [((2, 12, 7, 5), 3), ((1, 64, 20, 20), 16)])
def test_gradients_against_differences(shape, groups, act):
    """The slope of sum(y dy) along a direction, from two evaluations in 64 bits: differences of step h are off by h^2 and by rounding / h."""
    import gpu_util as g
    import mytorch_b200.nn.functional as F

    x, dy, gamma, beta = _inputs(shape, groups, 17)
    rng = np.random.default_rng(18)
    xt, gt, bt = g.dev(x, True), g.dev(gamma, True), g.dev(beta, True)
    (F.group_norm(xt, groups, gt, bt, activation=act) * g.dev(dy)).sum().backward()
    for t, values in ((xt, x), (gt, gamma), (bt, beta)):
        d = rng.standard_normal(values.shape)
        at = lambda s: (Oracle(*[(v.astype(np.float64) + s * d if v is values else v.astype(np.float64)) for v in (x,)], groups,
                               *[v.astype(np.float64) + (s * d if v is values else 0) for v in (gamma, beta)], 1e-5, act).y * dy).sum()
        h = 1e-4
        want, got = (at(h) - at(-h)) / (2 * h), float((g.host(t.grad).astype(np.float64) * d).sum())
        assert abs(want - got) <= 1e-5 * float(np.abs(g.host(t.grad).astype(np.float64) * d).sum()) + 1e-6


def test_the_layer_trains():
    import gpu_util as g
    import mytorch_b200 as mt
    import mytorch_b200.nn as nn

    x, dy, _, _ = _inputs((4, 16, 6, 6), 4, 31)
    layer = nn.GroupNorm(4, 16, activation="relu")
    layer.to("cuda:0")
    assert [k for k, _ in layer.named_parameters()] == ["weight", "bias"]
    o = Oracle(x, 4, np.ones(16, np.float32), np.zeros(16, np.float32), 1e-5, "relu")
    y = layer(g.dev(x))
    _check_forward(g.host(y), o)
    (y * g.dev(dy)).sum().backward()
    assert layer.weight.grad.shape == layer.bias.grad.shape == (16,)
    with mt.no_grad():
        assert not layer(g.dev(x)).requires_grad
    assert np.array_equal(g.host(layer.eval()(g.dev(x))), g.host(y))
    assert list(nn.GroupNorm(2, 4, affine=False).parameters()) == []
