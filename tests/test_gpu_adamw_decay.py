"""AdamW's weight decay of a millionth and less a step: what a parameter loses is right on average over many of them, though each is rounded to float32.

The mean of (p' - exact p') sign(p) over n values, relative to that of |p|.  Each rounding of the result is off by at most 2^-24 |p| and, as the steps' sizes are spread over many of its
last places, evenly: 8 standard deviations of a mean are 8 * 2^-24 / sqrt(3 n).  The steps' own roundings have the sign of the step, as often that of p as not: under 2^-20 of a step each,
the mean's share of them 8 * 2^-20 lr / sqrt(n).  The decay as a float32 and its product: 2^-23 of it."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("lr", [1e-4, 1e-5, 2e-6])
def test_small_decays_are_not_rounded_away(bits, offset, lr):
    import gpu_util as g
    from mytorch_b200.optim import AdamW
    from test_gpu_adamw import _window

    n, wd, eps, b1, b2 = 1 << 22, 0.01, 1.0, 0.5, 0.75
    rng = np.random.default_rng(7)
    p0 = (rng.uniform(1, 2, n) * rng.choice([-1, 1], n)).astype(np.float32)
    grad = rng.standard_normal(n).astype(np.float32)
    p = _window(p0, offset)
    p.requires_grad, p.grad = True, _window(grad, offset)
    AdamW([p], lr=lr, betas=(b1, b2), eps=eps, weight_decay=wd, state_bits=bits).step()
    g64, p64 = grad.astype(np.float64), p0.astype(np.float64)
    exact = p64 * (1 - lr * wd) - lr * g64 / (np.abs(g64) + eps)  # the first step: both corrections undo the moments' weights
    mean = ((g.host(p) - exact) * np.sign(p64)).mean() / np.abs(p64).mean()
    assert abs(mean) <= 8 * (2.0 ** -24 / np.sqrt(3 * n) + 2.0 ** -20 * lr / np.sqrt(n)) + 2.0 ** -23 * lr * wd


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("wd", [0.0, 0.1])
@pytest.mark.parametrize("eps", [1e-8, 1e-12])
def test_an_infinite_parameter_stays(bits, offset, wd, eps):
    """p (1 - lr wd) - step is infinite where p is, and no number where p is none."""
    import gpu_util as g
    from mytorch_b200.optim import AdamW
    from test_gpu_adamw import _window

    p0 = np.random.default_rng(3).standard_normal(2500).astype(np.float32)
    p0[7::50], p0[8::50], p0[9::50], p0[10::50] = np.inf, -np.inf, np.nan, np.finfo(np.float32).max
    grad = np.random.default_rng(4).standard_normal(2500).astype(np.float32)
    grad[::3] = 0
    p = _window(p0, offset)
    p.requires_grad, p.grad = True, _window(grad, offset)
    opt = AdamW([p], lr=0.01, weight_decay=wd, eps=eps, state_bits=bits)
    for _ in range(2):
        opt.step()
    got = g.host(p)
    assert np.array_equal(np.isnan(got), np.isnan(p0))
    infinite = np.isinf(p0)
    assert np.array_equal(got[infinite], p0[infinite]) and np.isfinite(got[~infinite & ~np.isnan(p0)]).all()
