"""token_log_probs: a row that no gradient reaches has gradient zero, whatever its logits; what reaches a row that is NaN leaves NaN."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,v", [(9, 5), (30, 700), (1300, 3001), (30, 3001), (30, 10007), (12, 40001)])
@pytest.mark.parametrize("top", [0, 3])
def test_ignored_rows_that_are_nan(n, v, top):
    import gpu_util as g
    import mytorch_b200.nn.functional as F

    rng = np.random.default_rng(n + v)
    z = rng.standard_normal((n, v)).astype(np.float32)
    z[0::6] = -np.inf
    z[1::6, v // 2] = np.nan
    z[2::6, v - 1] = np.inf
    dead = np.arange(n) % 6 < 3
    tokens = rng.integers(0, v, n)
    tokens[::2] = -100  # ignored: of each kind
    tokens[1::8] = v  # outside
    silent = (tokens == -100) | (tokens == v)
    op = g.op("token_log_probs_backward")

    x, t = g.dev(z, True), g.dev(tokens)
    out = F.token_log_probs(x, t, top, ignore_index=-100)
    stats, top_tokens = out.log_probs._grad_node.helpers
    out.log_probs.sum().backward()
    got = g.host(x.grad)
    assert not got[silent].any() and not np.isnan(got[silent]).any()
    assert not np.isfinite(got[dead & ~silent]).any() and np.isfinite(got[~dead]).all()

    # of the entropy and the alternatives too, in the rows that they are asked of
    asked = np.arange(n) % 5 == 0
    dentropy = g.dev(asked.astype(np.float32))
    got = g.host(op(None, dentropy, None, stats, top_tokens, x, t, -100)[0])
    assert not got[~asked].any() and not np.isfinite(got[asked & dead]).any() and np.isfinite(got[asked & ~dead]).all()
    if top:
        dtop = np.zeros((n, top), np.float32)
        dtop[asked] = 1, 0, -1  # what cancels is a gradient
        got = g.host(op(None, g.dev(np.zeros(n, np.float32)), g.dev(dtop), stats, top_tokens, x, t, -100)[0])
        assert not got[~asked].any() and not np.isnan(got[~asked]).any()
        assert not np.isfinite(got[asked & dead]).any() and (got[asked & ~dead] != 0).sum() == 2 * (asked & ~dead).sum()
