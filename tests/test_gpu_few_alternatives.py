"""token_log_probs of rows that have fewer values than alternatives are asked for, of which the others are all alike: by every kernel, the same every time."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rest", [-np.inf, np.finfo(np.float32).min, 0.0], ids=["masked", "lowest", "ties"])
@pytest.mark.parametrize("n,v", [(2000, 700), (2000, 3001), (1500, 20001), (4000, 40000), (700, 5003), (100, 10007), (40, 33000), (3, 131077)])
def test_first_places_of_what_is_alike(n, v, rest):
    import gpu_util as g
    import mytorch_b200.nn.functional as F

    rng = np.random.default_rng(n + v)
    z = np.full((n, v), rest, np.float32)
    left = rng.integers(0, 4, n)  # rows of nothing else, too
    want = np.empty((n, 32), np.int64)
    for i in range(n):
        places = rng.permutation(v)[: left[i]]
        z[i, places] = np.arange(left[i], 0, -1)
        others = np.setdiff1d(np.arange(32 + left[i]), places)
        want[i] = np.concatenate([places, others])[:32]
    x, tokens = g.dev(z), g.dev(np.zeros(n, np.int64))
    first = None
    for _ in range(6):
        out = F.token_log_probs(x, tokens, 32)
        assert np.array_equal(g.host(out.top_tokens), want)
        values = [g.host(t) for t in out[:3]]
        first = first or values
        assert all(np.array_equal(a, b, equal_nan=True) for a, b in zip(values, first))
