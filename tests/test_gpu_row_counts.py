"""token_log_probs on both sides of the row counts at which other kernels take over: by clusters of 8, 4 and 2 CTAs, by one, by eight, four and one warps."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,v", [(n, v) for v in (16389, 33001, 65537) for n in (60, 87, 111, 112, 172, 185, 222, 223, 370, 371, 444, 445)]
                         + [(n, v) for v in (1024, 1025, 2048, 2049, 4096, 4097) for n in (1184, 1185, 3699, 3700)] + [(1184, 28001), (1185, 28000), (3700, 28001), (3700, 56001)])
def test_on_both_sides(n, v):
    import gpu_util as g
    import mytorch_b200.nn.functional as F
    from test_gpu_token_log_probs import U, _check, _logits, _reference

    top = 5
    part = _logits("normal", min(n, 64), v, n + v)  # the same rows again and again
    z = np.resize(part, (n, v))
    tokens = np.random.default_rng(v).integers(0, v, n)
    got = F.token_log_probs(g.dev(z), g.dev(tokens), top)
    want = {k: np.concatenate([t] * (n // len(part) + 1))[:n] if isinstance(t, np.ndarray) and len(t) == len(part) else t
            for k, t in _reference(part, tokens[: len(part)], top, None).items()}
    _check(g.host(got.entropy), want["entropy"], want["tol_h"], "entropy")
    assert np.array_equal(g.host(got.top_tokens), want["top_tokens"])
    _check(g.host(got.top_log_probs), want["top_log_probs"], want["tol"][:, None] + 3 * U * np.abs(want["top_log_probs"]), "top")
    given = want["log_p"][np.arange(n), tokens]
    _check(g.host(got.log_probs), given, want["tol"] + 3 * U * np.abs(given), "log_probs")
