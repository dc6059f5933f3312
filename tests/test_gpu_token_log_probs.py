"""Log probabilities of given tokens, entropy and alternatives, and their gradient, against 64 bits.

Tolerances, u = 2^-24: z - m is off by u |d|; exp by that of its argument and 2^-22 of itself (two units in the last place); sums by u times the additions that one value
goes through, at most v / 32 + 32 in a row of a warp, v / 256 + 32 above 1024 values; log S by the sum's error and its own 2 units; what is added up behind them by u of
each term.  Weighted by the probabilities |d| is at most the entropy's T / S."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.fixture(autouse=True, scope="module")
def blocks_of_these_sizes_go_back_to_the_driver():
    """A later module's test of the memory pool counts on sizes that no earlier one left there."""
    yield
    from mytorch_b200.backends.cuda.env import CudaEnv

    CudaEnv.instance().lib.pool_trim()


def _chain(v):
    return (v / 32 if v <= 1024 else v / 256) + 32


def _reference(z, tokens, top, ignore_index):
    """Dict of what forward gives, its tolerances, and what backward needs."""
    z = z.astype(np.float64)
    n, v = z.shape
    with np.errstate(all="ignore"):
        m = z.max(1, keepdims=True)
        d = z - m
        e = np.exp(d)
        s = e.sum(1, keepdims=True)
        log_p = d - np.log(s)
        p = e / s
        weighted = np.where(p == 0, 0.0, p * d).sum(1)
        h = np.log(s[:, 0]) - weighted
        known = tokens != ignore_index if ignore_index is not None else np.ones(n, bool)
        inside = (tokens >= 0) & (tokens < v)
        given = np.where(inside, log_p[np.arange(n), np.where(inside, tokens, 0)], np.nan)
        order = np.argsort(np.where(np.isnan(z), -np.inf, -z), axis=1, kind="stable")[:, :top]
        common = U * (_chain(v) + 8 + np.abs(weighted) + 3 * np.log(s[:, 0]))
        return {"log_probs": np.where(known, given, 0.0), "entropy": h, "top_log_probs": np.take_along_axis(log_p, order, 1), "top_tokens": order, "p": p, "log_p": log_p,
                "d": d, "tol": common, "tol_h": common + U * (2 * _chain(v) + 8) * np.abs(weighted) + 2 * U * h, "known": known, "log_s": np.log(s[:, 0])}


def _check(got, want, tol, name):
    got, want, tol = np.broadcast_arrays(np.asarray(got, np.float64), want, tol)
    assert np.array_equal(np.isnan(got), np.isnan(want)), name
    fine = np.isfinite(want)
    tol = np.where(np.isnan(tol), 1e-300, tol)  # a value beside NaN, like that of a row without a token: equal
    assert np.array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)]), name
    off = np.abs(got[fine] - want[fine]) / tol[fine]
    assert not off.size or off.max() <= 1, (name, off.max())


def _logits(kind, n, v, seed):
    rng = np.random.default_rng(seed)
    z = (2 * rng.standard_normal((n, v))).astype(np.float32)
    if kind == "ties":
        z = np.round(z).astype(np.float32)
        z[:, ::3] *= 0  # zeros of both signs
        z[:, ::6] *= -1
    elif kind == "masked":  # rows with few tokens left, some with none
        z[rng.random((n, v)) < 0.9] = -np.inf
        z[::3] = -np.inf
        z[::3, v // 2] = 1.5
        z[4::5] = -np.inf
    elif kind == "lowest":  # masks of the type's lowest value, some rows of nothing else
        z[rng.random((n, v)) < 0.7] = np.finfo(np.float32).min
        z[2::3] = np.finfo(np.float32).min
    elif kind == "nan":
        z[1::2, v // 3] = np.nan
        z[2::4, v - 1] = np.inf
    elif kind == "ascending":
        z = np.sort(z, axis=1)
    elif kind == "peaked":
        z[:, v // 2] += 60
    elif kind == "large":
        z *= 3e4
    return z


CASES = [(n, v, top) for n, v, top in ((1, 1, 1), (1, 2, 2), (3, 5, 0), (7, 31, 4), (5, 32, 32), (4, 33, 32), (9, 127, 20), (2, 129, 1), (33, 1000, 5), (2, 1023, 8), (3, 1025, 31), (5, 4096, 16),
                                       (6, 5003, 7), (150, 2050, 20), (1, 8193, 20), (1, 50000, 32), (2, 131072, 20), (1, 262147, 11), (1300, 300, 3), (40, 20001, 2))]


@pytest.mark.parametrize("kind", ["normal", "ties", "masked", "lowest", "nan", "ascending", "peaked", "large"])
@pytest.mark.parametrize("n,v,top", CASES)
def test_forward(n, v, top, kind):
    import gpu_util as g
    import mytorch_b200.nn.functional as F

    z = _logits(kind, n, v, n * v)
    rng = np.random.default_rng(1)
    tokens = rng.integers(0, v, n).astype([np.int32, np.int64][v % 2])
    tokens[3::4], tokens[2::7] = -100, v
    got = F.token_log_probs(g.dev(z), g.dev(tokens), top, -100)
    want = _reference(z, tokens, top, -100)
    _check(g.host(got.log_probs), want["log_probs"], want["tol"] + 3 * U * np.abs(np.nan_to_num(want["log_probs"], posinf=0, neginf=0)), "log_probs")
    _check(g.host(got.entropy), want["entropy"], want["tol_h"], "entropy")
    if not top:
        assert got.top_tokens is None and got.top_log_probs is None
        return
    assert got.top_tokens.shape == got.top_log_probs.shape == (n, top)
    assert np.array_equal(g.host(got.top_tokens), want["top_tokens"])
    _check(g.host(got.top_log_probs), want["top_log_probs"], want["tol"][:, None] + 3 * U * np.abs(np.nan_to_num(want["top_log_probs"], posinf=0, neginf=0)), "top")


def _gradient(ref, tokens, g, gh, gt, top_tokens):
    """(gradient, tolerance)"""
    p, log_p, n = ref["p"], ref["log_p"], len(tokens)
    rows = np.arange(n)
    g = np.where(ref["known"], g, 0.0)
    inside = (tokens >= 0) & (tokens < p.shape[1])
    with np.errstate(all="ignore"):
        inner = np.where(p == 0, 0.0, log_p + ref["entropy"][:, None])
        dz = -p * (g + gt.sum(1))[:, None] - gh[:, None] * p * inner
        d = np.abs(np.where(p == 0, 0.0, ref["d"]))
        weight = p * (np.abs(g) + np.abs(gt).sum(1))[:, None] + np.abs(gh)[:, None] * p * np.abs(inner)
        tol = U * ((d + 24 + gt.shape[1]) * weight + p * np.abs(gh)[:, None] * (2 * d + 3 * ref["log_s"][:, None] + 3 * np.abs(ref["entropy"])[:, None] + 8)) + 1e-37
    dz[rows[inside], tokens[inside]] += g[inside]
    tol[rows[inside], tokens[inside]] += 3 * U * np.abs(g[inside])
    for k in range(gt.shape[1]):
        dz[rows, top_tokens[:, k]] += gt[:, k]
        tol[rows, top_tokens[:, k]] += 3 * U * np.abs(gt[:, k])
    return dz, tol + U * np.abs(dz)


@pytest.mark.parametrize("kind", ["normal", "ties", "masked", "lowest", "peaked"])
@pytest.mark.parametrize("n,v,top", CASES)
def test_backward(n, v, top, kind):
    import gpu_util as g
    import mytorch_b200.nn.functional as F

    z = _logits(kind, n, v, n + v)
    rng = np.random.default_rng(2)
    tokens = rng.integers(0, v, n).astype([np.int64, np.int32][v % 2])
    tokens[3::4] = -100
    alive = np.isfinite(z.max(1))  # a row of -inf only has no gradient but NaN
    x = g.dev(z, True)
    out = F.token_log_probs(x, g.dev(tokens), top, ignore_index=-100)
    ref = _reference(z, tokens, top, -100)
    grads = [rng.standard_normal(n).astype(np.float32), rng.standard_normal(n).astype(np.float32), rng.standard_normal((n, top)).astype(np.float32)]
    helpers = out.log_probs._grad_node.helpers
    for used in ((1, 1, 1), (1, 0, 0), (0, 1, 0), (0, 0, 1)):
        if not top and used == (0, 0, 1):
            continue
        given = [g.dev(a) if u and a.size else None for a, u in zip(grads, used)]
        got = g.host(g.op("token_log_probs_backward")(*given, *helpers, x, g.dev(tokens), -100)[0])
        values = [a * u for a, u in zip(grads, used)]
        want, tol = _gradient(ref, tokens, *values, ref["top_tokens"])
        off = np.abs(got[alive] - want[alive]) / tol[alive]
        assert not off.size or off.max() <= 1, (used, off.max())
        assert not np.isfinite(got[~alive]).any() or used == (0, 0, 0) or (~alive).sum() == 0 or _only_ignored(got[~alive], tokens[~alive], used)


def _only_ignored(got, tokens, used):
    """A row of -inf whose gradients are all zero may be zero."""
    return all(not np.isfinite(row).any() or (t == -100 and used == (1, 0, 0)) for row, t in zip(got, tokens))


def test_gradient_against_differences():
    """(f(z + e) - f(z - e)) / 2e in 64 bits of f = sum of w log_probs + q entropy + r top: the formula's error is e^2 / 6 times a third derivative, under 1e-7 here."""
    import gpu_util as g
    import mytorch_b200.nn.functional as F

    rng = np.random.default_rng(3)
    n, v, top = 4, 37, 3
    z = rng.standard_normal((n, v)).astype(np.float32)
    tokens = rng.integers(0, v, n)
    w, q, r = (rng.standard_normal(s).astype(np.float32) for s in ((n,), (n,), (n, top)))
    x = g.dev(z, True)
    out = F.token_log_probs(x, g.dev(tokens), top)
    loss = (out.log_probs * g.dev(w)).sum() + (out.entropy * g.dev(q)).sum() + (out.top_log_probs * g.dev(r)).sum()
    loss.backward()

    def f(a):
        ref = _reference(a, tokens, top, None)
        return (ref["log_probs"] * w).sum() + (ref["entropy"] * q).sum() + (ref["top_log_probs"] * r).sum()

    got, e = g.host(x.grad), 1e-4
    for i in range(n):
        for j in range(v):
            up, down = z.astype(np.float64), z.astype(np.float64)
            up[i, j] += e
            down[i, j] -= e
            assert abs((f(up) - f(down)) / (2 * e) - got[i, j]) <= 1e-5


def test_rows_without_a_token():
    """Tokens outside the row have log probability NaN, ignored ones 0; neither has a gradient from it, nor does a token that cannot be have one elsewhere than by p."""
    import gpu_util as g
    import mytorch_b200.nn.functional as F

    for v in (9, 2000, 40000):
        z = np.zeros((6, v), np.float32)
        z[5, 0] = -np.inf
        tokens = np.array([0, -1, v, -100, 2 ** 40, 0])
        x = g.dev(z, True)
        out = F.token_log_probs(x, g.dev(tokens), ignore_index=-100)
        got = g.host(out.log_probs)
        assert np.isfinite(got[0]) and np.isnan(got[[1, 2, 4]]).all() and got[3] == 0 and got[5] == -np.inf
        ones = g.dev(np.ones(6, np.float32))
        node = out.log_probs._grad_node
        dz = g.host(g.op("token_log_probs_backward")(ones, None, None, *node.helpers, x, g.dev(tokens), -100)[0])
        assert not dz[1:5].any() and abs(dz[0, 0] - (1 - 1 / v)) <= 1e-6 and abs(dz[5, 0] - 1) <= 1e-6 and abs(dz[5, 1] + 1 / (v - 1)) <= 1e-6


def test_shapes_strides_and_windows():
    """[B, L, V] like its rows, no rows at all, and logits that begin at any float."""
    import gpu_util as g
    import mytorch_b200 as mt
    import mytorch_b200.nn.functional as F
    from mytorch_b200.backends.cuda.env import CudaMemory, CudaMemoryView

    rng = np.random.default_rng(4)
    for v in (260, 3001, 40004):
        z, tokens = rng.standard_normal((2, 3, v)).astype(np.float32), rng.integers(0, v, (2, 3))
        got = F.token_log_probs(g.dev(z), g.dev(tokens), 4)
        flat = F.token_log_probs(g.dev(z.reshape(6, v)), g.dev(tokens.reshape(6)), 4)
        assert got.log_probs.shape == (2, 3) and got.top_tokens.shape == (2, 3, 4) and got.top_tokens.dtype is mt.int64
        for a, b in zip(got, flat):
            assert np.array_equal(g.host(a).reshape(-1), g.host(b).reshape(-1))
        ref = _reference(z.reshape(6, v), tokens.reshape(6), 4, None)
        for offset in (1, 2, 3):
            view = CudaMemoryView(CudaMemory(0, 4 * (z.size + 4)), 4 * offset, 4 * z.size, 0)
            view.write(z)
            x = mt.Tensor._on_device((6, v), mt.float32, got.log_probs.device, view)
            x.requires_grad = True
            off = F.token_log_probs(x, g.dev(tokens.reshape(6)), 4)
            _check(g.host(off.log_probs), ref["log_probs"], ref["tol"] + 3 * U * np.abs(ref["log_probs"]), "window")
            assert np.array_equal(g.host(off.top_tokens), ref["top_tokens"])
            (off.log_probs + off.entropy).sum().backward()
            one = np.ones(6)
            want, tol = _gradient(ref, tokens.reshape(6), one, one, np.zeros((6, 0)), ref["top_tokens"])
            assert (np.abs(g.host(x.grad) - want) <= tol).all()
    got = F.token_log_probs(g.dev(np.zeros((0, 5), np.float32)), g.dev(np.zeros(0, np.int64)), 2)
    assert got.log_probs.shape == (0,) and got.top_tokens.shape == (0, 2)


def test_rows_past_32_bits():
    """A row whose first value lies more than 2^31 values into the logits, forward and backward: the same as by itself."""
    import gpu_util as g
    import mytorch_b200 as mt
    import mytorch_b200.nn.functional as F
    from mytorch_b200.backends.cuda.env import CudaEnv, CudaMemoryView

    n, v = 5, (1 << 29) + 12345
    x = mt.Tensor(shape=(n, v), dtype=mt.float32, device="cuda:0", requires_grad=True)
    x.fill_(-20.0)
    rng = np.random.default_rng(5)
    peak = rng.standard_normal(7).astype(np.float32)
    at = 4 * ((n - 1) * v + v - 1000)
    CudaMemoryView(x._native_array, at, peak.nbytes, 0).write(peak)
    tokens = np.array([0, 0, 0, 0, v - 998])
    out = F.token_log_probs(x, g.dev(tokens), 3)
    others = (v - 7) * np.exp(-20.0)
    log_s = np.log(np.exp(peak.astype(np.float64)).sum() + others)
    # the sum of equal values in 32 bits: 2^29 additions by at most 2^18 threads
    assert abs(g.host(out.log_probs)[4] - (peak[2] - log_s)) <= U * 4096
    assert np.array_equal(g.host(out.top_tokens)[4], v - 1000 + np.argsort(-peak, kind="stable")[:3]) and np.array_equal(g.host(out.top_tokens)[0], [0, 1, 2])
    out.log_probs.sum().backward()
    got = CudaMemoryView(x.grad._native_array, at, peak.nbytes, 0).read((7,), np.float32)
    want = (np.arange(7) == 2) - np.exp(peak.astype(np.float64) - log_s)
    assert np.abs(got - want).max() <= U * 8192
    del out, x
    CudaEnv.instance().lib.pool_trim()


def test_captured_and_replayed():
    """Two graphs over the same leaves, replayed in turn with other logits, give the bits of calls outside."""
    import gpu_util as g
    import mytorch_b200 as mt
    import mytorch_b200.nn.functional as F
    from mytorch_b200.cuda_graph import StepGraph

    rng = np.random.default_rng(6)
    n, v = 37, 5003
    x, tokens = g.dev(rng.standard_normal((n, v)).astype(np.float32), True), g.dev(rng.integers(0, v, n))

    def step():
        x.grad = None
        out = F.token_log_probs(x, tokens, 6)
        (out.log_probs - out.entropy).sum().backward()
        return out, x.grad

    step()
    graphs = [StepGraph(step), StepGraph(step)]
    results = [gr.capture() for gr in graphs]
    for turn in range(4):
        z = rng.standard_normal((n, v)).astype(np.float32)
        x._native_array.write(z)
        graphs[turn % 2].replay()
        out, grad = results[turn % 2]
        got = [g.host(t) for t in (*out, grad)]
        y = g.dev(z, True)
        want = F.token_log_probs(y, tokens, 6)
        (want.log_probs - want.entropy).sum().backward()
        assert all(np.array_equal(a, g.host(b)) for a, b in zip(got, (*want, y.grad)))
    for gr in graphs:
        gr.destroy()
