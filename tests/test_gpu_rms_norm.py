"""RMS norm, the norms around a residual block with its gate, and their gradients, against 64 bits.

Tolerances, u = 2^-24: a sum over a row is off by u times the additions that one value goes through, at most c / 32 + 16; half of that in a reciprocal root, and 4 for
square, division, root and rounding; a product by u of itself for every factor.  What is subtracted is bounded by the sum of its terms' sizes.  Sums over rows go through
at most rows + 16 additions in 32 bits."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
EPS = 1e-6


@pytest.fixture(autouse=True, scope="module")
def blocks_of_these_sizes_go_back_to_the_driver():
    """A later module's test of the memory pool counts on sizes that no earlier one left there."""
    yield
    from mytorch_b200.backends.cuda.env import CudaEnv

    CudaEnv.instance().lib.pool_trim()


def _inputs(shape, post, gate, seed=0, scale=1.0):
    """shape: as the tensors have it; everything else [rows, c]."""
    rng = np.random.default_rng(seed)
    c = shape[1] if len(shape) == 4 else shape[-1]
    f32 = lambda *s: (scale * rng.standard_normal(s)).astype(np.float32)
    a = {"residual": f32(*shape) + np.float32(0.3), "block": f32(*shape), "weight": f32(c) + np.float32(1)}
    if post:
        a["post_weight"] = f32(c) + np.float32(1)
    if gate:
        a["gate"] = f32(*{"channel": (c,), "sample": (shape[0], c), "full": shape}[gate])
    a["dnew"], a["dy"] = f32(*shape), f32(*shape)
    return a


def _rows(a, c):
    """[rows, c] in 64 bits of a tensor of 2 to 4 dimensions."""
    a = a.astype(np.float64)
    return (a.transpose(0, 2, 3, 1) if a.ndim == 4 else a).reshape(-1, c)


def _gate_rows(a, shape, c, gate):
    if not gate:
        return np.ones((1, c))
    g = a["gate"].astype(np.float64)
    rows = int(np.prod(shape)) // c
    return g[None, :] if gate == "channel" else np.repeat(g, rows // shape[0], axis=0) if gate == "sample" else _rows(a["gate"], c)


def _forward(a, shape, post, gate, scale):
    c = shape[1] if len(shape) == 4 else shape[-1]
    k = c / 64 + 12
    b = _rows(a["block"], c)
    rb = 1 / np.sqrt((b * b).mean(1, keepdims=True) + EPS) if post else np.ones((len(b), 1))
    hat = b * rb
    inner = hat * (a["post_weight"].astype(np.float64) if post else 1)
    gr = _gate_rows(a, shape, c, gate)
    x = _rows(a["residual"], c)
    new = scale * x + gr * inner
    tol_new = U * (3 * np.abs(scale * x) + (k + 4) * np.abs(gr * inner))
    rho = 1 / np.sqrt((new * new).mean(1, keepdims=True) + EPS)
    w = a["weight"].astype(np.float64)
    # the mean's relative error from that of the values is at most twice their largest error against the root mean square
    tol_y = np.abs(w) * rho * tol_new + np.abs(new * rho * w) * (U * (k + 4) + (rho * np.sqrt((tol_new ** 2).mean(1, keepdims=True))))
    return {"c": c, "k": k, "hat": hat, "inner": inner, "gate": gr, "new": new, "rho": rho, "rb": rb, "w": w, "y": new * rho * w, "tol_new": tol_new, "tol_y": tol_y}


SHAPES = [(1, 1), (1, 8), (3, 5), (2, 33), (1, 1024), (7, 128), (5, 130), (64, 96), (300, 64), (3, 750), (2, 5, 36), (4, 37, 257), (1, 4096), (3, 4099), (2, 8192), (2, 3, 11111), (1, 16384),
          (5, 12, 3, 4), (2, 130, 5, 7), (1, 1, 1), (40, 50, 512), (1200, 2048), (2, 20000)]


@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("gate", [None, "channel", "sample", "full"])
@pytest.mark.parametrize("shape", SHAPES)
def test_forward(shape, gate, post):
    import gpu_util as g
    import mytorch_b200.nn.functional as F

    a = _inputs(shape, post, gate)
    scale = [1.0, 0.5][shape[0] % 2]
    t = {k: g.dev(v) for k, v in a.items()}
    new, y = F.add_rms_norm(t["residual"], t["block"], t["weight"], t.get("post_weight"), t.get("gate"), scale, EPS)
    want = _forward(a, shape, post, gate, scale)
    assert new.shape == y.shape == shape
    got_new, got_y = _rows(g.host(new), want["c"]), _rows(g.host(y), want["c"])
    assert (np.abs(got_new - want["new"]) <= want["tol_new"]).all()
    assert (np.abs(got_y - want["y"]) <= want["tol_y"]).all()


def _backward(f, a, shape, post, gate, scale, dnew, dy):
    """{name: (gradient, tolerance)} as rows, from the values that forward stored."""
    c, k, rows = f["c"], f["k"], len(f["new"])
    u, hat = dy * f["w"], f["new"] * f["rho"]
    mean, mean_abs = (u * hat).mean(1, keepdims=True), np.abs(u * hat).mean(1, keepdims=True)
    D = dnew + f["rho"] * (u - hat * mean)
    size = np.abs(dnew) + f["rho"] * (np.abs(u) + np.abs(hat) * mean_abs)
    K = 2 * k + 16
    tol = U * K * size
    long = U * (rows + 16)
    out = {"residual": (scale * D, np.abs(scale) * (tol + U * size)), "weight": ((dy * hat).sum(0), (long + U * K) * np.abs(dy * hat).sum(0))}
    pw = a["post_weight"].astype(np.float64) if post else 1.0
    dinner, dinner_size = f["gate"] * D, np.abs(f["gate"]) * size
    each, each_size = D * f["inner"], size * np.abs(f["inner"])
    n = shape[0]
    if gate == "full":
        out["gate"] = (each, U * 2 * K * each_size)
    elif gate:
        shaped = (1, rows, c) if gate == "channel" else (n, rows // n, c)
        total, of_size = each.reshape(shaped).sum(1), each_size.reshape(shaped).sum(1)
        out["gate"] = (total[0] if gate == "channel" else total, ((long + 2 * U * K) * of_size)[0 if gate == "channel" else slice(None)])
    if post:
        out["post_weight"] = ((dinner * f["hat"]).sum(0), (long + 2 * U * K) * (dinner_size * np.abs(f["hat"])).sum(0))
        t, t_size = dinner * pw, dinner_size * np.abs(pw)
        db = f["rb"] * (t - f["hat"] * (t * f["hat"]).mean(1, keepdims=True))
        out["block"] = (db, U * 3 * K * f["rb"] * (t_size + np.abs(f["hat"]) * (t_size * np.abs(f["hat"])).mean(1, keepdims=True)))
    else:
        out["block"] = (dinner, U * (K + 4) * dinner_size)
    return out


@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("gate", [None, "channel", "sample", "full"])
@pytest.mark.parametrize("shape", SHAPES)
def test_backward(shape, gate, post):
    import gpu_util as g
    import mytorch_b200.nn.functional as F

    a = _inputs(shape, post, gate, 1)
    scale = [0.5, 1.0][shape[0] % 2]
    operands = ("residual", "block", "weight", "post_weight", "gate")
    for use_new, use_y in ((1, 1), (1, 0), (0, 1)):
        t = {k: g.dev(a[k], True) for k in operands if k in a}
        new, y = F.add_rms_norm(*[t.get(k) for k in operands], scale, EPS)
        got_new = _rows(g.host(new), a["weight"].size)
        loss = None
        for used, out, grad in ((use_new, new, "dnew"), (use_y, y, "dy")):
            if used:
                term = (out * g.dev(a[grad])).reshape((int(np.prod(shape)),)).sum()
                loss = term if loss is None else loss + term
        loss.backward()
        f = _forward(a, shape, post, gate, scale)
        f["new"] = got_new  # as it was stored: the gradient is that at this point
        f["rho"] = 1 / np.sqrt((got_new * got_new).mean(1, keepdims=True) + EPS)
        want = _backward(f, a, shape, post, gate, scale, use_new * _rows(a["dnew"], f["c"]), use_y * _rows(a["dy"], f["c"]))
        for name, (value, tol) in want.items():
            if t[name].grad is None:
                assert name == "weight" and not use_y
                continue
            got = g.host(t[name].grad)
            got = (_rows(got, f["c"]) if got.ndim > 2 or value.shape[0] == len(f["new"]) and value.ndim == 2 else got).reshape(value.shape)
            off = np.abs(got - value) / (tol + 1e-37)
            assert off.max() <= 1, (name, off.max())


@pytest.mark.parametrize("c", [129, 191, 194, 255, 260, 383, 386, 511, 513, 575, 578, 580, 767, 770, 772, 1023, 1025, 1028, 1279, 1282, 1284, 1535, 1538, 2047, 2050, 2052, 2303, 2306, 2559, 2562,
                               3001, 3071, 3080, 4095, 4098, 4100, 4607, 4610, 6143, 6145, 6148, 8191, 8194, 10241, 16380, 16383, 16386, 24572, 24575, 24578, 32767, 32768, 32770])
def test_widths_about_the_ends_of_each_group(c):
    """The widest and the narrowest rows that a number of warps and values a thread holds."""
    test_backward((2, 5, c), "sample", True)


@pytest.mark.parametrize("c", [129, 255, 260, 383, 386, 511, 516, 575, 578, 767, 772, 1023, 1025, 1028, 1279, 1282, 1535, 1540, 2047, 2052, 2306, 2559, 2564, 3071, 3080])
def test_widths_of_many_rows(c):
    """As above, for a forward pass of more rows than would be spread over eight warps each."""
    test_forward((4, 300, c), "channel", True)


@pytest.mark.parametrize("shape", [(1, 1), (3, 5), (2, 64), (9, 1000), (2, 3, 4096), (2, 66, 3, 5)])
def test_the_norm_by_itself(shape):
    import gpu_util as g
    import mytorch_b200.nn as nn
    import mytorch_b200.nn.functional as F

    a = _inputs(shape, False, None, 2)
    c = a["weight"].size
    x, w = g.dev(a["residual"], True), g.dev(a["weight"], True)
    y = F.rms_norm(x, w, EPS)
    zero = dict(a, block=np.zeros_like(a["block"]))
    f = _forward(zero, shape, False, None, 1.0)
    assert (np.abs(_rows(g.host(y), c) - f["y"]) <= f["tol_y"]).all()
    (y * g.dev(a["dy"])).reshape((int(np.prod(shape)),)).sum().backward()
    want = _backward(f, zero, shape, False, None, 1.0, 0 * f["new"], _rows(a["dy"], c))
    for t, name in ((x, "residual"), (w, "weight")):
        got = g.host(t.grad)
        assert (np.abs((_rows(got, c) if name == "residual" else got) - want[name][0]) <= want[name][1] + 1e-37).all(), name
    layer = nn.RMSNorm(c, EPS)
    layer.to("cuda:0")
    plain = F.rms_norm(g.dev(a["residual"]), None, EPS)
    assert np.array_equal(g.host(layer(g.dev(a["residual"]))), g.host(plain)) and not plain.requires_grad


def test_gradient_against_differences():
    """In 64 bits by steps of 1e-4 either way: off by 1e-8 times third derivatives, which are of the order of the values (ones)."""
    import gpu_util as g
    import mytorch_b200.nn.functional as F

    shape = (2, 3, 7)
    a = _inputs(shape, True, "sample", 3)
    operands = ("residual", "block", "weight", "post_weight", "gate")
    t = {k: g.dev(a[k], True) for k in operands}
    new, y = F.add_rms_norm(*[t[k] for k in operands], 0.75, EPS)
    ((new * g.dev(a["dnew"])).reshape((42,)).sum() + (y * g.dev(a["dy"])).reshape((42,)).sum()).backward()

    def loss(values):
        f = _forward(values, shape, True, "sample", 0.75)
        return (f["new"] * _rows(a["dnew"], 7)).sum() + (f["y"] * _rows(a["dy"], 7)).sum()

    for k in operands:
        got = g.host(t[k].grad).reshape(-1)
        for i in range(a[k].size):
            sides = []
            for e in (1e-4, -1e-4):
                v = {n: x.astype(np.float64) for n, x in a.items()}
                v[k].reshape(-1)[i] += e
                sides.append(loss(v))
            assert abs((sides[0] - sides[1]) / 2e-4 - got[i]) <= 2e-5 * max(1, abs(got[i])), k


@pytest.mark.parametrize("offset", [1, 2, 3])
def test_windows_that_begin_at_any_float(offset):
    import gpu_util as g
    import mytorch_b200 as mt
    import mytorch_b200.nn.functional as F
    from mytorch_b200.backends.cuda.env import CudaMemory, CudaMemoryView

    def window(a):
        view = CudaMemoryView(CudaMemory(0, 4 * (a.size + 4)), 4 * offset, 4 * a.size, 0)
        view.write(a)
        t = mt.Tensor._on_device(a.shape, mt.float32, mt.Device("cuda:0"), view)
        t.requires_grad = True
        return t

    operands = ("residual", "block", "weight", "post_weight", "gate")
    for shape in ((9, 64), (5, 2000)):
        a = _inputs(shape, True, "channel", 4)
        for off in operands:  # one of them at a time, and all
            t = {k: window(a[k]) if k == off or off == "gate" else g.dev(a[k], True) for k in operands}
            new, y = F.add_rms_norm(*[t[k] for k in operands], 1.0, EPS)
            f = _forward(a, shape, True, "channel", 1.0)
            assert (np.abs(g.host(new) - f["new"]) <= f["tol_new"]).all() and (np.abs(g.host(y) - f["y"]) <= f["tol_y"]).all()
            f["new"] = g.host(new).astype(np.float64)
            f["rho"] = 1 / np.sqrt((f["new"] ** 2).mean(1, keepdims=True) + EPS)
            ((new * g.dev(a["dnew"])).reshape((a["dnew"].size,)).sum() + (y * g.dev(a["dy"])).reshape((a["dy"].size,)).sum()).backward()
            for name, (value, tol) in _backward(f, a, shape, True, "channel", 1.0, a["dnew"].astype(np.float64), a["dy"].astype(np.float64)).items():
                assert (np.abs(g.host(t[name].grad) - value) <= tol + 1e-37).all(), (name, off)


def test_rows_of_zeros_and_of_no_numbers():
    """A row of zeros is normed by 1 / sqrt(eps); what is not finite stays in its row."""
    import gpu_util as g
    import mytorch_b200.nn.functional as F

    for c in (6, 300, 5000):
        a = _inputs((4, c), True, None, 5)
        a["residual"][0] = a["block"][0] = 0
        a["residual"][1, c // 2], a["block"][2, 0] = np.nan, np.inf
        new, y = F.add_rms_norm(g.dev(a["residual"]), g.dev(a["block"]), g.dev(a["weight"]), g.dev(a["post_weight"]), eps=EPS)
        new, y = g.host(new), g.host(y)
        assert not new[0].any() and not y[0].any() and np.isnan(y[1]).all() and np.isnan(y[2]).all() and np.isfinite(new[3]).all() and np.isfinite(y[3]).all()
        assert np.isfinite(np.delete(new[1], c // 2)).all()


@pytest.mark.parametrize("gate", [None, "channel", "sample", "full"])
@pytest.mark.parametrize("c", [5, 64, 130, 1000, 4096, 20000])
def test_gradient_of_the_sum_alone_beside_infinite_values(c, gate):
    """Without a norm the sum's gradient does not know the block's values but in the gate's: those of the operands are finite, and products of at most two numbers."""
    import gpu_util as g
    import mytorch_b200.nn.functional as F

    a = _inputs((3, c), False, gate)
    a["block"][:, c // 2], a["residual"][1, c // 3] = np.inf, -np.inf
    t = {k: g.dev(v, k in ("residual", "block")) for k, v in a.items()}
    new, _ = F.add_rms_norm(t["residual"], t["block"], t["weight"], None, t.get("gate"), 0.5, EPS)
    (new * g.dev(a["dnew"])).reshape((3 * c,)).sum().backward()
    gr = _gate_rows(a, (3, c), c, gate)
    for name, factor in (("residual", 0.5), ("block", gr)):
        want = a["dnew"].astype(np.float64) * factor
        assert (np.abs(g.host(t[name].grad) - want) <= U * np.abs(want)).all()


def test_no_rows():
    import gpu_util as g
    import mytorch_b200.nn.functional as F

    operands = [g.dev(a, True) for a in (np.zeros((0, 6), np.float32), np.zeros((0, 6), np.float32), np.ones(6, np.float32), np.ones(6, np.float32), np.ones(6, np.float32))]
    new, y = F.add_rms_norm(*operands)
    assert new.shape == y.shape == (0, 6)
    got = g.op("add_rms_norm_backward")(new, y, new, y, y, *operands)
    assert got[0].shape == (0, 6) and all(not g.host(t).any() for t in got[2:])


def test_captured_and_replayed():
    """Two graphs over the same leaves and the same scratch, replayed in turn, while a tape of the same leaves lives; gradients as outside."""
    import gpu_util as g
    import mytorch_b200.nn as nn
    from mytorch_b200.cuda_graph import StepGraph

    rng = np.random.default_rng(6)
    layers = [nn.AddRMSNorm(96, gate=0.5), nn.AddRMSNorm(96, gate=0.25)]
    for layer in layers:
        layer.to("cuda:0")
    x, b = g.dev(rng.standard_normal((70, 96)).astype(np.float32), True), g.dev(rng.standard_normal((70, 96)).astype(np.float32), True)
    leaves = [x, b] + [p for layer in layers for p in layer.parameters()]

    def step():
        for t in leaves:
            t.grad = None
        new, y = layers[0](x, b)
        new, y = layers[1](new, y)
        (new * y).sum().backward()
        return [t.grad for t in leaves]

    step()
    kept = layers[0](x, b)
    graphs = [StepGraph(step), StepGraph(step)]
    results = [gr.capture() for gr in graphs]
    for turn in range(4):
        x._native_array.write(rng.standard_normal((70, 96)).astype(np.float32))
        graphs[turn % 2].replay()
        got = [g.host(t) for t in results[turn % 2]]
        want = [g.host(t) for t in step()]
        assert all(np.array_equal(p, q) for p, q in zip(got, want))
    assert kept[0].shape == (70, 96)
    for gr in graphs:
        gr.destroy()


def test_rows_past_32_bits():
    """The last rows of tensors of more than 2^31 values, forward and backward, where all others are zero."""
    import gpu_util as g
    import mytorch_b200 as mt
    import mytorch_b200.nn.functional as F
    from mytorch_b200.backends.cuda.env import CudaEnv, CudaMemoryView

    rows, c = (1 << 31) // 2000 + 5, 2000
    rng = np.random.default_rng(7)
    names = ("residual", "block", "dnew", "dy")
    last = {k: rng.standard_normal((2, c)).astype(np.float32) for k in names}
    weight = {k: rng.standard_normal(c).astype(np.float32) for k in ("weight", "post_weight", "gate")}
    at, size = 4 * (rows - 2) * c, 4 * 2 * c
    big = {}
    for k, a in last.items():
        big[k] = mt.Tensor(shape=(rows, c), dtype=mt.float32, device="cuda:0")
        big[k].fill_(0)
        CudaMemoryView(big[k]._native_array, at, size, 0).write(a)
    small = {k: g.dev(a) for k, a in weight.items()}
    end = lambda t: CudaMemoryView(t._native_array, at, size, 0).read((2, c), np.float32)
    new, y, rstd, block_rstd = g.op("add_rms_norm")(big["residual"], big["block"], *small.values())
    f = _forward({**last, **weight}, (2, c), True, "channel", 1.0)
    assert (np.abs(end(new) - f["new"]) <= f["tol_new"]).all() and (np.abs(end(y) - f["y"]) <= f["tol_y"]).all()
    del y
    got = g.op("add_rms_norm_backward")(big["dnew"], big["dy"], new, rstd, block_rstd, new, big["block"], *small.values())
    f["new"] = end(new).astype(np.float64)
    f["rho"] = 1 / np.sqrt((f["new"] ** 2).mean(1, keepdims=True) + EPS)
    want = _backward(f, last | weight, (2, c), True, "channel", 1.0, last["dnew"].astype(np.float64), last["dy"].astype(np.float64))
    for name, t in (("residual", got[0]), ("block", got[1])):
        assert (np.abs(end(t) - want[name][0]) <= want[name][1] + 1e-37).all(), name
    for name, t in (("weight", got[2]), ("post_weight", got[3]), ("gate", got[4])):  # zeros add nothing
        assert (np.abs(g.host(t) - want[name][0]) <= want[name][1] + 1e-37).all(), name
    del got, big, new
    CudaEnv.instance().lib.pool_trim()
