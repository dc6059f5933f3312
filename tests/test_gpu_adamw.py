"""AdamW with states in 32 bits against 64 bits, and in 8 bits against an emulation by what the codes stand for, whose codes have to be equal.

Tolerances, u = 2^-24: a coefficient that is rounded to float32, a product and a sum by u of themselves each."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
BLOCK = 256


@pytest.fixture(autouse=True, scope="module")
def blocks_of_these_sizes_go_back_to_the_driver():
    """A later module's test of the memory pool counts on sizes that no earlier one left there."""
    yield
    from mytorch_b200.backends.cuda.env import CudaEnv

    CudaEnv.instance().lib.pool_trim()


def _window(a, offset):
    import mytorch_b200 as mt
    from mytorch_b200.backends.cuda.env import CudaMemory, CudaMemoryView

    view = CudaMemoryView(CudaMemory(0, 4 * (a.size + 4)), 4 * offset, 4 * a.size, 0)
    view.write(a)
    return mt.Tensor._on_device(a.shape, mt.float32, mt.Device("cuda:0"), view)


def _params(sizes, offset, rng, size=1.0):
    made = []
    for n in sizes:
        p = _window((size * rng.standard_normal(n)).astype(np.float32), offset)
        p.requires_grad = True
        made.append(p)
    return made


def _give(params, rng, offset=0, size=1.0):
    """New gradients, of unequal size from value to value; returns them."""
    grads = [(size * np.exp(2 * rng.standard_normal(p.shape)) * rng.standard_normal(p.shape)).astype(np.float32) for p in params]
    for p, a in zip(params, grads):
        p.grad = _window(a, offset)
    return grads


SIZES = [[1], [5, 0, 3], [255], [256], [257, 1, 4096], [1000] * 7, [100003, 7, 64, 5, 30000, 2], [37] * 400, [2048, 2049, 4097]]
IDS = [f"{len(s)}x{s[0]}" for s in SIZES]


@pytest.mark.parametrize("limit", [None, 0.5], ids=["", "clipped"])
@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("sizes", SIZES, ids=IDS)
def test_32_bits(sizes, offset, limit):
    import gpu_util as g
    from mytorch_b200.optim import AdamW

    rng = np.random.default_rng(sum(sizes))
    params = _params(sizes, offset, rng)
    lr, b1, b2, eps, wd = 0.01, 0.9, 0.99, 1e-6, 0.1
    opt = AdamW(params, lr=lr, betas=(b1, b2), eps=eps, weight_decay=wd, max_grad_norm=limit, maximize=offset == 1)
    opt.grad_scale = 0.5
    m = v = [np.zeros(n) for n in sizes]
    tol_m = tol_v = [np.zeros(n) for n in sizes]
    for t in (1, 2, 3):
        p = [g.host(q).astype(np.float64) for q in params]
        grads = [0.5 * a.astype(np.float64) for a in _give(params, rng, offset)]
        opt.step()
        factor = 1.0
        if limit is not None:
            norm = math.sqrt(sum((a * a).sum() for a in grads))
            assert abs(g.host(opt.grad_norm)[0] - norm) <= 2 * U * norm
            factor = min(1.0, limit / (norm + 1e-6))
        for i, a in enumerate(grads):
            a = a * factor * (-1 if offset == 1 else 1)
            tol_m[i:i + 1] = [b1 * tol_m[i] + U * (4 * np.abs(b1 * m[i]) + 6 * np.abs((1 - b1) * a))]
            tol_v[i:i + 1] = [b2 * tol_v[i] + U * (4 * np.abs(b2 * v[i]) + 9 * (1 - b2) * a * a) + 1e-44]
            m = m[:i] + [b1 * m[i] + (1 - b1) * a] + m[i + 1:]
            v = v[:i] + [b2 * v[i] + (1 - b2) * a * a] + v[i + 1:]
            gm, gv = (g.host(opt.state[params[i]][k]).astype(np.float64) for k in ("exp_avg", "exp_avg_sq"))
            assert (np.abs(gm - m[i]) <= tol_m[i]).all() and (np.abs(gv - v[i]) <= tol_v[i]).all()
            step = lr / (1 - b1 ** t) * gm / (np.sqrt(gv / (1 - b2 ** t)) + eps)
            want = p[i] * (1 - lr * wd) - step
            assert (np.abs(g.host(params[i]) - want) <= U * (3 * np.abs(p[i]) + 16 * np.abs(step) + np.abs(want))).all()
            assert int(g.host(opt.state[params[i]]["step"])[0]) == t


# ------------------------------------------------------------------------------ 8 bits

def _mix(x):
    x = (x ^ (x >> 16)) * 0x6A09E667 & 0xFFFFFFFF
    x = (x ^ (x >> 15)) * 0xBB67AE85 & 0xFFFFFFFF
    return x ^ (x >> 16)


TABLES = [np.array([(1 - 2 * (c >> 7)) * math.ldexp((c & 7) + (8 if c & 120 else 0), max(c >> 3 & 15, 1) - 17) for c in range(256)]),
          np.array([math.ldexp((c & 7) + (8 if c >> 3 else 0), max(c >> 3, 1) - 33) for c in range(256)])]


def _decode(codes, scales, k, n):
    """[blocks, 512], [blocks, 2] -> the first n values"""
    with np.errstate(invalid="ignore", over="ignore"):
        unit = np.where(scales[:, k] == 255, np.nan, np.where(scales[:, k] == 0, 0.0, 2.0 ** (scales[:, k].astype(np.float64) - 127)))
        return (TABLES[k][codes[:, k * BLOCK:(k + 1) * BLOCK]] * unit[:, None]).reshape(-1)[:n]


def _encode(x, k, random16):
    """float32 values in blocks of 256 -> (codes, scales): the nearest multiple of the step below or above, by 16 random bits."""
    lowest, bottom = ((13, 0), (29, 1))[k]
    codes, scales = np.zeros(x.shape, np.int64), np.zeros(len(x), np.int64)
    for i, row in enumerate(np.abs(x.astype(np.float64))):
        if not np.isfinite(row).all():
            scales[i] = 255
            continue
        most = row.max()
        if most == 0:
            continue
        power = max(math.frexp(most)[1] - 1, -126)
        scales[i] = power + 127
        own = np.maximum(np.where(row > 0, np.frexp(row)[1] - 1, -2000), power - lowest)
        n = (np.rint(np.ldexp(row, 3 - own + 20)).astype(np.int64) + random16[i] * 16 + 8) >> 20  # eighths of 2^own; 16 is the next power
        field = own - (power - lowest) + 1
        carried = n == 16
        field, n = np.where(carried, field + 1, field), np.where(carried, 8, n)
        code = np.where(n >= 8, field * 8 + n - 8, n)
        codes[i] = np.where(row == 0, 0, np.maximum(code, bottom))
    if k == 0:
        codes = codes + 128 * (np.signbit(x) & np.isfinite(x).all(1, keepdims=True))
    return codes, scales


def _emulate(grad32, codes, scales, b1, b2, seed, ordinal, t):
    """One step of the moments of one tensor: (m, v as float32 before rounding, codes, scales).  grad32: what enters the moments."""
    n, blocks = grad32.size, len(codes)
    b1, b2 = (round(b * (1 << 20)) / (1 << 20) for b in (b1, b2))
    pad = lambda a: np.concatenate([a, np.zeros(blocks * BLOCK - n, a.dtype)]).reshape(blocks, BLOCK)
    with np.errstate(over="ignore", invalid="ignore"):
        g = grad32.reshape(-1).astype(np.float64)
        h = (grad32.reshape(-1) * np.float32(math.sqrt(1 - b2))).astype(np.float64)
        m = (b1 * _decode(codes, scales, 0, n) + (1 - b1) * g).astype(np.float32)
        v = (b2 * _decode(codes, scales, 1, n) + h * h).astype(np.float32)
    key = _mix((_mix((seed + 0x9E3779B1 * (ordinal + 1)) & 0xFFFFFFFF) + t) & 0xFFFFFFFF)
    r = np.array([_mix((key + i * 0x9E3779B1) & 0xFFFFFFFF) for i in range(blocks * BLOCK)], np.int64).reshape(blocks, BLOCK)
    cm, sm = _encode(pad(m), 0, r >> 16)
    cv, sv = _encode(pad(v), 1, r & 0xFFFF)
    return m, v, np.concatenate([cm, cv], 1), np.stack([sm, sv], 1)


def _states(opt, p):
    import gpu_util as g

    return g.host(opt.state[p]["moments"]), g.host(opt.state[p]["scales"])


@pytest.mark.parametrize("limit", [None, 0.5], ids=["", "clipped"])
@pytest.mark.parametrize("offset,size", [(0, 1.0), (1, 1e-6), (0, 1e-17), (3, 1e12)])
@pytest.mark.parametrize("sizes", [[1], [5, 0, 3], [255], [256], [257, 1, 4099], [1000] * 3, [9000, 7], [257, 600], [255, 700]], ids=lambda s: f"{len(s)}x{s[0]}")
def test_8_bits(sizes, offset, size, limit):
    import gpu_util as g
    from mytorch_b200.optim import AdamW

    rng = np.random.default_rng(sum(sizes))
    params = _params(sizes, offset, rng)
    lr, b1, b2, eps, wd, seed = 0.01, 0.9, 0.999, 1e-8, 0.1, 12345
    opt = AdamW(params, lr=lr, betas=(b1, b2), eps=eps, weight_decay=wd, max_grad_norm=limit, state_bits=8, seed=seed)
    q1, q2 = (round(b * (1 << 20)) / (1 << 20) for b in (b1, b2))
    held = [(np.zeros((-(-n // BLOCK), 2 * BLOCK), np.int64), np.zeros((-(-n // BLOCK), 2), np.int64)) for n in sizes]
    for t in (1, 2, 3):
        p = [g.host(q).astype(np.float64) for q in params]
        grads = _give(params, rng, offset, size)
        opt.step()
        factor = 1.0
        if limit is not None:
            norm = math.sqrt(sum((a.astype(np.float64) ** 2).sum() for a in grads))
            factor = min(1.0, limit / (norm + 1e-6))
        for i, a in enumerate(grads):
            m, v, codes, scales = _emulate(a * np.float32(factor), *held[i], b1, b2, seed, i, t)
            got_codes, got_scales = _states(opt, params[i])
            assert np.array_equal(got_scales, scales)
            assert np.array_equal(_decode(got_codes, got_scales, 0, a.size), _decode(codes, scales, 0, a.size))
            assert np.array_equal(got_codes[:, BLOCK:], codes[:, BLOCK:])
            held[i] = (got_codes.astype(np.int64), got_scales.astype(np.int64))
            step = lr / (1 - q1 ** t) * m / (np.sqrt(v.astype(np.float64) / (1 - q2 ** t)) + eps)
            want = p[i] * (1 - lr * wd) - step
            assert (np.abs(g.host(params[i]) - want) <= U * (3 * np.abs(p[i]) + 16 * np.abs(step) + np.abs(want)) + 1e-44).all()
            first, second = opt.moments(params[i])
            assert first.shape == params[i].shape
            assert np.array_equal(g.host(first), _decode(codes, scales, 0, a.size)) and np.array_equal(g.host(second), _decode(codes, scales, 1, a.size))
    flat = [g.host(t) for t in opt.moments()]
    for k in range(2):
        assert np.array_equal(flat[k], np.concatenate([g.host(opt.moments(p)[k]) for p in params]))


def test_8_bits_round_without_bias():
    """The mean of n rounded values is off by their rounding, at most an eighth of each at random: 5 standard deviations, and 2^-17 of a step of an eighth for the
    random number's 16 bits."""
    import gpu_util as g
    from mytorch_b200.optim import AdamW

    n = 1 << 18
    p = _window(np.zeros(n, np.float32), 0)
    p.requires_grad = True
    opt = AdamW([p], lr=0.0, betas=(0.5, 0.5), state_bits=8, seed=3)
    p.grad = _window(np.full(n, 1.3, np.float32), 0)
    opt.step()
    m, v = (g.host(t).astype(np.float64) for t in opt.moments())
    for got, want in ((m, 0.65), (v, 0.845)):
        assert len(np.unique(got)) == 2 and got.min() <= want <= got.max() and (got.max() - got.min()) <= want / 8
        spread = (got.max() - got.min()) / 2
        assert abs(got.mean() - want) <= 5 * spread / math.sqrt(n) + (got.max() - got.min()) * 2.0 ** -16


def test_8_bits_keep_second_moments_above_zero():
    """Values far under their block's largest one: the second moment stays at the lowest code, and the next step, of gradients of zero, moves nothing far."""
    import gpu_util as g
    from mytorch_b200.optim import AdamW

    a = np.full(256, 1e-9, np.float32)
    a[0] = 1e4
    p = _window(np.zeros(256, np.float32), 0)
    p.requires_grad = True
    opt = AdamW([p], lr=1e-3, weight_decay=0.0, eps=1e-30, state_bits=8)
    for t in range(4):
        p.grad = _window(a if t == 0 else 0 * a, 0)
        opt.step()
        m, v = (g.host(x) for x in opt.moments(p))
        assert (v > 0).all() and np.abs(g.host(p)).max() <= 4e-3 * (t + 1)


def test_8_bits_of_what_is_no_number():
    """A gradient that is not finite leaves its block of 256 NaN, and nothing else."""
    import gpu_util as g
    from mytorch_b200.optim import AdamW

    rng = np.random.default_rng(0)
    a = rng.standard_normal(1000).astype(np.float32)
    for bad in (np.nan, np.inf, -np.inf, 3e38):
        a[300] = bad
        p = _window(np.ones(1000, np.float32), 0)
        p.requires_grad, p.grad = True, _window(a, 0)
        opt = AdamW([p], state_bits=8)
        opt.step()
        m, v = (g.host(x) for x in opt.moments(p))
        inside = np.arange(1000) // 256 == 1
        assert np.isnan(v[inside]).all() and np.isfinite(v[~inside]).all() and np.isfinite(m[~inside]).all()
        assert np.isnan(m[inside]).all() == (bad != np.float32(3e38))
        assert np.isfinite(np.delete(g.host(p), 300)).all()


@pytest.mark.parametrize("bits", [8, 32])
def test_captured_and_replayed(bits):
    """Steps replayed from a graph count on: the same parameters and states as steps outside."""
    import gpu_util as g
    from mytorch_b200.cuda_graph import StepGraph
    from mytorch_b200.optim import AdamW

    results = []
    for captured in (False, True):
        rng = np.random.default_rng(7)
        params = _params([300, 5000, 3], 0, rng)
        opt = AdamW(params, lr=0.01, max_grad_norm=1.0, state_bits=bits)
        _give(params, rng)
        if captured:  # the state comes to be outside
            with pytest.raises(RuntimeError, match="eager optimizer step"):
                StepGraph(opt.step).capture()
            assert not opt.state
        opt.step()
        graph = None
        if captured:
            graph = StepGraph(lambda: (opt.step(), opt.grad_norm))
            graph.capture()
        for _ in range(5):
            for p in params:
                p.grad._native_array.write(rng.standard_normal(p.shape).astype(np.float32))
            if captured:
                graph.replay()
            else:
                opt.step()
        results.append([g.host(p) for p in params] + [g.host(t) for t in opt.moments()] + [g.host(opt.state[params[0]]["step"])])
        if graph:
            graph.destroy()
    assert results[0][-1][0] == 6 and all(np.array_equal(a, b) for a, b in zip(*results))


@pytest.mark.parametrize("bits", [8, 32])
def test_checkpoint_and_groups(bits, tmp_path):
    """Two groups with their own numbers, saved after two steps and continued in another optimizer: the same as going on."""
    import gpu_util as g
    import mytorch_b200 as mt
    import mytorch_b200.nn as nn
    from mytorch_b200 import serialization
    from mytorch_b200.optim import AdamW

    def make(arrays):
        params = [nn.Parameter(g.dev(a)) for a in arrays]
        return params, AdamW([{"params": params[:2], "lr": 0.1}, {"params": params[2:], "betas": (0.5, 0.75), "weight_decay": 0.0}], lr=0.01, state_bits=bits)

    rng = np.random.default_rng(8)
    shapes = [(300,), (8, 3, 3, 3), (17, 4)]
    arrays = [rng.standard_normal(s).astype(np.float32) for s in shapes]
    grads = [[rng.standard_normal(s).astype(np.float32) for s in shapes] for _ in range(4)]
    params, opt = make(arrays)

    def run(params, opt, some):
        for now in some:
            for p, a in zip(params, now):
                p.grad = g.dev(a)
            opt.step()

    run(params, opt, grads[:2])
    serialization.save({"opt": opt.state_dict(), "params": params}, tmp_path / "c.pt")
    run(params, opt, grads[2:])
    found = serialization.load(tmp_path / "c.pt")
    others, again = make([g.host(t) for t in found["params"]])
    again.load_state_dict(found["opt"])
    run(others, again, grads[2:])
    for p, q in zip(params, others):
        assert np.array_equal(g.host(p), g.host(q)) and opt.moments(p)[0].shape == p.shape
        assert all(np.array_equal(g.host(a), g.host(b)) for a, b in zip(opt.moments(p), again.moments(q)))
    assert int(g.host(again.state[others[2]]["step"])[0]) == 4
    assert isinstance(found["params"][0], mt.Tensor)


def test_what_is_wrong_is_said_before_anything_changes():
    import gpu_util as g
    import mytorch_b200 as mt
    import mytorch_b200.nn as nn
    from mytorch_b200.optim import AdamW

    for bits in (8, 32):
        p, q = nn.Parameter(g.dev(np.ones(8, np.float32))), nn.Parameter(g.dev(np.ones((2, 4), np.float32)))
        opt = AdamW([p, q], state_bits=bits)
        with pytest.raises(RuntimeError, match="no moments"):
            opt.moments()
        p.grad = g.dev(np.ones(8, np.float32))
        with pytest.raises(RuntimeError, match="no gradient"):
            opt.step()
        q.grad = g.dev(np.ones(8, np.float32))
        with pytest.raises(RuntimeError, match="Mismatched shape"):
            opt.step()
        assert not opt.state and (g.host(p) == 1).all()
        q.grad = g.dev(np.ones((2, 4), np.float32))
        opt.step()
        before = g.host(p)
        other = AdamW([p, q], state_bits=40 - bits)
        other.load_state_dict({"state": {id(t): s for t, s in opt.state.items()}, "param_groups": [{"params": [id(p), id(q)]}]})
        with pytest.raises(RuntimeError, match="state is not of its size"):
            other.step()
        opt.state[q]["step"] = mt.tensor(np.ones(1, np.int32), device="cuda:0")
        with pytest.raises(RuntimeError, match="state is not of its size"):
            opt.step()
        assert np.array_equal(g.host(p), before)
        a, b = nn.Parameter(g.dev(np.ones(8, np.float32))), nn.Parameter(g.dev(np.ones(8, np.float32)))
        a.grad = b.grad = g.dev(np.ones(8, np.float32))
        two = AdamW([{"params": [a]}, {"params": [b]}], state_bits=bits)
        two.step()
        two.state[b]["step"] = two.state[a]["step"]
        with pytest.raises(RuntimeError, match="share a step"):
            two.step()
        two.state[b]["step"] = mt.tensor(np.ones(1, np.int64), device="cuda:0")
        before = [g.host(t) for t in (a, b)]
        for wrong in ({"lr": -1.0}, {"betas": (0.9, 1.0)}, {"eps": float("nan")}, {"betas": (0.9, 1 - 1e-7)}):
            group = two.param_groups[1]  # the second: the first is not updated either
            held = dict(group)
            group.update(wrong)
            if bits == 32 and wrong == {"betas": (0.9, 1 - 1e-7)}:
                two.step()
            else:
                with pytest.raises(RuntimeError, match="betas from 0 to below 1"):
                    two.step()
                assert all(np.array_equal(g.host(t), x) for t, x in zip((a, b), before))
            group.update(held)


@pytest.mark.parametrize("bits", [8, 32])
def test_a_tensor_past_32_bits(bits):
    """The last values of a tensor of more than 2^31, whose other gradients are zero: those of a short one (the roundings of 8 bits know the place modulo 2^32)."""
    import gpu_util as g
    import mytorch_b200 as mt
    from mytorch_b200.backends.cuda.env import CudaEnv, CudaMemoryView
    from mytorch_b200.optim import AdamW

    n, last = (1 << 31) + 300, 700
    rng = np.random.default_rng(9)
    p, grad = (mt.Tensor(shape=(n,), dtype=mt.float32, device="cuda:0", requires_grad=k == 0) for k in range(2))
    values = [rng.standard_normal(last).astype(np.float32) for _ in range(2)]
    for t, a in zip((p, grad), values):
        t.fill_(0)
        CudaMemoryView(t._native_array, 4 * (n - last), 4 * last, 0).write(a)
    p.grad = grad
    opt = AdamW([p], lr=0.01, weight_decay=0.1, state_bits=bits)
    opt.step()
    b = (0.9, 0.999) if bits == 32 else tuple(round(x * 2 ** 20) / 2 ** 20 for x in (0.9, 0.999))
    x = values[1].astype(np.float64)
    step = 0.01 * x / (np.abs(x) + 1e-8)  # the first step: m / (1 - b1) and v / (1 - b2) are x and x^2
    want = values[0] * (1 - 0.001) - step
    got = CudaMemoryView(p._native_array, 4 * (n - last), 4 * last, 0).read((last,), np.float32)
    assert (np.abs(got - want) <= U * (4 * np.abs(values[0]) + 24 * np.abs(step))).all()
    if bits == 8:
        blocks = -(-n // BLOCK)
        codes = CudaMemoryView(opt.state[p]["moments"]._native_array, (blocks - 4) * 512, 4 * 512, 0).read((4, 512), np.uint8)
        scales = CudaMemoryView(opt.state[p]["scales"]._native_array, (blocks - 4) * 2, 8, 0).read((4, 2), np.uint8)
        part = 4 * BLOCK - (blocks * BLOCK - n)  # values of the last four blocks
        m = _decode(codes, scales, 0, part)[-last:]
        big = np.abs(m) > 2.0 ** -8 * np.abs(m).max()
        assert (np.abs(m - (1 - b[0]) * x)[big] <= np.abs((1 - b[0]) * x)[big] / 8).all()
    del opt, p, grad
    CudaEnv.instance().lib.pool_trim()
