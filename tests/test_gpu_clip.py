"""The norm of all gradients, clipping in place and in the SGD update, against 64 bits.

The norm is added up in 64 bits and rounded once: 2^-24 of itself, taken as 2^-23.  A clipped gradient is off by the factor's rounding and its own."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, scope="module")
def blocks_of_these_sizes_go_back_to_the_driver():
    """A later module's test of the memory pool counts on sizes that no earlier one left there."""
    yield
    from mytorch_b200.backends.cuda.env import CudaEnv

    CudaEnv.instance().lib.pool_trim()


U = 2.0 ** -24


def _params(arrays, offset=0):
    """Tensors without meaning whose gradients are `arrays`, each `offset` floats into its block."""
    import mytorch_b200 as mt
    from mytorch_b200.backends.cuda.env import CudaMemory, CudaMemoryView

    made = []
    for a in arrays:
        p = mt.Tensor(shape=a.shape, dtype=mt.float32, device="cuda:0", requires_grad=True)
        view = CudaMemoryView(CudaMemory(0, 4 * (a.size + 4)), 4 * offset, 4 * a.size, 0)
        view.write(a)
        p.grad = mt.Tensor._on_device(a.shape, mt.float32, p.device, view)
        made.append(p)
    return made


def _norm(arrays):
    return float(np.sqrt(sum((a.astype(np.float64) ** 2).sum() for a in arrays)))


SIZES = [[1], [3], [4, 1, 2], [1000], [190001 // 20] * 20, [100003, 7, 64, 5, 300000, 2], [37] * 400, [1, 0, 5], [5000000, 3], [2048] * 193]


@pytest.mark.parametrize("offset", [0, 1, 3])
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{s[0]}")
def test_norm_and_clipping(sizes, offset):
    import gpu_util as g
    from mytorch_b200.optim import clip_grad_norm_, grad_norm

    rng = np.random.default_rng(sum(sizes))
    arrays = [rng.standard_normal(s).astype(np.float32) for s in sizes]
    want = _norm(arrays)
    params = _params(arrays, offset)
    assert abs(g.host(grad_norm(params))[0] - want) <= 2 * U * want
    for limit in (2 * want, float("inf")):  # not reached: nothing changes
        assert abs(g.host(clip_grad_norm_(params, limit))[0] - want) <= 2 * U * want
        assert all(np.array_equal(g.host(p.grad), a) for p, a in zip(params, arrays))
    norm = clip_grad_norm_(params, want / 4)
    assert norm.shape == (1,) and abs(g.host(norm)[0] - want) <= 2 * U * want
    factor = want / 4 / (want + 1e-6)
    assert all((np.abs(g.host(p.grad) - a * factor) <= 4 * U * np.abs(a)).all() for p, a in zip(params, arrays))
    clip_grad_norm_(params, 0.0)
    assert not any(g.host(p.grad).any() for p in params)


@pytest.mark.parametrize("size", [1e30, 1e-30, 3e38, 1e-42])
def test_squares_that_leave_32_bits(size):
    import gpu_util as g
    from mytorch_b200.optim import clip_grad_norm_

    a = (np.sign(np.random.default_rng(1).standard_normal(5000)) * size).astype(np.float32)
    want = _norm([a])
    params = _params([a])
    got = g.host(clip_grad_norm_(params, want / 2))[0]
    assert got == np.float32(want) if want < 3e38 else np.isinf(got)
    factor = want / 2 / (want + 1e-6)
    assert (np.abs(g.host(params[0].grad) - a * factor) <= 4 * U * np.abs(a) + 2e-45).all()


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("at", [0, 4321, 9999])
def test_bad_values_show(bad, at):
    import gpu_util as g
    from mytorch_b200.optim import clip_grad_norm_

    a = np.ones(10000, np.float32)
    a[at] = bad
    params = _params([a, np.ones(3, np.float32)])
    norm = g.host(clip_grad_norm_(params, 1.0))[0]
    got = g.host(params[0].grad)
    if np.isnan(bad):
        assert np.isnan(norm) and np.isnan(got).all() and np.isnan(g.host(params[1].grad)).all()
    else:  # a factor of 0
        assert np.isinf(norm) and np.isnan(got[at]) and not np.delete(got, at).any() and not g.host(params[1].grad).any()


def test_the_same_bits_every_time():
    import gpu_util as g
    from mytorch_b200.optim import grad_norm

    rng = np.random.default_rng(3)
    params = _params([rng.standard_normal(s).astype(np.float32) for s in (100000, 77, 1234567)])
    assert len({g.host(grad_norm(params)).tobytes() for _ in range(5)}) == 1


def test_a_gradient_of_two_parameters_is_scaled_once():
    import gpu_util as g
    import mytorch_b200 as mt
    from mytorch_b200.optim import clip_grad_norm_

    p, q, r = (mt.tensor(np.full((3, 4), v, np.float32), device="cuda:0", requires_grad=True) for v in (1.0, 2.0, 3.0))
    ((p + q) * r).sum().backward()
    assert p.grad._native_array.ptr == q.grad._native_array.ptr
    want = _norm([g.host(t.grad) for t in (p, q, r)])
    before = [g.host(t.grad) for t in (p, q, r)]
    assert abs(g.host(clip_grad_norm_([p, q, r], 1.0))[0] - want) <= 2 * U * want
    for t, b in zip((p, q, r), before):
        assert (np.abs(g.host(t.grad) - b / (want + 1e-6)) <= 4 * U * np.abs(b)).all()


def test_parameters_without_gradients_count_nothing():
    import gpu_util as g
    import mytorch_b200 as mt
    from mytorch_b200.optim import clip_grad_norm_

    a = np.full(100, 2.0, np.float32)
    params = _params([a]) + [mt.Tensor(shape=(5,), dtype=mt.float32, device="cuda:0", requires_grad=True)]
    assert g.host(clip_grad_norm_(params, 10.0))[0] == 20.0
    assert (np.abs(g.host(params[0].grad) - 1.0) <= 1e-6).all()
    assert g.host(clip_grad_norm_(params[0], 100.0)).shape == (1,)  # one tensor instead of several


def _sgd(p, g, buf, factor, lr, decay, momentum, nesterov, maximize, scale, first):
    """(parameter, buffer) after an update, in 64 bits."""
    g = (-g if maximize else g) * scale * factor + decay * p
    buf = g if first else momentum * buf + g
    return p - lr * (g + momentum * buf if nesterov else buf), buf


@pytest.mark.parametrize("limit", [0.5, 1e6])
@pytest.mark.parametrize("scale,nesterov,maximize", [(1.0, False, False), (0.25, True, False), (1.0, False, True)])
@pytest.mark.parametrize("sizes", [[5], [1000, 3, 64], [70000, 13], [50] * 230])
def test_update_with_clipping(sizes, scale, nesterov, maximize, limit):
    import gpu_util as g
    import mytorch_b200.nn as nn
    from mytorch_b200.optim import SGD

    rng = np.random.default_rng(len(sizes) + sizes[0])
    values = [rng.standard_normal(s).astype(np.float32) for s in sizes]
    params = [nn.Parameter(g.dev(v)) for v in values]
    split = len(params) // 2
    groups = [{"params": params[:split], "lr": 0.5}, {"params": params[split:]}] if split else params
    opt = SGD(groups, lr=0.1, momentum=0.9, weight_decay=0.01, nesterov=nesterov, maximize=maximize, max_grad_norm=limit)
    opt.grad_scale = scale
    want, bufs = [v.astype(np.float64) for v in values], [np.zeros(s) for s in sizes]
    for step in range(3):
        grads = [rng.standard_normal(s).astype(np.float32) for s in sizes]
        for p, a in zip(params, grads):
            p.grad = g.dev(a)
        opt.step()
        norm = scale * _norm(grads)
        assert abs(g.host(opt.grad_norm)[0] - norm) <= 2 * U * norm
        factor = min(1.0, limit / (norm + 1e-6))
        for k, a in enumerate(grads):
            lr = 0.5 if k < split else 0.1
            want[k], bufs[k] = _sgd(want[k], a.astype(np.float64), bufs[k], factor, lr, 0.01, 0.9, nesterov, maximize, scale, step == 0)
            assert np.array_equal(g.host(params[k].grad), a)  # the gradients stay as they are
            # a dozen roundings a step of numbers no larger than these
            assert (np.abs(g.host(params[k]) - want[k]) <= 40 * U * (np.abs(want[k]) + 2 * np.abs(bufs[k]) + np.abs(a) + 1)).all()
            assert (np.abs(g.host(opt.state[params[k]]["momentum_buffer"]) - bufs[k]) <= 40 * U * (np.abs(bufs[k]) + np.abs(a) + 1)).all()


def test_under_the_limit_the_update_is_the_one_without():
    import gpu_util as g
    import mytorch_b200.nn as nn
    from mytorch_b200.optim import SGD

    rng = np.random.default_rng(5)
    values = [rng.standard_normal(s).astype(np.float32) for s in (1000, 77, 4)]
    grads = [rng.standard_normal(s).astype(np.float32) for s in (1000, 77, 4)]
    results = []
    for limit in (None, 1e3):
        params = [nn.Parameter(g.dev(v)) for v in values]
        opt = SGD(params, lr=0.1, momentum=0.9, weight_decay=1e-3, max_grad_norm=limit)
        for _ in range(2):
            for p, a in zip(params, grads):
                p.grad = g.dev(a)
            opt.step()
        results.append([g.host(p) for p in params])
        assert (opt.grad_norm is None) == (limit is None)
    assert all(np.array_equal(a, b) for a, b in zip(*results))


def test_in_a_captured_step():
    import gpu_util as g
    import mytorch_b200 as mt
    import mytorch_b200.nn as nn
    import mytorch_b200.nn.functional as F
    from mytorch_b200.cuda_graph import StepGraph
    from mytorch_b200.optim import SGD

    rng = np.random.default_rng(6)
    tokens, labels = rng.integers(0, 50, (16, 1, 12)), rng.integers(0, 4, 16)

    def make():
        mt.manual_seed(1)
        net = nn.Sequential(nn.Embedding(50, 32, channels_first=True), nn.Conv2d(32, 32, (1, 3), padding=(0, 1)), nn.GroupNorm(4, 32, activation="silu"))
        head = nn.Linear(32, 4)
        net.to("cuda:0")
        head.to("cuda:0")
        opt = SGD(list(net.parameters()) + list(head.parameters()), lr=0.1, momentum=0.9, max_grad_norm=0.1)
        x, t = g.dev(tokens), g.dev(labels)

        def step():
            loss = F.cross_entropy(head(net(x).mean(dim=(2, 3))), t)
            opt.zero_grad()
            loss.backward()
            opt.step()
            return loss, opt.grad_norm
        return step, list(net.parameters()) + list(head.parameters())

    step, params = make()
    for _ in range(4):
        loss, norm = step()
    want = [g.host(p) for p in params] + [g.host(loss), g.host(norm)]
    step, params = make()
    step()  # the optimizer's first step makes its buffers
    graph = StepGraph(step)
    loss, norm = graph.capture()
    for _ in range(3):
        graph.replay()
    got = [g.host(p) for p in params] + [g.host(loss), g.host(norm)]
    graph.destroy()
    for a, b in zip(want, got):
        assert np.array_equal(a, b)


def test_example_learns():
    from mytorch_b200.examples.token_cnn import train_token_cnn

    losses, accuracy = train_token_cnn(steps=300, log=lambda line: None)
    assert np.isfinite(losses).all() and np.mean(losses[-20:]) < 0.5 * np.mean(losses[:20]) and accuracy > 0.8


def test_parameters_that_join_later():
    """A group that joins after the first step has its first update among others that have had theirs."""
    import gpu_util as g
    import mytorch_b200.nn as nn
    from mytorch_b200.optim import SGD

    rng = np.random.default_rng(12)
    values = [rng.standard_normal(s).astype(np.float32) for s in (300, 5000, 9)]
    params = [nn.Parameter(g.dev(v)) for v in values]
    opt = SGD(params[:1], lr=0.1, momentum=0.9, max_grad_norm=0.5)
    want, bufs = [v.astype(np.float64) for v in values], [np.zeros(v.shape) for v in values]
    for step in range(3):
        if step == 1:
            opt.param_groups.append(dict(opt.param_groups[0], params=params[1:]))
        grads = [rng.standard_normal(v.shape).astype(np.float32) for v in values[:3 if step else 1]]
        for p, a in zip(params, grads):
            p.grad = g.dev(a)
        opt.step()
        factor = min(1.0, 0.5 / (_norm(grads) + 1e-6))
        for k, a in enumerate(grads):
            want[k], bufs[k] = _sgd(want[k], a.astype(np.float64), bufs[k], factor, 0.1, 0.0, 0.9, False, False, 1.0, step == (k > 0))
            assert (np.abs(g.host(params[k]) - want[k]) <= 40 * U * (np.abs(want[k]) + 2 * np.abs(bufs[k]) + np.abs(a) + 1)).all()


def test_refusals_of_a_step():
    import gpu_util as g
    import mytorch_b200 as mt
    import mytorch_b200.nn as nn
    from mytorch_b200.optim import SGD, clip_grad_norm_
    from mytorch_b200.tensor import InvalidDataTypeError, MismatchDevicesError

    p, q = nn.Parameter(g.dev(np.ones(8, np.float32))), nn.Parameter(g.dev(np.ones((2, 4), np.float32)))
    opt = SGD([p, q], lr=1.0, momentum=0.9, max_grad_norm=100.0)
    p.grad = g.dev(np.ones(8, np.float32))
    for wrong, error in ((np.ones((4, 2), np.float32), RuntimeError), (np.ones((2, 4), np.int64), InvalidDataTypeError)):
        q.grad = g.dev(wrong)
        with pytest.raises(error):
            opt.step()
        assert not opt.state and (g.host(p) == 1).all()
    with pytest.raises(InvalidDataTypeError):
        clip_grad_norm_([p, q], 1.0)
    q.grad = mt.tensor(np.ones((2, 4), np.float32))
    for call in (opt.step, lambda: clip_grad_norm_([p, q], 1.0)):
        with pytest.raises((RuntimeError, MismatchDevicesError)):
            call()
    assert (g.host(p.grad) == 1).all()
    q.grad = g.dev(np.ones((2, 4), np.float32))
    opt.step()
    opt.state[q]["momentum_buffer"] = g.dev(np.ones(3, np.float32))
    with pytest.raises(RuntimeError, match="momentum buffer"):
        opt.step()
    assert (g.host(p) == 0).all()
