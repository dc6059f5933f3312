"""Paths of the token operators that the operators' own tests do not reach: updates of tensors off 16 bytes, slabs through memory with values that strain the
statistics, two host threads on one device's scratch, a layer made on the device.  Bounds as in those tests."""
import threading

import numpy as np
import pytest
from test_gpu_clip import U, _norm, _sgd
from test_gpu_embedding import _gradient, _tokens
from test_gpu_group_norm import Oracle, _check_backward, _check_forward, _inputs

pytestmark = pytest.mark.gpu

THROUGH_MEMORY = [((2, 64, 200, 200), 2), ((1, 30, 260, 250), 1), ((40, 2052, 1, 1), 2)]


def _window(array, offset):
    """A tensor that begins `offset` floats into its block."""
    import mytorch_b200 as mt
    from mytorch_b200.backends.cuda.env import CudaMemory, CudaMemoryView

    view = CudaMemoryView(CudaMemory(0, 4 * (array.size + 4)), 4 * offset, 4 * array.size, 0)
    view.write(array)
    return mt.Tensor._on_device(array.shape, mt.float32, mt.Device("cuda:0"), view)


@pytest.mark.parametrize("offsets", [(1, 1, 1), (3, 3, 3), (2, 2, 2), (0, 1, 0), (1, 0, 0), (0, 0, 3), (1, 2, 3)])  # parameter, gradient, buffer
@pytest.mark.parametrize("first", [True, False])
@pytest.mark.parametrize("sizes", [[5, 1, 3], [2048, 2049, 2047], [30001, 70, 4097]])
def test_an_update_with_clipping_off_16_bytes(sizes, first, offsets):
    import gpu_util as g
    import mytorch_b200.nn as nn
    from mytorch_b200.optim import SGD

    rng = np.random.default_rng(sizes[0])
    f32 = lambda: [rng.standard_normal(s).astype(np.float32) for s in sizes]
    values, grads, bufs = f32(), f32(), f32()
    params = [nn.Parameter(_window(v, offsets[0])) for v in values]
    assert all(p._native_array.ptr % 16 == 4 * offsets[0] for p in params)
    opt = SGD(params, lr=0.1, momentum=0.9, weight_decay=0.01, max_grad_norm=0.5)
    for p, a, b in zip(params, grads, bufs):
        p.grad = _window(a, offsets[1])
        if not first:
            opt.state[p] = {"momentum_buffer": _window(b, offsets[2])}
    opt.step()
    norm = _norm(grads)
    assert abs(g.host(opt.grad_norm)[0] - norm) <= 2 * U * norm
    factor = min(1.0, 0.5 / (norm + 1e-6))
    for p, v, a, b in zip(params, values, grads, bufs):
        want, buf = _sgd(v.astype(np.float64), a.astype(np.float64), b.astype(np.float64), factor, 0.1, 0.01, 0.9, False, False, 1.0, first)
        assert (np.abs(g.host(p) - want) <= 40 * U * (np.abs(want) + 2 * np.abs(buf) + np.abs(a) + 1)).all()
        assert (np.abs(g.host(opt.state[p]["momentum_buffer"]) - buf) <= 40 * U * (np.abs(buf) + np.abs(a) + 1)).all()
        assert np.array_equal(g.host(p.grad), a)


def _device(a):
    import gpu_util as g

    return g.dev(a.reshape(a.shape[:2]) if a.shape[2:] == (1, 1) else a)


@pytest.mark.parametrize("shape,groups", THROUGH_MEMORY)
def test_a_mean_far_from_zero_through_memory(shape, groups):
    import gpu_util as g

    x, dy, gamma, beta = _inputs(shape, groups, 3, mean=1000.0)
    o = Oracle(x, groups, gamma, beta, 1e-5, "silu")
    xt, gt, bt = _device(x), g.dev(gamma), g.dev(beta)
    y, mean, rstd = g.op("group_norm")(xt, groups, gt, bt, 1e-5, "silu")
    _check_forward(g.host(y).reshape(shape), o)
    assert (np.abs(g.host(rstd) / o.rstd - 1) <= 1e-5).all()
    got = g.op("group_norm_backward")(_device(dy), mean, rstd, xt, gt, bt, groups, "silu")
    _check_backward([g.host(t).reshape(w) for t, w in zip(got, (shape, gamma.shape, beta.shape))], o, dy, "silu")


@pytest.mark.parametrize("shape,groups", THROUGH_MEMORY)
def test_one_value_far_from_the_others_through_memory(shape, groups):
    """Also as a thread's first value, from which it counts the others."""
    import gpu_util as g

    for at in (0, 5, -1):
        x, _, gamma, beta = _inputs(shape, groups, 4)
        x.reshape(shape[0], -1)[:, at] = 3e4
        o = Oracle(x, groups, gamma, beta, 1e-5, None)
        y, mean, rstd = g.op("group_norm")(_device(x), groups, g.dev(gamma), g.dev(beta), 1e-5, None)
        _check_forward(g.host(y).reshape(shape), o)
        assert (np.abs(g.host(rstd) / o.rstd - 1) <= 1e-5).all()


@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("shape,groups", [((2, 64, 200, 200), 2), ((40, 2052, 1, 1), 2)])
def test_a_bad_value_stays_in_its_group_through_memory(shape, groups, bad):
    import gpu_util as g

    x, dy, gamma, beta = _inputs(shape, groups, 11)
    gt, bt, dyt = g.dev(gamma), g.dev(beta), _device(dy)

    def both(x):
        xt = _device(x)
        y, mean, rstd = g.op("group_norm")(xt, groups, gt, bt, 1e-5, "silu")
        dx = g.op("group_norm_backward")(dyt, mean, rstd, xt, gt, bt, groups, "silu", (True, False, False))[0]
        return g.host(y).reshape(shape), g.host(dx).reshape(shape)

    clean = both(x)
    half = shape[1] // 2
    x[1, half + 3, shape[2] // 2, shape[3] // 3] = bad
    for got, want in zip(both(x), clean):
        assert np.isnan(got[1, half:]).all()
        got[1, half:] = want[1, half:]
        assert np.array_equal(got, want)


def test_two_threads_on_one_scratch():
    import gpu_util as g

    rng = np.random.default_rng(0)

    def norm(shape, groups):
        x, dy, gamma, beta = _inputs(shape, groups, shape[1])

        def run():
            xt, gt, bt = _device(x), g.dev(gamma), g.dev(beta)
            y, mean, rstd = g.op("group_norm")(xt, groups, gt, bt, 1e-5, "silu")
            return [y, mean, rstd, *g.op("group_norm_backward")(_device(dy), mean, rstd, xt, gt, bt, groups, "silu")]
        return run

    def embedding(count, rows, width):
        tokens = _tokens(rng, count, rows, "text")
        dy, table = rng.standard_normal((count, width), dtype=np.float32), np.zeros((rows, width), np.float32)
        return lambda: g.op("embedding_backward")(g.dev(dy), g.dev(tokens), g.dev(table), 1.0)

    cases = [norm((1, 30, 260, 250), 1), embedding(20000, 900, 24), norm((8, 32, 30, 30), 4), embedding(3000, 100, 40), norm((1500, 64, 1, 1), 4)]
    alone = [[g.host(t) for t in run()] for run in cases]
    wrong = []

    def worker(order):
        for _ in range(15):
            results = [(i, cases[i]()) for i in order]
            for i, tensors in results:
                if not all(np.array_equal(g.host(t), want) for t, want in zip(tensors, alone[i])):
                    wrong.append(i)

    threads = [threading.Thread(target=worker, args=(order,)) for order in ((0, 1, 2, 3, 4), (1, 4, 0, 3, 2))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_a_layer_made_on_the_device():
    import gpu_util as g
    import mytorch_b200.nn as nn

    layer = nn.Embedding(30, 8, padding_idx=4, device="cuda:0")
    rows = g.host(layer.weight)
    assert not rows[4].any() and np.delete(rows, 4, 0).all()
    tokens, dy = np.arange(60) % 30, np.ones((60, 8), np.float32)
    (layer(g.dev(tokens)) * g.dev(dy)).sum().backward()
    want, bound = _gradient(tokens, dy, 30, 1.0, 4)
    assert (np.abs(g.host(layer.weight.grad) - want) <= bound).all()
