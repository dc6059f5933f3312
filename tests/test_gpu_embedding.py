"""Embedding lookup (bit by bit) and its gradient (against 64 bits).

A gradient's value is a sum of k numbers added up in 32 bits in some fixed order, times the scale: off by at most (k + 2) 2^-24 times the sum of their
sizes (times the scale's)."""
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


def _tokens(rng, count, rows, skew):
    if skew == "same":
        return np.full(count, rows // 2)
    if skew == "uniform":
        return rng.integers(0, rows, count)
    order = rng.permutation(rows)
    return order[np.minimum(np.exp(rng.random(count) * np.log(rows + 1)).astype(np.int64) - 1, rows - 1)]


def _gradient(tokens, dy, rows, scale, padding=None):
    """(gradient, bound of what it may be off) in 64 bits; tokens outside the table count nothing."""
    t = tokens.reshape(-1).astype(np.int64)
    kept = (t >= 0) & (t < rows) & (t != (-1 if padding is None else padding))
    dy = dy.reshape(t.size, -1).astype(np.float64)[kept] * scale
    t = t[kept]
    order = np.argsort(t, kind="stable")
    starts = np.flatnonzero(np.diff(t[order], prepend=-1))
    want, size = np.zeros((2, rows, dy.shape[1]))
    if t.size:
        want[t[order][starts]] = np.add.reduceat(dy[order], starts)
        size[t[order][starts]] = np.add.reduceat(np.abs(dy[order]), starts)
    count = np.bincount(t, minlength=rows)[:, None]
    return want, (count + 2) * U * size


CASES = [  # tokens, rows, width, how they are distributed
    (1, 1, 1, "uniform"), (1, 5000, 64, "uniform"), (2, 3, 4, "same"), (33, 100, 3, "uniform"), (1000, 100, 32, "text"), (1000, 2, 300, "uniform"),
    (5000, 70001, 24, "text"), (8191, 10007, 300, "text"), (70000, 50, 8, "same"), (70000, 50000, 16, "uniform"), (3000, 300, 1025, "text"),
    (20000, 1000, 130, "same"), (40000, 300000, 4, "text"), (300, 20, 2048, "uniform"), (4097, 4097, 31, "text"), (140000, 900, 5, "text")]


@pytest.mark.parametrize("index", [np.int32, np.int64])
@pytest.mark.parametrize("count,rows,width,skew", CASES)
def test_lookup_and_gradient(count, rows, width, skew, index):
    import gpu_util as g
    import mytorch_b200.nn.functional as F

    rng = np.random.default_rng(count + rows + width)
    tokens = _tokens(rng, count, rows, skew).astype(index)
    table, dy = rng.standard_normal((rows, width), dtype=np.float32), rng.standard_normal((count, width), dtype=np.float32)
    scale = np.float32(width ** 0.5)
    tt, wt = g.dev(tokens), g.dev(table, True)
    out = F.embedding(tt, wt, scale=float(scale))
    assert out.shape == (count, width) and np.array_equal(g.host(out), table[tokens] * scale)
    want, bound = _gradient(tokens, dy, rows, float(scale))
    dyt = g.dev(dy)
    got = g.host(g.op("embedding_backward")(dyt, tt, wt, float(scale))[0])
    assert (np.abs(got - want) <= bound).all()
    assert np.array_equal(got, g.host(g.op("embedding_backward")(dyt, tt, wt, float(scale))[0]))  # the same bits every time


@pytest.mark.parametrize("padding", [0, 7, 99, -1, -100])
def test_padding_gets_no_gradient(padding):
    import gpu_util as g
    import mytorch_b200.nn.functional as F

    rng = np.random.default_rng(4)
    tokens = _tokens(rng, 2000, 100, "text")
    tokens[::3] = padding % 100
    table, dy = rng.standard_normal((100, 20), dtype=np.float32), rng.standard_normal((2000, 20), dtype=np.float32)
    wt = g.dev(table, True)
    out = F.embedding(g.dev(tokens), wt, padding_idx=padding)
    assert np.array_equal(g.host(out), table[tokens])
    (out * g.dev(dy)).sum().backward()
    want, bound = _gradient(tokens, dy, 100, 1.0, padding % 100)
    got = g.host(wt.grad)
    assert not got[padding].any() and (np.abs(got - want) <= bound).all()


@pytest.mark.parametrize("index", [np.int32, np.int64])
def test_tokens_outside_the_table(index):
    """Their rows are NaN and their gradient is nobody's, also where the low 32 bits of a token name a row."""
    import gpu_util as g
    import mytorch_b200.nn.functional as F

    rng = np.random.default_rng(5)
    tokens = rng.integers(0, 50, 600).astype(index)
    outside = [-1, 50, 51, 2 ** 31 - 1, -2 ** 31] + ([2 ** 32, 2 ** 32 + 3, -2 ** 32, 2 ** 62] if index is np.int64 else [])
    for i, v in enumerate(outside):
        tokens[10 + 40 * i] = v
    table, dy = rng.standard_normal((50, 36), dtype=np.float32), rng.standard_normal((600, 36), dtype=np.float32)
    bad = (tokens < 0) | (tokens >= 50)
    got = g.host(F.embedding(g.dev(tokens), g.dev(table)))
    assert np.isnan(got[bad]).all() and np.array_equal(got[~bad], table[tokens[~bad]])
    want, bound = _gradient(tokens, dy, 50, 1.0)
    assert (np.abs(g.host(g.op("embedding_backward")(g.dev(dy), g.dev(tokens), g.dev(table))[0]) - want) <= bound).all()
    nobody = g.dev(np.full(100, 50, index))
    assert not g.host(g.op("embedding_backward")(g.dev(dy[:100]), nobody, g.dev(table))[0]).any()


@pytest.mark.parametrize("shape", [(), (5,), (3, 4), (2, 3, 4), (2, 1, 9), (2, 2, 3, 2)])
@pytest.mark.parametrize("channels_first", [False, True])
def test_shapes(shape, channels_first):
    import gpu_util as g
    import mytorch_b200 as mt
    import mytorch_b200.nn.functional as F

    if channels_first and len(shape) != 3:
        pytest.skip("channels_first takes three dimensions")
    rng = np.random.default_rng(6)
    tokens = rng.integers(0, 11, shape)
    table = rng.standard_normal((11, 12), dtype=np.float32)
    wt = g.dev(table, True)
    out = F.embedding(mt.tensor(tokens, device="cuda:0"), wt, channels_first=channels_first)
    want = table[tokens]
    if channels_first:
        want = want.transpose(0, 3, 1, 2)
    assert out.shape == want.shape and np.array_equal(g.host(out), want)
    if shape:
        dy = rng.standard_normal(out.shape).astype(np.float32)
        (out * g.dev(dy)).sum().backward()
        rows = dy.transpose(0, 2, 3, 1) if channels_first else dy
        expected, bound = _gradient(tokens, np.ascontiguousarray(rows), 11, 1.0)
        assert (np.abs(g.host(wt.grad) - expected) <= bound).all()


def test_no_tokens():
    import gpu_util as g
    import mytorch_b200.nn.functional as F

    wt = g.dev(np.ones((5, 3), np.float32), True)
    out = F.embedding(g.dev(np.zeros((0,), np.int64)), wt)
    assert out.shape == (0, 3)
    assert not g.host(g.op("embedding_backward")(out, g.dev(np.zeros((0,), np.int64)), wt)[0]).any()


@pytest.mark.parametrize("offset", [1, 2, 3])
@pytest.mark.parametrize("width", [32, 30])
def test_windows_at_any_float(width, offset):
    import gpu_util as g
    import mytorch_b200 as mt
    from mytorch_b200.backends.cuda.env import CudaMemory, CudaMemoryView

    def window(array):
        view = CudaMemoryView(CudaMemory(0, 4 * (array.size + 4)), 4 * offset, 4 * array.size, 0)
        view.write(array)
        return mt.Tensor._on_device(array.shape, mt.float32, mt.Device("cuda:0"), view)

    rng = np.random.default_rng(7)
    tokens = _tokens(rng, 700, 90, "text")
    table, dy = rng.standard_normal((90, width), dtype=np.float32), rng.standard_normal((700, width), dtype=np.float32)
    wt = window(table)
    assert np.array_equal(g.host(g.op("embedding")(g.dev(tokens), wt, 2.0)), table[tokens] * 2)
    want, bound = _gradient(tokens, dy, 90, 2.0)
    assert (np.abs(g.host(g.op("embedding_backward")(window(dy), g.dev(tokens), wt, 2.0)[0]) - want) <= bound).all()


def test_gradient_against_differences():
    """sum(out dy) is linear in the table: its slope along a direction is a difference of two lookups."""
    import gpu_util as g
    import mytorch_b200.nn.functional as F

    rng = np.random.default_rng(8)
    tokens = _tokens(rng, 500, 60, "text")
    table, d, dy = rng.standard_normal((60, 16), dtype=np.float32), rng.standard_normal((60, 16)), rng.standard_normal((500, 16), dtype=np.float32)
    wt = g.dev(table, True)
    (F.embedding(g.dev(tokens), wt, scale=4.0) * g.dev(dy)).sum().backward()
    want = (4 * ((table + d)[tokens] - (table - d)[tokens]) / 2 * dy.astype(np.float64)).sum()
    assert abs((g.host(wt.grad) * d).sum() - want) <= 1e-5 * np.abs(g.host(wt.grad) * d).sum()


def test_the_layer_and_a_table_used_twice():
    import gpu_util as g
    import mytorch_b200 as mt
    import mytorch_b200.nn as nn

    mt.manual_seed(3)
    layer = nn.Embedding(20, 8, padding_idx=2)
    assert not layer.weight._numpy()[2].any() and layer.weight._numpy()[3].any()
    layer.to("cuda:0")
    rng = np.random.default_rng(9)
    a, b = rng.integers(0, 20, (2, 30))
    dy = rng.standard_normal((2, 30, 8), dtype=np.float32)
    (layer(g.dev(a)) * g.dev(dy[0]) + layer(g.dev(b)) * g.dev(dy[1])).sum().backward()
    want, bound = _gradient(np.concatenate([a, b]), dy, 20, 1.0, 2)
    assert (np.abs(g.host(layer.weight.grad) - want) <= 2 * bound).all()


@pytest.mark.parametrize("count", [511, 512, 513, 2048, 4095, 4096, 4098])
@pytest.mark.parametrize("skew", ["uniform", "same", "text"])
def test_as_many_tokens_as_one_block_orders(count, skew):
    import gpu_util as g

    rng = np.random.default_rng(count)
    tokens = _tokens(rng, count, 3000, skew)
    table, dy = np.zeros((3000, 6), np.float32), rng.standard_normal((count, 6), dtype=np.float32)
    want, bound = _gradient(tokens, dy, 3000, 1.0)
    got = g.host(g.op("embedding_backward")(g.dev(dy), g.dev(tokens), g.dev(table), 1.0)[0])
    assert (np.abs(got - want) <= bound).all()


@pytest.mark.parametrize("count", [1300000, 1310000, 1212415])
def test_shares_larger_than_shared_memory(count):
    """Where a CTA's share of the tokens is written straight to memory, the last one's rest is too."""
    import gpu_util as g

    rng = np.random.default_rng(count)
    tokens, dy = rng.integers(0, 5000, count), rng.standard_normal((count, 4), dtype=np.float32)
    want, bound = _gradient(tokens, dy, 5000, 1.0)
    got = g.host(g.op("embedding_backward")(g.dev(dy), g.dev(tokens), g.dev(np.zeros((5000, 4), np.float32)), 1.0)[0])
    assert (np.abs(got - want) <= bound).all()


@pytest.mark.parametrize("count,width", [(33000, 512), (50000, 337)])
def test_results_larger_than_half_of_l2(count, width):
    import gpu_util as g
    import mytorch_b200.nn.functional as F

    rng = np.random.default_rng(width)
    tokens, table = rng.integers(-1, 301, count), rng.standard_normal((300, width), dtype=np.float32)
    out = g.host(F.embedding(g.dev(tokens), g.dev(table), scale=2.0))
    inside = (tokens >= 0) & (tokens < 300)
    assert np.array_equal(out[inside], 2 * table[tokens[inside]]) and np.isnan(out[~inside]).all()


@pytest.mark.parametrize("count,width", [(2100001, 1023), (8400001, 1024)])
def test_offsets_beyond_32_bits(count, width):
    """2^31 values and more, 2^31 vectors of four and more: whole numbers, whose sums are exact."""
    import gpu_util as g
    import mytorch_b200 as mt
    import mytorch_b200.nn.functional as F
    from mytorch_b200.backends.cuda.env import CudaEnv, CudaMemoryView

    rng = np.random.default_rng(1)
    tokens, table = rng.integers(0, 700, count).astype(np.int32), rng.integers(-3, 4, (700, width)).astype(np.float32)
    tt, wt = g.dev(tokens), g.dev(table)
    out = F.embedding(tt, wt)
    rows = 5
    for first in (0, count // 2, count - rows):
        part = CudaMemoryView(out._native_array, 4 * first * width, 4 * rows * width, 0)
        assert np.array_equal(g.host(mt.Tensor._on_device((rows, width), mt.float32, out.device, part)), table[tokens[first:first + rows]])
    got = g.host(g.op("embedding_backward")(out, tt, wt, 1.0)[0])
    assert np.array_equal(got, np.bincount(tokens, minlength=700)[:, None] * table)
    del out
    CudaEnv.instance().lib.pool_trim()
