"""A tensor that a call takes in two roles gets its window of the flat buffer for one of the two gradients: they are written side by side, and added up by the tape."""
import numpy as np
import pytest

import mytorch_b200 as mt
from mytorch_b200.backends.cuda import ops


class _Library:
    def __init__(self):
        self.given = {}

    def __getattr__(self, name):
        def call(*args):
            self.given[name] = args
            return 0
        return call


class _Env:
    def __init__(self):
        self.lib = _Library()

    def workspace(self, need):
        return 0, 0

    def stream(self):
        return 0


def _t(*shape):
    t = mt.tensor(np.ones(shape, np.float32))
    t.requires_grad = True
    return t


def _add_rms_norm(w):
    x, row = _t(4, 6), _t(4)
    return ops.cuda_add_rms_norm_backward(x, x, x, row, row, x, x, w, w, w)[2:]


def _group_norm(w):
    x, row = _t(4, 6), _t(4, 2)
    return ops.cuda_group_norm_backward(x, row, row, x, w, w, 2, None)[1:]


def _batch_norm(w):
    x, c = _t(2, 6, 3, 3), _t(6)
    return ops.cuda_batch_norm2d_backward(x, c, c, x, w, w, 1e-5)[1:]


def _batch_norm_add_relu(w):
    x, c = _t(2, 6, 3, 3), _t(6)
    return ops.cuda_batch_norm2d_add_relu_backward(x, c, c, x, x, w, w, 1e-5)[2:]


@pytest.mark.parametrize("call", [_add_rms_norm, _group_norm, _batch_norm, _batch_norm_add_relu])
def test_a_window_once_a_call(monkeypatch, call):
    env = _Env()
    monkeypatch.setattr(ops, "_env", lambda t: env)
    monkeypatch.setattr(ops, "_new", lambda shape, like, dtype=None: mt.tensor(np.zeros(shape, np.float32)))
    monkeypatch.setattr(ops, "_aligned", lambda *t: False)
    w = _t(6)
    w._grad_slot = object()
    got = call(w)
    assert len(got) >= 2 and got[0]._native_array is w._grad_slot
    assert all(t._native_array is not w._grad_slot for t in got[1:])
    written = [id(t) for args in env.lib.given.values() for t in args if any(t is r for r in got)]
    assert len(set(written)) == len(got)  # each is written to, in a place of its own
    w.grad = _t(6)  # there is a gradient already: none goes to the window
    assert all(t._native_array is not w._grad_slot for t in call(w))


@pytest.mark.parametrize("shape", [(4, 0, 6), (4, 6, 0, 3)])
def test_a_gate_of_no_rows_is_cleared(monkeypatch, shape):
    """A row of the gate a sample, and samples without a position: no kernel writes its gradient."""
    env = _Env()
    monkeypatch.setattr(ops, "_env", lambda t: env)
    monkeypatch.setattr(ops, "_new", lambda shape, like, dtype=None: mt.tensor(np.full(shape, 7, np.float32)))
    x, row, gate = _t(*shape), _t(0), _t(4, 6)
    dgate = ops.cuda_add_rms_norm_backward(x, x, x, row, row, x, x, None, None, gate)[4]
    assert dgate.shape == (4, 6)
    cleared = env.lib.given.get("memset_async")
    assert cleared is not None and cleared[0] is dgate and cleared[1:3] == (0, 4 * 24)
