"""What group_norm, embedding and gradient clipping refuse, before anything reaches the GPU."""
import numpy as np
import pytest

import mytorch_b200 as mt
import mytorch_b200.nn as nn
import mytorch_b200.nn.functional as F
from mytorch_b200.backends.cuda.env import LIBRARY_PATH, NativeError, _binding
from mytorch_b200.optim import SGD, clip_grad_norm_, grad_norm
from mytorch_b200.tensor import InvalidDataTypeError, InvalidShapeError, MismatchDataTypesError, MismatchShapesError

ADDRESS = 1 << 20  # never dereferenced


def _f32(*shape):
    return mt.tensor(np.zeros(shape, np.float32))


def test_group_norm_refuses():
    x, w = _f32(2, 8, 3, 3), _f32(8)
    with pytest.raises(RuntimeError, match="expects an input"):
        F.group_norm(_f32(2, 8, 3), 2)
    for groups in (3, 0, -2, 16, 2.0):
        with pytest.raises(RuntimeError, match="no .* groups"):
            F.group_norm(x, groups)
    with pytest.raises(RuntimeError, match="activation"):
        F.group_norm(x, 2, activation="tanh")
    with pytest.raises(MismatchShapesError):
        F.group_norm(x, 2, _f32(4))
    with pytest.raises(MismatchShapesError):
        F.group_norm(x, 2, w, _f32(8, 1))
    with pytest.raises(MismatchDataTypesError):
        F.group_norm(x, 2, mt.tensor(np.zeros(8)))
    with pytest.raises(RuntimeError, match="no function registered for group_norm on cpu"):
        F.group_norm(x, 2, w, w)
    with pytest.raises(RuntimeError, match="groups"):
        nn.GroupNorm(3, 8)


def test_embedding_refuses():
    table = _f32(10, 4)
    for dtype in (np.float32, np.int16, np.uint8):
        with pytest.raises(InvalidDataTypeError):
            F.embedding(mt.tensor(np.zeros(3, dtype)), table)
    tokens = mt.tensor(np.zeros((2, 3), np.int64))
    with pytest.raises(InvalidShapeError):
        F.embedding(tokens, _f32(10))
    with pytest.raises(RuntimeError, match="channels_first"):
        F.embedding(tokens, table, channels_first=True)
    for padding in (10, -11):
        with pytest.raises(RuntimeError, match="padding_idx"):
            F.embedding(tokens, table, padding_idx=padding)
        with pytest.raises(RuntimeError, match="padding_idx"):
            nn.Embedding(10, 4, padding_idx=padding)
    with pytest.raises(RuntimeError, match="no function registered for embedding on cpu"):
        F.embedding(tokens, table)


def test_clipping_refuses():
    p = nn.Parameter(_f32(4))
    for call in (lambda: grad_norm([p]), lambda: clip_grad_norm_([], 1.0)):
        with pytest.raises(RuntimeError, match="no gradient"):
            call()
    p.grad = _f32(4)
    for limit in (-1.0, float("nan")):
        with pytest.raises(RuntimeError, match="max_norm"):
            clip_grad_norm_([p], limit)
        with pytest.raises(RuntimeError, match="max_grad_norm"):
            SGD([p], max_grad_norm=limit)
    with pytest.raises(RuntimeError, match="no function registered for clip_gradients on cpu"):
        clip_grad_norm_([p], 1.0)
    opt = SGD([p], max_grad_norm=1.0)
    with pytest.raises(RuntimeError, match="one CUDA device"):
        opt.step()
    assert not opt.state  # nothing was made for a step that did not happen


def test_entry_points_refuse_bad_arguments():
    _binding.load(LIBRARY_PATH, NativeError)
    lib, a = _binding, ADDRESS
    big = 1 << 40
    refused = [
        lambda: lib.group_norm_forward_f32(2, 8, 9, 3, a, a, a, 1e-5, 0, a, a, a, a, big, None),
        lambda: lib.group_norm_forward_f32(2, 8, 9, 0, a, a, a, 1e-5, 0, a, a, a, a, big, None),
        lambda: lib.group_norm_forward_f32(-1, 8, 9, 2, a, a, a, 1e-5, 0, a, a, a, a, big, None),
        lambda: lib.group_norm_forward_f32(2, 8, 9, 2, a, a, a, 1e-5, 3, a, a, a, a, big, None),
        lambda: lib.group_norm_forward_f32(2, 8, 9, 2, None, a, a, 1e-5, 0, a, a, a, a, big, None),
        lambda: lib.group_norm_backward_f32(2, 8, 9, 3, a, a, a, a, a, a, 0, a, a, a, a, big, None),
        lambda: lib.group_norm_backward_f32(2, 8, 9, 2, a, a, a, a, a, a, -1, a, a, a, a, big, None),
        lambda: lib.group_norm_backward_f32(2, 8, 9, 2, None, a, a, a, a, a, 0, a, a, a, a, big, None),
        lambda: lib.group_norm_backward_f32(2, 8, 9, 2, a, a, a, a, a, a, 0, a, a, a, a, 8, None),
        lambda: lib.embedding_forward_f32(2, a, 4, 10, 4, a, 1.0, a, None),
        lambda: lib.embedding_forward_f32(0, a, -1, 10, 4, a, 1.0, a, None),
        lambda: lib.embedding_forward_f32(0, None, 4, 10, 4, a, 1.0, a, None),
        lambda: lib.embedding_forward_f32(0, a, 4, 0, 4, a, 1.0, a, None),
        lambda: lib.embedding_backward_f32(2, a, 4, 10, 4, a, 1.0, -1, a, a, big, None),
        lambda: lib.embedding_backward_f32(1, a, 4, 10, 4, None, 1.0, -1, a, a, big, None),
        lambda: lib.embedding_backward_f32(1, a, 4, 10, 4, a, 1.0, -1, None, a, big, None),
        lambda: lib.embedding_backward_f32(1, a, 4, 10, 4, a, 1.0, -1, a, a, 8, None),
        lambda: lib.grad_norm_f32(1, None, None, None, None),
        lambda: lib.clip_grads_f32(1, None, None, a, 1, 1.0, a, None),
        lambda: lib.sgd_multi_clipped_f32(0, None, None, None, None, None, 0.1, 0.0, 0.0, 0.0, 0, 0, 1.0, None, 0, 1.0, a, None),
    ]
    for call in refused:
        with pytest.raises(NativeError):
            call()
    # over no elements: nothing to do, and no GPU needed
    assert lib.group_norm_forward_f32(0, 8, 9, 2, None, None, None, 1e-5, 0, None, None, None, None, 0, None) == 0
    assert lib.embedding_forward_f32(1, None, 0, 10, 4, None, 1.0, None, None) == 0
