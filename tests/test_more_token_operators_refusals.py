"""What token_log_probs, the norms around a block and AdamW refuse, before anything reaches the GPU."""
import ctypes

import numpy as np
import pytest

import mytorch_b200 as mt
import mytorch_b200.nn as nn
import mytorch_b200.nn.functional as F
from mytorch_b200.backends.cuda.env import LIBRARY_PATH, NativeError, _binding
from mytorch_b200.optim import AdamW
from mytorch_b200.tensor import InvalidDataTypeError, InvalidShapeError, MismatchDataTypesError, MismatchShapesError

ADDRESS = 1 << 20  # never dereferenced


def _f32(*shape):
    return mt.tensor(np.zeros(shape, np.float32))


def test_token_log_probs_refuses():
    logits, tokens = _f32(3, 5), mt.tensor(np.zeros(3, np.int64))
    for shape in ((5,), (2, 3, 4, 5), (3, 0)):
        with pytest.raises(InvalidShapeError):
            F.token_log_probs(_f32(*shape), tokens)
    for dtype in (np.float32, np.int16, np.uint8):
        with pytest.raises(InvalidDataTypeError):
            F.token_log_probs(logits, mt.tensor(np.zeros(3, dtype)))
    for shape in ((4,), (3, 1), (1, 3)):
        with pytest.raises(MismatchShapesError):
            F.token_log_probs(logits, mt.tensor(np.zeros(shape, np.int64)))
    for top in (-1, 6, 33, 2.0, None):
        with pytest.raises(RuntimeError, match="top is from 0 to 32"):
            F.token_log_probs(logits, tokens, top)
    with pytest.raises(RuntimeError, match="top is from 0 to 32"):
        F.token_log_probs(_f32(3, 50), tokens, 33)
    with pytest.raises(RuntimeError, match="ignore_index"):
        F.token_log_probs(logits, tokens, ignore_index=0.5)
    with pytest.raises(RuntimeError, match="no function registered for token_log_probs on cpu"):
        F.token_log_probs(logits, tokens, 2)


def test_norms_refuse():
    x, w = _f32(2, 3, 8), _f32(8)
    for shape in ((8,), (1, 2, 3, 4, 5), (2, 0)):
        with pytest.raises(InvalidShapeError):
            F.rms_norm(_f32(*shape))
        with pytest.raises(InvalidShapeError):
            F.add_rms_norm(_f32(*shape), _f32(*shape))
    with pytest.raises(MismatchShapesError):
        F.rms_norm(x, _f32(3))
    with pytest.raises(MismatchShapesError):
        F.add_rms_norm(x, _f32(6, 8))
    for name, shape in (("weight", (1, 8)), ("post_weight", (3,)), ("gate", (3, 8)), ("gate", (2, 1, 8)), ("gate", (1,)), ("gate", (6, 8))):
        with pytest.raises(MismatchShapesError):
            F.add_rms_norm(x, x, **{name: _f32(*shape)})
    with pytest.raises(MismatchDataTypesError):
        F.add_rms_norm(x, x, mt.tensor(np.zeros(8)))
    with pytest.raises(RuntimeError, match="eps"):
        F.rms_norm(x, w, -1e-6)
    with pytest.raises(RuntimeError, match="eps"):
        F.add_rms_norm(x, x, eps=float("nan"))
    for call in (lambda: F.rms_norm(x, w), lambda: F.add_rms_norm(x, x, w, w, w), lambda: nn.RMSNorm(8)(x), lambda: nn.AddRMSNorm(8)(x, x)):
        with pytest.raises(RuntimeError, match="no function registered for add_rms_norm on cpu"):
            call()
    with pytest.raises(RuntimeError, match="a gate of its own"):
        nn.AddRMSNorm(8, gate=1.0)(x, x, w)
    assert {k: t.shape for k, t in nn.AddRMSNorm(8, gate=0.5).named_parameters()} == {"weight": (8,), "post_weight": (8,), "gate": (8,)}
    assert [k for k, _ in nn.AddRMSNorm(8, post_norm=False).named_parameters()] == ["weight"] and not list(nn.RMSNorm(8, affine=False).parameters())
    assert (nn.AddRMSNorm(8, gate=0.5).gate._numpy() == 0.5).all()


def test_adamw_refuses():
    p = nn.Parameter(_f32(4))
    for wrong in (dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(betas=(0.9,)), dict(lr=-1.0), dict(eps=-1.0), dict(weight_decay=float("nan"))):
        with pytest.raises(RuntimeError, match="betas are two numbers"):
            AdamW([p], **wrong)
        with pytest.raises(RuntimeError, match="betas are two numbers"):
            AdamW([{"params": [p], **wrong}])
    for bits in (4, 16, "8"):
        with pytest.raises(RuntimeError, match="state_bits"):
            AdamW([p], state_bits=bits)
    for limit in (-1.0, float("nan")):
        with pytest.raises(RuntimeError, match="max_grad_norm"):
            AdamW([p], max_grad_norm=limit)
    for bits in (8, 32):
        opt = AdamW([p], state_bits=bits)
        p.grad = _f32(4)
        with pytest.raises(RuntimeError, match="one CUDA device"):
            opt.step()
        assert not opt.state  # nothing was made for a step that did not happen


def test_entry_points_refuse_bad_arguments():
    _binding.load(LIBRARY_PATH, NativeError)
    lib, a, big = _binding, ADDRESS, 1 << 40
    five, four, one, two = (ctypes.c_void_p * 5)(a, a, a, a, a), (ctypes.c_void_p * 4)(a, a, a, a), (ctypes.c_longlong * 1)(300), (ctypes.c_longlong * 2)(300, 1)
    without = [(ctypes.c_void_p * 5)(*[None if i == k else a for i in range(5)]) for k in range(5)]
    off = [(ctypes.c_void_p * 5)(a, a, a + 4, a, a), (ctypes.c_void_p * 5)(a, a, a, a + 1, a)]
    numbers = (0.1, 0.9, 0.99, 1e-8, 0.0, 1.0)
    refused = [
        lambda: lib.token_log_probs_forward_f32(-1, 5, a, 0, a, 0, 0, 0, a, a, a, a, a, None),
        lambda: lib.token_log_probs_forward_f32(1 << 31, 5, a, 0, a, 0, 0, 0, a, a, a, a, a, None),
        lambda: lib.token_log_probs_forward_f32(2, 0, a, 0, a, 0, 0, 0, a, a, a, a, a, None),
        lambda: lib.token_log_probs_forward_f32(2, 5, a, 2, a, 0, 0, 0, a, a, a, a, a, None),
        lambda: lib.token_log_probs_forward_f32(2, 5, a, 0, a, 0, 0, 6, a, a, a, a, a, None),
        lambda: lib.token_log_probs_forward_f32(2, 50, a, 0, a, 0, 0, 33, a, a, a, a, a, None),
        lambda: lib.token_log_probs_forward_f32(2, 5, a, 0, a, 0, 0, 2, a, a, a, a, None, None),
        lambda: lib.token_log_probs_forward_f32(2, 5, a, 0, None, 0, 0, 2, a, a, a, a, a, None),
        lambda: lib.token_log_probs_backward_f32(2, 5, a, 0, a, 0, 0, 6, a, a, a, a, a, a, None),
        lambda: lib.token_log_probs_backward_f32(2, 5, a, 0, a, 0, 0, 2, a, a, a, a, None, a, None),
        lambda: lib.token_log_probs_backward_f32(2, 5, a, 0, a, 0, 0, 2, a, a, a, None, a, a, None),
        lambda: lib.token_log_probs_backward_f32(2, 5, a, 0, a, 0, 0, 2, a, a, a, a, a, None, None),
        lambda: lib.add_rms_norm_forward_f32(-1, 8, a, a, a, a, a, 1, 1.0, 1e-6, a, a, a, a, None),
        lambda: lib.add_rms_norm_forward_f32(1 << 31, 8, a, a, a, a, a, 1, 1.0, 1e-6, a, a, a, a, None),
        lambda: lib.add_rms_norm_forward_f32(6, 0, a, a, a, a, a, 1, 1.0, 1e-6, a, a, a, a, None),
        lambda: lib.add_rms_norm_forward_f32(6, 8, a, a, a, a, a, 4, 1.0, 1e-6, a, a, a, a, None),
        lambda: lib.add_rms_norm_forward_f32(6, 8, a, a, a, a, a, 0, 1.0, 1e-6, a, a, a, a, None),
        lambda: lib.add_rms_norm_forward_f32(6, 8, a, a, a, a, a, 1, 1.0, -1.0, a, a, a, a, None),
        lambda: lib.add_rms_norm_forward_f32(6, 8, a, a, a, a, a, 1, 1.0, 1e-6, None, a, a, a, None),
        lambda: lib.add_rms_norm_forward_f32(6, 8, a, None, a, a, None, 1, 1.0, 1e-6, a, a, a, a, None),
        lambda: lib.add_rms_norm_forward_f32(6, 8, a, None, a, None, a, 1, 1.0, 1e-6, a, a, a, a, None),
        lambda: lib.add_rms_norm_backward_f32(6, 8, a, a, None, a, a, a, a, a, a, 1, 1.0, a, a, a, a, a, a, big, None),
        lambda: lib.add_rms_norm_backward_f32(6, 8, a, a, a, a, a, None, a, a, a, 1, 1.0, a, a, a, a, a, a, big, None),
        lambda: lib.add_rms_norm_backward_f32(6, 8, a, a, a, a, a, a, a, a, a, 5, 1.0, a, a, a, a, a, a, big, None),
        lambda: lib.add_rms_norm_backward_f32(6, 8, a, a, a, a, a, a, a, a, a, 1, 1.0, a, a, a, a, a, a, 8, None),
        lambda: lib.adamw_f32(1, None, one, *numbers, None, 0, -1.0, None, a, None),
        lambda: lib.adamw_f32(1, five, one, *numbers, None, 0, -1.0, None, None, None),
        lambda: lib.adamw_f32(1, five, one, *numbers, a, 0, 1.0, None, a, None),
        lambda: lib.adamw_f32(1, five, one, 0.1, 1.0, 0.99, 1e-8, 0.0, 1.0, None, 0, -1.0, None, a, None),
        lambda: lib.adamw8_f32(1, five, two, 0.1, 0.9, 1 - 1e-7, 1e-8, 0.0, 1.0, None, 0, -1.0, None, a, None),
        lambda: lib.adamw8_f32(1, five, (ctypes.c_longlong * 2)(-1, 0), *numbers, None, 0, -1.0, None, a, None),
        lambda: lib.adamw8_moments_f32(1, None, one, None),
        lambda: lib.adamw8_moments_f32(1, (ctypes.c_void_p * 4)(a + 8, a, a, a), one, None),
        lambda: lib.adamw8_moments_f32(1, (ctypes.c_void_p * 4)(a, a, a, None), one, None),
    ]
    refused += [lambda t=t: lib.adamw_f32(1, t, one, *numbers, None, 0, -1.0, None, a, None) for t in without]
    refused += [lambda t=t: lib.adamw8_f32(1, t, two, *numbers, None, 0, -1.0, None, a, None) for t in without + off]
    for call in refused:
        with pytest.raises(NativeError):
            call()
    # over nothing: nothing to do, and no GPU needed
    assert lib.token_log_probs_forward_f32(0, 5, None, 0, None, 0, 0, 2, None, None, None, None, None, None) == 0
    assert lib.token_log_probs_backward_f32(0, 5, None, 0, None, 0, 0, 2, None, None, None, None, None, None, None) == 0
    assert lib.add_rms_norm_forward_f32(0, 8, None, None, None, None, None, 1, 1.0, 1e-6, None, None, None, None, None) == 0
    assert lib.adamw_f32(0, None, None, *numbers, None, 0, -1.0, None, None, None) == 0 and lib.adamw8_moments_f32(0, four, one, None) == 0
