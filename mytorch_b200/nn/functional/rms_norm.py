"""The norm of the channels of a position by their root mean square, by itself and around a residual block (no counterpart in the reference)."""
from mytorch_b200.ops._common import dispatch, grad_enabled, record, tracker
from mytorch_b200.tensor import InvalidShapeError, MismatchDataTypesError, MismatchDevicesError, MismatchShapesError, Tensor


def _channels(x):
    if len(x.shape) not in (2, 3, 4):
        raise InvalidShapeError(x.shape)
    channels = x.shape[1] if len(x.shape) == 4 else x.shape[-1]
    if channels < 1:
        raise InvalidShapeError(x.shape)
    return channels


def _check(x, eps, *others):
    """others: (tensor or None, the shapes that it may have)"""
    for t, shapes in others:
        if t is not None:
            if t.shape not in shapes:
                raise MismatchShapesError([x.shape, t.shape])
            if t.device is not x.device:
                raise MismatchDevicesError([x.device, t.device])
            if t.dtype is not x.dtype:
                raise MismatchDataTypesError([x.dtype, t.dtype])
    if not eps >= 0:
        raise RuntimeError(f"rms_norm: eps is a number from 0 up: {eps}")


def rms_norm(x: Tensor, weight=None, eps=1e-6) -> Tensor:
    """weight * x / sqrt(mean(x^2) + eps) over the channels of every position: the last dimension of [N, C] and [B, L, C], dimension 1 of an image [N, C, H, W]."""
    _check(x, eps, (weight, [(_channels(x),)]))
    wanted = grad_enabled(x, weight)
    _, y, rstd, _ = dispatch(x.device, "add_rms_norm")(x, None, weight, eps=eps, keep=wanted)
    y.requires_grad = wanted
    return record("rms_norm", [x, weight], y, [rstd])


@tracker.register_backward_function("rms_norm")
def rms_norm_backward(dy, rstd, x, weight):
    needed = (x.requires_grad, False, weight is not None and weight.requires_grad, False, False)
    grads = dispatch(x.device, "add_rms_norm_backward")(None, dy, x, rstd, None, x, None, weight, needed=needed)
    return [grads[0], grads[2]]


def add_rms_norm(residual: Tensor, block: Tensor, weight=None, post_weight=None, gate=None, scale=1.0, eps=1e-6):
    """What lies between two blocks of a residual network, in one pass: (new, rms_norm(new, weight, eps)) with
    new = scale * residual + gate * rms_norm(block, post_weight, eps), or without ``post_weight`` new = scale * residual + gate * block.

    ``gate``: None, or [C], or one row a sample [first dimension, C], or a value for each of the block's.  Shapes as in ``rms_norm``."""
    channels = _channels(residual)
    _check(residual, eps, (block, [residual.shape]), (weight, [(channels,)]), (post_weight, [(channels,)]),
           (gate, [(channels,), (residual.shape[0], channels), residual.shape]))
    operands = (residual, block, weight, post_weight, gate)
    wanted = grad_enabled(*operands)
    new, y, rstd, block_rstd = dispatch(residual.device, "add_rms_norm")(*operands, scale, eps, wanted)
    if wanted:
        new.requires_grad = y.requires_grad = True
        # another object over the sum's memory: a node that held its own output would never be freed without a backward
        tracker.add_node("add_rms_norm", [*operands, scale], [new, y], [Tensor(tensor=new), rstd, block_rstd])
    return new, y


@tracker.register_backward_function("add_rms_norm")
def add_rms_norm_backward(dnew, dy, new, rstd, block_rstd, residual, block, weight, post_weight, gate, scale):
    operands = (residual, block, weight, post_weight, gate)
    needed = tuple(t is not None and t.requires_grad for t in operands)
    return dispatch(residual.device, "add_rms_norm_backward")(dnew, dy, new, rstd, block_rstd, *operands, scale, needed)
