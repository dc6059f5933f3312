"""The norm of all gradients together, and clipping by it (no counterpart in the reference)."""
from mytorch_b200.dtype import float32
from mytorch_b200.ops._common import dispatch
from mytorch_b200.tensor import InvalidDataTypeError, MismatchDevicesError, Tensor


def grad_norm(params):
    """sqrt of the sum of squares of all gradients of ``params`` (a tensor or several; those without a gradient count nothing), as a tensor of one
    element on their device.  Nothing waits for it."""
    return _clip(params, None)


def clip_grad_norm_(params, max_norm):
    """Multiplies the gradients of ``params`` by min(1, max_norm / (norm + 1e-6)) in place and returns their norm before that, as ``grad_norm`` does.
    Memory that holds the gradients of several parameters (addition hands one tensor to both of its operands) counts for each and is multiplied once.
    Norms that are infinite or no number show in the gradients: the factor is then 0 or no number."""
    max_norm = float(max_norm)
    if not max_norm >= 0:
        raise RuntimeError(f"clip_grad_norm_: max_norm is a number from 0 up: {max_norm}")
    return _clip(params, max_norm)


def _clip(params, max_norm):
    params = [params] if isinstance(params, Tensor) else list(params)
    for p in params:
        if p.grad is not None:
            norm = dispatch(p.grad.device, "clip_gradients")(params, max_norm)
            if norm is not None:
                return norm
            break
    else:
        raise RuntimeError("there is no gradient to take the norm of")
    grads = [p.grad for p in params if p.grad is not None]  # what is wrong with one of them
    for g in grads:
        if g.device is not grads[0].device:
            raise MismatchDevicesError([grads[0].device, g.device])
    raise InvalidDataTypeError([g.dtype for g in grads if g.dtype is not float32])
