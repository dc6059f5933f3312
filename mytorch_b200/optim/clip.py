"""The norm of all gradients together, and clipping by it (no counterpart in the reference)."""
from mytorch_b200.ops._common import dispatch
from mytorch_b200.tensor import MismatchDevicesError, Tensor


def grad_norm(params):
    """sqrt of the sum of squares of all gradients of ``params`` (a tensor or several; those without a gradient count nothing), as a tensor of one
    element on their device.  Nothing waits for it."""
    return _clip(params, None)


def clip_grad_norm_(params, max_norm):
    """Multiplies the gradients of ``params`` by min(1, max_norm / (norm + 1e-6)) in place and returns their norm before that, as ``grad_norm`` does.
    A tensor that holds the gradient of several parameters (addition hands one to both of its operands) counts for each and is multiplied once.
    Norms that are infinite or no number show in the gradients: the factor is then 0 or no number."""
    max_norm = float(max_norm)
    if not max_norm >= 0:
        raise RuntimeError(f"clip_grad_norm_: max_norm is a number from 0 up: {max_norm}")
    return _clip(params, max_norm)


def _clip(params, max_norm):
    grads, again, known = [], [], set()
    device = None
    for p in [params] if isinstance(params, Tensor) else params:
        grad = p.grad
        if grad is None:
            continue
        if device is None:
            device = grad.device
        elif grad.device is not device:
            raise MismatchDevicesError([device, grad.device])
        memory = grad._native_array
        at = id(grad) if memory is None else memory.ptr
        if at in known and 0 not in grad.shape:
            again.append(grad)
        else:
            known.add(at)
            grads.append(grad)
    if device is None:
        raise RuntimeError("there is no gradient to take the norm of")
    return dispatch(device, "clip_gradients")(grads, again, max_norm)
