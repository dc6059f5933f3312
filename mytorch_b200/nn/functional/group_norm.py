"""Group normalisation with an activation behind it, as one operator (no counterpart in the reference)."""
from mytorch_b200.ops._common import dispatch, grad_enabled, record, tracker
from mytorch_b200.tensor import MismatchDataTypesError, MismatchDevicesError, MismatchShapesError, Tensor

ACTIVATIONS = (None, "relu", "silu")


def group_norm(input: Tensor, num_groups, weight=None, bias=None, eps=1e-5, activation=None) -> Tensor:
    """activation(weight * (input - mean) / sqrt(var + eps) + bias) for an input [N, C, H, W] or [N, C]: mean and (biased) variance are those of the
    C / num_groups channels of a group at all positions of one image.  ``activation``: None, "relu" or "silu" (z / (1 + exp(-z))).
    Neither the normalised tensor nor the activation's input is stored; backward computes them again from the input."""
    shape = input.shape
    if len(shape) not in (2, 4):
        raise RuntimeError(f"group_norm expects an input [N, C, H, W] or [N, C], got shape {shape}")
    channels = shape[1]
    if not isinstance(num_groups, int) or num_groups < 1 or channels % num_groups:
        raise RuntimeError(f"group_norm: {channels} channels are no {num_groups} groups")
    if activation not in ACTIVATIONS:
        raise RuntimeError(f"group_norm: activation is one of {ACTIVATIONS}: {activation}")
    for t in (weight, bias):
        if t is not None:
            if t.shape != (channels,):
                raise MismatchShapesError([shape, t.shape])
            if t.device is not input.device:
                raise MismatchDevicesError([input.device, t.device])
            if t.dtype is not input.dtype:
                raise MismatchDataTypesError([input.dtype, t.dtype])
    out, mean, rstd = dispatch(input.device, "group_norm")(input, num_groups, weight, bias, eps, activation)
    out.requires_grad = grad_enabled(input, weight, bias)
    return record("group_norm", [input, weight, bias, num_groups, activation], out, [mean, rstd])


@tracker.register_backward_function("group_norm")
def group_norm_backward(output_grad, mean, rstd, input, weight, bias, num_groups, activation):
    needed = [t is not None and t.requires_grad for t in (input, weight, bias)]
    return dispatch(input.device, "group_norm_backward")(output_grad, mean, rstd, input, weight, bias, num_groups, activation, needed)
