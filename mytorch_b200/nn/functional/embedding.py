"""Embedding lookup (no counterpart in the reference)."""
from mytorch_b200.dtype import int32, int64
from mytorch_b200.ops._common import dispatch, grad_enabled, record, tracker
from mytorch_b200.tensor import InvalidDataTypeError, InvalidShapeError, MismatchDevicesError, Tensor


def embedding(tokens: Tensor, weight: Tensor, scale=1.0, padding_idx=None, channels_first=False) -> Tensor:
    """``scale`` times the rows of ``weight`` [rows, width] that the int32 or int64 ``tokens`` name: tokens.shape + (width,).  ``channels_first``: tokens
    [N, H, W] become an image [N, width, H, W] (text: [N, 1, L]), which in the channels-last storage of images is the rows as they are.
    ``padding_idx``: a row that gets no gradient (counted from the end where negative).  A token outside the table reads nothing: its row is NaN."""
    if tokens.dtype is not int32 and tokens.dtype is not int64:
        raise InvalidDataTypeError(tokens.dtype)
    if len(weight.shape) != 2:
        raise InvalidShapeError(weight.shape)
    if tokens.device is not weight.device:
        raise MismatchDevicesError([tokens.device, weight.device])
    if channels_first and len(tokens.shape) != 3:
        raise RuntimeError(f"embedding: channels_first takes tokens [N, H, W], got shape {tokens.shape}")
    if padding_idx is not None:
        rows = weight.shape[0]
        if not -rows <= padding_idx < rows:
            raise RuntimeError(f"embedding: padding_idx {padding_idx} is outside a table of {rows} rows")
        padding_idx %= rows
    out = dispatch(weight.device, "embedding")(tokens, weight, scale, channels_first)
    if not grad_enabled(weight):
        return out
    out.requires_grad = True
    return record("embedding", [tokens, weight, scale, padding_idx, channels_first], out)


@tracker.register_backward_function("embedding")
def embedding_backward(output_grad, tokens, weight, scale, padding_idx, channels_first):
    return [None, dispatch(weight.device, "embedding_backward")(output_grad, tokens, weight, scale, padding_idx, channels_first)[0]]
