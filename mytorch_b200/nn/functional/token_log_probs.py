"""Log probabilities of given tokens, with the entropy and the most likely alternatives of every row (no counterpart in the reference)."""
from typing import NamedTuple, Optional

from mytorch_b200.dtype import int32, int64
from mytorch_b200.ops._common import dispatch, grad_enabled, tracker
from mytorch_b200.tensor import InvalidDataTypeError, InvalidShapeError, MismatchDevicesError, MismatchShapesError, Tensor

MOST_ALTERNATIVES = 32


class TokenLogProbs(NamedTuple):
    log_probs: Tensor
    entropy: Tensor
    top_log_probs: Optional[Tensor]
    top_tokens: Optional[Tensor]


def token_log_probs(logits: Tensor, tokens: Tensor, top=0, ignore_index=None) -> TokenLogProbs:
    """Of ``logits`` [N, V] or [B, L, V] and one int32 or int64 token a row, in one pass over the logits: log softmax(logits)[token] and the entropy of the row's
    distribution, of the shape of ``tokens``; with ``top`` (at most 32) also the log probabilities and int64 indices of the most likely tokens, in descending order, equal
    ones by index, of shape tokens.shape + (top,).  The first three have gradients.

    ``ignore_index``: a row with this token has log probability 0 and no gradient from it; entropy and alternatives are those of its logits.  Another token outside [0, V)
    has log probability NaN and no gradient from it either.  A logit of -inf is a token that cannot be; a row of nothing else, or with NaN or +inf in it, is NaN, its alternatives in the order of
    its logits (NaN first), and so is its gradient.  A row that no gradient reaches, as one of an ignored token where nothing is made of its entropy and alternatives, has
    gradient zero, whatever its logits."""
    if len(logits.shape) not in (2, 3) or logits.shape[-1] < 1:
        raise InvalidShapeError(logits.shape)
    if tokens.dtype is not int32 and tokens.dtype is not int64:
        raise InvalidDataTypeError(tokens.dtype)
    if tokens.shape != logits.shape[:-1]:
        raise MismatchShapesError([logits.shape, tokens.shape])
    if tokens.device is not logits.device:
        raise MismatchDevicesError([logits.device, tokens.device])
    if not isinstance(top, int) or not 0 <= top <= min(MOST_ALTERNATIVES, logits.shape[-1]):
        raise RuntimeError(f"token_log_probs: top is from 0 to {MOST_ALTERNATIVES} and not above {logits.shape[-1]}: {top}")
    if ignore_index is not None and not isinstance(ignore_index, int):
        raise RuntimeError(f"token_log_probs: ignore_index is a number or None: {ignore_index}")
    wanted = grad_enabled(logits)
    log_probs, entropy, top_log_probs, top_tokens, stats = dispatch(logits.device, "token_log_probs")(logits, tokens, top, ignore_index, wanted)
    if wanted:
        outputs = [t for t in (log_probs, entropy, top_log_probs) if t is not None]
        for t in outputs:
            t.requires_grad = True
        tracker.add_node("token_log_probs", [logits, tokens, ignore_index], outputs, [stats, top_tokens])
    return TokenLogProbs(log_probs, entropy, top_log_probs, top_tokens)


@tracker.register_backward_function("token_log_probs")
def token_log_probs_backward(dlog_probs, dentropy, *rest):
    *dtop, stats, top_tokens, logits, tokens, ignore_index = rest
    return dispatch(logits.device, "token_log_probs_backward")(dlog_probs, dentropy, dtop[0] if dtop else None, stats, top_tokens, logits, tokens, ignore_index)
