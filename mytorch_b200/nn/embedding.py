"""Embedding (no counterpart in the reference): rows N(0, 1), the padding row zero."""
import mytorch_b200 as mytorch
from mytorch_b200.dtype import float32
from mytorch_b200.nn.functional.embedding import embedding
from mytorch_b200.nn.module import Module
from mytorch_b200.nn.parameter import Parameter
from mytorch_b200.tensor import Tensor


class Embedding(Module):
    """``scale``, ``padding_idx`` and ``channels_first`` as in ``functional.embedding``."""

    def __init__(self, num_embeddings, embedding_dim, padding_idx=None, scale=1.0, channels_first=False, device="cpu", dtype=float32):
        super().__init__()
        if padding_idx is not None and not -num_embeddings <= padding_idx < num_embeddings:
            raise RuntimeError(f"Embedding: padding_idx {padding_idx} is outside a table of {num_embeddings} rows")
        self.num_embeddings, self.embedding_dim, self.padding_idx = num_embeddings, embedding_dim, padding_idx
        self.scale, self.channels_first = scale, channels_first
        self.register_parameter("weight", Parameter(Tensor(shape=(num_embeddings, embedding_dim), dtype=dtype, device=device)))
        self.reset_parameters()

    def reset_parameters(self, std=1):
        """Rows N(0, std^2), the padding row zero."""
        self.weight.normal_(0, std)
        if self.padding_idx is not None:
            rows = self.weight._host_array().copy()
            rows[self.padding_idx] = 0
            self.weight.copy_(mytorch.tensor(rows, dtype=self.weight.dtype))

    def forward(self, tokens):
        return embedding(tokens, self.weight, self.scale, self.padding_idx, self.channels_first)
