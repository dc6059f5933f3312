from .conv import conv2d
from .cross_entropy import cross_entropy
from .embedding import embedding
from .group_norm import group_norm
from .linear import linear
from .pool_ops import max_pool2d
from .relu import add_relu, relu
from .rms_norm import add_rms_norm, rms_norm
from .token_log_probs import TokenLogProbs, token_log_probs
