from .clip import clip_grad_norm_, grad_norm
from .optimizer import Optimizer
from .sgd import SGD
