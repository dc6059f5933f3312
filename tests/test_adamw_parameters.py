"""AdamW updates all parameters of a group at once, so none may be there twice: two updates of the same memory would run side by side."""
import numpy as np
import pytest

import mytorch_b200 as mt
import mytorch_b200.nn as nn
from mytorch_b200.optim import AdamW


@pytest.mark.parametrize("bits", [32, 8])
def test_a_parameter_twice_is_refused(bits):
    p, q = (nn.Parameter(mt.tensor(np.zeros(3, np.float32))) for _ in range(2))
    with pytest.raises(RuntimeError, match="occurs twice"):
        AdamW([p, q, p], state_bits=bits)
    with pytest.raises(RuntimeError, match="occurs twice"):
        AdamW([{"params": [q]}, {"params": [p, p]}], state_bits=bits)
    with pytest.raises(RuntimeError, match="overlap"):
        AdamW([{"params": [p]}, {"params": [q, p]}], state_bits=bits)
    AdamW([p, q], state_bits=bits)
