"""The token example's padding: its row of the table is zero, as nn.Embedding leaves it."""
import numpy as np

from mytorch_b200 import nn
from mytorch_b200.examples.token_cnn import TokenCNN


def test_the_padding_row_is_zero():
    net = TokenCNN(vocabulary=50, width=16)
    rows = net.embed.weight._numpy()
    assert not rows[0].any() and (rows[1:].std(1) > 0.1).all() and abs(rows[1:].std() * 4 - 1) < 0.2


def test_rows_of_any_deviation():
    layer = nn.Embedding(1000, 8, padding_idx=-3)
    layer.reset_parameters(0.25)
    rows = layer.weight._numpy()
    assert not rows[-3].any() and abs(np.delete(rows, 997, 0).std() * 4 - 1) < 0.1
