"""The norms' gradient of rows that a cluster of CTAs holds, more of them than two turns of the resident clusters: each goes on to other rows, whose values come while it works, and to
rows of another row of the gate."""
import pytest

from test_gpu_rms_norm import test_backward as _gradients

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape,gate,post", [((700, 8200), None, True), ((700, 8200), "channel", True), ((620, 8201), "full", True), ((350, 2, 8200), "sample", True),
                                             ((350, 2, 8202), "sample", False), ((130, 5, 8193), "sample", True), ((300, 12292), "channel", False), ((240, 16384), "full", True),
                                             ((130, 2, 16384), "sample", True)])
def test_gradients_of_many_rows(shape, gate, post):
    _gradients(shape, gate, post)
