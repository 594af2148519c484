"""What the windowed operators' Python side refuses before any CUDA call."""

import math

import pytest

from lsrm_sparse import ops


@pytest.mark.parametrize("scale", [-1.0, -0.125, -1e-30, 1e-50, 1e39, math.nan, math.inf, -math.inf])
def test_softmax_scales_that_are_no_scale(scale):
    """They used to select 1 / sqrt(head_dim), as 0 does."""
    with pytest.raises(ValueError, match="softmax_scale"):
        ops._scale("window_sink_attention", scale)


def test_softmax_scales():
    assert ops._scale("x", None) == 0.0 and ops._scale("x", 0) == 0.0 and ops._scale("x", 0.25) == 0.25
