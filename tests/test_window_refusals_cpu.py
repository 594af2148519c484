"""What the windowed operators' Python side refuses before any CUDA call."""

import ctypes
import math

import pytest

from lsrm_sparse import ops
from tests.test_abi_cpu import lib  # noqa: F401  (builds and loads the library)


@pytest.mark.parametrize("scale", [-1.0, -0.125, -1e-30, 1e-50, 1e39, math.nan, math.inf, -math.inf])
def test_softmax_scales_that_are_no_scale(scale):
    """They used to select 1 / sqrt(head_dim), as 0 does."""
    with pytest.raises(ValueError, match="softmax_scale"):
        ops._scale("window_sink_attention", scale)


def test_softmax_scales():
    assert ops._scale("x", None) == 0.0 and ops._scale("x", 0) == 0.0 and ops._scale("x", 0.25) == 0.25


def test_any_number_of_sequences(lib):  # noqa: F811
    """The backward takes as many sequences as the forward (no token: nothing is launched)."""
    sh = lib.WindowShape(70000, 0, 0, 4, 2, 64, 1, 8, 2, 1, 256, 128, 128, 0.0)
    p, h = 1 << 20, lib.lib()
    assert h.lsrm_window_attn_fwd(ctypes.byref(sh), p, p, p, p, p, p, p, p, None, None) == 0
    assert h.lsrm_window_attn_bwd(ctypes.byref(sh), p, p, p, p, p, p, p, p, p, p, p, p, p, 1 << 40, None, None) == 0
