"""The 8-bit norm of rows that hold a NaN or an infinity: no finite number may
come out of them, and no other row or group may change."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BAD = [math.nan, math.inf, -math.inf]


@pytest.mark.parametrize("out", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("group", [0, 32, 128])
@pytest.mark.parametrize("rows,cols", [(6, 200), (6, 1024), (6, 2048), (6, 1001), (6, 333), (4000, 1024), (3000, 257)])
def test_rows_that_hold_no_number(rows, cols, group, out):
    from lsrm_sparse import api

    g = torch.Generator(device="cuda").manual_seed(rows + cols + group)
    x = torch.randn(rows, cols, device="cuda", generator=g).bfloat16()
    res = torch.randn(rows, cols, device="cuda", generator=g)
    clean = api.residual_rms_norm_8bit(x, res, None, dtype=out, group=group)
    at = [0, cols // 2, cols - 1]
    for i, v in enumerate(BAD):
        res[i + 1, at[i]] = v
    q, scales, h = api.residual_rms_norm_8bit(x, res, None, dtype=out, group=group)
    H = x.float() + res
    y = H * (H.square().mean(1, keepdim=True) + 1e-6).rsqrt()  # NaN all over a NaN's row, at an infinity, else 0
    width = group or cols
    bad = torch.stack([~torch.isfinite(p).all(1) for p in y.split(width, 1)], 1)
    assert bad[1].all() and bad[2:4].any(1).all()
    assert torch.equal(torch.isnan(scales), bad)
    back = api.dequantize_8bit(q, scales, torch.float32)
    wide = bad.repeat_interleave(width, 1)[:, :cols]
    assert torch.equal(torch.isnan(back), wide)
    # beside the infinity of a row stand zeros; the other rows are what they were
    assert (back[2:4][~wide[2:4]] == 0).all()
    rest = [0] + list(range(4, rows))
    for a, b in zip((q, scales, h), clean):
        assert torch.equal(a[rest].view(torch.uint8), b[rest].view(torch.uint8))


@pytest.mark.parametrize("out", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("cols", [512, 515])
@pytest.mark.parametrize("bad", BAD)
def test_a_weight_that_is_no_number(cols, bad, out):
    from lsrm_sparse import api

    x = torch.randn(40, cols, device="cuda").bfloat16()
    w = torch.ones(cols, device="cuda").bfloat16()
    w[70] = bad
    for group in (0, 64):
        q, scales, _ = api.residual_rms_norm_8bit(x, None, w, dtype=out, group=group)
        back = api.dequantize_8bit(q, scales, torch.bfloat16)
        lo, hi = (0, cols) if group == 0 else (64, 128)
        assert torch.isnan(back[:, lo:hi]).all()
        assert torch.isfinite(back[:, :lo]).all() and torch.isfinite(back[:, hi:]).all()


@pytest.mark.parametrize("cols", [256, 250])
def test_the_largest_and_smallest_scales(cols):
    """y from its largest finite values (a scale near 2^128 / 127) down to ones whose scale would have no reciprocal."""
    from lsrm_sparse import api

    x = torch.ones(3, cols, device="cuda").bfloat16()
    for w, zero in ((3.3e38, False), (1e-30, False), (1e-38, True)):
        wt = torch.full((cols,), w, device="cuda")
        for out in (torch.int8, torch.float8_e4m3fn):
            q, scales, _ = api.residual_rms_norm_8bit(x, None, wt, dtype=out)
            assert torch.isfinite(scales).all()
            back = api.dequantize_8bit(q, scales, torch.float32).double()
            # a whole step where the scale stands at its least (2^-126), else half a step
            assert ((back - w).abs() <= (2.0**-126 if zero else 2.0**-4 * w)).all()
