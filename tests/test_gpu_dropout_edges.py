"""Dropout of infinities, of values at the ends of a type's range and of p close
to 1; the same element must come out the same wherever it lies in the tensor."""

import math

import pytest
import torch

from tests.philox_oracle import keep, words
from tests.test_gpu_residual_norm import philox_words

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("p", [0.1, 0.3, 0.5])
def test_infinities_stay_infinite(dtype, p):
    """In whole chunks of eight and in the rest of a tensor, forward and backward."""
    from lsrm_sparse import api

    n = 1027
    x = torch.full((n,), math.inf, device="cuda", dtype=dtype)
    x[::2] = -math.inf
    x.requires_grad_()
    y = api.dropout(x, p, 21)
    (dx,) = torch.autograd.grad(y, x, x.detach())
    want = torch.where(keep((n,), p, 21), x.detach(), 0.0)
    assert torch.equal(y.detach(), want) and torch.equal(dx, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("p", [0.1, 0.3, 0.5, 0.9, 0.99999])
def test_rounded_once_over_the_whole_range(dtype, p):
    """Powers of two with odd mantissas from the least subnormal to the largest number: the 32-bit product, rounded to
    the type (the scale is 1 / (1 - p) in 32 bits)."""
    from lsrm_sparse import api

    n = 8195 if p < 0.99 else (1 << 20) + 3  # some are kept
    info = torch.finfo(dtype)
    lo, hi = math.log2(info.smallest_normal) - (10 if dtype == torch.float16 else 6), math.log2(info.max)
    g = torch.Generator(device="cuda").manual_seed(3)
    e = torch.rand(n, device="cuda", generator=g, dtype=torch.float64) * (hi - lo) + lo
    sign = torch.randint(0, 2, (n,), device="cuda", generator=g) * 2 - 1
    x = (torch.exp2(e) * sign).to(dtype)
    got = api.dropout(x, p, 8)
    scale = torch.tensor(1.0 / (1.0 - p), device="cuda", dtype=torch.float32)
    mask = keep((n,), p, 8)
    assert mask.any()
    assert torch.equal(got, torch.where(mask, x.float() * scale, 0.0).to(dtype))


def test_the_mask_oracle_is_the_generator():
    for seed, offset in ((0, 0), (2**63 + 12345, 2**40 + 7), (2**64 - 1, 2**64 - 100), (5, 2**32 - 3)):
        assert words(0, 803, seed, offset).tolist() == philox_words(803, seed, offset)
        assert words(400, 403, seed, offset).tolist() == philox_words(803, seed, offset)[400:]
