"""Norm, dropout and dequantisation over more rows than the GPU holds at once:
teams take several rows, threads several chunks, counters pass 32 bits midway.
Bounds as in test_gpu_residual_norm."""

import pytest
import torch

from tests.philox_oracle import keep
from tests.test_gpu_residual_norm import BF, FF, HF, REL, TINY, UNIT, _grid8, close

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF, HF, FF])
@pytest.mark.parametrize("offset", [3, 2**32 - 2_000_000, 2**64 - 1_000_000])
def test_dropout(dtype, offset):
    from lsrm_sparse import api

    n, p, seed = (1 << 24) + 5, 0.3, 2**40 + 1
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(n, device="cuda", generator=g).to(dtype)
    scale = torch.tensor(1.0 / (1.0 - p), device="cuda")
    want = torch.where(keep((n,), p, seed, offset), x.float() * scale, 0.0).to(dtype)
    assert torch.equal(api.dropout(x, p, seed, offset), want)


@pytest.mark.parametrize("rows,cols", [(30000, 1024), (20000, 1001), (60000, 256), (50000, 200), (30000, 63), (6000, 4096)])
@pytest.mark.parametrize("dtype,stream,p", [(BF, BF, 0.1), (HF, FF, 0.25), (BF, FF, 0.0), (HF, HF, 0.0)])
def test_norm_forward_and_gradients(rows, cols, dtype, stream, p):
    from lsrm_sparse import api

    seed, offset = 11, 2**32 - 500_000
    g = torch.Generator(device="cuda").manual_seed(rows + cols)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    x, res = r(rows, cols).to(dtype).requires_grad_(), (2 * r(rows, cols)).to(stream).requires_grad_()
    w = (1 + 0.3 * r(cols)).to(stream).requires_grad_()
    dy, dh = r(rows, cols).to(dtype), r(rows, cols).to(stream)
    y, h = api.residual_rms_norm(x, res, w, p=p, seed=seed, offset=offset, eps=1e-5)
    dx, dres, dw = torch.autograd.grad((y, h), (x, res, w), (dy, dh))
    f = torch.where(keep((rows, cols), p, seed, offset), 1 / (1 - p), 0.0).double() if p else 1.0
    X, R, W = x.detach().double() * f, res.detach().double(), w.detach().double()
    H = X + R
    rs = (H.square().mean(1, keepdim=True) + 1e-5).rsqrt()
    u, us = UNIT[dtype], UNIT[stream]
    eh = 2.0**-22 * (X.abs() + R.abs())
    close(h.detach(), H, us * H.abs() + eh + TINY[stream], "h")
    Y = H * rs * W
    close(y.detach(), Y, (u + REL) * Y.abs() + eh * rs * W.abs() + TINY[dtype], "y")
    del X, R, Y, eh
    G = dy.double() * W
    mean = (G * H).mean(1, keepdim=True)
    D = rs * (G - H * rs**2 * mean) + dh.double()
    slack = (us + REL) * rs**3 * H.abs() * (mean.abs() + (G * H).abs().mean(1, keepdim=True)) \
        + REL * (rs * G.abs() + dh.double().abs())
    close(dres, D, us * D.abs() + slack + TINY[stream], "dresidual")
    close(dx, D * f, (u * D.abs() + slack) * f + TINY[dtype], "dx")
    t = dy.double() * H * rs
    close(dw, t.sum(0), us * t.sum(0).abs() + (us + REL) * t.abs().sum(0) + TINY[stream], "dweight")


@pytest.mark.parametrize("rows,cols,group", [(30000, 1024, 0), (30000, 1040, 128), (20000, 1001, 64), (20000, 1001, 0),
                                             (60000, 200, 32), (60000, 72, 32), (6000, 4096, 128)])
@pytest.mark.parametrize("out,dtype,stream", [(torch.int8, BF, BF), (torch.float8_e4m3fn, HF, FF)])
def test_norm_8bit_and_dequantize(rows, cols, group, out, dtype, stream):
    from lsrm_sparse import api

    g = torch.Generator(device="cuda").manual_seed(rows + cols)
    x = torch.randn(rows, cols, device="cuda", generator=g).to(dtype)
    res = torch.randn(rows, cols, device="cuda", generator=g).to(stream)
    w = (1 + 0.3 * torch.randn(cols, device="cuda", generator=g)).to(dtype)
    q, scales, h = api.residual_rms_norm_8bit(x, res, w, dtype=out, group=group)
    H = x.double() + res.double()
    close(h, H, UNIT[stream] * H.abs() + 2.0**-22 * (x.double().abs() + res.double().abs()) + TINY[stream], "h")
    Y = H * (H.square().mean(1, keepdim=True) + 1e-6).rsqrt() * w.double()
    top, width = 448.0 if out == torch.float8_e4m3fn else 127.0, group or cols
    for i, part in enumerate(Y.split(width, 1)):
        sc = part.abs().amax(1) / top
        assert ((scales[:, i].double() - sc).abs() <= 2.0**-17 * sc).all()
        t = part / sc[:, None]
        ref, step = _grid8(t, out)
        got = q[:, i * width:i * width + part.shape[1]].double()
        assert ((got - t).abs() <= 0.5 * step + 2.0**-16 * t.abs()).all()
        assert (got != ref).double().mean() <= 0.01
    for to in (BF, HF, FF):
        back = api.dequantize_8bit(q, scales, to)
        ref = (q.float() * scales.repeat_interleave(width, 1)[:, :cols]).to(to)  # one product in 32 bits, rounded once
        assert torch.equal(back, ref)
