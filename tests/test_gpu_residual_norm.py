"""Residual RMS norm (forward, backward, 8-bit output) and counter-based dropout
against 64-bit evaluations.

Bounds: u is the output type's unit roundoff (2^-8 bf16, 2^-11 fp16, 2^-24
fp32); 32-bit arithmetic over C columns is taken as 2^-18 of the terms' sum,
that of residual + x / (1 - p) as 2^-22 of its two terms (which may cancel);
h is stored rounded (u_s), which reaches the gradients through h once."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

UNIT = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0**-25, torch.float32: 0.0}
REL = 2.0**-18
BF, HF, FF = torch.bfloat16, torch.float16, torch.float32


def philox_words(n, seed, offset):
    """Word e % 4 of block offset + e // 4 for e < n (Python integers: no shared arithmetic with the kernels)."""
    out = []
    for b in range(-(-n // 4)):
        c = (offset + b) % 2**64
        x = [c % 2**32, c >> 32, 0, 0]
        for r in range(10):
            k0, k1 = (seed + r * 0x9E3779B9) % 2**32, ((seed >> 32) + r * 0xBB67AE85) % 2**32
            a, d = x[0] * 0xD2511F53, x[2] * 0xCD9E8D57
            x = [(d >> 32) ^ x[1] ^ k0, d % 2**32, (a >> 32) ^ x[3] ^ k1, a % 2**32]
        out += x
    return out[:n]


def keep_mask(shape, p, seed, offset=0):
    w = torch.tensor(philox_words(math.prod(shape), seed, offset), dtype=torch.int64)
    return (w >= int(p * 2**32)).view(shape).cuda()


def close(x, ref, bound, what=""):
    assert torch.isfinite(x).all(), what
    over = ((x.double() - ref).abs() - bound).max().item() if x.numel() else 0.0
    assert over <= 1e-13, f"{what}: {over:.3g} beyond the bound"


def test_generator_known_answers():
    """The generator's published test vectors for an all-zero and an all-one counter and key need words 2 and 3 of the
    counter, which are zero here: the zero vector is checked, then words against the Python form at a large offset."""
    assert philox_words(4, 0, 0) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    from lsrm_sparse import api

    x = torch.ones(4096, device="cuda")
    for seed, offset in ((0, 0), (2**63 + 12345, 2**40 + 7), (2**64 - 1, 2**64 - 100)):
        for p in (0.25, 0.5):
            y = api.dropout(x, p, seed, offset)
            assert torch.equal(y > 0, keep_mask((4096,), p, seed, offset))


@pytest.mark.parametrize("dtype", [BF, HF, FF])
@pytest.mark.parametrize("shape,p", [((1,), 0.5), ((7,), 0.9), ((3, 1001), 0.1), ((5, 4, 64), 0.3), ((2, 33, 8), 0.05)])
def test_dropout(shape, p, dtype):
    from lsrm_sparse import api

    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(*shape, device="cuda", generator=g).to(dtype).requires_grad_()
    dy = torch.randn(*shape, device="cuda", generator=g).to(dtype)
    y = api.dropout(x, p, 77, 5)
    (dx,) = torch.autograd.grad(y, x, dy)
    keep = keep_mask(shape, p, 77, 5)
    for got, t in ((y.detach(), x.detach()), (dx, dy)):
        ref = torch.where(keep, t.double() / (1 - p), 0.0)
        close(got, ref, (UNIT[dtype] + 2.0**-22) * ref.abs() + TINY[dtype])
        assert torch.equal(got != 0, keep & (t != 0))


def test_dropout_share_strides_and_dropped_values():
    from lsrm_sparse import api

    x = torch.ones(1 << 20, device="cuda")
    for p in (0.05, 0.3, 0.9):
        kept = (api.dropout(x, p, 3) != 0).double().mean().item()
        assert abs(kept - (1 - p)) <= 6 * math.sqrt(p * (1 - p) / x.numel())
    # a view is dropped as its contiguous copy is; what is dropped does not matter
    v = torch.randn(64, 48, device="cuda").bfloat16().t()[3:]
    assert torch.equal(api.dropout(v, 0.5, 9), api.dropout(v.contiguous(), 0.5, 9))
    bad = torch.full((4096,), math.nan, device="cuda")
    keep = keep_mask((4096,), 0.5, 4)
    assert torch.equal(torch.isnan(api.dropout(bad, 0.5, 4)), keep)
    assert api.dropout(bad, 0.0, 4) is bad
    assert api.dropout(torch.empty(0, 5, device="cuda"), 0.5, 1).shape == (0, 5)
    for p in (1.0, -0.1, math.nan):
        with pytest.raises(ValueError):
            api.dropout(x, p, 1)
    with pytest.raises(ValueError):
        api.dropout(torch.ones(4), 0.5, 1)
    with pytest.raises(ValueError):
        api.dropout(torch.ones(4, device="cuda", dtype=torch.float64), 0.5, 1)


SHAPES = [(1, 1), (3, 33), (1, 1024), (8, 1001), (37, 64), (700, 8), (5, 4096), (2, 16384), (3, 16383), (1300, 1000),
          (700, 1025), (2000, 257), (4500, 128)]


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("dtype,stream,wtype,p", [(BF, BF, BF, 0.1), (BF, FF, FF, 0.0), (HF, FF, HF, 0.25),
                                                  (HF, HF, None, 0.0), (BF, None, FF, 0.5)])
def test_norm_forward_and_gradients(rows, cols, dtype, stream, wtype, p):
    from lsrm_sparse import api

    if p and rows * cols > 70000:
        pytest.skip("the Python generator is slow there")
    g = torch.Generator(device="cuda").manual_seed(rows + cols)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    x = r(rows, cols).to(dtype).requires_grad_()
    res = (2 * r(rows, cols)).to(stream).requires_grad_() if stream else None
    w = (1 + 0.3 * r(cols)).to(wtype).requires_grad_() if wtype else None
    st = stream or dtype
    dy, dh = r(rows, cols).to(dtype), r(rows, cols).to(st)
    y, h = api.residual_rms_norm(x, res, w, p=p, seed=11, offset=3, eps=1e-5)
    inputs = [t for t in (x, res, w) if t is not None]
    got = dict(zip([n for n, t in (("dx", x), ("dres", res), ("dw", w)) if t is not None],
                   torch.autograd.grad((y, h), inputs, (dy, dh))))
    f = torch.where(keep_mask((rows, cols), p, 11, 3), 1 / (1 - p), 0.0).double() if p else 1.0
    X, W = x.detach().double(), w.detach().double() if wtype else 1.0
    H = X * f + (res.detach().double() if stream else 0.0)
    rs = (H.square().mean(1, keepdim=True) + 1e-5).rsqrt()
    u, us = UNIT[dtype], UNIT[st]
    eh = 2.0**-22 * ((X * f).abs() + (H - X * f).abs())
    close(h.detach(), H, us * H.abs() + eh + TINY[st], "h")
    Y, W1 = H * rs * W, W.abs() if wtype else 1.0
    close(y.detach(), Y, (u + REL) * Y.abs() + eh * rs * W1 + TINY[dtype], "y")
    G = dy.double() * W
    mean = (G * H).mean(1, keepdim=True)
    D = rs * (G - H * rs**2 * mean) + dh.double()
    # h reaches the gradient rounded: in its own factor and in the mean
    slack = (us + REL) * rs**3 * (H.abs() * mean.abs() + H.abs() * (G * H).abs().mean(1, keepdim=True)) \
        + REL * (rs * G.abs() + dh.double().abs())
    if stream:
        close(got["dres"], D, us * D.abs() + slack + TINY[st], "dresidual")
    close(got["dx"], D * f, (u * D.abs() + slack) * f + TINY[dtype], "dx")
    if wtype:
        t = dy.double() * H * rs
        uw = UNIT[wtype]
        close(got["dw"], t.sum(0), uw * t.sum(0).abs() + (us + REL) * t.abs().sum(0) + TINY[wtype], "dweight")


def test_norm_gradients_against_differences():
    from lsrm_sparse import api

    rows, cols = 6, 40
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(rows, cols, device="cuda", generator=g).half().requires_grad_()
    res, w, = (torch.randn(*s, device="cuda", generator=g).requires_grad_() for s in ((rows, cols), (cols,)))
    dy, dh = torch.randn(2, rows, cols, device="cuda", generator=g)
    y, h = api.residual_rms_norm(x, res, w, p=0.25, seed=5)
    grads = torch.autograd.grad((y, h), (x, res, w), (dy.half(), dh))
    f = torch.where(keep_mask((rows, cols), 0.25, 5), 1 / 0.75, 0.0).double()
    base = [t.detach().double() for t in (x, res, w)]

    def loss(a, b, c):
        hh = a * f + b
        return ((hh / (hh.square().mean(1, keepdim=True) + 1e-6).sqrt() * c * dy.half().double()).sum()
                + (hh * dh.double()).sum()).item()

    for i, grad in enumerate(grads):
        step = torch.randn(base[i].shape, device="cuda", generator=g, dtype=torch.float64)
        up, down = (loss(*[b + s * 1e-5 * step if j == i else b for j, b in enumerate(base)]) for s in (1, -1))
        diff = (up - down) / 2e-5
        tol = (6 * UNIT[grad.dtype] + 1e-5) * (grad.double() * step).norm().item() + 1e-6 * abs(diff)
        assert abs((grad.double() * step).sum().item() - diff) <= tol, i


def test_norm_uses_one_output_only():
    from lsrm_sparse import api

    x = torch.randn(9, 72, device="cuda").bfloat16().requires_grad_()
    res = torch.randn(9, 72, device="cuda").bfloat16().requires_grad_()
    w = torch.ones(72, device="cuda").bfloat16().requires_grad_()
    d = torch.randn(9, 72, device="cuda").bfloat16()
    y, h = api.residual_rms_norm(x, res, w, p=0.5, seed=1)
    zero = torch.zeros_like(d)
    a = torch.autograd.grad(y, (x, res, w), d, retain_graph=True)
    b = torch.autograd.grad((y, h), (x, res, w), (d, zero), retain_graph=True)
    assert all(torch.equal(s, t) for s, t in zip(a, b))
    a = torch.autograd.grad(h, (x, res, w), d, retain_graph=True, allow_unused=True)
    b = torch.autograd.grad((y, h), (x, res, w), (zero, d))
    assert all(torch.equal(s, t) for s, t in zip(a, b))


def test_norm_zero_rows_and_no_rows():
    from lsrm_sparse import api

    x = torch.zeros(5, 96, device="cuda").bfloat16().requires_grad_()
    w = torch.ones(96, device="cuda").bfloat16().requires_grad_()
    y, h = api.residual_rms_norm(x, None, w)
    dx, dw = torch.autograd.grad(y, (x, w), torch.ones_like(y))
    assert (y == 0).all() and (h == 0).all() and (dw == 0).all() and torch.isfinite(dx).all()
    x = torch.empty(0, 96, device="cuda").bfloat16().requires_grad_()
    y, h = api.residual_rms_norm(x, None, w)
    dx, dw = torch.autograd.grad(y, (x, w), torch.ones_like(y))
    assert dx.shape == (0, 96) and (dw == 0).all()
    q, s, h = api.residual_rms_norm_8bit(x, None, w)
    assert q.shape == (0, 96) and s.shape == (0, 1)


def _grid8(t, out):
    step = torch.ones_like(t)
    if out == torch.float8_e4m3fn:
        step = torch.exp2(torch.floor(torch.log2(t.abs().clamp(min=2.0**-6))) - 3)
    return torch.round(t / step) * step, step


@pytest.mark.parametrize("rows,cols", [(1, 1), (8, 1024), (3, 1001), (700, 33), (5, 4100), (1200, 128), (2, 16384),
                                       (601, 1023)])
@pytest.mark.parametrize("out,group,dtype,stream", [(torch.float8_e4m3fn, 0, BF, BF), (torch.int8, 128, BF, FF),
                                                    (torch.float8_e4m3fn, 32, HF, HF), (torch.int8, 64, HF, None),
                                                    (torch.int8, 0, BF, None)])
def test_norm_8bit(rows, cols, out, group, dtype, stream):
    from lsrm_sparse import api

    g = torch.Generator(device="cuda").manual_seed(rows + cols)
    x = torch.randn(rows, cols, device="cuda", generator=g).to(dtype)
    res = torch.randn(rows, cols, device="cuda", generator=g).to(stream) if stream else None
    w = (1 + 0.3 * torch.randn(cols, device="cuda", generator=g)).to(dtype)
    x[0] = 0.0
    if stream:
        res[0] = 0.0
    q, scales, h = api.residual_rms_norm_8bit(x, res, w, dtype=out, group=group)
    H = x.double() + (res.double() if stream else 0.0)
    close(h, H, (UNIT[stream or dtype] + 2.0**-22) * H.abs() + TINY[stream or dtype], "h")
    Y = H * (H.square().mean(1, keepdim=True) + 1e-6).rsqrt() * w.double()
    top = 448.0 if out == torch.float8_e4m3fn else 127.0
    width = group or cols
    assert scales.shape == (rows, -(-cols // width)) and q.shape == x.shape and q.dtype == out
    for i, part in enumerate(Y.split(width, 1)):
        amax = part.abs().amax(1)
        sc = torch.where(amax > 0, amax / top, 1.0)
        assert ((scales[:, i].double() - sc).abs() <= 2.0**-17 * sc).all()
        t = part / sc[:, None]
        ref, step = _grid8(t, out)
        got = q[:, i * width:i * width + part.shape[1]].double()
        # half a step from the value (a hair more where 32-bit arithmetic moved it), on the grid
        assert ((got - t).abs() <= 0.5 * step + 2.0**-16 * t.abs()).all()
        assert ((got != ref).double().mean() <= 0.01)
    for to in (BF, HF, FF):
        y = api.dequantize_8bit(q, scales, to)
        ref = q.double() * scales.double().repeat_interleave(width, 1)[:, :cols]
        close(y, ref, (UNIT[to] + 2.0**-22) * ref.abs() + TINY[to], "dequantize")


def test_layouts_and_refusals():
    from lsrm_sparse import api

    x = torch.randn(40, 64, device="cuda").bfloat16()
    res = torch.randn(40, 64, device="cuda").bfloat16()
    w = torch.randn(64, device="cuda").bfloat16()
    y, h = api.residual_rms_norm(x, res, w, p=0.5, seed=2)
    wide = torch.randn(40, 128, device="cuda").bfloat16()
    wide[:, 3:67] = x
    y2, h2 = api.residual_rms_norm(wide[:, 3:67], res.t().contiguous().t(), w, p=0.5, seed=2)
    assert torch.equal(y, y2) and torch.equal(h, h2)
    y3, h3 = api.residual_rms_norm(x.view(2, 20, 64), res.view(2, 20, 64), w, p=0.5, seed=2)
    assert torch.equal(y, y3.view(40, 64)) and torch.equal(h, h3.view(40, 64))
    for bad in (lambda: api.residual_rms_norm(x.float()), lambda: api.residual_rms_norm(x, res[:1], w),
                lambda: api.residual_rms_norm(x, res.half(), w), lambda: api.residual_rms_norm(x, res, w[:63]),
                lambda: api.residual_rms_norm(x, res, w.half()), lambda: api.residual_rms_norm(x.cpu()),
                lambda: api.residual_rms_norm(x, res, w, p=1.0),
                lambda: api.residual_rms_norm_8bit(x, res, w, group=48),
                lambda: api.residual_rms_norm_8bit(x, res, w, dtype=torch.uint8),
                lambda: api.dequantize_8bit(*api.residual_rms_norm_8bit(x, res, w)[:2], torch.float64)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError, match="cols"):
        api.residual_rms_norm(torch.zeros(1, 16392, device="cuda").bfloat16())
