"""Tensors of more than 2^31 elements: the same bits as the part that lies past
them gives alone."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _room():
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB")
    yield
    torch.cuda.empty_cache()


def _normal(*shape, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, device="cuda", generator=g).bfloat16()


def test_windowed_attention():
    """Sequences at the end of 270000 tokens of 64 heads of 128 channels (2.2e9 elements), forward and backward."""
    from lsrm_sparse import api

    n, m, hq, hkv, d = 270_000, 700, 64, 8, 128
    cut = torch.tensor([0, 300, m], dtype=torch.int32, device="cuda")
    cu = torch.cat([torch.zeros(1, dtype=torch.int32, device="cuda"), cut + n - m])
    q, do = (torch.zeros(n, hq, d, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    k, v = (torch.zeros(n, hkv, d, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    for i, t in enumerate((q, k, v, do)):
        t[n - m:] = _normal(m, t.shape[1], d, seed=i)

    def run(q, k, v, do, cu):
        q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
        out = api.window_sink_attention(q, k, v, cu, window=96, sinks=4)
        return (out.detach(), *torch.autograd.grad(out, (q, k, v), do))

    big = run(q, k, v, do, cu)
    for a, b in zip(big, run(*(t[n - m:].contiguous() for t in (q, k, v, do)), cut)):
        assert torch.equal(a[n - m:], b)


def test_decode():
    """The window's slots lie past 2^31 elements of one sequence's cache, and wrap."""
    from lsrm_sparse import api
    from tests.test_gpu_window_attn import _decode_ref

    cap, hkv, d, window, sinks = 2_200_000, 8, 128, 3000, 4
    kc, vc = (torch.zeros(1, cap, hkv, d, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    for c, s in ((kc, 1), (vc, 2)):
        c[0, :2000] = _normal(2000, hkv, d, seed=s)
        c[0, cap - 4000:] = _normal(4000, hkv, d, seed=s + 10)
    q, kn, vn = _normal(1, 32, d, seed=3), _normal(1, hkv, d, seed=4), _normal(1, hkv, d, seed=5)
    for n in (cap - 2, cap + 1000):
        ln = torch.tensor([n], dtype=torch.int32, device="cuda")
        out = api.window_sink_decode(q, kn, vn, kc, vc, ln, window=window, sinks=sinks)
        slot = sinks + (n - sinks) % (cap - sinks)
        assert torch.equal(kc[0, slot], kn[0]) and torch.equal(vc[0, slot], vn[0])
        ref, bound = _decode_ref(q, kn, vn, kc, vc, ln, window, sinks)
        assert ((out.double() - ref).abs() <= bound).all()


def test_norm_and_dropout():
    """The last rows of 2.2e9 elements: norm forward and backward with dropout, to 8 bits and back, dropout alone."""
    from lsrm_sparse import api

    cols, m = 1001, 5000  # as many rows as give a row the same team as in the whole
    rows = 2_200_000
    first = rows - m
    first -= first % 8  # rows that start on a counter block and a chunk, as the part alone does
    m = rows - first
    x, res, dy = (torch.zeros(rows, cols, device="cuda", dtype=torch.bfloat16) for _ in range(3))
    for i, t in enumerate((x, res, dy)):
        t[first:] = _normal(m, cols, seed=i)
    w = _normal(cols, seed=9)

    def run(x, res, dy, offset):
        x, res = x.detach().requires_grad_(), res.detach().requires_grad_()
        y, h = api.residual_rms_norm(x, res, w, p=0.2, seed=3, offset=offset)
        dx, dres = torch.autograd.grad((y, h), (x, res), (dy, dy))
        q, s, _ = api.residual_rms_norm_8bit(x.detach(), res.detach(), w, group=64)
        return [t.detach()[-m:].clone() for t in (y, h, dx, dres, q.view(torch.uint8), s,
                                                  api.dequantize_8bit(q, s), api.dropout(x.detach(), 0.2, 3, offset))]

    a, b = run(x, res, dy, 0), run(x[first:], res[first:], dy[first:], first * cols // 4)
    assert [torch.equal(s, t) for s, t in zip(a, b)] == [True] * len(a)
