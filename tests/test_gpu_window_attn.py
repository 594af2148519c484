"""Windowed attention with sinks (training and single-token forms) against the
64-bit definition, within the bounds that tests/window_oracle.py derives."""

import math

import pytest
import torch

from tests import window_oracle as oracle

pytestmark = pytest.mark.gpu


def _cu(lens):
    return torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32, device="cuda")


def _inputs(nq, nk, hq, hkv, d, dtype, seed=0, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda n, h: (torch.randn(n, h, d, device="cuda", generator=g) * std).to(dtype)  # noqa: E731
    return r(nq, hq), r(nk, hkv), r(nk, hkv), r(nq, hq)


def _check(got, ref, names):
    for n in names:
        x, y, b = got[n].double(), ref[n], ref["b_" + n]
        assert torch.isfinite(x).all(), n
        over = ((x - y).abs() - b).max().item() if x.numel() else 0.0
        assert over <= 1e-12, f"{n}: {over:.3g} beyond the bound"


def _run(q, k, v, do, cu_q, cu_k, **kw):
    from lsrm_sparse import api, ops

    q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
    out, lse = api.window_sink_attention(q, k, v, cu_q, cu_k, return_lse=True, **kw)
    dq, dk, dv = torch.autograd.grad(out, (q, k, v), do)
    assert ops.read_errors() == 0
    return {"out": out.detach(), "lse": lse.t(), "dq": dq, "dk": dk, "dv": dv}


CASES = [
    # lens_q, lens_k (None: the same), Hq, Hkv, D, window, sinks, causal, dtype
    ([1], None, 1, 1, 64, 1, 0, True, torch.bfloat16),
    ([1, 77, 222], None, 8, 4, 64, 128, 4, True, torch.bfloat16),
    ([700], None, 4, 4, 64, 128, 16, False, torch.bfloat16),
    ([513], None, 4, 1, 128, 64, 7, True, torch.float16),
    ([300, 0, 45, 1], None, 6, 2, 32, 33, 1, True, torch.float16),
    ([129, 255], None, 5, 1, 128, 1000, 0, True, torch.bfloat16),
    ([640], None, 2, 2, 128, 1, 128, True, torch.bfloat16),
    ([500], None, 3, 1, 64, 100, 128, False, torch.float16),
    ([1000], None, 16, 1, 64, 200, 4, True, torch.bfloat16),
    ([260], None, 28, 4, 64, 50, 2, True, torch.bfloat16),
    ([900], None, 1, 1, 32, 2, 3, False, torch.bfloat16),
    # chunks of queries at the end of longer key sequences, and more queries than keys (rows that see nothing)
    ([5, 130, 64], [700, 130, 0], 4, 2, 64, 96, 4, True, torch.bfloat16),
    ([300, 40], [100, 41], 2, 1, 128, 64, 8, True, torch.bfloat16),
    ([300, 40], [100, 41], 2, 1, 64, 64, 8, False, torch.float16),
    ([33, 200], [333, 1200], 8, 1, 64, 256, 64, False, torch.bfloat16),
]


@pytest.mark.parametrize("lens_q,lens_k,hq,hkv,d,window,sinks,causal,dtype", CASES)
def test_forward_and_gradients(lens_q, lens_k, hq, hkv, d, window, sinks, causal, dtype):
    cu_q = _cu(lens_q)
    cu_k = cu_q if lens_k is None else _cu(lens_k)
    q, k, v, do = _inputs(int(cu_q[-1]), int(cu_k[-1]), hq, hkv, d, dtype, seed=hq + d)
    got = _run(q, k, v, do, cu_q, cu_k, window=window, sinks=sinks, causal=causal)
    ref = oracle.attention(q, k, v, cu_q, cu_k, window, sinks, causal, dout=do, bounds=True)
    _check(got, ref, ("out", "dq", "dk", "dv"))
    live = torch.isfinite(ref["lse"])
    assert torch.equal(torch.isfinite(got["lse"]), live)
    # scores up to ~30 from sums of d products in 32 bits
    assert (got["lse"].double() - ref["lse"])[live].abs().max().item() <= 1e-4 if live.any() else True


@pytest.mark.parametrize("std", [0.05, 6.0])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_flat_and_peaked_scores(std, dtype):
    """Nearly uniform rows, and rows that one key takes (scores of hundreds: the running maximum moves far)."""
    cu = _cu([400])
    q, k, v, do = _inputs(400, 400, 4, 2, 64, dtype, seed=3, std=std)
    got = _run(q, k, v, do, cu, cu, window=150, sinks=4, causal=True)
    _check(got, oracle.attention(q, k, v, cu, cu, 150, 4, True, dout=do, bounds=True), ("out", "dq", "dk", "dv"))


def test_rising_scores():
    """Scores that rise along the keys: every tile sets a new maximum."""
    n, d = 600, 64
    cu = _cu([n])
    q, k, v, do = _inputs(n, n, 2, 1, d, torch.bfloat16, seed=4)
    q = q.abs()
    k = (k.abs() * torch.linspace(0.0, 8.0, n, device="cuda")[:, None, None]).to(k.dtype)
    got = _run(q, k, v, do, cu, cu, window=n, sinks=0, causal=True)
    _check(got, oracle.attention(q, k, v, cu, cu, n, 0, True, dout=do, bounds=True), ("out", "dq", "dk", "dv"))


@pytest.mark.parametrize("scale", [0.01, 0.5])
def test_softmax_scale(scale):
    cu = _cu([200])
    q, k, v, do = _inputs(200, 200, 2, 2, 64, torch.bfloat16, seed=5)
    got = _run(q, k, v, do, cu, cu, window=64, sinks=4, causal=True, softmax_scale=scale)
    _check(got, oracle.attention(q, k, v, cu, cu, 64, 4, True, scale=scale, dout=do, bounds=True),
           ("out", "dq", "dk", "dv"))


@pytest.mark.parametrize("d,hq,hkv", [(64, 4, 2), (128, 3, 1), (32, 8, 8)])
def test_packed_projection_views(d, hq, hkv):
    """q, k and v as slices of one [N, (Hq + 2 Hkv) D] projection give what contiguous tensors give, bit for bit."""
    n = 333
    cu = _cu([100, n - 100])
    g = torch.Generator(device="cuda").manual_seed(d)
    qkv = torch.randn(n, (hq + 2 * hkv) * d, device="cuda", generator=g).bfloat16()
    q, k, v = (t.unflatten(1, (-1, d)) for t in qkv.split([hq * d, hkv * d, hkv * d], 1))
    do = torch.randn(n, hq, d, device="cuda", generator=g).bfloat16()
    a = _run(q, k, v, do, cu, cu, window=60, sinks=2, causal=True)
    b = _run(q.contiguous(), k.contiguous(), v.contiguous(), do, cu, cu, window=60, sinks=2, causal=True)
    assert all(torch.equal(a[x], b[x]) for x in a)
    # a layout that the kernels do not take as it is: heads outside tokens
    c = _run(q.transpose(0, 1).contiguous().transpose(0, 1), k, v, do, cu, cu, window=60, sinks=2, causal=True)
    assert all(torch.equal(a[x], c[x]) for x in a)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("d", [32, 64, 128])
def test_tokens_outside_the_sequences_do_not_matter(causal, d):
    """NaN and infinities after the last sequence reach no output, and get zero outputs and gradients."""
    lens, n, pad = [150, 67], 217, 90
    cu = _cu(lens)
    q, k, v, do = _inputs(n + pad, n + pad, 4, 2, d, torch.bfloat16, seed=6)
    for t in (q, k, v, do):
        t[n:] = math.nan
        t[n + 1::3] = math.inf
    got = _run(q, k, v, do, cu, cu, window=40, sinks=3, causal=causal)
    ref = oracle.attention(q[:n], k[:n], v[:n], cu, cu, 40, 3, causal, dout=do[:n], bounds=True)
    _check({x: got[x][:n] for x in ("out", "dq", "dk", "dv")}, ref, ("out", "dq", "dk", "dv"))
    for x in ("out", "dq", "dk", "dv"):
        assert (got[x][n:] == 0).all(), x


def test_a_neighbour_sequence_does_not_matter():
    """A sequence's results do not depend on what its neighbours hold, NaN included."""
    lens = [100, 61, 200]
    cu = _cu(lens)
    q, k, v, do = _inputs(361, 361, 2, 2, 64, torch.bfloat16, seed=7)
    a = _run(q, k, v, do, cu, cu, window=48, sinks=4, causal=True)
    for t in (q, k, v, do):
        t[100:161] = math.nan
    b = _run(q, k, v, do, cu, cu, window=48, sinks=4, causal=True)
    for x in ("out", "dq", "dk", "dv"):
        assert torch.equal(a[x][:100], b[x][:100]) and torch.equal(a[x][161:], b[x][161:]), x
        assert torch.isnan(b[x][100:161]).any()


def test_gradients_against_differences():
    """Directional differences of the 64-bit loss against the kernels' gradients."""
    cu = _cu([90, 38])
    q, k, v, do = _inputs(128, 128, 4, 2, 64, torch.float16, seed=8)
    got = _run(q, k, v, do, cu, cu, window=30, sinks=4, causal=True)
    g = torch.Generator(device="cuda").manual_seed(9)
    base = [t.double() for t in (q, k, v)]

    def loss(*t):
        return (oracle.attention(*t, cu, cu, 30, 4, True)["out"] * do.double()).sum().item()

    for i, name in enumerate(("dq", "dk", "dv")):
        step = torch.randn(base[i].shape, device="cuda", generator=g, dtype=torch.float64)
        h = 1e-4
        up, down = (loss(*[b + s * h * step if j == i else b for j, b in enumerate(base)]) for s in (1, -1))
        diff = (up - down) / (2 * h)
        grad = got[name].double()
        # each gradient element is off by a few units of 2^-11: random signs against the step add in quadrature
        tol = 6 * 3 * 2.0**-11 * (grad * step).norm().item() + 1e-5 * abs(diff)
        assert abs((grad * step).sum().item() - diff) <= tol, name


def test_same_bits_twice_and_on_another_stream():
    cu = _cu([257, 1000])
    q, k, v, do = _inputs(1257, 1257, 8, 2, 64, torch.bfloat16, seed=10)
    kw = dict(window=128, sinks=4, causal=True)
    a = _run(q, k, v, do, cu, cu, **kw)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b = _run(q, k, v, do, cu, cu, **kw)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a[x], b[x]) for x in a)


def test_many_short_sequences():
    lens = [1 + (7 * i) % 23 for i in range(400)]
    cu = _cu(lens)
    n = int(cu[-1])
    q, k, v, do = _inputs(n, n, 4, 2, 64, torch.bfloat16, seed=11)
    got = _run(q, k, v, do, cu, cu, window=5, sinks=2, causal=True)
    _check(got, oracle.attention(q, k, v, cu, cu, 5, 2, True, dout=do, bounds=True), ("out", "dq", "dk", "dv"))


def test_no_tokens():
    from lsrm_sparse import api

    cu = torch.zeros(3, dtype=torch.int32, device="cuda")
    q = torch.empty(0, 4, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    kv = torch.empty(0, 2, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    out = api.window_sink_attention(q, kv, kv, cu, window=8)
    dq, dk = torch.autograd.grad(out, (q, kv), out.detach())
    assert out.shape == (0, 4, 64) and dq.shape == q.shape and dk.shape == kv.shape


def test_offsets_that_leave_the_tensors_are_reported():
    from lsrm_sparse import api, ops

    q, k, v, _ = _inputs(100, 100, 2, 2, 64, torch.bfloat16)
    cu = torch.tensor([0, 60, 130], dtype=torch.int32, device="cuda")
    api.window_sink_attention(q, k, v, cu, window=8)
    assert ops.read_errors() & 0x8
    assert ops.read_errors() == 0


def test_matches_the_sliding_band():
    """Without sinks, the symmetric form is the band of ``sliding_window_attention``."""
    from lsrm_sparse import api

    cu = _cu([300, 212])
    q, k, v, _ = _inputs(512, 512, 4, 4, 64, torch.bfloat16, seed=12)
    a = api.window_sink_attention(q, k, v, cu, window=64, causal=False)
    b = api.sliding_window_attention(q, k, v, cu, 64)
    ref = oracle.attention(q, k, v, cu, cu, 64, 0, False, bounds=True)
    assert ((a.double() - b.double()).abs() <= 2 * ref["b_out"]).all()


# ------------------------------ single token ---------------------------------


def _decode_ref(q, k_new, v_new, kc, vc, lengths, window, sinks, scale=None):
    b, hq, d = q.shape
    hkv, cap = k_new.shape[1], kc.shape[1]
    u = oracle.UNIT[q.dtype]
    out = torch.zeros(b, hq, d, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    for i, n in enumerate(lengths.tolist()):
        if n < 0:
            continue
        pos = sorted(set(range(min(sinks, n + 1))) | set(range(max(0, n + 1 - window), n + 1)))
        slot = [j if j < sinks else sinks + (j - sinks) % (cap - sinks) for j in pos]
        kc[i, slot[-1] if pos[-1] == n else slot[pos.index(n)]] = k_new[i]
        vc[i, slot[-1] if pos[-1] == n else slot[pos.index(n)]] = v_new[i]
        k, v = kc[i, slot].double(), vc[i, slot].double()
        for h in range(hq):
            s = k[:, h // (hq // hkv)] @ q[i, h].double() * (scale or d**-0.5)
            p = torch.softmax(s, 0)
            vv = v[:, h // (hq // hkv)]
            out[i, h] = p @ vv
            bound[i, h] = u * out[i, h].abs() + (u + 2.0**-14) * (p @ vv.abs()) + (
                2.0**-25 * vv.abs().sum(0) if q.dtype == torch.float16 else 0.0)
    return out, bound


DECODE = [
    # lengths, Hq, Hkv, D, window, sinks, slack (capacity past sinks + window), dtype
    ([0], 1, 1, 64, 1, 0, 0, torch.bfloat16),
    ([0, 1, 2, 3, 4, 5, 100], 8, 4, 64, 16, 4, 0, torch.bfloat16),
    ([700, 15, -1, 16, 17, 3000], 16, 2, 128, 512, 4, 0, torch.bfloat16),
    ([1000], 16, 16, 64, 2000, 0, 0, torch.float16),
    ([5000, 63, 64, 65], 12, 4, 32, 1000, 64, 37, torch.float16),
    ([257, 9], 28, 4, 128, 256, 1, 5, torch.bfloat16),
    ([9000, 31], 64, 1, 64, 8192, 16, 0, torch.bfloat16),
    ([130, 0, 4], 5, 5, 128, 64, 130, 0, torch.bfloat16),
]


@pytest.mark.parametrize("lengths,hq,hkv,d,window,sinks,slack,dtype", DECODE)
def test_decode(lengths, hq, hkv, d, window, sinks, slack, dtype):
    from lsrm_sparse import api

    b, cap = len(lengths), sinks + window + slack
    g = torch.Generator(device="cuda").manual_seed(hq + d)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g).to(dtype)  # noqa: E731
    q, kn, vn = r(b, hq, d), r(b, hkv, d), r(b, hkv, d)
    kc, vc = r(b, cap, hkv, d), r(b, cap, hkv, d)
    for i, n in enumerate(lengths):  # slots that no position fills hold anything
        if n < cap:
            kc[i, max(n, 0):] = math.nan
            vc[i, max(n, 0):] = math.nan
    ln = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    kr, vr = kc.clone(), vc.clone()
    out = api.window_sink_decode(q, kn, vn, kc, vc, ln, window=window, sinks=sinks)
    ref, bound = _decode_ref(q, kn, vn, kr, vr, ln, window, sinks)
    assert torch.equal(kc.view(torch.int16), kr.view(torch.int16)), "k_cache"
    assert torch.equal(vc.view(torch.int16), vr.view(torch.int16)), "v_cache"
    assert ((out.double() - ref).abs() <= bound).all()


def test_decode_strided_caches_and_scale():
    """Caches interleaved in one [B, capacity, 2, Hkv, D] buffer, q / k / v from one projection."""
    from lsrm_sparse import api

    b, hq, hkv, d, window, sinks = 3, 8, 2, 64, 100, 4
    g = torch.Generator(device="cuda").manual_seed(1)
    both = torch.randn(b, sinks + window, 2, hkv, d, device="cuda", generator=g).bfloat16()
    kc, vc = both[:, :, 0], both[:, :, 1]
    qkv = torch.randn(b, hq + 2 * hkv, d, device="cuda", generator=g).bfloat16()
    q, kn, vn = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    ln = torch.tensor([50, 104, 999], dtype=torch.int32, device="cuda")
    kr, vr = kc.clone(), vc.clone()
    out = api.window_sink_decode(q, kn, vn, kc, vc, ln, window=window, sinks=sinks, softmax_scale=0.3)
    ref, bound = _decode_ref(q, kn, vn, kr, vr, ln, window, sinks, 0.3)
    assert torch.equal(kc, kr) and torch.equal(vc, vr)
    assert ((out.double() - ref).abs() <= bound).all()


def test_decode_continues_a_prompt():
    """Tokens answered one by one over the ring give the rows of the packed causal form."""
    from lsrm_sparse import api

    n, hq, hkv, d, window, sinks = 90, 4, 2, 64, 24, 3
    cu = _cu([n])
    q, k, v, _ = _inputs(n, n, hq, hkv, d, torch.bfloat16, seed=13)
    ref = oracle.attention(q, k, v, cu, cu, window, sinks, True, bounds=True)
    kc = torch.full((1, sinks + window, hkv, d), math.nan, device="cuda", dtype=torch.bfloat16)
    vc = kc.clone()
    for i in range(n):
        ln = torch.tensor([i], dtype=torch.int32, device="cuda")
        out = api.window_sink_decode(q[i:i + 1], k[i:i + 1], v[i:i + 1], kc, vc, ln, window=window, sinks=sinks)
        assert ((out.double() - ref["out"][i]).abs() <= ref["b_out"][i]).all(), i


@pytest.mark.parametrize("change,error", [
    (dict(q=lambda t: t.float()), (TypeError, ValueError)),
    (dict(q=lambda t: t[..., :48]), ValueError),
    (dict(q=lambda t: t.cpu()), ValueError),
    (dict(k=lambda t: t[:-1]), ValueError),
    (dict(window=0), ValueError),
    (dict(sinks=-1), ValueError),
    (dict(sinks=129), RuntimeError),
    (dict(q=lambda t: t[:, :3]), RuntimeError),
    (dict(cu=lambda t: t.long()), ValueError),
])
def test_refusals(change, error):
    from lsrm_sparse import api

    q, k, v, _ = _inputs(64, 64, 4, 2, 64, torch.bfloat16)
    a = dict(q=q, k=k, v=v, cu=_cu([64]), window=8, sinks=2)
    for n, f in change.items():
        a[n] = f(a[n]) if callable(f) else f
    with pytest.raises(error):
        api.window_sink_attention(a["q"], a["k"], a["v"], a["cu"], window=a["window"], sinks=a["sinks"])


def test_decode_refusals():
    from lsrm_sparse import api

    g = lambda *s: torch.zeros(*s, device="cuda", dtype=torch.bfloat16)  # noqa: E731
    ln = torch.zeros(2, dtype=torch.int32, device="cuda")
    args = [g(2, 4, 64), g(2, 2, 64), g(2, 2, 64), g(2, 20, 2, 64), g(2, 20, 2, 64), ln]
    api.window_sink_decode(*args, window=16, sinks=4)
    with pytest.raises(RuntimeError, match="capacity"):
        api.window_sink_decode(*args, window=17, sinks=4)
    for i, bad in ((0, g(3, 4, 64)), (1, g(2, 2, 32)), (3, g(2, 20, 2, 64).transpose(1, 2)), (5, ln.long()),
                   (4, g(2, 19, 2, 64))):
        with pytest.raises(ValueError):
            api.window_sink_decode(*[bad if j == i else t for j, t in enumerate(args)], window=16, sinks=4)
