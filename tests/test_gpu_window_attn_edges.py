"""Windowed attention with sinks where the sequences do not fill the tensors, at
strides that are no multiple of a head, with no queries or no keys."""

import math

import pytest
import torch

from tests import window_oracle as oracle
from tests.test_gpu_window_attn import _check, _cu, _inputs, _run

pytestmark = pytest.mark.gpu

NAMES = ("out", "dq", "dk", "dv")


def _poison():
    """Memory that the allocator hands out next holds NaN."""
    for n in (1 << 12, 1 << 16, 1 << 20, 1 << 23):
        del_me = [torch.full((n,), math.nan, device="cuda") for _ in range(8)]
        del del_me


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("d,hq,hkv", [(32, 16, 1), (64, 4, 2), (128, 2, 2)])
@pytest.mark.parametrize("lead_q,lead_k,trail", [(1, 1, 0), (64, 64, 3), (130, 130, 70), (300, 17, 0), (17, 300, 1), (0, 5, 0)])
def test_tokens_before_the_first_sequence(causal, d, hq, hkv, lead_q, lead_k, trail):
    """They get zero outputs and gradients, and what they hold (NaN, infinities) reaches nothing."""
    lens = [150, 0, 67]
    n = sum(lens)
    cu = _cu(lens)
    q, _, _, do = _inputs(lead_q + n + trail, 1, hq, hkv, d, torch.bfloat16, seed=lead_q)
    _, k, v, _ = _inputs(1, lead_k + n + trail, hq, hkv, d, torch.bfloat16, seed=lead_k + 1)
    for t, lead in ((q, lead_q), (do, lead_q), (k, lead_k), (v, lead_k)):
        t[:lead] = math.nan
        t[1:lead:3] = math.inf
        t[lead + n:] = math.nan
    _poison()
    got = _run(q, k, v, do, cu + lead_q, cu + lead_k, window=40, sinks=3, causal=causal)
    sq, sk = slice(lead_q, lead_q + n), slice(lead_k, lead_k + n)
    ref = oracle.attention(q[sq], k[sk], v[sk], cu, cu, 40, 3, causal, dout=do[sq], bounds=True)
    _check({x: got[x][sq if x in ("out", "dq") else sk] for x in NAMES}, ref, NAMES)
    for x in NAMES:
        s = sq if x in ("out", "dq") else sk
        assert (got[x][:s.start] == 0).all() and (got[x][s.stop:] == 0).all(), x
    assert (got["lse"][:lead_q] == -math.inf).all()


def test_no_sequence_at_all():
    """Offsets of no sequence: every token is outside."""
    for at in (0, 30, 77):
        cu = torch.tensor([at], dtype=torch.int32, device="cuda")
        q, k, v, do = _inputs(77, 77, 2, 1, 64, torch.bfloat16)
        _poison()
        got = _run(q, k, v, do, cu, cu, window=8, sinks=2, causal=True)
        assert all((got[x] == 0).all() for x in NAMES)


def test_softmax_scale_refusals():
    from lsrm_sparse import api

    q, k, v, _ = _inputs(64, 64, 4, 2, 64, torch.bfloat16)
    kc, vc = (torch.zeros(64, 10, 2, 64, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    ln = torch.zeros(64, dtype=torch.int32, device="cuda")
    for scale in (-0.125, math.nan, math.inf):
        with pytest.raises(ValueError, match="softmax_scale"):
            api.window_sink_attention(q, k, v, _cu([64]), window=8, softmax_scale=scale)
        with pytest.raises(ValueError, match="softmax_scale"):
            api.window_sink_decode(q, k, v, kc, vc, ln, window=8, softmax_scale=scale)
    a = api.window_sink_attention(q, k, v, _cu([64]), window=8)
    assert torch.equal(a, api.window_sink_attention(q, k, v, _cu([64]), window=8, softmax_scale=0.0))


@pytest.mark.parametrize("window,sinks,slack", [(1, 0, 0), (16, 4, 3), (200, 1, 0)])
def test_decode_at_the_largest_lengths(window, sinks, slack):
    from lsrm_sparse import api
    from tests.test_gpu_window_attn import _decode_ref

    g = torch.Generator(device="cuda").manual_seed(2)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g).bfloat16()  # noqa: E731
    cap = sinks + window + slack
    q, kn, vn, kc, vc = r(3, 4, 64), r(3, 2, 64), r(3, 2, 64), r(3, cap, 2, 64), r(3, cap, 2, 64)
    ln = torch.tensor([2**31 - 1, 2**31 - 2, 2**30], dtype=torch.int32, device="cuda")
    kr, vr = kc.clone(), vc.clone()
    # the oracle counts positions one by one: the same slots as at lengths a whole number of rings smaller
    ring = cap - sinks
    small = torch.tensor([sinks + window + (n - sinks - window) % ring for n in ln.tolist()], device="cuda")
    out = api.window_sink_decode(q, kn, vn, kc, vc, ln, window=window, sinks=sinks)
    ref, bound = _decode_ref(q, kn, vn, kr, vr, small, window, sinks)
    assert torch.equal(kc, kr) and torch.equal(vc, vr)
    assert ((out.double() - ref).abs() <= bound).all()


def test_more_sequences_than_a_grid_dimension():
    """70001 sequences of one token, each its own sink: out = v, dv = do, and the scores' gradients cancel."""
    n, hq, hkv, d = 70001, 2, 1, 32
    cu = torch.arange(n + 1, device="cuda", dtype=torch.int32)
    q, k, v, do = _inputs(n, n, hq, hkv, d, torch.bfloat16, seed=14)
    _poison()
    got = _run(q, k, v, do, cu, cu, window=4, sinks=1, causal=True)
    assert torch.equal(got["out"], v.expand(n, hq, d))
    # a sum of two 16-bit values, rounded once
    assert torch.equal(got["dv"], do.float().sum(1, keepdim=True).bfloat16())
    big = (do.double().abs() * v.double().abs()).sum(2).amax(1, keepdim=True)[..., None] * d**-0.5 * 2.0**-14
    assert (got["dq"].double().abs() <= big * k.double().abs()).all()
    assert (got["dk"].double().abs() <= hq * big * q.double().abs().amax(1, keepdim=True)).all()


@pytest.mark.parametrize("d,hq,hkv", [(32, 6, 2), (64, 4, 4), (128, 3, 1)])
def test_token_strides_that_are_no_multiple_of_a_head(d, hq, hkv):
    """Rows padded by eight elements, and by a head and eight: the bits of contiguous tensors."""
    cu = _cu([100, 1, 232])
    q, k, v, do = _inputs(333, 333, hq, hkv, d, torch.bfloat16, seed=15)

    def padded(t, pad):
        n, h, _ = t.shape
        return torch.full((n, h * d + pad), math.nan, device="cuda", dtype=t.dtype)[:, :h * d].unflatten(1, (h, d)).copy_(t)

    a = _run(q, k, v, do, cu, cu, window=60, sinks=2, causal=True)
    b = _run(padded(q, 8), padded(k, d + 8), padded(v, 24), padded(do, 8), cu, cu, window=60, sinks=2, causal=True)
    assert all(torch.equal(a[x], b[x]) for x in a)


@pytest.mark.parametrize("d,hq,hkv", [(32, 8, 1), (64, 4, 2), (128, 2, 2)])
def test_no_queries_or_no_keys(d, hq, hkv):
    """One side empty: the other side's outputs and gradients are zero."""
    zero, some = _cu([0, 0]), _cu([70, 61])
    for cu_q, cu_k in ((zero, some), (some, zero)):
        nq, nk = int(cu_q[-1]), int(cu_k[-1])
        q, k, v, do = _inputs(nq, nk, hq, hkv, d, torch.float16, seed=16)
        _poison()
        got = _run(q, k, v, do, cu_q, cu_k, window=8, sinks=2, causal=False)
        assert all((got[x] == 0).all() for x in NAMES)
        assert got["dk"].shape[0] == nk and got["out"].shape[0] == nq


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_delta_does_not_inherit_the_outputs_rounding(dtype):
    """Keys and values around a large common one, nearly uniform rows of a hundred keys and more: the rounding of the
    output then moves delta, and with it dq, by more than everything else does.  The 64-bit error of a delta from the
    rounded output predicts the backward without what the rounding left over; with it the error is a small part of that:
    p's roundings, which a row averages (1 / sqrt(100)), and ds's, which meet the values' spread (1/16) alone."""
    from lsrm_sparse import ops

    n, hq, hkv, d, window = 600, 4, 2, 64, 300
    g = torch.Generator(device="cuda").manual_seed(17)
    r = lambda h: torch.randn(n, h, d, device="cuda", generator=g)  # noqa: E731
    q, k, v, do = ((0.3 * r(hq)).to(dtype), (1 + 0.3 * r(hkv)).to(dtype), (4 + 0.25 * r(hkv)).to(dtype), r(hq).to(dtype))
    cu = _cu([n])
    args = (cu, cu, window, 4, True)
    ref = oracle.attention(q, k, v, cu, cu, window, 4, True, dout=do)
    out, lse, rest = ops.window_attn_fwd(q, k, v, *args, need_rest=True)
    # what an error of delta does to dq: - scale * error * sum_j p_j k_j
    vis = oracle.visible(n, n, window, 4, True, "cuda")
    moved = torch.empty_like(ref["dq"])
    off = (do.double() * (ref["out"].to(dtype).double() - ref["out"])).sum(2)
    for h in range(hq):
        s = (q[:, h].double() @ k[:, h // 2].double().T * d**-0.5).masked_fill(~vis, -math.inf)
        moved[:, h] = -d**-0.5 * off[:, h, None] * (torch.softmax(s, 1) @ k[:, h // 2].double())
    rows = slice(100, None)  # a hundred keys at least
    err = {}
    for name, left in (("without", None), ("with", rest)):
        dq, dk, dv = ops.window_attn_bwd(q, k, v, out, left, lse, do, *args)
        err[name] = (dq.double() - ref["dq"])[rows].norm().item()
    predicted = moved[rows].norm().item()
    assert 0.7 * predicted <= err["without"] <= 1.4 * predicted
    assert err["with"] <= 0.35 * predicted


FEW = [
    # lens, Hq, Hkv, D, window, sinks, causal
    ([81, 40], 1, 1, 32, 1, 7, False),
    ([1005], 2, 2, 64, 8, 7, True),
    ([1, 2, 3, 9, 40, 64, 33, 50], 16, 8, 64, 3000, 1, True),
    ([5, 17, 64, 3], 64, 4, 64, 3000, 16, False),
    ([700, 130], 6, 2, 128, 20, 40, True),   # the sinks in a tile of their own
    ([900], 4, 1, 32, 40, 23, False),        # 20 + 20 + 1 + 23 keys: the most that counts as few
    ([466, 30], 8, 1, 128, 50, 14, True),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens,hq,hkv,d,window,sinks,causal", FEW)
def test_rows_of_few_keys_keep_what_rounding_p_leaves_over(lens, hq, hkv, d, window, sinks, causal, dtype):
    """Up to 64 keys a row, P enters the output's product unrounded to 2^-16: out is off by its own rounding, and dq and
    dk by dS's and theirs.  Scores of some units from sums of up to 128 products in 32 bits, and the exponentials, are
    within 2^-17."""
    u = oracle.UNIT[dtype]
    tiny = 2.0**-25 if dtype == torch.float16 else 0.0
    rel, left = 2.0**-17, 2.0**-16
    cu = _cu(lens)
    n = int(cu[-1])
    q, k, v, do = _inputs(n, n, hq, hkv, d, dtype, seed=18)
    got = _run(q, k, v, do, cu, cu, window=window, sinks=sinks, causal=causal)
    ref = oracle.attention(q, k, v, cu, cu, window, sinks, causal, dout=do)
    bound = {x: u * ref[x].abs() + tiny for x in ("out", "dq", "dk")}
    scale = d**-0.5
    at = 0
    for length in lens:
        s = slice(at, at + length)
        at += length
        vis = oracle.visible(length, length, window, sinks, causal, "cuda")
        for h in range(hq):
            qq, kk, vv, dd = q[s, h].double(), k[s, h // (hq // hkv)].double(), v[s, h // (hq // hkv)].double(), do[s, h].double()
            p = torch.softmax((qq @ kk.T * scale).masked_fill(~vis, -math.inf), 1)
            spread = p @ vv.abs()
            bound["out"][s, h] += (left + rel) * spread + tiny * (vis.double() @ vv.abs())
            dp, delta = dd @ vv.T, (dd * ref["out"][s, h]).sum(1, keepdim=True)
            big = (dd.abs() * spread).sum(1, keepdim=True)
            ds = u * (p * (dp - delta)).abs() + p * ((left + rel) * big + 2 * rel * (dd.abs() @ vv.abs().T + big)) + tiny * vis
            bound["dq"][s, h] += ds @ kk.abs() * scale
            bound["dk"][s, h // (hq // hkv)] += ds.T @ qq.abs() * scale
    for x in ("out", "dq", "dk"):
        over = ((got[x].double() - ref[x]).abs() - bound[x]).max().item()
        assert over <= 1e-12, f"{x}: {over:.3g} beyond the bound"
