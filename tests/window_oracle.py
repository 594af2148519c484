"""Attention with a sliding window and sinks in 64 bits, from the definition,
with bounds on how far a kernel that rounds its probabilities and results to
16 bits may be from it.

u is the 16-bit type's unit roundoff (2^-8 bf16, 2^-11 fp16).  With scores,
statistics and sums in 32 bits, and the probabilities p, the score gradients ds
and the results each rounded once,

    |out - o|   <= u |o|  + u sum_j p |v|
    |dv' - dv|  <= u |dv| + u sum_i p |do|
    |dq' - dq|  <= u |dq| + scale sum_j (u |ds| + u p D_i) |k|
    |dk' - dk|  <= u |dk| + scale sum_i (u |ds| + u p D_i) |q|

where D_i = sum_d |do o| bounds what the rounded output does to delta.  32-bit
arithmetic adds at most 2^-14 of the same sums (p, ds up to |p (|dp| + D)|), and
a value below the 16-bit type's normal range is off by at most 2^-25 (fp16).
"""

import math

import torch

UNIT = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}


def visible(lq, lk, window, sinks, causal, device="cpu"):
    pos = torch.arange(lq, device=device)[:, None] + lk - lq
    j = torch.arange(lk, device=device)[None]
    if causal:
        return (j <= pos) & ((pos - j < window) | (j < sinks))
    return ((pos - j).abs() <= window // 2) | (j < sinks)


def attention(q, k, v, cu_q, cu_k, window, sinks, causal, scale=None, dout=None, bounds=False):
    """q [Nq, Hq, D] etc. of any dtype; returns a dict of float64 tensors: out, lse [Nq, Hq] and, with dout, dq, dk,
    dv; with ``bounds`` also their elementwise bounds under "b_" names."""
    u = UNIT.get(q.dtype, 0.0)
    tiny = 2.0**-25 if q.dtype == torch.float16 else 0.0
    rel = 2.0**-14
    q, k, v = q.detach().double(), k.detach().double(), v.detach().double()
    hq, hkv, d = q.shape[1], k.shape[1], q.shape[2]
    g = hq // hkv
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    r = {"out": torch.zeros_like(q), "lse": torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=q.device)}
    names = ["out"]
    if dout is not None:
        do = dout.detach().double()
        r.update(dq=torch.zeros_like(q), dk=torch.zeros_like(k), dv=torch.zeros_like(v))
        names += ["dq", "dk", "dv"]
    if bounds:
        r.update({"b_" + n: torch.zeros_like(r[n]) for n in names})
    cq, ck = cu_q.tolist(), cu_k.tolist()
    for a, b, c, e in zip(cq[:-1], cq[1:], ck[:-1], ck[1:]):
        vis = visible(b - a, e - c, window, sinks, causal, q.device)
        for h in range(hq):
            kk, vv, qq = k[c:e, h // g], v[c:e, h // g], q[a:b, h]
            s = (qq @ kk.T * scale).masked_fill(~vis, -math.inf)
            lse = torch.logsumexp(s, 1) if e > c else torch.full((b - a,), -math.inf, dtype=s.dtype, device=s.device)
            p = torch.where(vis, (s - lse[:, None].clamp(min=-1e300)).exp(), torch.zeros_like(s))
            o = p @ vv
            r["out"][a:b, h], r["lse"][a:b, h] = o, lse
            vf = vis.double()
            if bounds:
                r["b_out"][a:b, h] = tiny + u * o.abs() + (u + rel) * (p @ vv.abs()) + tiny * (vf @ vv.abs())
            if dout is None:
                continue
            dd = do[a:b, h]
            dp = dd @ vv.T
            ds = p * (dp - (dd * o).sum(1, keepdim=True))
            r["dq"][a:b, h] = ds @ kk * scale
            r["dk"][c:e, h // g] += ds.T @ qq * scale
            r["dv"][c:e, h // g] += p.T @ dd
            if bounds:
                big = (dd * o).abs().sum(1, keepdim=True)
                es = u * ds.abs() + u * p * big + rel * p * (dd.abs() @ vv.abs().T + big) + tiny * vf
                r["b_dq"][a:b, h] = es @ kk.abs() * scale
                r["b_dk"][c:e, h // g] += es.T @ qq.abs() * scale
                r["b_dv"][c:e, h // g] += ((u + rel) * p + tiny * vf).T @ dd.abs()
    if bounds and dout is not None:
        for n in ("dq", "dk", "dv"):
            r["b_" + n] += u * r[n].abs() + tiny
    return r
