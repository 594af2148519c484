"""What the decoder-layer operators are measured on: attention with a sliding window and sinks (training pass and
single-token form over a ring cache), the residual RMS norm with its branch dropout and 8-bit output, and dropout from
a counter-based generator.

``run`` computes a case in elementary torch operations in 32 bits, or, where ``own`` is true, through
``lsrm_sparse.api``.
"""

import math
import os
import sys

import numpy as np
import torch

own = False

_PACKAGE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                        "large-sparse-reconstruction-model_b200")
_CHUNK = 512  # queries that the plain attention takes against one band of keys
_MOST_SCORES = 131072 * 16 * 1024 * 1.02  # scores of the largest listed case's bands
_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32,
       "e4m3": torch.float8_e4m3fn, "int8": torch.int8}
_Q8_MAX = {"e4m3": 448.0, "int8": 127.0}


def _api():
    if _PACKAGE not in sys.path:
        sys.path.insert(0, _PACKAGE)
    from lsrm_sparse import api

    return api


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------


def listed():
    return [
        # a training step's shortest sequences: three ragged ones, one of a single token
        {"name": "attn_short", "op": "attn", "tokens": 300, "seqs": 3, "hq": 8, "hkv": 4, "d": 64, "window": 128,
         "sinks": 4, "causal": True, "dtype": "bf16"},
        # the decoder's voxel tokens: one sequence, symmetric window, first tokens visible to all
        {"name": "attn_voxel", "op": "attn", "tokens": 131072, "seqs": 1, "hq": 16, "hkv": 16, "d": 64, "window": 512,
         "sinks": 16, "causal": False, "dtype": "bf16"},
        # long causal sequences, grouped heads of 128 channels, a wide window
        {"name": "attn_long", "op": "attn", "tokens": 16384, "seqs": 2, "hq": 32, "hkv": 8, "d": 128, "window": 2048,
         "sinks": 4, "causal": True, "dtype": "bf16"},
        # many packed sequences of uneven lengths, the decoder's default 32 query and 2 kv heads
        {"name": "attn_ragged", "op": "attn", "tokens": 20011, "seqs": 40, "hq": 32, "hkv": 2, "d": 32, "window": 256,
         "sinks": 1, "causal": True, "dtype": "f16"},
        # one sequence answered token by token: latency
        {"name": "decode_one", "op": "decode", "batch": 1, "hq": 16, "hkv": 16, "d": 64, "window": 512, "sinks": 4,
         "longest": 3000, "dtype": "bf16"},
        # a served batch at the full window, lengths from zero to well past the ring's end
        {"name": "decode_batch", "op": "decode", "batch": 64, "hq": 32, "hkv": 8, "d": 128, "window": 8192, "sinks": 4,
         "longest": 20000, "dtype": "bf16"},
        # the norm in front of 8-bit projections while serving a few tokens: latency
        {"name": "norm_few", "op": "norm8", "rows": 8, "cols": 1024, "group": 0, "out": "e4m3", "weight": True,
         "dtype": "bf16"},
        # the same for a long prompt of a wide model, scales per 128 columns
        {"name": "norm_wide", "op": "norm8", "rows": 16384, "cols": 4096, "group": 128, "out": "int8", "weight": True,
         "dtype": "bf16"},
        # the decoder's training step between attention and MLP
        {"name": "norm_train", "op": "norm", "rows": 131072, "cols": 1024, "p": 0.1, "weight": True, "dtype": "bf16",
         "stream": "bf16"},
        # an odd width, 32-bit residual stream and weight
        {"name": "norm_odd", "op": "norm", "rows": 5003, "cols": 1001, "p": 0.25, "weight": True, "dtype": "f16",
         "stream": "f32"},
        # dropout of a ragged batch's embeddings
        {"name": "drop_odd", "op": "drop", "rows": 77, "cols": 1001, "p": 0.1, "dtype": "bf16"},
        # dropout of the decoder's MLP hidden units, forward and backward
        {"name": "drop_hidden", "op": "drop", "rows": 131072, "cols": 4096, "p": 0.1, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attn", "attn", "attn", "decode", "decode", "norm", "norm8", "drop"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if op == "attn":
        while True:
            hkv, g, d = rng.choice([1, 2, 3, 4, 8, 16]), rng.choice([1, 1, 2, 3, 4, 5, 8, 16]), rng.choice([32, 64, 128])
            c = {"op": op, "tokens": _log(rng, 64, 65536), "seqs": _log(rng, 1, 48), "hq": hkv * g, "hkv": hkv, "d": d,
                 "window": _log(rng, 1, 4096), "sinks": rng.choice([0, 1, 4, 7, 16, 64, 128]),
                 "causal": rng.random() < 0.6, "dtype": dtype}
            scores = c["tokens"] * c["hq"] * (_CHUNK + c["window"] + c["seqs"] * c["sinks"])
            if (c["hq"] <= 64 and c["seqs"] <= c["tokens"] and c["seqs"] * c["sinks"] <= 1024
                    and scores * d <= _MOST_SCORES * 64):
                return c
    if op == "decode":
        while True:
            hkv, g, d = rng.choice([1, 2, 4, 8, 16]), rng.choice([1, 2, 3, 4, 7, 8, 16]), rng.choice([32, 64, 128])
            w = _log(rng, 64, 8192)
            c = {"op": op, "batch": _log(rng, 1, 64), "hq": hkv * g, "hkv": hkv, "d": d, "window": w,
                 "sinks": rng.choice([0, 1, 4, 16, 64]), "longest": _log(rng, 1, 3 * w), "dtype": dtype}
            if c["batch"] * w * hkv * d <= 64 * 8192 * 8 * 128:
                return c
    if op == "norm8":
        rows = _log(rng, 1, 16384)
        cols = min(_log(rng, 33, 8192), 16384 * 4096 // rows)
        return {"op": op, "rows": rows, "cols": cols, "group": rng.choice([0, 32, 64, 128]),
                "out": rng.choice(["e4m3", "int8"]), "weight": rng.random() < 0.8, "dtype": dtype}
    if op == "norm":
        rows = _log(rng, 1, 131072)
        cols = min(_log(rng, 33, 8192), 131072 * 1024 // rows)
        return {"op": op, "rows": rows, "cols": cols, "p": rng.choice([0.0, 0.1, 0.25, 0.5]),
                "weight": rng.random() < 0.8, "dtype": dtype, "stream": rng.choice([dtype, "f32"])}
    rows = _log(rng, 1, 131072)
    return {"op": op, "rows": rows, "cols": min(_log(rng, 1, 8192), 131072 * 2048 // rows),
            "p": rng.choice([0.05, 0.1, 0.3, 0.5, 0.9]), "dtype": rng.choice(["bf16", "f16", "f32"])}


def _cuts(case, seed):
    """Offsets of the ragged sequences: random cuts, one sequence of a single token where there are three or more."""
    n, b = case["tokens"], case["seqs"]
    r = np.random.RandomState(seed % (1 << 31))
    cuts = np.sort(r.choice(np.arange(1, n), b - 1, replace=False)) if b > 1 else np.zeros(0, np.int64)
    if b >= 3 and 1 not in cuts:
        cuts[0] = 1
    return np.concatenate([[0], cuts, [n]]).astype(np.int64)


def _reach(case):
    return (case["window"] - 1, 0) if case["causal"] else (case["window"] // 2, case["window"] // 2)


def _capacity(case):
    return case["sinks"] + case["window"]


def _lengths(case, seed):
    """Tokens before the new one, per sequence: one empty, one at the longest, the rest spread between."""
    r = np.random.RandomState(seed % (1 << 31))
    n = r.randint(0, case["longest"] + 1, case["batch"])
    n[0] = case["longest"]
    if case["batch"] > 1:
        n[1] = 0
    return n.astype(np.int32)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    s = {"case": dict(case), "seed": int(seed)}
    op, dt = case["op"], _DT[case["dtype"]]

    def normal(*shape, std=1.0, dtype=dt):
        return torch.randn(*shape, device=dev, generator=g).mul_(std).to(dtype)

    if op == "attn":
        n, hq, hkv, d = case["tokens"], case["hq"], case["hkv"], case["d"]
        s["cu"] = torch.from_numpy(_cuts(case, seed).astype(np.int32)).to(dev)
        s["q"], s["k"], s["v"] = (normal(n, h, d).requires_grad_() for h in (hq, hkv, hkv))
        s["dout"] = normal(n, hq, d, std=0.1)
    elif op == "decode":
        b, hq, hkv, d, cap = case["batch"], case["hq"], case["hkv"], case["d"], _capacity(case)
        s["lengths"] = torch.from_numpy(_lengths(case, seed)).to(dev)
        s["k_cache"], s["v_cache"] = normal(b, cap, hkv, d), normal(b, cap, hkv, d)
        s["q"], s["k_new"], s["v_new"] = normal(b, hq, d), normal(b, hkv, d), normal(b, hkv, d)
    elif op in ("norm", "norm8"):
        n, c = case["rows"], case["cols"]
        stream = _DT[case.get("stream", case["dtype"])]
        s["x"] = normal(n, c)
        s["residual"] = normal(n, c, std=2.0, dtype=stream)
        s["weight"] = (1.0 + 0.2 * torch.randn(c, device=dev, generator=g)).to(stream) if case["weight"] else None
        if op == "norm":
            s["dy"], s["dh"] = normal(n, c, std=0.1), normal(n, c, std=0.1, dtype=stream)
            for t in (s["x"], s["residual"], s["weight"]):
                if t is not None:
                    t.requires_grad_()
    else:
        s["x"] = normal(case["rows"], case["cols"]).requires_grad_()
        s["dy"] = normal(case["rows"], case["cols"], std=0.1)
    return s


def work(case):
    op = case["op"]
    size = {"bf16": 2, "f16": 2, "f32": 4}
    e = size[case["dtype"]]
    if op == "attn":
        left, right = _reach(case)
        pairs = 0
        cu = _cuts(case, 1)
        for a, b in zip(cu[:-1], cu[1:]):
            i = np.arange(b - a)
            lo, hi = np.maximum(i - left, 0), np.minimum(i + right, b - a - 1)
            seen = np.minimum(case["sinks"], i + 1 if case["causal"] else b - a)
            pairs += int((hi - lo + 1).sum() + np.minimum(seen, lo).sum())
        n, hq, hkv, d = case["tokens"], case["hq"], case["hkv"], case["d"]
        # read q, k, v and the output's gradient; write the output and the three gradients
        return {"bytes": e * n * d * (4 * hq + 4 * hkv), "flops": 14.0 * pairs * hq * d}
    if op == "decode":
        n = _lengths(case, 1).astype(np.int64) + 1
        seen = int(np.minimum(n, case["window"] + case["sinks"]).sum())
        b, hq, hkv, d = case["batch"], case["hq"], case["hkv"], case["d"]
        return {"bytes": e * d * (2 * seen * hkv + 2 * b * hq + 4 * b * hkv), "flops": 4.0 * seen * hq * d}
    n, c = case["rows"], case["cols"]
    if op == "drop":  # x -> y and dy -> dx
        return {"bytes": 4 * e * n * c, "flops": 2.0 * n * c}
    st = size[case.get("stream", case["dtype"])]
    if op == "norm":  # read x, residual, dy, dh; write y, h, dx, dresidual
        return {"bytes": n * c * (4 * e + 4 * st) + 3 * st * c, "flops": 16.0 * n * c}
    groups = 1 if case["group"] == 0 else -(-c // case["group"])
    # read x, residual; write h, the 8-bit values with their scales, and the values that they stand for
    return {"bytes": n * c * (3 * e + 1 + e) + 4 * n * groups + e * c, "flops": 8.0 * n * c}


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------


def run(s):
    op = s["case"]["op"]
    return {"attn": _attn, "decode": _decode, "norm": _norm, "norm8": _norm8, "drop": _drop}[op](s)


def _attn(s):
    c = s["case"]
    if own:
        out = _api().window_sink_attention(s["q"], s["k"], s["v"], s["cu"], window=c["window"], sinks=c["sinks"],
                                           causal=c["causal"])
        dq, dk, dv = torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["dout"])
        return {"out": out.detach(), "dq": dq, "dk": dk, "dv": dv}
    with torch.no_grad():
        return _plain_attn(s)


def _plain_attn(s):
    """Queries in chunks, each chunk against the band of keys that its window can reach and against every sequence's
    first tokens; masked softmax and the gradients by their formulas."""
    c = s["case"]
    n, hq, hkv, d = c["tokens"], c["hq"], c["hkv"], c["d"]
    grp, scale = hq // hkv, 1.0 / math.sqrt(d)
    left, right = (min(t, n) for t in _reach(c))
    dev = s["q"].device
    size = min(_CHUNK, n)
    chunks = -(-n // size)
    cu = s["cu"].long()
    tok = torch.arange(chunks * size, device=dev)
    seq = torch.searchsorted(cu, tok.clamp(max=n - 1), right=True) - 1
    qi = tok.view(chunks, size)
    # [chunks, keys]: the band's tokens, then every sequence's first ones
    band = qi[:, :1] - left + torch.arange(size + left + right, device=dev)
    sink = (cu[:-1, None] + torch.arange(c["sinks"], device=dev)).reshape(-1)
    sink_ok = (torch.arange(c["sinks"], device=dev) < (cu[1:] - cu[:-1])[:, None]).reshape(-1)
    band_ok = (band >= 0) & (band < n)
    kidx = torch.cat([band.clamp(0, n - 1), sink.clamp(max=n - 1).expand(chunks, -1)], 1)
    seq_q, seq_k = seq.view(chunks, size), seq[kidx]
    near = (kidx[:, None] >= qi[..., None] - left) & (kidx[:, None] <= qi[..., None] + right)
    is_sink = torch.arange(kidx.shape[1], device=dev) >= band.shape[1]
    seen = torch.where(is_sink, ~near & torch.cat([band_ok, sink_ok.expand(chunks, -1)], 1)[:, None],
                       near & torch.cat([band_ok, sink_ok.expand(chunks, -1)], 1)[:, None])
    seen &= (seq_q[..., None] == seq_k[:, None]) & (qi[..., None] < n)
    if c["causal"]:
        seen &= kidx[:, None] <= qi[..., None]
    seen = seen[:, None, None]  # [chunks, 1, 1, size, keys]

    def rows(t):  # [n, hq, d] -> [chunks, hkv, grp, size, d]
        t = torch.nn.functional.pad(t.float(), (0, 0, 0, 0, 0, chunks * size - n))
        return t.view(chunks, size, hkv, grp, d).permute(0, 2, 3, 1, 4)

    def back(t):
        return t.permute(0, 3, 1, 2, 4).reshape(chunks * size, hq, d)[:n].to(s["q"].dtype)

    def gather(t):  # [n, hkv, d] -> [chunks, hkv, 1, keys, d]
        return t.float()[kidx].permute(0, 2, 1, 3).unsqueeze(2)

    q, do = rows(s["q"]), rows(s["dout"])
    k, v = gather(s["k"]), gather(s["v"])
    p = torch.matmul(q, k.transpose(-1, -2)).mul_(scale).masked_fill_(~seen, -math.inf)
    p = p.sub_(p.amax(-1, keepdim=True).clamp_(min=-1e30)).exp_()
    p = p.div_(p.sum(-1, keepdim=True).clamp_(min=1e-30))
    out = torch.matmul(p, v)
    dv = torch.matmul(p.transpose(-1, -2), do).sum(2)
    ds = torch.matmul(do, v.transpose(-1, -2)).sub_((do * out).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    dq = torch.matmul(ds, k)
    dk = torch.matmul(ds.transpose(-1, -2), q).sum(2)

    def spread(t):  # [chunks, hkv, keys, d] -> [n, hkv, d]
        z = torch.zeros(n, hkv, d, device=dev)
        return z.index_add_(0, kidx.reshape(-1), t.permute(0, 2, 1, 3).reshape(-1, hkv, d)).to(s["k"].dtype)

    return {"out": back(out), "dq": back(dq), "dk": spread(dk), "dv": spread(dv)}


def _decode(s):
    c = s["case"]
    if own:
        out = _api().window_sink_decode(s["q"], s["k_new"], s["v_new"], s["k_cache"], s["v_cache"], s["lengths"],
                                        window=c["window"], sinks=c["sinks"])
        return {"out": out, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    b, hq, hkv, d, w, sk = c["batch"], c["hq"], c["hkv"], c["d"], c["window"], c["sinks"]
    cap = _capacity(c)
    n = s["lengths"].long()
    row = torch.arange(b, device=n.device)
    slot = torch.where(n < sk, n, sk + (n - sk).clamp(min=0) % (cap - sk))
    s["k_cache"][row, slot] = s["k_new"]
    s["v_cache"][row, slot] = s["v_new"]
    # the sinks' positions, then the window's last ones from the newest back
    pos = torch.cat([torch.arange(sk, device=n.device).expand(b, -1), n[:, None] - torch.arange(w, device=n.device)], 1)
    first = torch.arange(sk + w, device=n.device) < sk
    seen = torch.where(first, pos <= n[:, None], pos >= sk)
    at = torch.where(pos < sk, pos.clamp(min=0), sk + (pos - sk).clamp(min=0) % (cap - sk))
    k, v = (t[row[:, None], at].float().transpose(1, 2) for t in (s["k_cache"], s["v_cache"]))  # [b, hkv, keys, d]
    v = v.masked_fill(~seen[:, None, :, None], 0.0)
    p = torch.matmul(s["q"].float().view(b, hkv, hq // hkv, d), k.transpose(-1, -2)) / math.sqrt(d)
    p = p.masked_fill(~seen[:, None, None], -math.inf)
    p = torch.exp(p - p.amax(-1, keepdim=True))
    out = torch.matmul(p / p.sum(-1, keepdim=True), v).reshape(b, hq, d).to(s["q"].dtype)
    return {"out": out, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _philox(n, seed, offset, device):
    """Word e % 4 of block e // 4 of Philox4x32-10 for e < n, as int64 values below 2^32."""
    low = 0xFFFFFFFF
    block = torch.arange(-(-n // 4), device=device) + offset
    x0, x1, x2, x3 = block & low, block >> 32, torch.zeros_like(block), torch.zeros_like(block)
    k0, k1 = seed & low, (seed >> 32) & low
    for _ in range(10):
        a, b = x0 * 0xD2511F53, x2 * 0xCD9E8D57  # 64-bit products, kept modulo 2^64
        x0, x1, x2, x3 = ((b >> 32) & low) ^ x1 ^ k0, b & low, ((a >> 32) & low) ^ x3 ^ k1, a & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack([x0, x1, x2, x3], 1).view(-1)[:n]


def _keep(shape, p, seed, device):
    return (_philox(math.prod(shape), seed, 0, device) >= int(p * 2.0**32)).view(shape)


def _norm(s):
    c = s["case"]
    p = c["p"]
    if own:
        y, h = _api().residual_rms_norm(s["x"], s["residual"], s["weight"], p=p, seed=s["seed"])
        wanted = [t for t in (s["x"], s["residual"], s["weight"]) if t is not None]
        grads = torch.autograd.grad((y, h), wanted, (s["dy"], s["dh"]))
        return {"y": y.detach(), "h": h.detach(), "dx": grads[0], "dresidual": grads[1],
                "dweight": grads[2] if c["weight"] else None}
    with torch.no_grad():
        x, dt, st = s["x"].float(), s["x"].dtype, s["residual"].dtype
        keep = _keep(x.shape, p, s["seed"], x.device) if p else None
        drop = (lambda t: torch.where(keep, t / (1.0 - p), 0.0)) if p else (lambda t: t)
        w = s["weight"].float() if c["weight"] else 1.0
        h = s["residual"].float() + drop(x)
        r = torch.rsqrt((h * h).mean(-1, keepdim=True) + 1e-6)
        y = h * r * w
        g = s["dy"].float() * w
        dh = r * (g - h * r * r * (g * h).mean(-1, keepdim=True)) + s["dh"].float()
        dw = (s["dy"].float() * h * r).sum(0).to(st) if c["weight"] else None
        return {"y": y.to(dt), "h": h.to(st), "dx": drop(dh).to(dt), "dresidual": dh.to(st), "dweight": dw}


def _norm8(s):
    c = s["case"]
    if own:
        api = _api()
        q, scale, h = api.residual_rms_norm_8bit(s["x"], s["residual"], s["weight"], dtype=_DT[c["out"]],
                                                 group=c["group"])
        return {"y": api.dequantize_8bit(q, scale, s["x"].dtype), "scale": scale, "h": h}
    n, cols = c["rows"], c["cols"]
    top = _Q8_MAX[c["out"]]
    h = s["residual"].float() + s["x"].float()
    y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + 1e-6)
    if c["weight"]:
        y = y * s["weight"].float()
    width = c["group"] or cols
    groups = -(-cols // width)
    y = torch.nn.functional.pad(y, (0, groups * width - cols)).view(n, groups, width)
    amax = y.abs().amax(-1, keepdim=True)
    scale = torch.where(amax > 0, amax / top, 1.0)
    y = (y * (1.0 / scale)).clamp(-top, top)
    y = (y.round() if c["out"] == "int8" else y.to(torch.float8_e4m3fn).float()) * scale
    return {"y": y.view(n, -1)[:, :cols].to(s["x"].dtype), "scale": scale.view(n, groups), "h": h.to(s["x"].dtype)}


def _drop(s):
    c = s["case"]
    if own:
        y = _api().dropout(s["x"], c["p"], s["seed"])
        (dx,) = torch.autograd.grad(y, s["x"], s["dy"])
        return {"y": y.detach(), "dx": dx}
    with torch.no_grad():
        keep = _keep(s["x"].shape, c["p"], s["seed"], s["x"].device)
        y, dx = (torch.where(keep, t.float() / (1.0 - c["p"]), 0.0).to(t.dtype) for t in (s["x"], s["dy"]))
        return {"y": y, "dx": dx}


# ---------------------------------------------------------------------------
# The same in 64 bits, from the definitions
# ---------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "attn":
        return _exact_attn(case, s)
    if op == "decode":
        return _exact_decode(case, s)
    if op == "drop":
        f = _exact_factor(case["rows"], case["cols"], case["p"], s)
        return {"y": s["x"].detach().double() * f, "dx": s["dy"].double() * f}
    x, res = s["x"].detach().double(), s["residual"].detach().double()
    w = s["weight"].detach().double() if case["weight"] else torch.ones(case["cols"], device=x.device).double()
    if op == "norm8":
        h = res + x
        return {"h": h, **_exact_8bit(case, h / (h.pow(2).sum(-1, keepdim=True) / case["cols"] + 1e-6).sqrt() * w)}
    f = _exact_factor(case["rows"], case["cols"], case["p"], s) if case["p"] else torch.ones((), device=x.device).double()
    x, res, w = x.requires_grad_(), res.requires_grad_(), w.requires_grad_()
    h = res + x * f
    y = h / (h.pow(2).sum(-1, keepdim=True) / case["cols"] + 1e-6).sqrt() * w
    dx, dres, dw = torch.autograd.grad((y, h), (x, res, w), (s["dy"].double(), s["dh"].double()))
    return {"y": y.detach(), "h": h.detach(), "dx": dx, "dresidual": dres, "dweight": dw if case["weight"] else None}


def _exact_factor(rows, cols, p, s):
    """What dropout multiplies each value by: 0 or 1 / (1 - p), from Philox4x32-10 on 16-bit limbs."""
    dev = s["x"].device
    out = torch.empty(rows * cols, device=dev, dtype=torch.float64)
    mask32 = (1 << 32) - 1

    def mulhilo(m, t):
        lo = m * (t & 0xFFFF)
        hi = m * (t >> 16) + (lo >> 16)
        return hi >> 16, ((hi & 0xFFFF) << 16) | (lo & 0xFFFF)

    step = 1 << 26
    for at in range(0, rows * cols, step):
        e = torch.arange(at, min(at + step, rows * cols), device=dev)
        words = [torch.div(e, 4, rounding_mode="floor") & mask32, e >> 34, torch.zeros_like(e), torch.zeros_like(e)]
        for r in range(10):
            k0 = (s["seed"] + r * 0x9E3779B9) & mask32
            k1 = ((s["seed"] >> 32) + r * 0xBB67AE85) & mask32
            h0, l0 = mulhilo(0xD2511F53, words[0])
            h1, l1 = mulhilo(0xCD9E8D57, words[2])
            words = [h1 ^ words[1] ^ k0, l1, h0 ^ words[3] ^ k1, l0]
        own_word = torch.stack(words)[e % 4, torch.arange(e.numel(), device=dev)]
        out[at:at + e.numel()] = (own_word >= math.floor(p * 4294967296)).double() / (1 - p)
    return out.view(rows, cols)


def _exact_8bit(case, y):
    """Scales and values of y on the 8-bit grid: whole steps of the scale, or three fraction bits down to 2^-9."""
    width = case["group"] or case["cols"]
    scales, values = [], []
    for part in y.split(width, 1):
        top = part.abs().max(1, keepdim=True).values
        sc = torch.where(top == 0, torch.ones_like(top), top / _Q8_MAX[case["out"]])
        t = part / sc
        step = torch.ones_like(t)
        if case["out"] == "e4m3":
            step = torch.exp2(torch.floor(torch.log2(t.abs().clamp(min=2.0**-6))) - 3)
        scales.append(sc)
        values.append(torch.round(t / step) * step * sc)
    return {"y": torch.cat(values, 1), "scale": torch.cat(scales, 1)}


def _exact_attn(case, s):
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    left, right = _reach(case)
    q, k, v, do = (s[x].detach().double() for x in ("q", "k", "v", "dout"))
    out, dq, dk, dv = (torch.zeros_like(x) for x in (q, q, k, v))
    cu = s["cu"].tolist()
    step = max(64, min(1024, int(1.5e9 // (hq * (left + right + 1200)))))
    for a, b in zip(cu[:-1], cu[1:]):
        for i0 in range(a, b, step):
            i1 = min(b, i0 + step)
            lo, hi = max(a, i0 - left), min(b, i1 + right)
            j = torch.unique(torch.cat([torch.arange(a, min(b, a + case["sinks"])), torch.arange(lo, hi)])).to(q.device)
            i = torch.arange(i0, i1, device=q.device)
            gap = i[:, None] - j[None]
            vis = (gap <= left) & (gap >= -right) | (j - a < case["sinks"])[None]
            if case["causal"]:
                vis &= gap >= 0
            for h in range(hkv):
                hs = slice(h * (hq // hkv), (h + 1) * (hq // hkv))
                leaf = [t.clone().requires_grad_() for t in (q[i0:i1, hs], k[j, h], v[j, h])]
                with torch.enable_grad():
                    sc = torch.einsum("igd,jd->gij", leaf[0], leaf[1]) / d**0.5
                    pr = torch.softmax(sc.masked_fill(~vis, -math.inf), -1)
                    o = torch.einsum("gij,jd->igd", pr, leaf[2])
                    gq, gk, gv = torch.autograd.grad(o, leaf, do[i0:i1, hs])
                out[i0:i1, hs], dq[i0:i1, hs] = o.detach(), gq
                dk[:, h].index_add_(0, j, gk)
                dv[:, h].index_add_(0, j, gv)
    return {"out": out, "dq": dq, "dk": dk, "dv": dv}


def _exact_decode(case, s):
    hq, hkv, d, w, sk = case["hq"], case["hkv"], case["d"], case["window"], case["sinks"]
    ring = _capacity(case) - sk
    out = torch.zeros(case["batch"], hq, d, device=s["q"].device, dtype=torch.float64)
    for b, n in enumerate(s["lengths"].tolist()):
        pos = sorted(set(range(min(sk, n + 1))) | set(range(max(0, n + 1 - w), n + 1)))
        slots = [j if j < sk else sk + (j - sk) % ring for j in pos]
        at = slots[pos.index(n)]
        s["k_cache"][b, at], s["v_cache"][b, at] = s["k_new"][b], s["v_new"][b]
        idx = torch.tensor(slots, device=out.device)
        k, v = s["k_cache"][b, idx].double(), s["v_cache"][b, idx].double()
        q = s["q"][b].double().view(hkv, hq // hkv, d)
        pr = torch.softmax(torch.einsum("hgd,jhd->hgj", q, k) / d**0.5, -1)
        out[b] = torch.einsum("hgj,jhd->hgd", pr, v).reshape(hq, d)
    return {"out": out, "k_cache": s["k_cache"].double(), "v_cache": s["v_cache"].double()}
