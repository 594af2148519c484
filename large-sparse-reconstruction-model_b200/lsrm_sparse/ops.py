"""Thin torch-tensor wrappers over the C ABI (include/lsrm_sparse.h).

Tensors must live on a CUDA device; every call enqueues on the current torch
stream and never synchronises, except where a function says so.  Device-side
error bits accumulate in a per-device word that ``read_errors()`` returns and
clears (with a synchronisation).
"""

from __future__ import annotations

import ctypes
import math
from typing import List, Optional, Sequence, Tuple

import torch

from . import _lib
from ._lib import AttnShape, Varlen, check

_ERR_WORDS = {}


def _err_word(device: torch.device) -> torch.Tensor:
    key = device.index if device.index is not None else torch.cuda.current_device()
    w = _ERR_WORDS.get(key)
    if w is None:
        w = torch.zeros(1, dtype=torch.int32, device=device)
        _ERR_WORDS[key] = w
    return w


def read_errors(device=None, clear: bool = True) -> int:
    """Synchronise and return the OR of device error bits (LSRM_ERR_*)."""
    dev = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
    w = _err_word(dev)
    v = int(w.item())
    if clear and v:
        w.zero_()
    return v


def _stream() -> ctypes.c_void_p:
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def _ptr(t: Optional[torch.Tensor]):
    return ctypes.c_void_p(t.data_ptr()) if t is not None else None


def _dtype_code(t: torch.Tensor) -> int:
    if t.dtype == torch.bfloat16:
        return 1
    if t.dtype == torch.float16:
        return 0
    raise TypeError(f"only bf16/fp16 are supported, got {t.dtype}")


def _i32(t: torch.Tensor) -> torch.Tensor:
    if t.dtype != torch.int32:
        t = t.to(torch.int32)
    return t.contiguous()


class Meta:
    """Device int32 metadata of one varlen problem (keeps the tensors alive)."""

    def __init__(self, cu_seqlens_q, cu_seqlens_k, cu_seqblocks, cu_block_include_tokens, total_q=None, total_k=None):
        self.cu_seqlens_q = _i32(cu_seqlens_q)
        self.cu_seqlens_k = _i32(cu_seqlens_k)
        self.cu_seqblocks = _i32(cu_seqblocks)
        self.cu_block_include_tokens = _i32(cu_block_include_tokens)
        self.num_seqs = self.cu_seqlens_q.numel() - 1
        self.num_blocks = self.cu_block_include_tokens.numel() - 1
        self.total_q = int(total_q) if total_q is not None else None
        self.total_k = int(total_k) if total_k is not None else None

    def struct(self, total_q: int, total_k: int) -> Varlen:
        return Varlen(
            self.num_seqs, int(total_q), int(total_k), self.num_blocks,
            self.cu_seqlens_q.data_ptr(), self.cu_seqlens_k.data_ptr(), self.cu_seqblocks.data_ptr(),
            self.cu_block_include_tokens.data_ptr(),
        )


def _shape(q: torch.Tensor, k: torch.Tensor, softmax_scale: Optional[float]) -> AttnShape:
    assert q.dim() == 3 and k.dim() == 3, "q/k must be [tokens, heads, head_dim]"
    assert q.stride(-1) == 1 and q.stride(-2) == q.shape[-1], "q must have contiguous [heads, head_dim]"
    assert k.stride(-1) == 1 and k.stride(-2) == k.shape[-1], "k must have contiguous [heads, head_dim]"
    return AttnShape(
        q.shape[1], k.shape[1], q.shape[2], _dtype_code(q), q.stride(0), k.stride(0),
        float(softmax_scale) if softmax_scale else 0.0,
    )


def _rows(*ts):
    """The kernels address q, out, dout and dq with q's token stride and k, v,
    dk and dv with k's: hand them dense [tokens, heads, head_dim] tensors (a
    no-op for contiguous inputs; a copy for any other layout)."""
    return tuple(t if t is None or t.is_contiguous() else t.contiguous() for t in ts)


def _workspace(nbytes: int, device) -> torch.Tensor:
    return torch.empty(max(int(nbytes), 256), dtype=torch.uint8, device=device)


# ---------------------------------------------------------------------------
# Selected-block attention
# ---------------------------------------------------------------------------


def _check_block_topk(block_topk, num_kv_heads: int, rows: int):
    """The kernels read block_topk as [num_kv_heads, rows, topk]: reject any
    other shape before it reaches them."""
    if block_topk.dim() != 3 or tuple(block_topk.shape[:2]) != (num_kv_heads, rows):
        raise ValueError(f"block_topk must be [num_kv_heads={num_kv_heads}, {rows}, topk], got "
                         f"{tuple(block_topk.shape)}")


def select_attn_fwd(q, k, v, block_topk, meta: Meta, softmax_scale=None, cu_query_blocks=None,
                    workspace: Optional[torch.Tensor] = None):
    """Returns (out [Nq,Hq,D], lse_log2 [Hq,Nq] fp32, workspace)."""
    L = _lib.lib()
    assert q.dtype == k.dtype == v.dtype
    q, k, v = _rows(q, k, v)
    block_topk = _i32(block_topk)
    topk = block_topk.shape[-1]
    nqb = 0 if cu_query_blocks is None else cu_query_blocks.numel() - 1
    _check_block_topk(block_topk, k.shape[1], nqb if nqb > 0 else q.shape[0])
    cqb = _i32(cu_query_blocks) if cu_query_blocks is not None else None
    vl = meta.struct(q.shape[0], k.shape[0])
    sh = _shape(q, k, softmax_scale)
    need = L.lsrm_select_workspace_bytes(ctypes.byref(vl), ctypes.byref(sh), topk, nqb)
    if need == 0:
        raise _lib.LsrmError("invalid selection problem: " + L.lsrm_last_error().decode())
    if workspace is None or workspace.numel() < need:
        workspace = _workspace(need, q.device)
    out = torch.empty_like(q)
    lse = torch.empty(q.shape[1], q.shape[0], dtype=torch.float32, device=q.device)
    rc = L.lsrm_select_attn_fwd(
        ctypes.byref(vl), ctypes.byref(sh), _ptr(q), _ptr(k), _ptr(v), _ptr(block_topk), topk, _ptr(cqb), nqb,
        _ptr(out), _ptr(lse), _ptr(workspace), workspace.numel(), _ptr(_err_word(q.device)), _stream(),
    )
    check(rc, "lsrm_select_attn_fwd")
    return out, lse, workspace


def select_attn_bwd(q, k, v, out, lse, dout, block_topk, meta: Meta, softmax_scale=None, cu_query_blocks=None,
                    workspace: Optional[torch.Tensor] = None):
    """Returns (dq, dk, dv)."""
    L = _lib.lib()
    q, k, v, out, dout = _rows(q, k, v, out, dout)
    block_topk = _i32(block_topk)
    topk = block_topk.shape[-1]
    nqb = 0 if cu_query_blocks is None else cu_query_blocks.numel() - 1
    _check_block_topk(block_topk, k.shape[1], nqb if nqb > 0 else q.shape[0])
    cqb = _i32(cu_query_blocks) if cu_query_blocks is not None else None
    vl = meta.struct(q.shape[0], k.shape[0])
    sh = _shape(q, k, softmax_scale)
    need = L.lsrm_select_workspace_bytes(ctypes.byref(vl), ctypes.byref(sh), topk, nqb)
    if workspace is None or workspace.numel() < need:
        workspace = _workspace(need, q.device)
    dq = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    dk = torch.empty(k.shape, dtype=k.dtype, device=k.device)
    dv = torch.empty(v.shape, dtype=v.dtype, device=v.device)
    delta = torch.empty(q.shape[1], q.shape[0], dtype=torch.float32, device=q.device)
    rc = L.lsrm_select_attn_bwd(
        ctypes.byref(vl), ctypes.byref(sh), _ptr(q), _ptr(k), _ptr(v), _ptr(out), _ptr(lse), _ptr(dout),
        _ptr(block_topk), topk, _ptr(cqb), nqb, _ptr(dq), _ptr(dk), _ptr(dv), _ptr(delta), _ptr(workspace),
        workspace.numel(), _ptr(_err_word(q.device)), _stream(),
    )
    check(rc, "lsrm_select_attn_bwd")
    return dq, dk, dv


# ---------------------------------------------------------------------------
# Dense-range branches
# ---------------------------------------------------------------------------

DENSE_COMPRESSED = _lib.DENSE_COMPRESSED
DENSE_INTRA_BLOCK = _lib.DENSE_INTRA_BLOCK
DENSE_SLIDING = _lib.DENSE_SLIDING


def dense_attn_fwd(q, k, v, meta: Meta, mode: int, window: int = 0, softmax_scale=None):
    """Returns (out, lse).  lse is natural-log for DENSE_COMPRESSED, log2
    otherwise; [Hq, Nq] fp32."""
    L = _lib.lib()
    q, k, v = _rows(q, k, v)
    vl = meta.struct(q.shape[0], k.shape[0])
    sh = _shape(q, k, softmax_scale)
    need = L.lsrm_dense_workspace_bytes(ctypes.byref(vl), ctypes.byref(sh), mode)
    if need == 0:
        raise _lib.LsrmError("invalid dense problem: " + L.lsrm_last_error().decode())
    ws = _workspace(need, q.device)
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty(q.shape[1], q.shape[0], dtype=torch.float32, device=q.device)
    rc = L.lsrm_dense_attn_fwd(ctypes.byref(vl), ctypes.byref(sh), mode, int(window), _ptr(q), _ptr(k), _ptr(v),
                               _ptr(out), _ptr(lse), _ptr(ws), ws.numel(), _ptr(_err_word(q.device)), _stream())
    check(rc, "lsrm_dense_attn_fwd")
    return out, lse


def dense_attn_bwd(q, k, v, out, lse, dout, meta: Meta, mode: int, window: int = 0, softmax_scale=None):
    L = _lib.lib()
    q, k, v, out, dout = _rows(q, k, v, out, dout)
    vl = meta.struct(q.shape[0], k.shape[0])
    sh = _shape(q, k, softmax_scale)
    need = L.lsrm_dense_workspace_bytes(ctypes.byref(vl), ctypes.byref(sh), mode)
    ws = _workspace(need, q.device)
    dq = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    dk = torch.empty(k.shape, dtype=k.dtype, device=k.device)
    dv = torch.empty(v.shape, dtype=v.dtype, device=v.device)
    delta = torch.empty(q.shape[1], q.shape[0], dtype=torch.float32, device=q.device)
    rc = L.lsrm_dense_attn_bwd(ctypes.byref(vl), ctypes.byref(sh), mode, int(window), _ptr(q), _ptr(k), _ptr(v),
                               _ptr(out), _ptr(lse), _ptr(dout), _ptr(dq), _ptr(dk), _ptr(dv), _ptr(delta), _ptr(ws),
                               ws.numel(), _ptr(_err_word(q.device)), _stream())
    check(rc, "lsrm_dense_attn_bwd")
    return dq, dk, dv


def umma_selftest(a, b, p, v):
    L = _lib.lib()
    D = a.shape[1]
    c1 = torch.empty(128, 128, dtype=torch.float32, device=a.device)
    c2 = torch.empty(128, D, dtype=torch.float32, device=a.device)
    rc = L.lsrm_umma_selftest(D, _ptr(a), _ptr(b), _ptr(p), _ptr(v), _ptr(c1), _ptr(c2), _ptr(_err_word(a.device)),
                              _stream())
    check(rc, "lsrm_umma_selftest")
    return c1, c2


# ---------------------------------------------------------------------------
# Scoring, compression, gated merge
# ---------------------------------------------------------------------------


def block_topk(q, ck, lse_ln, topk: int, meta: Meta, cu_query_blocks=None, force_self: bool = False,
               sm_scale: Optional[float] = None):
    """Deterministic block selection; returns int32 [Hkv, rows, topk]."""
    L = _lib.lib()
    q, ck = _rows(q, ck)
    vl = meta.struct(q.shape[0], ck.shape[0])
    sh = _shape(q, ck, None)
    nqb = 0 if cu_query_blocks is None else cu_query_blocks.numel() - 1
    rows = nqb if nqb else q.shape[0]
    out = torch.empty(ck.shape[1], rows, topk, dtype=torch.int32, device=q.device)
    cqb = _i32(cu_query_blocks) if cu_query_blocks is not None else None
    lse_ln = lse_ln.float().contiguous()
    nbytes = L.lsrm_block_topk_workspace_bytes(ctypes.byref(vl), ctypes.byref(sh), int(topk), nqb)
    ws = _workspace(nbytes, q.device) if nbytes else None
    rc = L.lsrm_block_topk(ctypes.byref(vl), ctypes.byref(sh), _ptr(q), _ptr(ck), _ptr(lse_ln), int(topk), _ptr(cqb),
                           nqb, int(bool(force_self)), float(sm_scale) if sm_scale else 0.0, _ptr(out), _ptr(ws),
                           int(nbytes), _ptr(_err_word(q.device)), _stream())
    check(rc, "lsrm_block_topk")
    return out


def block_mean_fwd(x: torch.Tensor, cu_block_include_tokens: torch.Tensor) -> torch.Tensor:
    """x [N, C] (row stride may exceed C) -> [nb, C]."""
    L = _lib.lib()
    assert x.dim() == 2 and x.stride(1) == 1
    cu_ = _i32(cu_block_include_tokens)
    nb = cu_.numel() - 1
    out = torch.empty(nb, x.shape[1], dtype=x.dtype, device=x.device)
    rc = L.lsrm_block_mean_fwd(nb, x.shape[1], _dtype_code(x), _ptr(cu_), _ptr(x), x.stride(0), _ptr(out), _stream())
    check(rc, "lsrm_block_mean_fwd")
    return out


def block_mean_bwd(dout: torch.Tensor, cu_block_include_tokens: torch.Tensor, total_tokens: int) -> torch.Tensor:
    L = _lib.lib()
    dout = dout.contiguous()
    cu_ = _i32(cu_block_include_tokens)
    dx = torch.empty(total_tokens, dout.shape[1], dtype=dout.dtype, device=dout.device)
    rc = L.lsrm_block_mean_bwd(cu_.numel() - 1, dout.shape[1], _dtype_code(dout), _ptr(cu_), int(total_tokens),
                               _ptr(dout), _ptr(dx), _stream())
    check(rc, "lsrm_block_mean_bwd")
    return dx


def resnorm_mean_fwd(x, h, cu_block_include_tokens, eps: float = 1e-5, want_y: bool = False):
    """Returns (block_mean [nb, C], y or None, mean [N], rstd [N])."""
    L = _lib.lib()
    x = x.contiguous()
    h = h.contiguous()
    cu_ = _i32(cu_block_include_tokens)
    nb = cu_.numel() - 1
    N, C = x.shape
    out = torch.empty(nb, C, dtype=x.dtype, device=x.device)
    y = torch.empty_like(x) if want_y else None
    mean = torch.empty(N, dtype=torch.float32, device=x.device)
    rstd = torch.empty(N, dtype=torch.float32, device=x.device)
    rc = L.lsrm_resnorm_mean_fwd(nb, N, C, _dtype_code(x), _ptr(cu_), _ptr(x), _ptr(h), float(eps), _ptr(y),
                                 _ptr(out), _ptr(mean), _ptr(rstd), _stream())
    check(rc, "lsrm_resnorm_mean_fwd")
    return out, y, mean, rstd


def resnorm_mean_bwd(x, h, cu_block_include_tokens, mean, rstd, dout):
    L = _lib.lib()
    cu_ = _i32(cu_block_include_tokens)
    N, C = x.shape
    dr = torch.empty_like(x)
    rc = L.lsrm_resnorm_mean_bwd(cu_.numel() - 1, N, C, _dtype_code(x), _ptr(cu_), _ptr(x), _ptr(h), _ptr(mean),
                                 _ptr(rstd), _ptr(dout.contiguous()), _ptr(dr), _stream())
    check(rc, "lsrm_resnorm_mean_bwd")
    return dr


def _ptr_array(ts):
    arr = (ctypes.c_void_p * len(ts))(*[t.data_ptr() for t in ts])
    return arr


def gate_merge_fwd(z, branches: Sequence[torch.Tensor], per_head: bool = False, head_dim: int = 0):
    L = _lib.lib()
    z = z.contiguous()
    branches = [b.contiguous() for b in branches]
    N, C = branches[0].shape
    out = torch.empty(N, C, dtype=branches[0].dtype, device=z.device)
    arr = _ptr_array(branches)
    rc = L.lsrm_gate_merge_fwd(N, C, len(branches), int(per_head), int(head_dim), _dtype_code(z), _ptr(z), arr,
                               _ptr(out), _stream())
    check(rc, "lsrm_gate_merge_fwd")
    return out


def gate_merge_bwd(z, branches: Sequence[torch.Tensor], dout, per_head: bool = False, head_dim: int = 0):
    L = _lib.lib()
    z = z.contiguous()
    branches = [b.contiguous() for b in branches]
    N, C = branches[0].shape
    dz = torch.empty_like(z)
    dbr = [torch.empty_like(b) for b in branches]
    rc = L.lsrm_gate_merge_bwd(N, C, len(branches), int(per_head), int(head_dim), _dtype_code(z), _ptr(z),
                               _ptr_array(branches), _ptr(dout.contiguous()), _ptr(dz), _ptr_array(dbr), _stream())
    check(rc, "lsrm_gate_merge_bwd")
    return dz, dbr


def ulysses_pack(x: torch.Tensor, world: int) -> torch.Tensor:
    """[n, H, D] -> [W, n, hp, D]: the head slice of every rank, rank-major
    (hp = H/W, or one replicated head when H < W)."""
    L = _lib.lib()
    n, H, D = x.shape
    if x.stride(2) != 1 or x.stride(1) != D:
        x = x.contiguous()
    hp = H // world if H >= world else 1
    out = torch.empty(world, n, hp, D, dtype=x.dtype, device=x.device)
    rc = L.lsrm_ulysses_pack(n, H, D, world, _dtype_code(x), x.stride(0), _ptr(x), _ptr(out), _stream())
    check(rc, "lsrm_ulysses_pack")
    return out


def ulysses_unpack(y: torch.Tensor, num_heads: int) -> torch.Tensor:
    """[W, n, hp, D] -> [n, H, D]; replicas of one head are summed in rank
    order (fp32)."""
    L = _lib.lib()
    world, n, hp, D = y.shape
    y = y.contiguous()
    out = torch.empty(n, num_heads, D, dtype=y.dtype, device=y.device)
    rc = L.lsrm_ulysses_unpack(n, num_heads, D, world, _dtype_code(y), _ptr(y), out.stride(0), _ptr(out), _stream())
    check(rc, "lsrm_ulysses_unpack")
    return out


def head_layernorm_pack(x: torch.Tensor, world: int = 1, eps: float = 1e-5) -> torch.Tensor:
    """Per-head non-affine LayerNorm (fp32, cast back) of x [n, H, D] written
    straight into the Ulysses send layout [W, n, H/W, D] (W = 1: [1, n, H, D])."""
    L = _lib.lib()
    n, H, D = x.shape
    if x.stride(2) != 1 or x.stride(1) != D:
        x = x.contiguous()
    out = torch.empty(world, n, H // world, D, dtype=x.dtype, device=x.device)
    rc = L.lsrm_head_layernorm_pack(n, H, D, world, _dtype_code(x), x.stride(0), float(eps), _ptr(x), _ptr(out),
                                    _stream())
    check(rc, "lsrm_head_layernorm_pack")
    return out


def head_layernorm_pack_bwd(x: torch.Tensor, grad_packed: torch.Tensor, eps: float = 1e-5) -> torch.Tensor:
    """Gradient of ``head_layernorm_pack`` with respect to x [n, H, D]."""
    L = _lib.lib()
    n, H, D = x.shape
    if x.stride(2) != 1 or x.stride(1) != D:
        x = x.contiguous()
    world = grad_packed.shape[0]
    g = grad_packed.contiguous()
    out = torch.empty(n, H, D, dtype=x.dtype, device=x.device)
    rc = L.lsrm_head_layernorm_pack_bwd(n, H, D, world, _dtype_code(x), x.stride(0), float(eps), _ptr(x), _ptr(g),
                                        _ptr(out), _stream())
    check(rc, "lsrm_head_layernorm_pack_bwd")
    return out


# ---------------------------------------------------------------------------
# Projection GEMM with the per-head LayerNorm in its epilogue
# ---------------------------------------------------------------------------


def _addr(t: Optional[torch.Tensor]):
    return t.data_ptr() if t is not None else None


def qkv_norm_fwd(x: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor], segments, head_dim: int,
                 eps: float = 1e-5):
    """x [M, K] bf16 (row stride >= K), w [N, K] bf16 (stacked Linear
    weights), ``segments`` a list of (cols, raw, norm) in column order.
    Returns (outputs, rstd): per segment the bf16 result [M, cols] if ``raw``
    and its per-head LayerNorm [M, cols] if ``norm`` (None otherwise), and
    rstd [M, N / head_dim] fp32."""
    L = _lib.lib()
    assert x.dim() == 2 and x.stride(1) == 1 and x.dtype == torch.bfloat16, "x must be [M, K] bf16, unit column stride"
    w = w.contiguous()
    M, K = x.shape
    N = w.shape[0]
    dev = x.device
    segs = (_lib.QkvSegment * len(segments))()
    outs = []
    for i, (cols, raw, norm) in enumerate(segments):
        o = torch.empty(M, cols, dtype=x.dtype, device=dev) if raw else None
        on = torch.empty(M, cols, dtype=x.dtype, device=dev) if norm else None
        segs[i] = _lib.QkvSegment(int(cols), 0, _addr(o), _addr(on))
        outs.append((o, on))
    rstd = torch.empty(M, N // head_dim, dtype=torch.float32, device=dev)
    b = bias.contiguous() if bias is not None else None
    rc = L.lsrm_qkv_norm_fwd(M, K, N, int(head_dim), _ptr(x), x.stride(0), _ptr(w), _ptr(b), segs, len(segments),
                             float(eps), _ptr(rstd), _ptr(_err_word(dev)), _stream())
    check(rc, "lsrm_qkv_norm_fwd")
    return outs, rstd


def qkv_norm_bwd(M: int, N: int, head_dim: int, segments, rstd: torch.Tensor, device, dtype=torch.bfloat16):
    """``segments``: per segment (cols, out_norm, grad_out, grad_norm) with
    None for absent tensors.  Returns the gradient of the pre-norm result
    [M, N]."""
    L = _lib.lib()
    segs = (_lib.QkvGradSegment * len(segments))()
    keep = []
    for i, (cols, on, go, gn) in enumerate(segments):
        go = go.contiguous() if go is not None else None
        gn = gn.contiguous() if gn is not None else None
        keep += [go, gn]
        segs[i] = _lib.QkvGradSegment(int(cols), 0, _addr(on), _addr(go), _addr(gn))
    out = torch.empty(M, N, dtype=dtype, device=device)
    rc = L.lsrm_qkv_norm_bwd(M, N, int(head_dim), segs, len(segments), _ptr(rstd), _ptr(out), _stream())
    check(rc, "lsrm_qkv_norm_bwd")
    return out


# ---------------------------------------------------------------------------
# Windowed attention with sinks, residual RMS norm, counter-based dropout
# ---------------------------------------------------------------------------

_DTYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2, torch.float8_e4m3fn: 3, torch.int8: 4}


def _need(cond: bool, msg: str):
    if not cond:
        raise ValueError(msg)


def _scale(name: str, scale) -> float:
    """What the entry points take for ``softmax_scale``: None and 0 select 1/sqrt(head_dim)."""
    if not scale:
        return 0.0
    _need(2.0**-126 <= scale < 2.0**127, f"{name}: softmax_scale ({scale}) must be positive and finite in 32 bits")
    return float(scale)


def _cuda(name: str, *ts):
    """All tensors (None passes) on one CUDA device, which is returned."""
    dev = None
    for t in ts:
        if t is None:
            continue
        _need(t.is_cuda, f"{name}: tensors must be on a CUDA device, got {t.device}")
        _need(dev is None or t.device == dev, f"{name}: tensors are on {dev} and {t.device}")
        dev = t.device
    return dev


def _run(dev: torch.device, name: str, *args):
    """Call the entry point ``name`` on the current stream of ``dev`` (its raw
    handle: building a Stream object takes longer than the smallest kernels)."""
    fn, i = getattr(_lib.lib(), name), dev.index
    if i == torch._C._cuda_getDevice():
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(i))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(i))
    if rc:
        check(rc, name)


def _flat(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """Contiguous and 16-byte aligned (a copy for any other layout)."""
    if t is None:
        return None
    if not t.is_contiguous():
        t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)


def _token_rows(t: torch.Tensor):
    """[n, heads, head_dim] with contiguous heads in aligned rows, as is or
    copied, and the row stride."""
    n, h, d = t.shape
    lead, per_head, unit = t.stride()
    ok = unit == 1 and (h == 1 or per_head == d) and t.data_ptr() % 16 == 0
    if ok and n <= 1:
        return t, h * d
    if ok and lead >= h * d and lead % 8 == 0:
        return t, lead
    return _flat(t), h * d


def _window_shape(q, k, v, cu_q, window, sinks, causal, scale):
    q, qs = _token_rows(q)
    k, ks = _token_rows(k)
    v, vs = _token_rows(v)
    sh = _lib.WindowShape(cu_q.numel() - 1, q.shape[0], k.shape[0], q.shape[1], k.shape[1], q.shape[2],
                          _dtype_code(q), min(int(window), 2**31 - 1), int(sinks), int(bool(causal)), qs, ks, vs,
                          _scale("window_sink_attention", scale))
    return sh, q, k, v


def check_window_attn(q, k, v, cu_seqlens_q, cu_seqlens_k, window, sinks):
    name = "window_sink_attention"
    _cuda(name, q, k, v, cu_seqlens_q, cu_seqlens_k)
    _need(q.dim() == k.dim() == v.dim() == 3, f"{name}: q, k and v must be [tokens, heads, head_dim]")
    _need(k.shape == v.shape and q.shape[2] == k.shape[2],
          f"{name}: shapes {tuple(q.shape)}, {tuple(k.shape)} and {tuple(v.shape)} do not go together")
    _need(q.dtype == k.dtype == v.dtype, f"{name}: q, k and v must have one dtype")
    for t in (cu_seqlens_q, cu_seqlens_k):
        _need(t.dim() == 1 and t.numel() >= 1 and t.dtype == torch.int32,
              f"{name}: cu_seqlens must be int32 [sequences + 1]")
    _need(cu_seqlens_q.numel() == cu_seqlens_k.numel(), f"{name}: cu_seqlens_q and cu_seqlens_k differ in length")
    _need(int(window) >= 1, f"{name}: window ({window}) must be at least 1")
    _need(int(sinks) >= 0, f"{name}: sinks ({sinks}) must not be negative")


def window_attn_fwd(q, k, v, cu_q, cu_k, window: int, sinks: int, causal: bool, softmax_scale=None,
                    need_rest: bool = False):
    """Returns (out [Nq, Hq, D], lse [Nq, Hq] fp32, natural log), and with
    ``need_rest`` what out's rounding left over, for the backward."""
    sh, q, k, v = _window_shape(q, k, v, cu_q, window, sinks, causal, softmax_scale)
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    rest = torch.empty_like(out) if need_rest else None
    lse = torch.empty(q.shape[0], q.shape[1], dtype=torch.float32, device=q.device)
    cu_q, cu_k = cu_q.contiguous(), cu_k.contiguous()
    _run(q.device, "lsrm_window_attn_fwd", ctypes.byref(sh), _addr(cu_q), _addr(cu_k), _addr(q), _addr(k), _addr(v),
         _addr(out), _addr(rest), _addr(lse), _addr(_err_word(q.device)))
    return (out, lse, rest) if need_rest else (out, lse)


def window_attn_bwd(q, k, v, out, rest, lse, dout, cu_q, cu_k, window: int, sinks: int, causal: bool,
                    softmax_scale=None):
    """Returns (dq, dk, dv); ``rest`` is the forward's, or None."""
    sh, q, k, v = _window_shape(q, k, v, cu_q, window, sinks, causal, softmax_scale)
    dout = _flat(dout)
    dq = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    dk = torch.empty(k.shape, dtype=k.dtype, device=k.device)
    dv = torch.empty(v.shape, dtype=v.dtype, device=v.device)
    cu_q, cu_k = cu_q.contiguous(), cu_k.contiguous()
    ws = _workspace(_lib.lib().lsrm_window_attn_workspace_bytes(ctypes.byref(sh)), q.device)
    _run(q.device, "lsrm_window_attn_bwd", ctypes.byref(sh), _addr(cu_q), _addr(cu_k), _addr(q), _addr(k), _addr(v),
         _addr(out), _addr(rest), _addr(lse), _addr(dout), _addr(dq), _addr(dk), _addr(dv), _addr(ws), ws.numel(),
         _addr(_err_word(q.device)))
    return dq, dk, dv


def window_decode(q, k_new, v_new, k_cache, v_cache, lengths, window: int, sinks: int, softmax_scale=None):
    """One token a sequence over a ring cache, which is updated in place.
    q [B, Hq, D], k_new / v_new [B, Hkv, D], caches [B, capacity, Hkv, D],
    lengths [B] int32.  Returns out [B, Hq, D]."""
    name = "window_sink_decode"
    dev = _cuda(name, q, k_new, v_new, k_cache, v_cache, lengths)
    _need(q.dim() == 3 and k_new.dim() == 3 and k_cache.dim() == 4,
          f"{name}: q and k_new must be [batch, heads, head_dim], the caches [batch, capacity, heads, head_dim]")
    b, hkv, d = k_new.shape
    _need(k_new.shape == v_new.shape and k_cache.shape == v_cache.shape and q.shape[0] == b and q.shape[2] == d
          and (k_cache.shape[0], *k_cache.shape[2:]) == (b, hkv, d),
          f"{name}: shapes {tuple(q.shape)}, {tuple(k_new.shape)} and {tuple(k_cache.shape)} do not go together")
    _need(q.dtype == k_new.dtype == v_new.dtype == k_cache.dtype == v_cache.dtype, f"{name}: tensors must have one dtype")
    _need(lengths.dtype == torch.int32 and tuple(lengths.shape) == (b,), f"{name}: lengths must be int32 [batch]")
    strides = []
    for c in (k_cache, v_cache):  # written in place: no copy may stand in
        sb, sl, sh, sd = c.stride()
        if b == 1:  # the stride of a single sequence says nothing
            sb = sl
        _need(sd == 1 and (hkv == 1 or sh == d) and sl % 8 == 0 and sb % 8 == 0 and sl >= hkv * d and sb >= hkv * d
              and c.data_ptr() % 16 == 0,
              f"{name}: the caches need contiguous heads and strides of 8 elements, aligned to 16 bytes")
        strides += [sb, sl]
    (q, qs), (k_new, ks), (v_new, vs) = _token_rows(q), _token_rows(k_new), _token_rows(v_new)
    lengths = lengths.contiguous()
    sh = _lib.WindowDecodeShape(b, q.shape[1], hkv, d, _dtype_code(q), k_cache.shape[1], min(int(window), 2**31 - 1),
                                int(sinks), qs, ks, vs, *strides, _scale(name, softmax_scale))
    out = torch.empty(b, q.shape[1], d, dtype=q.dtype, device=dev)
    _run(dev, "lsrm_window_decode", ctypes.byref(sh), _addr(q), _addr(k_new), _addr(v_new), _addr(k_cache),
         _addr(v_cache), _addr(lengths), _addr(out))
    return out


def _seed(v: int) -> int:
    return int(v) & (2**64 - 1)


def dropout(x: torch.Tensor, p: float, seed: int, offset: int = 0) -> torch.Tensor:
    """x / (1 - p) where the counter-based generator keeps the element, else 0."""
    dev = _cuda("dropout", x)
    _need(x.dtype in (torch.bfloat16, torch.float16, torch.float32), f"dropout: dtype {x.dtype} is not supported")
    x = _flat(x)
    y = torch.empty(x.shape, dtype=x.dtype, device=dev)
    _run(dev, "lsrm_dropout", x.numel(), _DTYPES[x.dtype], float(p), _seed(seed), _seed(offset), _addr(x), _addr(y))
    return y


def _check_norm(name, x, residual, weight):
    dev = _cuda(name, x, residual, weight)
    _need(x.dim() >= 1, f"{name}: x must have at least one dimension")
    stream = x.dtype if residual is None else residual.dtype
    _need(x.dtype in (torch.bfloat16, torch.float16), f"{name}: x must be bf16 or fp16, got {x.dtype}")
    _need(stream in (x.dtype, torch.float32), f"{name}: the residual must have x's dtype or fp32, got {stream}")
    _need(residual is None or residual.shape == x.shape, f"{name}: the residual must have x's shape")
    _need(weight is None or (tuple(weight.shape) == tuple(x.shape[-1:]) and weight.dtype in (x.dtype, torch.float32)),
          f"{name}: the weight must be [{x.shape[-1]}] of x's dtype or fp32")
    return dev, stream


def _rows_of(x):
    c = x.shape[-1]
    return (x.numel() // c if c else 0), c


def residual_rms_norm_fwd(x, residual, weight, eps: float, p: float, seed: int, offset: int, need_rstd: bool = True):
    """Returns (y, h, rstd [rows] fp32 or None)."""
    dev, stream = _check_norm("residual_rms_norm", x, residual, weight)
    x, residual, weight = _flat(x), _flat(residual), _flat(weight)
    rows, c = _rows_of(x)
    y = torch.empty(x.shape, dtype=x.dtype, device=dev)
    h = torch.empty(x.shape, dtype=stream, device=dev)
    rstd = torch.empty(rows, dtype=torch.float32, device=dev) if need_rstd else None
    _run(dev, "lsrm_residual_rms_norm_fwd", rows, c, _DTYPES[x.dtype], _DTYPES[stream],
         _DTYPES[x.dtype if weight is None else weight.dtype], float(eps), float(p), _seed(seed), _seed(offset),
         _addr(x), _addr(residual), _addr(weight), _addr(y), _addr(h), _addr(rstd))
    return y, h, rstd


def residual_rms_norm_bwd(h, rstd, weight, dy, dh, p: float, seed: int, offset: int, need_dw: bool = True):
    """Gradients (dx, dresidual, dweight) from dy and dh (None: zero); dx is
    dresidual itself where the two are equal."""
    dev = h.device
    weight, dy, dh = _flat(weight), _flat(dy), _flat(dh)
    rows, c = _rows_of(h)
    same = p == 0.0 and dy.dtype == h.dtype
    dres = torch.empty(h.shape, dtype=h.dtype, device=dev)
    dx = dres if same else torch.empty(h.shape, dtype=dy.dtype, device=dev)
    need_dw = need_dw and weight is not None
    dw = torch.empty_like(weight) if need_dw else None
    ws = _workspace(_lib.lib().lsrm_residual_rms_norm_workspace_bytes(rows, c), dev) if need_dw else None
    _run(dev, "lsrm_residual_rms_norm_bwd", rows, c, _DTYPES[dy.dtype], _DTYPES[h.dtype],
         _DTYPES[dy.dtype if weight is None else weight.dtype], float(p), _seed(seed), _seed(offset), _addr(h),
         _addr(rstd), _addr(weight), _addr(dy), _addr(dh), None if same else _addr(dx), _addr(dres), _addr(dw),
         _addr(ws), ws.numel() if ws is not None else 0)
    return dx, dres, dw


def residual_rms_norm_8bit(x, residual, weight, eps: float, dtype: torch.dtype, group: int):
    """Returns (values [.., C] in ``dtype``, scales [.., groups] fp32, h)."""
    dev, stream = _check_norm("residual_rms_norm_8bit", x, residual, weight)
    _need(dtype in (torch.float8_e4m3fn, torch.int8), f"residual_rms_norm_8bit: dtype {dtype} is not e4m3 or int8")
    x, residual, weight = _flat(x), _flat(residual), _flat(weight)
    rows, c = _rows_of(x)
    groups = -(-c // group) if group > 0 else 1
    q = torch.empty(x.shape, dtype=dtype, device=dev)
    scales = torch.empty(*x.shape[:-1], groups, dtype=torch.float32, device=dev)
    h = torch.empty(x.shape, dtype=stream, device=dev)
    _run(dev, "lsrm_residual_rms_norm_8bit", rows, c, _DTYPES[x.dtype], _DTYPES[stream],
         _DTYPES[x.dtype if weight is None else weight.dtype], float(eps), _DTYPES[dtype], int(group), _addr(x),
         _addr(residual), _addr(weight), _addr(q), _addr(scales), _addr(h))
    return q, scales, h


def dequantize_8bit(values, scales, dtype: torch.dtype, group: int):
    dev = _cuda("dequantize_8bit", values, scales)
    _need(values.dtype in (torch.float8_e4m3fn, torch.int8) and scales.dtype == torch.float32
          and dtype in (torch.bfloat16, torch.float16, torch.float32), "dequantize_8bit: unsupported dtypes")
    values, scales = _flat(values), scales.contiguous()
    rows, c = _rows_of(values)
    y = torch.empty(values.shape, dtype=dtype, device=dev)
    _run(dev, "lsrm_dequantize_8bit", rows, c, _DTYPES[values.dtype], _DTYPES[dtype], int(group), _addr(values),
         _addr(scales), _addr(y))
    return y
