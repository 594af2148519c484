"""The windowed attention's, norm's and dropout's C entry points refuse bad
arguments on the host, before any CUDA call, with a message; and the 64-bit
attention of the GPU tests agrees with a plain softmax on the CPU."""

import ctypes
import math

import pytest
import torch

from tests import window_oracle as oracle
from tests.test_abi_cpu import lib  # noqa: F401  (builds and loads the library)

INVALID, WORKSPACE = -1, -5


def _shape(L, **kw):
    v = dict(num_seqs=1, total_q=64, total_k=64, num_q_heads=4, num_kv_heads=2, head_dim=64, dtype=1, window=8, sinks=2,
             causal=1, q_token_stride=256, k_token_stride=128, v_token_stride=128, softmax_scale=0.0)
    v.update(kw)
    return L.WindowShape(*[v[n] for n, _ in L.WindowShape._fields_])


@pytest.mark.parametrize("change,text", [
    (dict(num_q_heads=3), "multiple"), (dict(head_dim=48), "head_dim"), (dict(dtype=2), "dtype"),
    (dict(window=0), "window"), (dict(sinks=129), "sinks"), (dict(sinks=-1), "sinks"),
    (dict(q_token_stride=128), "strides"), (dict(k_token_stride=132), "multiples of 8"),
    (dict(num_q_heads=130, q_token_stride=130 * 64), "query heads"), (dict(total_q=-1), "negative"),
])
def test_window_attn_arguments(lib, change, text):  # noqa: F811
    h = lib.lib()
    sh = _shape(lib, **change)
    p = 1 << 20  # never dereferenced: the checks come first
    assert h.lsrm_window_attn_fwd(ctypes.byref(sh), p, p, p, p, p, p, p, p, None, None) == INVALID
    assert text in h.lsrm_last_error().decode()
    assert h.lsrm_window_attn_bwd(ctypes.byref(sh), p, p, p, p, p, p, p, p, p, p, p, p, p, 1 << 30, None, None) == INVALID


def test_window_attn_pointers_and_workspace(lib):  # noqa: F811
    h = lib.lib()
    sh, p = _shape(lib), 1 << 20
    fwd = [ctypes.byref(sh), p, p, p, p, p, p, None, p, None, None]
    for i in (1, 2, 3, 4, 5, 6, 8):
        assert h.lsrm_window_attn_fwd(*[None if j == i else a for j, a in enumerate(fwd)]) == INVALID
    assert h.lsrm_window_attn_fwd(*[p + 8 if j == 3 else a for j, a in enumerate(fwd)]) == INVALID
    need = h.lsrm_window_attn_workspace_bytes(ctypes.byref(sh))
    # delta of every row, the sinks' own sums, and one slot of partial sums more than the tokens fill
    row = 2 * 2 * 2 * 64 * 4
    assert need >= 64 * 4 * 4 + row + 2 * row
    assert h.lsrm_window_attn_bwd(ctypes.byref(sh), p, p, p, p, p, p, p, p, p, p, p, p, p, need - 1, None,
                                  None) == WORKSPACE
    assert h.lsrm_window_attn_fwd(None, *fwd[1:]) == INVALID
    empty = _shape(lib, total_q=0, total_k=0)
    assert h.lsrm_window_attn_fwd(ctypes.byref(empty), p, p, None, None, None, None, None, None, None, None) == 0


@pytest.mark.parametrize("change,text", [
    (dict(capacity=9), "capacity"), (dict(window=0), "window"), (dict(num_q_heads=3), "multiple"),
    (dict(head_dim=256), "head_dim"), (dict(k_slot_stride=100), "strides"), (dict(k_slot_stride=132), "multiples"),
    (dict(batch=70000), "batch"), (dict(dtype=3), "dtype"),
])
def test_window_decode_arguments(lib, change, text):  # noqa: F811
    v = dict(batch=2, num_q_heads=4, num_kv_heads=2, head_dim=64, dtype=1, capacity=10, window=8, sinks=2, q_stride=256,
             k_new_stride=128, v_new_stride=128, k_batch_stride=1280, k_slot_stride=128, v_batch_stride=1280,
             v_slot_stride=128, softmax_scale=0.0)
    v.update(change)
    sh = lib.WindowDecodeShape(*[v[n] for n, _ in lib.WindowDecodeShape._fields_])
    p = 1 << 20
    assert lib.lib().lsrm_window_decode(ctypes.byref(sh), p, p, p, p, p, p, p, None) == INVALID
    assert text in lib.lib().lsrm_last_error().decode()


def test_norm_and_dropout_arguments(lib):  # noqa: F811
    h, p = lib.lib(), 1 << 20

    def fwd(rows=4, cols=64, dt=1, st=1, wt=1, drop=0.0, x=p, y=p):
        return h.lsrm_residual_rms_norm_fwd(rows, cols, dt, st, wt, 1e-6, drop, 0, 0, x, p, p, y, p, p, None)

    for bad in (dict(rows=-1), dict(cols=0), dict(cols=16385), dict(dt=2), dict(st=0), dict(wt=0), dict(drop=1.0),
                dict(drop=-0.1), dict(drop=math.nan), dict(x=p + 2), dict(y=None)):
        assert fwd(**bad) == INVALID, bad
    assert fwd(rows=0) == 0
    assert h.lsrm_residual_rms_norm_bwd(4, 64, 1, 2, 1, 0.0, 0, 0, p, p, p, p, p, None, p, p, p, 1 << 20, None) == INVALID
    assert h.lsrm_residual_rms_norm_bwd(4, 64, 1, 1, 1, 0.0, 0, 0, p, p, p, p, p, None, p, p, p, 16, None) == WORKSPACE
    assert h.lsrm_residual_rms_norm_8bit(4, 64, 1, 1, 1, 1e-6, 3, 48, p, p, p, p, p, p, None) == INVALID
    assert h.lsrm_residual_rms_norm_8bit(4, 64, 1, 1, 1, 1e-6, 2, 0, p, p, p, p, p, p, None) == INVALID
    assert h.lsrm_dequantize_8bit(4, 64, 1, 1, 0, p, p, p, None) == INVALID
    assert h.lsrm_dropout(-1, 1, 0.5, 0, 0, p, p, None) == INVALID
    assert h.lsrm_dropout(8, 3, 0.5, 0, 0, p, p, None) == INVALID
    assert h.lsrm_dropout(8, 1, 1.0, 0, 0, p, p, None) == INVALID
    assert h.lsrm_dropout(8, 1, 0.5, 0, 0, p + 4, p, None) == INVALID
    assert h.lsrm_dropout(0, 1, 0.5, 0, 0, None, None, None) == 0


@pytest.mark.parametrize("causal", [True, False])
def test_the_oracle_is_a_masked_softmax(causal):
    g = torch.Generator().manual_seed(0)
    cu_q, cu_k = torch.tensor([0, 7, 20]), torch.tensor([0, 30, 38])
    q, k, v, do = (torch.randn(n, h, 8, generator=g, dtype=torch.float64) for n, h in ((20, 4), (38, 2), (38, 2), (20, 4)))
    r = oracle.attention(q, k, v, cu_q, cu_k, 5, 2, causal, dout=do)
    leaf = [t.clone().requires_grad_() for t in (q, k, v)]
    outs = []
    for b in range(2):
        i = torch.arange(int(cu_q[b + 1] - cu_q[b]))
        j = torch.arange(int(cu_k[b + 1] - cu_k[b]))
        gap = i[:, None] + len(j) - len(i) - j
        mask = (gap >= 0) & ((gap < 5) | (j < 2)) if causal else (gap.abs() <= 2) | (j < 2)
        qq, kk, vv = leaf[0][cu_q[b]:cu_q[b + 1]], leaf[1][cu_k[b]:cu_k[b + 1]], leaf[2][cu_k[b]:cu_k[b + 1]]
        for h in range(4):
            s = (qq[:, h] @ kk[:, h // 2].T / 8**0.5).masked_fill(~mask, -1e300)
            p = torch.softmax(s, 1) * mask.any(1, keepdim=True)
            outs.append((b, h, p @ vv[:, h // 2]))
    loss = sum((o * do[cu_q[b]:cu_q[b + 1], h]).sum() for b, h, o in outs)
    grads = torch.autograd.grad(loss, leaf)
    for b, h, o in outs:
        assert torch.allclose(o, r["out"][cu_q[b]:cu_q[b + 1], h], atol=1e-12)
    for x, n in zip(grads, ("dq", "dk", "dv")):
        assert torch.allclose(x, r[n], atol=1e-12), n
