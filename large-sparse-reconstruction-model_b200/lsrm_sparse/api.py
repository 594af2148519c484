"""The reference's op-level API (``sparse.ops``), same names, argument order
and return conventions, backed by the sm_100a kernels.

* ``get_block_score``            — sparse/ops/block_score.py:16-98
* ``spatial_selection_attention`` — sparse/ops/triton_native_sparse_attention.py:17-41
* ``native_sparse_attend``       — sparse/ops/triton_native_sparse_attention_impl_kvcentric.py:1382-1435
* ``set_variant``                — kvcentric.py:1275 (accepted, no effect)
* ``sparse_window_attention``    — sparse/ops/block_window_attention.py:14-31
* ``compressed_attention``       — the flash_attn_varlen_func call of the
                                   compressed branch (spatial_sparse_attention.py:121-143)

Differences from the reference, all documented in the repository's design
notes: ties in top-k go to the lowest block id; a block listed twice for one
query raises (the reference attends it twice); selection entries outside
``[0, blocks_in_sequence)`` are skipped wherever they appear.
"""

from __future__ import annotations

import math
from typing import Optional

import torch

from . import functional as F
from . import ops

_LSE_CHECK = False


def _raise_on_device_errors():
    if _LSE_CHECK:
        e = ops.read_errors()
        if e:
            raise ops._lib.LsrmError(f"device error bits 0x{e:x}")


def get_block_score(q, compressed_k, lse, topk, cu_seqlens_q, compressed_cu_seqlens, seqlens_q=None,
                    compressed_seqlens=None, sm_scale=None, *, cu_query_blocks=None, force_self_block=False):
    """Top-k compressed blocks per query token ([Hkv, Nq, topk] int32,
    ascending, -1 padded).  With ``cu_query_blocks`` (extension) one selection
    per query block: [Hkv, n_query_blocks, topk]."""
    nb = compressed_k.shape[0]
    dummy_blocks = torch.arange(nb + 1, dtype=torch.int32, device=q.device)
    meta = ops.Meta(cu_seqlens_q, cu_seqlens_q, compressed_cu_seqlens, dummy_blocks)
    with torch.no_grad():
        return ops.block_topk(q, compressed_k, lse, int(topk), meta, cu_query_blocks=cu_query_blocks,
                              force_self=force_self_block, sm_scale=sm_scale)


def native_sparse_attend(q, k, v, topk_idx, cu_seqblocks, cu_block_include_tokens, cu_seqlens_q, cu_seqlens_k,
                         softmax_scale: Optional[float] = None, return_lse: bool = False, *, cu_query_blocks=None):
    """Variable-block selected attention; LSE (optional) is log2-based
    [Hq, Nq] fp32 as in the reference."""
    assert q.dtype in (torch.float16, torch.bfloat16), "Only fp16/bf16 supported"
    assert q.dtype == k.dtype == v.dtype
    assert topk_idx.dtype == torch.int32
    assert cu_seqlens_q.dtype == torch.int32 and cu_seqlens_k.dtype == torch.int32
    q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    if softmax_scale is None:
        softmax_scale = 1.0 / math.sqrt(q.shape[-1])
    meta = ops.Meta(cu_seqlens_q, cu_seqlens_k, cu_seqblocks, cu_block_include_tokens)
    out, lse = F.select_attention(q, k, v, topk_idx, meta, softmax_scale, cu_query_blocks)
    _raise_on_device_errors()
    return (out, lse) if return_lse else out


def spatial_selection_attention(q, k, v, block_topk, cu_seqblocks, cu_block_include_tokens, cu_seqlens_q,
                                cu_seqlens_k, seqlens_q=None, seqlens_k=None, softmax_scale=None):
    """Drop-in replacement with the original function signature."""
    return native_sparse_attend(q, k, v, block_topk, cu_seqblocks, cu_block_include_tokens, cu_seqlens_q,
                                cu_seqlens_k, softmax_scale=softmax_scale)


def set_variant(variant: str):
    """Accepted for compatibility; the backward has a single deterministic
    implementation."""
    return None


def sparse_window_attention(q, k, v, cu_block_include_tokens, softmax_scale=None):
    """Self-attention independently within each block."""
    n = q.shape[0]
    two = torch.arange(2, dtype=torch.int32, device=q.device)  # built on the device: no host synchronisation
    cu_seq = two * n
    cu_sb = two * (cu_block_include_tokens.numel() - 1)
    meta = ops.Meta(cu_seq, cu_seq, cu_sb, cu_block_include_tokens)
    out, _ = F.dense_attention(q.contiguous(), k.contiguous(), v.contiguous(), meta, ops.DENSE_INTRA_BLOCK, 0,
                               softmax_scale)
    return out


def sliding_window_attention(q, k, v, cu_seqlens, window: int, softmax_scale=None):
    """Extension: band attention |i - j| <= window // 2 inside each sequence."""
    nb = cu_seqlens.numel() - 1
    cu_blocks = cu_seqlens
    cu_sb = torch.arange(nb + 1, dtype=torch.int32, device=q.device)
    meta = ops.Meta(cu_seqlens, cu_seqlens, cu_sb, cu_blocks)
    out, _ = F.dense_attention(q.contiguous(), k.contiguous(), v.contiguous(), meta, ops.DENSE_SLIDING, int(window),
                               softmax_scale)
    return out


def compressed_attention(q, compressed_k, compressed_v, cu_seqlens_q, compressed_cu_seqlens, return_lse=False,
                         softmax_scale=None):
    """Every query attends to all compressed blocks of its sequence; LSE is
    natural-log [Hq, Nq] (flash-attn's convention)."""
    nb = compressed_k.shape[0]
    dummy_blocks = torch.arange(nb + 1, dtype=torch.int32, device=q.device)
    meta = ops.Meta(cu_seqlens_q, cu_seqlens_q, compressed_cu_seqlens, dummy_blocks)
    out, lse = F.dense_attention(q.contiguous(), compressed_k.contiguous(), compressed_v.contiguous(), meta,
                                 ops.DENSE_COMPRESSED, 0, softmax_scale)
    return (out, lse) if return_lse else out


# ---------------------------------------------------------------------------
# A decoder layer's other operators (extensions: no reference counterpart)
# ---------------------------------------------------------------------------


def window_sink_attention(q, k, v, cu_seqlens_q, cu_seqlens_k=None, *, window: int, sinks: int = 0,
                          causal: bool = True, softmax_scale: Optional[float] = None, return_lse: bool = False):
    """Attention with a sliding window and a few first tokens that stay
    visible, over packed sequences: q [Nq, Hq, D], k / v [Nk, Hkv, D] (bf16 /
    fp16; D 32, 64 or 128; Hq a multiple of Hkv), int32 offsets [sequences + 1]
    (``cu_seqlens_k`` defaults to ``cu_seqlens_q``).  Query i of a sequence
    stands at position i + Lk - Lq and sees key j when

    * causal:    j <= pos and (pos - j < window or j < sinks)
    * symmetric: |pos - j| <= window // 2 or j < sinks (``sliding_window_attention``'s
      band, with sinks)

    A query that sees nothing gives 0, and so do tokens outside the sequences.
    ``sinks`` is at most 128, Hq at most 64 times Hkv; ``softmax_scale`` None or 0
    selects 1 / sqrt(D), a negative one is refused.  Differentiable in q, k and v
    (the scores' gradients pass through the operand type: fp16 wants the usual
    loss scale).  With ``return_lse`` also the natural-log LSE [Hq, Nq] fp32.  A
    value that is no finite number stays within its sequence, where it may reach
    queries that do not see it (0 times it, in a shared tile of keys)."""
    cu_k = cu_seqlens_q if cu_seqlens_k is None else cu_seqlens_k
    out, lse = F.window_sink_attention(q, k, v, cu_seqlens_q, cu_k, window, sinks, causal, softmax_scale)
    _raise_on_device_errors()
    return (out, lse.t()) if return_lse else out


def window_sink_decode(q, k_new, v_new, k_cache, v_cache, lengths, *, window: int, sinks: int = 0,
                       softmax_scale: Optional[float] = None):
    """The causal form for one new token of each sequence over a ring cache:
    q [B, Hq, D], k_new / v_new [B, Hkv, D], caches [B, capacity, Hkv, D] with
    capacity >= sinks + window, lengths [B] int32 (tokens before the new one;
    negative: an idle row).  Writes the new key and value to their slot (position
    j lives in slot j below ``sinks``, else in sinks + (j - sinks) % (capacity -
    sinks)) and returns the attention's output [B, Hq, D].  ``sinks`` has no limit
    here; ``softmax_scale`` as in ``window_sink_attention``.  ``lengths`` is not
    advanced.  Not differentiable."""
    with torch.no_grad():
        return ops.window_decode(q, k_new, v_new, k_cache, v_cache, lengths, window, sinks, softmax_scale)


def dropout(x, p: float, seed: int, offset: int = 0):
    """Dropout whose mask is a function of (seed, offset, element index) and is
    never stored: the backward, or a second call, regenerates it.  Element e
    draws word e % 4 of the Philox4x32-10 block ``offset + e // 4``, so calls that
    must differ take other seeds, or offsets at least ceil(numel / 4) apart.  p in
    [0, 1).  Seed and offset are host integers: a captured CUDA graph replays the
    masks of its capture, so a step that draws new ones is launched or captured anew."""
    if not 0.0 <= p < 1.0:
        raise ValueError(f"dropout: p ({p}) must be in [0, 1)")
    return F.dropout(x, float(p), seed, offset)


def residual_rms_norm(x, residual=None, weight=None, *, eps: float = 1e-6, p: float = 0.0, seed: int = 0,
                      offset: int = 0):
    """The step between a block's branches: h = residual + dropout(x) and
    y = h / sqrt(mean(h**2) + eps) * weight over the last dimension.  Returns
    (y, h): y in x's dtype, h in the residual's (x's or fp32).  Differentiable in
    x, residual and weight; the dropout is ``dropout``'s, with its mask (and its
    host-side seed).  The backward reads h as it was stored."""
    if not 0.0 <= p < 1.0:
        raise ValueError(f"residual_rms_norm: p ({p}) must be in [0, 1)")
    return F.residual_rms_norm(x, residual, weight, float(eps), float(p), seed, offset)


def residual_rms_norm_8bit(x, residual=None, weight=None, *, eps: float = 1e-6, dtype=torch.float8_e4m3fn,
                           group: int = 0):
    """``residual_rms_norm`` (without dropout) with y in 8 bits: returns
    (values, scales, h).  ``dtype`` is float8_e4m3fn or int8; one fp32 scale per
    row, or per ``group`` (32, 64, 128) columns; y ~ values * scale.  The scale of
    a row or group whose y holds a NaN or an infinity is NaN.  Not differentiable."""
    if group not in (0, 32, 64, 128):
        raise ValueError(f"residual_rms_norm_8bit: group ({group}) must be 0, 32, 64 or 128")
    with torch.no_grad():
        return ops.residual_rms_norm_8bit(x, residual, weight, eps, dtype, group)


def dequantize_8bit(values, scales, dtype=torch.bfloat16):
    """values * scale of ``residual_rms_norm_8bit``, in ``dtype``."""
    groups, c = scales.shape[-1], values.shape[-1]
    if scales.shape[:-1] != values.shape[:-1]:
        raise ValueError(f"dequantize_8bit: scales {tuple(scales.shape)} do not go with values {tuple(values.shape)}")
    group = 0 if groups == 1 else next((g for g in (32, 64, 128) if -(-c // g) == groups), None)
    if group is None:
        raise ValueError(f"dequantize_8bit: {groups} scales do not divide {c} columns")
    with torch.no_grad():
        return ops.dequantize_8bit(values, scales, dtype, group)
