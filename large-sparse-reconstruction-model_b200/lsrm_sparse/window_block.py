"""A transformer stack over packed sequences whose attention sees a sliding
window and the sequence's first tokens: trained on whole sequences, then run
token by token over a ring cache of fixed size.

* ``WindowBlock`` — RMS norm, windowed attention with sinks, RMS norm, MLP
* ``WindowStack`` — the layer loop with the residual stream, the final norm,
  ``prefill`` and ``step``
* ``WindowCache`` — one layer's ring of keys and values

The residual stream is carried apart from the branch that is still to be added
to it: a block's first act is ``residual_rms_norm(branch, stream)``, which adds
(with the branch's dropout) and norms in one pass.  Dropout masks are a function
of the step's seed and the place in the stack, so activation recomputation and
the backward see the forward's masks.  ``quantize_()`` turns the Linears that
follow a norm into 8-bit ones (e4m3 weights and activations, a scale per row)
for inference: the norm then writes their operand in 8 bits directly.  Such a
stack takes no dropout and no gradient: its parameters are frozen, and a
backward pass through it raises.  The Linears themselves are library GEMMs, as
in the decoder.
"""

from __future__ import annotations

from typing import List, Optional

import torch
import torch.nn as nn

from . import api

_SITE = 1 << 40  # counter blocks between two dropout sites: more than any tensor's


class Linear8(nn.Module):
    """A Linear for 8-bit inference: e4m3 weights with a scale per output, fed
    with the (values, scales) of ``residual_rms_norm_8bit``."""

    def __init__(self, linear: nn.Linear):
        super().__init__()
        w = linear.weight.detach().float()
        scale = w.abs().amax(1, keepdim=True).clamp_(min=1e-12) / 448.0
        self.register_buffer("weight", (w / scale).to(torch.float8_e4m3fn))
        self.register_buffer("scale", scale.t().contiguous())  # [1, out]
        self.bias = linear.bias

    def forward(self, values, scales, dtype):
        # bf16 whatever ``dtype``: the library's fp16 form with a scale per row gives wrong products, and next to
        # e4m3's rounding (2^-4) bf16's (2^-9) is small
        y = torch._scaled_mm(values, self.weight.t(), scale_a=scales, scale_b=self.scale, out_dtype=torch.bfloat16)
        y = y.to(dtype)
        return y if self.bias is None else y + self.bias


class _NoGradient(torch.autograd.Function):
    """``t``, behind the ``sources`` that no gradient reaches."""

    @staticmethod
    def forward(ctx, t, *sources):
        return t.view_as(t)

    @staticmethod
    def backward(ctx, _):
        raise RuntimeError("8-bit Linears are for inference: no gradient passes through the norm in front of them")


class WindowCache:
    """Keys and values of one layer: [batch, sinks + window, heads, head_dim],
    position j in slot j below ``sinks``, else in the ring behind them."""

    def __init__(self, batch: int, window: int, sinks: int, num_kv_heads: int, head_dim: int, dtype, device):
        shape = (batch, sinks + window, num_kv_heads, head_dim)
        self.k, self.v = (torch.empty(shape, dtype=dtype, device=device) for _ in range(2))
        self.window, self.sinks = window, sinks

    def fill(self, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor):
        """Keep what later tokens can see of packed prompts k / v [N, heads, head_dim].
        Tokens before the first and after the last sequence are padding, as in
        ``window_sink_attention``.  Selecting the tokens waits for the GPU, so a
        prefill cannot be captured in a CUDA graph."""
        n = cu_seqlens.numel() - 1
        if n == 0:
            return
        cu = cu_seqlens.long()
        tok = torch.arange(k.shape[0], device=k.device)
        seq = torch.searchsorted(cu, tok, right=True) - 1
        inside = (seq >= 0) & (seq < n)
        seq = seq.clamp(0, n - 1)
        pos, left = tok - cu[seq], cu[seq + 1] - tok
        inside &= (pos >= 0) & (left > 0)  # offsets that are out of order write nothing out of range
        kept = inside & ((pos < self.sinks) | (left <= self.window))
        tok, seq, pos = tok[kept], seq[kept], pos[kept]
        slot = torch.where(pos < self.sinks, pos, self.sinks + (pos - self.sinks) % self.window)
        self.k[seq, slot], self.v[seq, slot] = k[tok], v[tok]


class WindowBlock(nn.Module):
    def __init__(self, dim: int, num_q_heads: int, num_kv_heads: int, window: int, sinks: int = 0, causal: bool = True,
                 mlp_ratio: float = 4.0, dropout: float = 0.0, eps: float = 1e-6, act_layer=nn.GELU):
        super().__init__()
        self.num_q_heads, self.num_kv_heads, self.head_dim = num_q_heads, num_kv_heads, dim // num_q_heads
        self.window, self.sinks, self.causal, self.dropout, self.eps = window, sinks, causal, dropout, eps
        self.norm_attn, self.norm_mlp = (nn.Parameter(torch.ones(dim)) for _ in range(2))
        self.qkv = nn.Linear(dim, (num_q_heads + 2 * num_kv_heads) * self.head_dim, bias=False)
        self.proj = nn.Linear(dim, dim, bias=False)
        self.fc1, self.act, self.fc2 = nn.Linear(dim, int(dim * mlp_ratio)), act_layer(), nn.Linear(int(dim * mlp_ratio), dim)

    def quantize_(self):
        if not isinstance(self.qkv, Linear8):
            self.qkv, self.fc1 = Linear8(self.qkv), Linear8(self.fc1)
        return self.requires_grad_(False)

    def _norm_linear(self, branch, stream, weight, linear, p, seed, offset):
        """(linear(norm(stream + dropout(branch))), the new stream)."""
        if isinstance(linear, Linear8):
            if p:
                raise ValueError("8-bit Linears are for inference: the norm in front of them has no dropout (call eval())")
            values, scales, h = api.residual_rms_norm_8bit(branch, stream, weight, eps=self.eps)
            if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (branch, stream)):
                h = _NoGradient.apply(h, branch, stream)
            return linear(values, scales, branch.dtype), h
        y, stream = api.residual_rms_norm(branch, stream, weight, eps=self.eps, p=p, seed=seed, offset=offset)
        return linear(y), stream

    def _split(self, qkv):
        hq, hkv, d = self.num_q_heads, self.num_kv_heads, self.head_dim
        return (t.unflatten(1, (-1, d)) for t in qkv.split([hq * d, hkv * d, hkv * d], 1))

    def _check_causal(self):
        if not self.causal:
            raise ValueError("the single-token form is causal: a stack with causal=False has no prefill and no step")

    def forward(self, branch, stream, cu_seqlens, seed: int = 0, site: int = 0, first: bool = False,
                cache: Optional[WindowCache] = None):
        """branch and stream [N, dim] (stream None at the stack's start); returns
        the next (branch, stream).  ``site`` counts the stack's dropout sites."""
        if cache is not None:
            self._check_causal()
        p = self.dropout if self.training and cache is None else 0.0
        qkv, stream = self._norm_linear(branch, stream, self.norm_attn, self.qkv, 0.0 if first else p, seed,
                                        site * _SITE)
        q, k, v = self._split(qkv)
        if cache is not None:
            cache.fill(k, v, cu_seqlens)
        o = api.window_sink_attention(q, k, v, cu_seqlens, window=self.window, sinks=self.sinks, causal=self.causal)
        hidden, stream = self._norm_linear(self.proj(o.flatten(1)), stream, self.norm_mlp, self.fc1, p, seed,
                                           (site + 1) * _SITE)
        return self.fc2(api.dropout(self.act(hidden), p, seed, (site + 2) * _SITE)), stream

    def step(self, branch, stream, cache: WindowCache, lengths):
        """One token of each sequence ([batch, dim]) over the cache (causal blocks)."""
        self._check_causal()
        qkv, stream = self._norm_linear(branch, stream, self.norm_attn, self.qkv, 0.0, 0, 0)
        q, k, v = self._split(qkv)
        o = api.window_sink_decode(q, k, v, cache.k, cache.v, lengths, window=self.window, sinks=self.sinks)
        hidden, stream = self._norm_linear(self.proj(o.flatten(1)), stream, self.norm_mlp, self.fc1, 0.0, 0, 0)
        return self.fc2(self.act(hidden)), stream


class WindowStack(nn.Module):
    """``depth`` blocks and a final norm over packed tokens [N, dim]."""

    def __init__(self, depth: int, dim: int, num_q_heads: int, num_kv_heads: int, window: int, sinks: int = 0,
                 causal: bool = True, mlp_ratio: float = 4.0, dropout: float = 0.0, eps: float = 1e-6):
        super().__init__()
        self.eps = eps
        self.blocks = nn.ModuleList([WindowBlock(dim, num_q_heads, num_kv_heads, window, sinks, causal, mlp_ratio,
                                                 dropout, eps) for _ in range(depth)])
        self.norm = nn.Parameter(torch.ones(dim))

    def quantize_(self):
        for b in self.blocks:
            b.quantize_()
        return self

    def make_caches(self, batch: int, dtype, device) -> List[WindowCache]:
        return [WindowCache(batch, b.window, b.sinks, b.num_kv_heads, b.head_dim, dtype, device) for b in self.blocks]

    def forward(self, x, cu_seqlens, seed: int = 0, caches: Optional[List[WindowCache]] = None):
        """x [N, dim] of sequences at cu_seqlens (int32).  ``seed`` picks the
        step's dropout masks; ``caches`` are filled for ``step`` (which, like it,
        takes no dropout in any mode)."""
        branch, stream = x, None
        for i, b in enumerate(self.blocks):
            branch, stream = b(branch, stream, cu_seqlens, seed, 3 * i, i == 0, caches[i] if caches else None)
        p = self.blocks[0].dropout if self.training and not caches else 0.0
        return api.residual_rms_norm(branch, stream, self.norm, eps=self.eps, p=p, seed=seed,
                                     offset=3 * len(self.blocks) * _SITE)[0]

    @torch.no_grad()
    def prefill(self, x, cu_seqlens):
        """Whole prompts (causal stacks): (outputs [N, dim], caches, lengths)."""
        caches = self.make_caches(cu_seqlens.numel() - 1, x.dtype, x.device)
        y = self.forward(x, cu_seqlens, caches=caches)
        return y, caches, cu_seqlens.diff().int()

    @torch.no_grad()
    def step(self, x, caches, lengths):
        """The next token of each sequence, x [batch, dim], with ``lengths`` tokens
        before it; returns its output and the new lengths.  A negative length marks
        an idle row: its caches and its length stay as they are."""
        branch, stream = x, None
        for b, c in zip(self.blocks, caches):
            branch, stream = b.step(branch, stream, c, lengths)
        y = api.residual_rms_norm(branch, stream, self.norm, eps=self.eps)[0]
        return y, lengths + (lengths >= 0).to(lengths.dtype)
