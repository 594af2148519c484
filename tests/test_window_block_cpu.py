"""The windowed stack's host side, on CPU tensors: which keys and values a
prompt leaves in the ring cache."""

import pytest
import torch

from lsrm_sparse.window_block import WindowCache, WindowStack


def _filled(cu, n, window, sinks):
    """(cache after fill, cache expected): token t's key is t + 1, untouched slots hold 0."""
    batch = len(cu) - 1
    cache = WindowCache(batch, window, sinks, 1, 1, torch.float32, "cpu")
    cache.k.zero_()
    cache.v.zero_()
    k = torch.arange(1.0, n + 1)[:, None, None]
    cache.fill(k, -k, torch.tensor(cu, dtype=torch.int32))
    want = torch.zeros(batch, sinks + window, 1, 1)
    for b in range(batch):
        length = cu[b + 1] - cu[b]
        for pos in range(length):
            if pos < sinks or length - pos <= window:
                want[b, pos if pos < sinks else sinks + (pos - sinks) % window] = cu[b] + pos + 1
    return cache, want


@pytest.mark.parametrize("cu,n", [
    ([0, 5, 5, 30], 30),
    ([0, 5, 12], 20),     # tokens after the last sequence
    ([4, 9, 21], 21),     # and before the first
    ([3, 3], 8),          # an empty sequence between padding
    ([0], 6),             # no sequence at all
    ([0], 0),
])
@pytest.mark.parametrize("window,sinks", [(4, 2), (1, 0), (40, 3)])
def test_cache_keeps_what_later_tokens_see(cu, n, window, sinks):
    cache, want = _filled(cu, n, window, sinks)
    assert torch.equal(cache.k, want) and torch.equal(cache.v, -want)


def test_offsets_out_of_order_stay_inside_the_cache():
    """Such offsets are an error of the caller's that the attention reports; the cache's indices stay in range."""
    for cu in ([0, 9, 4, 12], [8, 2, 30], [-3, 40]):
        cache = WindowCache(len(cu) - 1, 4, 2, 1, 1, torch.float32, "cpu")
        cache.fill(torch.ones(12, 1, 1), torch.ones(12, 1, 1), torch.tensor(cu, dtype=torch.int32))


def test_symmetric_stacks_have_no_single_token_form():
    stack = WindowStack(1, 64, 2, 1, window=4, causal=False)
    x, cu = torch.zeros(3, 64), torch.tensor([0, 3], dtype=torch.int32)
    caches = stack.make_caches(1, torch.float32, "cpu")
    for call in (lambda: stack.prefill(x, cu), lambda: stack(x, cu, caches=caches),
                 lambda: stack.step(x[:1], caches, torch.zeros(1, dtype=torch.int32))):
        with pytest.raises(ValueError, match="causal"):
            call()


def test_quantize_twice():
    stack = WindowStack(2, 64, 2, 1, window=4).quantize_()
    before = [b.clone() for b in stack.buffers()]
    stack.quantize_()
    assert len(before) == 8 and all(torch.equal(a.float(), b.float()) for a, b in zip(before, stack.buffers()))
    assert [n for n, p in stack.named_parameters() if p.requires_grad] == ["norm"]
