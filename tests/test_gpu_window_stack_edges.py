"""The windowed stack away from the plain case: padded prompts, idle rows, modes
that have no single-token form, 8-bit Linears outside inference."""

import pytest
import torch

from tests.test_gpu_window_block import _reference, _stack

pytestmark = pytest.mark.gpu


def test_padded_prompts_then_tokens():
    """Tokens outside the sequences (any finite value) leave the sequences' outputs and caches as they are."""
    stack = _stack().eval()
    lens, before, after, extra = [40, 3, 0, 25], 7, 21, 4
    n = sum(lens)
    starts = torch.tensor([0] + lens).cumsum(0) + before
    cu = starts.to(torch.int32).cuda()
    full = torch.randn(len(lens), max(lens) + extra, 256, device="cuda").bfloat16()
    prompt = torch.randn(before + n + after, 256, device="cuda").bfloat16()
    for i, m in enumerate(lens):
        prompt[starts[i]:starts[i] + m] = full[i, :m]
    y, caches, lengths = stack.prefill(prompt, cu)
    assert lengths.tolist() == lens
    for i, m in enumerate(lens):
        if m:
            c = torch.tensor([0, m], dtype=torch.int32, device="cuda")
            ref = _reference(stack, full[i, :m], c)
            got = y[starts[i]:starts[i] + m].double()
            assert (got - ref).norm() <= 10 * 2.0**-8 * ref.norm(), i
    for t in range(extra):
        x = torch.stack([full[i, m + t] for i, m in enumerate(lens)])
        y, lengths = stack.step(x, caches, lengths)
        for i, m in enumerate(lens):
            c = torch.tensor([0, m + t + 1], dtype=torch.int32, device="cuda")
            ref = _reference(stack, full[i, :m + t + 1], c)[-1]
            assert (y[i].double() - ref).norm() <= 10 * 2.0**-8 * ref.norm(), (i, t)
