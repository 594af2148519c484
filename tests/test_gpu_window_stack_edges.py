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


def test_idle_rows_stay_idle():
    """A row of negative length keeps it and its caches over several steps; the others go on as if it were not there."""
    stack = _stack().eval()
    full = torch.randn(3, 12, 256, device="cuda").bfloat16()
    caches = stack.make_caches(3, torch.bfloat16, "cuda")
    for c in caches:
        c.k.fill_(float("nan"))
        c.v.fill_(float("nan"))
    lengths = torch.tensor([0, -1, 0], dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, 6], dtype=torch.int32, device="cuda")
    outs = []
    for t in range(6):
        y, lengths = stack.step(full[:, t], caches, lengths)
        outs.append(y)
    assert lengths.tolist() == [6, -1, 6] and lengths.dtype == torch.int32
    for c in caches:
        assert torch.isnan(c.k[1]).all() and torch.isnan(c.v[1]).all()
    for i in (0, 2):
        ref = _reference(stack, full[i, :6], cu)
        got = torch.stack(outs, 1)[i].double()
        assert (got - ref).norm() <= 10 * 2.0**-8 * ref.norm(), i
    # taken up later, the row starts from its own position
    lengths[1] = 0
    y, lengths = stack.step(full[:, 6], caches, lengths)
    ref = _reference(stack, full[1, 6:7], torch.tensor([0, 1], dtype=torch.int32, device="cuda"))
    assert lengths.tolist() == [7, 1, 7]
    assert (y[1:2].double() - ref).norm() <= 10 * 2.0**-8 * ref.norm()
