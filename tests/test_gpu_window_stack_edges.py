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


def test_8bit_stack_takes_no_gradient():
    """A backward pass raises where it would leave gradients out; without one the stack runs in any mode."""
    stack = _stack().quantize_()
    cu = torch.tensor([0, 64, 100], dtype=torch.int32, device="cuda")
    x = torch.randn(100, 256, device="cuda").bfloat16()
    with torch.no_grad():
        ref = stack(x, cu)
    y = stack(x, cu)  # training mode without dropout; only the final norm's weight takes a gradient
    assert torch.equal(y.detach(), ref)
    y.float().sum().backward()
    assert stack.norm.grad is not None and stack.norm.grad.abs().sum() > 0
    leaf = x.clone().requires_grad_()
    y = stack(leaf, cu)
    assert torch.equal(y.detach(), ref)
    with pytest.raises(RuntimeError, match="inference"):
        y.float().sum().backward()


def test_8bit_stack_takes_no_dropout():
    stack = _stack(dropout=0.2).quantize_()
    cu = torch.tensor([0, 100], dtype=torch.int32, device="cuda")
    x = torch.randn(100, 256, device="cuda").bfloat16()
    with torch.no_grad(), pytest.raises(ValueError, match="dropout"):
        stack(x, cu, seed=1)
    with torch.no_grad():
        stack.eval()(x, cu)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_linear8_is_the_product_of_its_operands(dtype):
    """Linear8 against the 64-bit product of the numbers that its 8-bit operands stand for: one rounding to bf16 (and one
    to fp16), sums of 512 products in 32 bits; and the weights within half a step of the Linear's."""
    from lsrm_sparse import api
    from lsrm_sparse.window_block import Linear8

    g = torch.Generator(device="cuda").manual_seed(5)
    lin = torch.nn.Linear(512, 192, device="cuda", dtype=dtype)
    lin8 = Linear8(lin)
    x = torch.randn(70, 512, device="cuda", generator=g).to(dtype)
    values, scales, _ = api.residual_rms_norm_8bit(x, None, None)
    with torch.no_grad():
        y = lin8(values, scales, dtype)
    a = values.double() * scales.double()
    w = lin8.weight.double() * lin8.scale.double().t()
    assert ((w - lin.weight.double()).abs() <= 2.0**-4 * lin.weight.double().abs() + 2.0**-10 * lin8.scale.double().t()).all()
    bias = lin.bias.detach().double()
    ref = a @ w.t()
    # the product's rounding, then the sum's with the bias (both at most 2^-8, bf16)
    bound = 2.0**-8 * (ref.abs() + (ref + bias).abs()) + 2.0**-12 * (a.abs() @ w.abs().t()) + 2.0**-25
    assert y.dtype == dtype and ((y.double() - ref - bias).abs() <= bound).all()


def test_8bit_stack_error_is_the_formats():
    """e4m3 is off by at most 2^-4 of a value, 2^-4 / sqrt(3) in the mean square, and so is a long product of two such
    operands by sqrt(2) of that; four of them on branches no larger than the stream add in quadrature, next to ten 16-bit roundings."""
    stack = _stack().eval()
    cu = torch.tensor([0, 64, 160], dtype=torch.int32, device="cuda")
    x = torch.randn(160, 256, device="cuda").bfloat16()
    ref = _reference(stack, x, cu)
    with torch.no_grad():
        y = stack.quantize_()(x, cu)
    bound = 4**0.5 * 2**0.5 * 2.0**-4 / 3**0.5 + 10 * 2.0**-8
    assert (y.double() - ref).norm() <= bound * ref.norm()


def test_prefill_takes_no_dropout():
    """As step: whatever the mode, the prompt's outputs and caches are those of the stack without dropout."""
    stack = _stack(dropout=0.3).train()
    cu = torch.tensor([0, 40], dtype=torch.int32, device="cuda")
    x = torch.randn(40, 256, device="cuda").bfloat16()
    y, caches, _ = stack.prefill(x, cu)
    ref, want, _ = stack.eval().prefill(x, cu)
    assert torch.equal(y, ref)
    for a, b in zip(caches, want):
        assert torch.equal(a.k[:, :27], b.k[:, :27]) and torch.equal(a.v[:, :27], b.v[:, :27])
