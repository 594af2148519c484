"""The windowed stack: a training step against the same layers in 64 bits, tokens
run one by one over the ring cache against the packed forward, dropout's masks
across a recomputation, and the 8-bit Linears."""

import pytest
import torch

from tests import window_oracle as oracle

pytestmark = pytest.mark.gpu


def _stack(dtype=torch.bfloat16, **kw):
    from lsrm_sparse import WindowStack

    torch.manual_seed(0)
    args = dict(depth=2, dim=256, num_q_heads=4, num_kv_heads=2, window=24, sinks=3)
    args.update(kw)
    return WindowStack(**args).cuda().to(dtype)


def _reference(stack, x, cu):
    """Outputs in 64 bits, from the stack's parameters."""
    w = {n: t.detach().double() for n, t in stack.named_parameters()}

    def norm(h, g):
        return h / (h.square().mean(1, keepdim=True) + stack.eps).sqrt() * g

    h = x.double()
    for i, b in enumerate(stack.blocks):
        p = f"blocks.{i}."
        q, k, v = (norm(h, w[p + "norm_attn"]) @ w[p + "qkv.weight"].T).split(
            [b.num_q_heads * b.head_dim] + [b.num_kv_heads * b.head_dim] * 2, 1)
        o = oracle.attention(*(t.reshape(len(x), -1, b.head_dim) for t in (q, k, v)), cu, cu, b.window, b.sinks,
                             b.causal)["out"]
        h = h + o.flatten(1) @ w[p + "proj.weight"].T
        m = torch.nn.functional.gelu(norm(h, w[p + "norm_mlp"]) @ w[p + "fc1.weight"].T + w[p + "fc1.bias"])
        h = h + m @ w[p + "fc2.weight"].T + w[p + "fc2.bias"]
    return norm(h, w["norm"])


@pytest.mark.parametrize("causal", [True, False])
def test_forward_against_64_bits(causal):
    stack = _stack(causal=causal).eval()
    cu = torch.tensor([0, 90, 91, 200], dtype=torch.int32, device="cuda")
    x = torch.randn(200, 256, device="cuda").bfloat16()
    with torch.no_grad():
        y = stack(x, cu)
    ref = _reference(stack, x, cu)
    # some ten 16-bit roundings of 2^-8 in a row, each relative to the whole
    assert (y.double() - ref).norm() <= 10 * 2.0**-8 * ref.norm()


def test_tokens_one_by_one_match_the_packed_forward():
    stack = _stack().eval()
    lens, extra = [40, 3, 0, 25], 37
    b = len(lens)
    full = torch.randn(b, max(lens) + extra, 256, device="cuda").bfloat16()
    cu = torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32, device="cuda")
    prompt = torch.cat([full[i, :n] for i, n in enumerate(lens)])
    _, caches, lengths = stack.prefill(prompt, cu)
    got = []
    for t in range(extra):
        x = torch.stack([full[i, n + t] for i, n in enumerate(lens)])
        y, lengths = stack.step(x, caches, lengths)
        got.append(y)
    got = torch.stack(got, 1)
    for i, n in enumerate(lens):
        c = torch.tensor([0, n + extra], dtype=torch.int32, device="cuda")
        ref = _reference(stack, full[i, :n + extra], c)[n:]
        assert (got[i].double() - ref).norm() <= 10 * 2.0**-8 * ref.norm(), i
    assert lengths.tolist() == [n + extra for n in lens]


def test_training_step_reaches_every_parameter_and_repeats():
    stack = _stack(dropout=0.1).train()
    cu = torch.tensor([0, 64, 150], dtype=torch.int32, device="cuda")
    x = torch.randn(150, 256, device="cuda").bfloat16()

    def grads(seed):
        stack.zero_grad()
        stack(x, cu, seed=seed).float().square().mean().backward()
        return [p.grad.clone() for p in stack.parameters()]

    a, b, c = grads(1), grads(1), grads(2)
    assert all(torch.isfinite(g).all() and g.abs().sum() > 0 for g in a)
    assert all(torch.equal(s, t) for s, t in zip(a, b))  # the same masks, the same order of every sum
    assert not all(torch.equal(s, t) for s, t in zip(a, c))


def test_recomputed_activations_see_the_same_masks():
    from torch.utils.checkpoint import checkpoint

    stack = _stack(dropout=0.2).train()
    cu = torch.tensor([0, 130], dtype=torch.int32, device="cuda")
    x = torch.randn(130, 256, device="cuda").bfloat16()

    def grads(run):
        stack.zero_grad()
        run(x).float().square().mean().backward()
        return [p.grad.clone() for p in stack.parameters()]

    a = grads(lambda t: stack(t, cu, seed=5))
    b = grads(lambda t: checkpoint(lambda u: stack(u, cu, seed=5), t, use_reentrant=False))
    assert all(torch.equal(s, t) for s, t in zip(a, b))


def test_8bit_linears():
    stack = _stack().eval()
    cu = torch.tensor([0, 64, 160], dtype=torch.int32, device="cuda")
    x = torch.randn(160, 256, device="cuda").bfloat16()
    with torch.no_grad():
        ref = stack(x, cu)
        y = stack.quantize_()(x, cu)
    # e4m3 rounds by 2^-4; two quantised products a block, each a branch beside the stream
    assert (y.float() - ref.float()).norm() <= 4 * 2.0**-4 * ref.float().norm()
