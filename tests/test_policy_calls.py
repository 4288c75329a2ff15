"""Calls of the scoring and policy-loss operators as a trainer around the engine makes them: tensors that inference made,
numbers that only fp32 finds too large, values given as tensors or not at all."""
import pytest
import torch

from climbing_gym_amd import ops

gpu = pytest.mark.gpu
DEV = "cuda"


@gpu
def test_tokens_and_temperatures_that_inference_made_go_through_autograd():
    g = torch.Generator().manual_seed(1)
    host, picks, heat = torch.randn(6, 300, generator=g), torch.randint(0, 300, (6,), generator=g), 0.5 + torch.rand(6, generator=g)
    def grads(targets, temperature):
        leaf = host.to(DEV).requires_grad_()
        logprobs, entropy = ops.token_logprobs(leaf, targets, temperature=temperature, entropy=True)
        (logprobs.sum() + 0.1 * entropy.sum()).backward()
        return logprobs.detach(), entropy.detach(), leaf.grad
    want = grads(picks.to(DEV), heat.to(DEV))
    with torch.inference_mode():
        targets, temperature = picks.to(DEV), heat.to(DEV)
    assert targets.is_inference() and temperature.is_inference()
    for a, b in zip(grads(targets, temperature), want):
        assert torch.equal(a, b)
    with torch.inference_mode():
        scores = host.to(DEV)
    assert scores.is_inference() and torch.equal(ops.token_logprobs(scores, targets, temperature=temperature), want[0])   # no graph
    with torch.inference_mode():      # the losses' arguments from inference too
        old, advantages = want[0] - 0.1, want[0] * 0 + 1.0
    logprobs = want[0].clone().requires_grad_()
    loss, _ = ops.policy_loss(logprobs, old, advantages)
    loss.backward()
    assert torch.equal(logprobs.grad, ops.policy_loss_forward(want[0], old, advantages)[2])


@gpu
def test_without_tokens_the_results_are_fp32_whatever_the_default_type_is():
    row, logits = torch.zeros(0, device=DEV), torch.zeros(0, 9, device=DEV, dtype=torch.bfloat16)
    targets = torch.zeros(0, device=DEV, dtype=torch.long)
    torch.set_default_dtype(torch.float64)
    try:
        results = [*ops.policy_loss_forward(row, row, row, entropy=row), *ops.policy_gradient(logits, targets, row, row)[:3],
                   ops.policy_loss(row.clone().requires_grad_(), row, row)[0]]
    finally:
        torch.set_default_dtype(torch.float32)
    assert all(t.dtype == torch.float32 and (t == 0).all() for t in results)
    assert [tuple(t.shape) for t in results] == [(), (7,), (0,), (0,), (), (7,), (0,), ()]
