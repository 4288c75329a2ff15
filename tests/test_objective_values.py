"""The numbers that `policy_objective` takes beside the completions: lists, arrays and tensors of them, and what it refuses before
any work on the device."""
import numpy as np
import pytest
import torch

from climbing_gym_amd import ops
from climbing_gym_amd.engine import LFM25Engine

PROMPTS, COMPLETIONS = [[1], [2, 3], [4]], [[5, 6], [7], [8, 9, 10]]
OLD = [[-1.0, -2.0], [-3.0], [-0.5, -0.25, -0.125]]


class Reached(Exception):
    pass


class Engine(LFM25Engine):
    """Stops where the first prefill would begin, with what the loss would be given."""
    def __init__(self):
        self.device = torch.device("cpu")

    def _completion_rows(self, *args):
        raise Reached


def _values(monkeypatch, *args, **kw):
    """(old, advantages, ref, per_sequence) as they arrive at the loss."""
    seen = {}
    monkeypatch.setattr(Engine, "_completion_rows", lambda self, *a: iter(()))
    def loss(logprobs, old, advantages, *, ref_logprobs, per_sequence, **rest):
        seen.update(old=old, advantages=advantages, ref=ref_logprobs, per_sequence=per_sequence)
        return torch.zeros(()), torch.zeros(7), None, None
    monkeypatch.setattr(ops, "policy_loss_forward", loss)
    Engine().policy_objective(PROMPTS, COMPLETIONS, *args, **kw)
    return seen


@pytest.mark.parametrize("form", (list, tuple, np.array, torch.tensor, lambda v: [torch.tensor(x) for x in v], lambda v: [np.float64(x) for x in v]))
def test_one_advantage_per_completion(monkeypatch, form):
    seen = _values(monkeypatch, OLD, form([1.0, -0.5, 0.25]))
    assert seen["per_sequence"] and torch.equal(seen["advantages"], torch.tensor([1.0, -0.5, 0.25]))
    assert torch.equal(seen["old"], torch.tensor(sum(OLD, []))) and seen["ref"] is None


@pytest.mark.parametrize("form", (list, tuple, np.array, torch.tensor))
def test_values_per_token(monkeypatch, form):
    rows = [form(row) for row in OLD]
    seen = _values(monkeypatch, rows, [form([1.0, 2.0]), form([3.0]), form([4.0, 5.0, 6.0])], ref_logprobs=rows)
    assert not seen["per_sequence"] and seen["advantages"].tolist() == [1, 2, 3, 4, 5, 6]
    assert torch.equal(seen["old"], torch.tensor(sum(OLD, []))) and torch.equal(seen["ref"], seen["old"])


def test_one_token_each_as_a_matrix(monkeypatch):
    monkeypatch.setattr("test_objective_values.COMPLETIONS", [[5], [6], [7]])
    seen = _values(monkeypatch, torch.zeros(3, 1), torch.ones(3, 1))
    assert not seen["per_sequence"] and seen["advantages"].tolist() == [1, 1, 1]


@pytest.mark.parametrize("args, kw, text", [
    ((None, [1.0] * 3), {}, "old_logprobs"), ((OLD, None), {}, "advantages"), ((OLD[:2], [1.0] * 3), {}, "old_logprobs"),
    ((OLD, [1.0] * 2), {}, "advantages"), ((OLD, torch.ones(4)), {}, "advantages"), ((OLD, [1.0, [1.0], 1.0]), {}, "advantages"),
    (([-1.0, -2.0, -3.0], [1.0] * 3), {}, "old_logprobs"), ((OLD, [1.0] * 3), dict(ref_logprobs=OLD[::-1]), "ref_logprobs"),
    ((OLD, [1.0] * 3), dict(config=ops.PolicyLossConfig(kl_coef=0.1)), "ref_logprobs"),
    ((OLD, [1.0] * 3), dict(temperature=0.0), "temperature"), ((OLD, [1.0] * 3), dict(temperature=float("nan")), "temperature")])
def test_refused_before_any_prefill(args, kw, text):
    with pytest.raises(ValueError, match=text):
        Engine().policy_objective(PROMPTS, COMPLETIONS, *args, **kw)


def test_what_is_right_gets_as_far_as_the_prefill():
    with pytest.raises(Reached):
        Engine().policy_objective(PROMPTS, COMPLETIONS, OLD, torch.ones(3))


def test_the_package_offers_what_a_call_returns():
    import climbing_gym_amd
    from climbing_gym_amd.engine import LFM25PolicyObjective
    assert climbing_gym_amd.LFM25PolicyObjective is LFM25PolicyObjective and "LFM25PolicyObjective" in climbing_gym_amd.__all__
    assert all(hasattr(climbing_gym_amd, name) for name in climbing_gym_amd.__all__)
