"""Decoding and scoring that share a prompt between its completions: fork and generate with one copy of the prompt's keys and
values, and the policy objective of given completions, against the CPU oracle.

Logits are held to 2e-2 (bf16) and 6e-2 (e4m3 history) of the fp32 oracle, as everywhere for this engine."""
import math
from types import SimpleNamespace

import pytest
import torch

from climbing_gym_amd.config import LFM25SamplingConfig
from oracle import lfm2_oracle as O
from test_engine_gpu import _engine, _flat

gpu = pytest.mark.gpu
PROMPTS = [[1, 2, 3], [1, 4], [1, *range(20, 95)], [1, 5, 6, 7, 8]]


def test_a_decoder_refuses_shared_prefixes_it_cannot_keep():
    from climbing_gym_amd.decoder import LFM25HIPDecoder
    engine = SimpleNamespace(dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="adaptive"):
        LFM25HIPDecoder(engine, shared_prefix=True, adaptive_batching=True)
    with pytest.raises(ValueError, match="bf16 or fp16"):
        LFM25HIPDecoder(SimpleNamespace(dtype=torch.float32), shared_prefix=True)


def _oracle_logprobs(oracle, prompt, completion):
    cache, logits = oracle.prefill([prompt], cap=len(prompt) + len(completion) + 1)
    out = []
    for t in completion:
        out.append(float(logits[0].log_softmax(-1)[t]))
        logits = oracle.append_tokens(cache, torch.tensor([0]), torch.tensor([t]))
    return out


@gpu
@torch.inference_mode()
def test_fork_with_a_shared_prefix_decodes_as_copies_do():
    engine, ocfg, state = _engine()
    oracle = O.OracleEngine(ocfg, state, torch.float32, 256)
    repeats, steps = 3, 6
    ids, cu, longest = _flat(PROMPTS)
    g = torch.Generator().manual_seed(3)
    forced = torch.randint(0, 257, (steps, len(PROMPTS) * repeats), generator=g)
    prefix = engine.prefill(ids, cu, longest, max_cache_len=128)
    state = engine.fork(prefix, repeats, share_prefix=True)
    keys = state.cache.k_cache
    for i, prompt in enumerate(PROMPTS):
        assert torch.equal(keys[:, i * repeats, :len(prompt)], prefix.cache.k_cache[:, i, :len(prompt)])
        assert (keys[:, i * repeats + 1:(i + 1) * repeats] == 0).all()       # no other copy
    caches = [oracle.prefill([PROMPTS[int(i)]], cap=128)[0] for i in state.prompt_indices]
    for step in range(steps):
        if step == 3:     # a batch without the first prompt's leader, the second prompt, and a later row
            state.active_slot_ids = torch.tensor([1, 2, 6, 7, 9, 11], device="cuda")
        rows = state.active_slot_ids.cpu()
        out = engine.decode_step(state, forced[step][rows], LFM25SamplingConfig(temperature=0.0))
        for at, row in enumerate(rows.tolist()):
            want = oracle.append_tokens(caches[row], torch.tensor([0]), forced[step][row:row + 1])
            torch.testing.assert_close(out.logits[at].float().cpu(), want[0], atol=2e-2, rtol=0)
    state.active_slot_ids = torch.tensor([2, 1], device="cuda")
    with pytest.raises(ValueError, match="ascending"):
        engine.decode_step(state, torch.tensor([1, 1]))


@gpu
@pytest.mark.parametrize("flags,bound", ((dict(), 2e-2), (dict(capture=False), 2e-2), (dict(fp8_kv=True), 6e-2),
                                         (dict(fp8_kv=True, fp8_mlp=True, fp8_operators=True, fp8_lm_head=True), 6e-2)))
@torch.inference_mode()
def test_generate_with_shared_prefixes(flags, bound):
    """Log-probabilities of what it draws, with rows that stop at different steps, the first repeat of a prompt among them."""
    engine, ocfg, state = _engine()
    oracle = O.OracleEngine(ocfg, state, torch.float32, 256)
    engine.enable_cuda_graphs(shared_prefix=True, **flags)
    repeats = 5
    stops = tuple(range(0, 257, 9))
    early = set()
    for seed, prompts in ((7, PROMPTS), (8, PROMPTS[::-1]), (9, [[1, 9, 9], [1, 4, 3, 2], [1] * 40, [1, 2]])):   # one graph serves them all
        sampling = LFM25SamplingConfig(temperature=1.0, max_new_tokens=24, seed=seed, stop_token_ids=stops, return_logprobs=True, ignore_eos=True)
        ids, cu, _ = _flat(prompts)
        out = engine.generate(ids, cu, 76, repeats, sampling)
        for i, prompt in enumerate(prompts):
            for j in range(repeats):
                n = int(out.lengths[i, j])
                tokens = out.token_ids[i, j, :n].cpu().tolist()
                assert n == 24 or tokens[-1] in stops
                assert not any(t in stops for t in tokens[:-1])
                if j == 0 and n < 24:
                    early.add(i)
                want = torch.tensor(_oracle_logprobs(oracle, prompt, tokens))
                # a log-probability moves by at most twice what its logits move by
                torch.testing.assert_close(out.logprobs[i, j, :n].cpu(), want, atol=2 * bound, rtol=0)
    assert early and len(engine._cuda_decoder.graphs) == 1
    one = engine.generate(*_flat(PROMPTS), 2, LFM25SamplingConfig(temperature=0.0, max_new_tokens=1))
    assert one.token_ids.shape == (4, 2, 1)
    with pytest.raises(ValueError, match="share prefixes"):
        engine.generate(*_flat([[1, 2]]), 4097, LFM25SamplingConfig(temperature=0.0, max_new_tokens=2))


@gpu
@torch.inference_mode()
def test_policy_objective_of_given_completions():
    from climbing_gym_amd import ops
    engine, ocfg, state = _engine()
    oracle = O.OracleEngine(ocfg, state, torch.float32, 256)
    completions = [[9, 10], [11, 12, 13], [14], list(range(100, 140))]
    want = [_oracle_logprobs(oracle, p, c) for p, c in zip(PROMPTS, completions)]
    g = torch.Generator().manual_seed(5)
    old = [[v + 0.3 * float(torch.randn((), generator=g)) for v in row] for row in want]
    ref = [[v + 0.2 * float(torch.randn((), generator=g)) for v in row] for row in want]
    per_token = [[float(torch.randn((), generator=g)) for _ in row] for row in want]
    config = ops.PolicyLossConfig(clip_high=0.28, kl="k3", kl_coef=0.1, entropy_coef=0.01, aggregate="sequence")
    for advantages in ([1.0, -0.5, 0.25, -2.0], per_token):
        got = engine.policy_objective(PROMPTS, completions, old, advantages, ref_logprobs=ref, config=config, max_prefill_tokens=50,
                                      head_chunk_size=7)
        policy = kl = size = 0.0
        for i, row in enumerate(got.logprobs):
            torch.testing.assert_close(torch.tensor(row), torch.tensor(want[i]), atol=4e-2, rtol=0)
            for t, lp in enumerate(row):
                o, r = (float(torch.tensor(x, dtype=torch.float32)) for x in (old[i][t], ref[i][t]))
                a = float(torch.tensor(advantages[i] if advantages is not per_token else advantages[i][t], dtype=torch.float32))
                ratio, w = math.exp(lp - o), 1.0 / (len(row) * 4)
                policy += w * -min(ratio * a, min(max(ratio, 0.8), 1.28) * a)
                kl += w * (math.exp(r - lp) - 1 - (r - lp))
                size += w * (abs(ratio * a) + abs(a) + 0.1 * math.exp(r - lp) + 1)
        # terms in fp32: the ratio's argument and exponential and a product, the cut's constant, 16 half steps in all
        slack = 16 * 2.0 ** -24 * size
        assert abs(got.stats[0] - policy) <= slack and abs(got.stats[1] - kl) <= 10 * slack
        assert abs(got.loss - (policy + 0.1 * kl - 0.01 * got.stats[2])) <= 2 * slack
        assert got.stats[6] == 46 and 0 < got.stats[2] <= math.log(257)
    with pytest.raises(ValueError, match="old_logprobs"):
        engine.policy_objective(PROMPTS, completions, old[:-1], [1.0] * 4)
    with pytest.raises(ValueError, match="advantages"):
        engine.policy_objective(PROMPTS, completions, old, [1.0] * 3)
    with pytest.raises(ValueError, match="ref_logprobs"):
        engine.policy_objective(PROMPTS, completions, old, [1.0] * 4, config=config)
    with pytest.raises(ValueError, match="at least one"):
        engine.policy_objective([], [], [], [])
