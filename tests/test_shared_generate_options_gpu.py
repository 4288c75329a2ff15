"""Every way of drawing that `generate` has, with shared prefixes and with copies, and a history of either type.

Logits of both are within 2e-2 (bf16) or 6e-2 (e4m3 history) of the same oracle's, so within twice that of each other, and a
log-probability moves by at most twice what its logits move by: 4 times the bound, as long as the histories are the same."""
import pytest
import torch

from climbing_gym_amd.config import LFM25SamplingConfig
from test_engine_gpu import _engine, _flat

pytestmark = pytest.mark.gpu
PROMPTS = [[1, 2, 3], [1, 4], [1, *range(20, 95)], [1, 5, 6, 7, 8]]
STOPS = (3, 9, 27, 81, 100, 120, 140)
OPTIONS = {"greedy": dict(temperature=0.0), "repetition penalty": dict(temperature=0.0, repetition_penalty=1.3), "top k": dict(temperature=1.0, top_k=5, seed=3),
           "top p": dict(temperature=1.0, top_p=0.8, seed=4), "behavior head": dict(temperature=1.0, seed=6, behavior_topk=4),
           "stop sequences": dict(temperature=1.0, seed=7, stop_token_sequences=tuple((a, b) for a in range(0, 257, 3) for b in (1, 50, 200))),
           "stop tokens": dict(temperature=1.0, seed=5, stop_token_ids=STOPS), "to the end of text": dict(temperature=1.0, seed=8, ignore_eos=False)}


@pytest.fixture(scope="module", params=(False, True), ids=("model dtype", "e4m3"))
def pair(request):
    engines = []
    for share in (False, True):
        engine = _engine()[0]
        engine.enable_cuda_graphs(shared_prefix=share, fp8_kv=request.param, max_graphs=1)
        engines.append(engine)
    return engines, 6e-2 if request.param else 2e-2


@pytest.mark.parametrize("repeats", (2, 5))
@pytest.mark.parametrize("option", OPTIONS)
@torch.inference_mode()
def test_draws_like_copies_do(pair, option, repeats):
    engines, bound = pair
    sampling = LFM25SamplingConfig(**{**dict(max_new_tokens=20, return_logprobs=True, ignore_eos=True), **OPTIONS[option]})
    plain, shared = [e.generate(*_flat(PROMPTS), repeats, sampling) for e in engines]
    steps = torch.arange(20, device="cuda")
    together = (plain.token_ids == shared.token_ids).cumprod(-1).bool() & (steps < torch.minimum(plain.lengths, shared.lengths)[..., None])
    assert together[..., 0].all()                                       # the first draw is the prefill's
    # the first draw that differs was still made after the same tokens, but is another token: its log-probability says nothing
    apart = (plain.logprobs - shared.logprobs).abs()
    assert (apart[together] <= 4 * bound).all(), apart[together].max()
    if plain.topk_logprobs is not None:
        same = together[..., None] & (plain.topk_token_ids == shared.topk_token_ids)
        apart = (plain.topk_logprobs - shared.topk_logprobs).abs()
        assert (apart[same] <= 4 * bound).all()
    whole = (plain.token_ids == shared.token_ids).all(-1)
    assert torch.equal(plain.lengths[whole], shared.lengths[whole]) and torch.equal(plain.finish_reasons[whole], shared.finish_reasons[whole])
    for out in (plain, shared):                                         # rows end where they say
        lengths, reasons = out.lengths.flatten().tolist(), out.finish_reasons.flatten().tolist()
        for row, n, reason in zip(out.token_ids.flatten(0, 1).tolist(), lengths, reasons):
            assert 1 <= n <= 20 and (n == 20 or reason in (1, 2))
            if option == "stop tokens":
                assert not any(t in STOPS for t in row[:n - 1]) and (n == 20 or row[n - 1] in STOPS)
