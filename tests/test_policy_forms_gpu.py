"""The forms of the scoring and policy kernels that only large calls take: logits that no cache holds, rows held in registers up
to 128 KiB and longer ones that are read twice, in place and inside wider matrices, batches of many sequences."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def ops():
    from climbing_gym_amd import ops as module
    return module


@pytest.mark.parametrize("rows, v, dtype", ((1792, 65536, torch.bfloat16), (4000, 29999, torch.float16), (1800, 32771, torch.float32),
                                            (14700, 8192, torch.bfloat16), (20000, 3001, torch.float32)))
@pytest.mark.parametrize("entropy", (False, True))
def test_logits_that_no_cache_holds(ops, rows, v, dtype, entropy):
    """More than 224 MB are loaded with the non-temporal hint, parts of them without: the same arithmetic, the same bits."""
    assert rows * v * dtype.itemsize >= 224 << 20
    g = torch.Generator(device=DEV).manual_seed(rows)
    logits = (3 * torch.randn(rows, v, device=DEV, generator=g)).to(dtype)
    targets = torch.randint(-1, v, (rows,), device=DEV, generator=g)
    whole = ops.token_logprobs_forward(logits, targets, entropy=entropy, temperature=0.9)
    step = 500
    for a in range(0, rows, step):
        part = ops.token_logprobs_forward(logits[a:a + step], targets[a:a + step], entropy=entropy, temperature=0.9)
        for x, y in zip(whole, part):
            assert (x is None and y is None) or torch.equal(x[a:a + step].nan_to_num(nan=7.0), y.nan_to_num(nan=7.0))


def test_rows_of_a_very_wide_matrix(ops):
    """64 rows of 65536 values, 4 MiB apart: 8 MB in all, whatever the matrix around them holds."""
    g = torch.Generator(device=DEV).manual_seed(1)
    wide = torch.empty(64, (1 << 21) + 64, device=DEV, dtype=torch.bfloat16)
    logits = wide[:, :65536]
    logits.copy_(3 * torch.randn(64, 65536, device=DEV, generator=g))
    targets = torch.randint(0, 65536, (64,), device=DEV, generator=g)
    for x, y in zip(ops.token_logprobs_forward(logits, targets, entropy=True), ops.token_logprobs_forward(logits.contiguous(), targets, entropy=True)):
        assert torch.equal(x, y)
