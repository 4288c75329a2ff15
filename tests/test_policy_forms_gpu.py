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


# --------------------------------------------------------------------------------------------- long rows of policy_gradient
# Roundings, u = 2^-24 each, of a row with d = (z - m) / T, M1 and M2 the means of |d| and d^2 under p, l = log V:
#   d takes z - m and the factor log2(e) / T, which is itself off by 2: 3 |d|, and one of the product with it: a term e^d is off
#   by 4 |d| + 2 (the hardware exponential is right to one unit in the last place, 2 u);
#   a sum in the kernels' order adds at most 152 (a thread's 128 values one by one, then 6 + 8 joins, or fewer values and
#   the joins of the online form), and means over p weigh the terms: log s is off by S = 4 M1 + 154 + 2 l, its logarithm included;
#   log p_t = d_t - log s adds 2 |d_t| and its own rounding |d_t| + l: 3 |d_t| + l + S;
#   p = 2^(d log2 e - log2 s) is off by 4 |d| + 3 l + 4 + S, and so is log p (which is no larger than |d| + l);
#   H = log s - sum(e d) / s: S + 4 M2 + 160 M1 + 2 l;
#   the slope of the loss by 16 of w (|A| r + kl (1 + e^x)) (exponentials 2 each after arguments right to a rounding of at
#   most 2, products and constants 1 each), the factors 1 / T, w and the sums 8.
def _check_long_rows(ops, dtype, v, entropy_coef, rows=12, seed=1, bounds=None, aggregate="sequence"):
    from test_policy_gpu import U, _definition, _plain
    g = torch.Generator(device=DEV).manual_seed(seed + v)
    logits = (3 * torch.randn(rows, v, device=DEV, generator=g)).to(dtype)
    targets = torch.randint(0, v, (rows,), device=DEV, generator=g)
    targets[0], targets[1], targets[5] = v - 1, 0, -1
    bounds = bounds or [0, 4, 4, rows - 1]                             # one row behind the last sequence
    mask = torch.ones(rows, dtype=torch.bool, device=DEV)
    mask[2] = False
    t = 0.9
    lp, h, d, logs, p, _ = _plain(logits, targets, t)
    normal = lambda: torch.randn(rows, device=DEV, generator=g)
    old, ref, adv = (lp + 0.2 * normal()).float(), (lp + 0.2 * normal()).float(), normal()
    cfg = ops.PolicyLossConfig(clip_low=0.2, clip_high=0.3, kl_coef=0.1, entropy_coef=entropy_coef, aggregate=aggregate)
    kw = dict(mask=mask, ref_logprobs=ref, cu_seqlens=torch.tensor(bounds, dtype=torch.int32, device=DEV), config=cfg, temperature=t)
    loss, stats, logprobs, grad = ops.policy_gradient(logits, targets, old, adv, **kw)
    live = mask & (targets >= 0)
    live[bounds[-1]:] = False
    assert int(live.sum()) == rows - 3 and stats[6].item() == rows - 3
    assert (logprobs[~live] == 0).all() and (grad[~live] == 0).all()

    l, m1, m2 = math.log(v), (p * d.abs()).sum(1), (p * d * d).sum(1)
    s = U * (4 * m1 + 154 + 2 * l)
    dt = d.gather(1, targets.clamp_min(0)[:, None])[:, 0].abs()
    assert ((logprobs.double() - lp).abs() <= U * (3 * dt + l) + s)[live].all()

    # the kernel's own log-probabilities in the definition
    cpu = lambda x: x.double().cpu()
    x, hh = cpu(logprobs).requires_grad_(), cpu(h).requires_grad_()
    want, want_stats = _definition(x, cpu(old), cpu(adv), live.cpu(), cpu(ref), hh if entropy_coef else None, bounds, cfg)
    slope, hslope = torch.autograd.grad(want, (x, hh), allow_unused=True)
    host = live.cpu()
    counts = [int(host[a:b].sum()) for a, b in zip(bounds[:-1], bounds[1:])]
    total, used = sum(counts), sum(c > 0 for c in counts)
    w = torch.zeros(rows, dtype=torch.float64)
    for a, b, c in zip(bounds[:-1], bounds[1:], counts):
        w[a:b] = {"sequence": 1.0 / (max(c, 1) * used), "token": 1.0 / total, "sum": 1.0}[aggregate]
    w = torch.where(live, w.to(DEV), 0.0)
    ratio, other = (logprobs.double() - old.double()).exp(), (ref.double() - logprobs.double()).exp()
    size = w * (adv.double().abs() * ratio + 0.1 * (1 + other))
    eh = s + U * (4 * m2 + 160 * m1 + 2 * l)
    slack = (16 * U * size).sum() + entropy_coef * (w * (eh + 3 * U * h)).sum() + U * want.abs().item()
    assert abs(loss.double().item() - want.item()) <= slack.item()

    gg, c = slope.to(DEV)[:, None], w[:, None] * entropy_coef
    hot = torch.zeros_like(p).scatter_(1, targets.clamp_min(0)[:, None], 1.0)
    logp = d - logs
    wanted = (gg * (hot - p) + c * p * (logp + h[:, None])) / t
    off = U * (4 * d.abs() + 3 * l + 4) + s[:, None]
    bound = gg.abs() * p * (off + 8 * U) + gg.abs() * hot * 8 * U + 16 * U * size[:, None] * (p + hot)
    bound = bound + c * p * ((logp + h[:, None]).abs() * (off + 8 * U) + off + eh[:, None] + U * (logp.abs() + h[:, None]))
    half, tiny = torch.finfo(dtype).eps / 2, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    bound = bound / t * (1 + 2.0 ** -7) + half * wanted.abs() * (1 + 2.0 ** -7) + tiny
    error = (grad.double() - wanted).abs()
    assert (error <= bound)[live].all(), (error / bound)[live].max()
    return logits, targets, old, adv, kw, grad


@pytest.mark.parametrize("entropy_coef", (0.0, 0.02))
@pytest.mark.parametrize("dtype, v", [(t, v) for t in (torch.bfloat16, torch.float16) for v in (8192, 8200, 32768, 65536, 65537, 65543, 65544, 131075)]
                         + [(torch.float32, v) for v in (4096, 4100, 16384, 32768, 32769, 32771, 32772, 65536, 131075)])
def test_policy_gradient_of_long_rows(ops, dtype, v, entropy_coef):
    _check_long_rows(ops, dtype, v, entropy_coef)


@pytest.mark.parametrize("dtype, v", ((torch.bfloat16, 8192), (torch.float16, 32768), (torch.bfloat16, 65536), (torch.bfloat16, 65537), (torch.bfloat16, 65544),
                                      (torch.float16, 131075), (torch.float32, 32769), (torch.float32, 65536)))
@pytest.mark.parametrize("entropy_coef", (0.0, 0.02))
def test_policy_gradient_of_long_rows_in_place_and_inside_a_wider_matrix(ops, dtype, v, entropy_coef):
    logits, targets, old, adv, kw, grad = _check_long_rows(ops, dtype, v, entropy_coef, seed=2)
    wide = torch.full((len(old), v + 9), 5.0, device=DEV, dtype=dtype)
    got = ops.policy_gradient(logits, targets, old, adv, out=wide[:, 3:v + 3], **kw)[3]
    assert torch.equal(got, grad) and (wide[:, :3] == 5).all() and (wide[:, v + 3:] == 5).all()
    wide.fill_(7.0)
    inside = wide[:, 1:v + 1]
    inside.copy_(logits)
    loss, stats, logprobs, _ = ops.policy_gradient(logits, targets, old, adv, **kw)
    again = ops.policy_gradient(inside, targets, old, adv, out=inside, **kw)
    assert torch.equal(inside, grad) and (wide[:, :1] == 7).all() and (wide[:, v + 1:] == 7).all()
    assert again[3] is inside
    for x, y in zip(again[:3], (loss, stats, logprobs)):
        assert torch.equal(x, y)


# --------------------------------------------------------------------------------------------- many sequences
def _random_bounds(n, sequences, end):
    g = torch.Generator().manual_seed(sequences)
    return [0, *torch.randint(0, end + 1, (sequences - 1,), generator=g).sort().values.tolist(), end]


@pytest.mark.parametrize("n, sequences", ((3000, 512), (3000, 513), (3000, 4097), (9000, 20000)))
@pytest.mark.parametrize("aggregate", ("token", "sequence", "sum"))
def test_policy_gradient_over_many_sequences(ops, n, sequences, aggregate):
    _check_long_rows(ops, torch.float32, 37, 0.02, rows=n, bounds=_random_bounds(n, sequences, n - 1), aggregate=aggregate)


@pytest.mark.parametrize("n, sequences", ((3000, 4097), (20000, 4096), (20000, 4097), (70001, 6000), (5000, 70000)))
@pytest.mark.parametrize("aggregate", ("token", "sequence", "sum"))
@pytest.mark.parametrize("masked, per_sequence", ((False, False), (True, True)))
def test_policy_loss_over_many_sequences(ops, n, sequences, aggregate, masked, per_sequence):
    from test_policy_gpu import U, _definition, _tokens
    lp, old, a, mask, _, _ = _tokens(n, sequences)
    bounds = _random_bounds(n, sequences, n - 7)
    which = torch.zeros(n, dtype=torch.long)
    for i, (s, e) in enumerate(zip(bounds[:-1], bounds[1:])):
        which[s:e] = i
    adv = torch.randn(sequences, generator=torch.Generator().manual_seed(n)) if per_sequence else a
    token_adv = adv[which] if per_sequence else adv
    cfg = ops.PolicyLossConfig(aggregate=aggregate)
    x = lp.double().requires_grad_()
    want, stats = _definition(x, old.double(), token_adv.double(), mask if masked else torch.ones(n, dtype=torch.bool), None, None, bounds, cfg)
    slope, = torch.autograd.grad(want, x)
    got = ops.policy_loss_forward(lp.to(DEV), old.to(DEV), adv.to(DEV), mask=mask.to(DEV) if masked else None, per_sequence=per_sequence, config=cfg,
                                  cu_seqlens=torch.tensor(bounds, dtype=torch.int32, device=DEV))
    # a token's slope: exponential |d| + 2 <= 10, products 2: 12 u; a loss of as many terms, none larger than r |A| w or 1.2 |A| w
    assert ((got[2].double().cpu() - slope).abs() <= 12 * U * slope.abs()).all() and (got[2][bounds[-1]:] == 0).all()
    counted = (mask if masked else torch.ones(n, dtype=torch.bool)).double()
    counted[bounds[-1]:] = 0
    w = {"sum": counted, "token": counted / counted.sum()}.get(aggregate)
    if w is None:
        per = torch.zeros(sequences, dtype=torch.float64).index_add_(0, which[:bounds[-1]], counted[:bounds[-1]])
        w = counted / (per.clamp_min(1)[which] * (per > 0).sum())
    size = (w * (lp.double() - old.double()).exp().clamp_min(1.2) * token_adv.double().abs()).sum()
    assert abs(got[0].double().cpu() - want.detach()) <= 12 * U * size + U * want.abs()
    assert got[1][6].item() == counted.sum()


def test_policy_loss_of_one_sequence_of_many_tokens(ops):
    """More blocks of counted tokens than a workgroup sweeps, without sequences: 2^24 + 2^13 tokens."""
    from test_policy_gpu import U
    n = (1 << 24) + (1 << 13) + 5
    g = torch.Generator(device=DEV).manual_seed(3)
    normal = lambda: torch.randn(n, device=DEV, generator=g)
    old, adv, mask = -normal().abs(), normal(), normal() > -0.5
    lp = old + 0.1 * normal()
    loss, stats, grad, _ = ops.policy_loss_forward(lp, old, adv, mask=mask, config=ops.PolicyLossConfig(clip_high=0.25, clip_low=0.25))
    ratio, a, w = (lp.double() - old.double()).exp(), adv.double(), mask.double() / mask.sum()
    gain = torch.minimum(ratio * a, ratio.clamp(0.75, 1.25) * a)
    want = -(w * gain).sum()
    assert stats[6].item() == mask.sum()
    assert abs(loss.double() - want) <= 12 * U * (w * gain.abs()).sum() + U * want.abs()
    slope = torch.where(ratio.clamp(0.75, 1.25) * a < ratio * a, 0.0, -w * ratio * a)
    assert ((grad.double() - slope).abs() <= 12 * U * slope.abs()).all()
