"""Loss and statistics of long batches, each against its own size: a bound that grows with the number of tokens only as the
sum of the terms' roundings does.

Per token, u = 2^-24: the log ratio is right to u (64-bit difference, rounded once), its exponential to |d| + 2, products with
advantage and clip constants 2 more: 12 u of |gain| for |d| < 8.  k1 takes 1, k2 3 and x its own, e^x - 1 - x up to 14
(expf's error against a value of 0.72 at x = 1): 16 u of kl.  A weight is right to u, the entropy is the input.  Sums are
64-bit; each result is rounded once."""
import pytest
import torch

from test_policy_gpu import BOUNDS, U, _definition, _tokens

DEV = "cuda"
VARIANTS = [dict(), dict(kl="k1", kl_coef=0.1), dict(kl="k2", kl_coef=0.1, dual_clip=1.5), dict(kl_coef=0.2, entropy_coef=0.05)]


def _case(n, aggregate, layout, number):
    """(arguments, config, loss and statistics in 64 bits, their bounds)"""
    from climbing_gym_amd import ops
    lp, old, a, mask, ref, h = _tokens(n, n + number)
    bounds = BOUNDS[layout](n) if layout else [0, n]
    cfg = ops.PolicyLossConfig(clip_low=0.2, clip_high=0.3, aggregate=aggregate, **VARIANTS[number])
    if number % 2 == 0:
        mask = None
    m = torch.ones(n, dtype=torch.bool) if mask is None else mask
    ref, h = ref if cfg.kl_coef else None, h if cfg.entropy_coef else None
    wide = lambda t: None if t is None else t.double()
    want, stats = _definition(wide(lp), wide(old), wide(a), m, wide(ref), wide(h), bounds, cfg)
    # the same sums of the terms' sizes
    live = m & (torch.arange(n) < bounds[-1])
    d = lp.double() - old.double()
    r, adv = d.exp(), a.double()
    assert d.abs().max() < 8
    size = torch.maximum((r * adv).abs(), r.clamp(1 - cfg.clip_low, 1 + cfg.clip_high) * adv.abs())   # at least |gain|
    if cfg.dual_clip:
        size = torch.maximum(size, cfg.dual_clip * adv.abs())
    kl = torch.zeros(n, dtype=torch.float64)
    if ref is not None:
        x = ref.double() - lp.double()
        kl = {"k1": x.abs(), "k2": x * x / 2, "k3": torch.expm1(x) - x}[cfg.kl]
    entropy = torch.zeros(n, dtype=torch.float64) if h is None else h.double()
    if aggregate == "sum":
        w = live.double()
    elif aggregate == "token":
        w = live.double() / live.sum().clamp_min(1)
    else:
        w = torch.zeros(n, dtype=torch.float64)
        counts = [int(live[s:e].sum()) for s, e in zip(bounds[:-1], bounds[1:])]
        for (s, e), c in zip(zip(bounds[:-1], bounds[1:]), counts):
            if c:
                w[s:e] = live[s:e].double() / (c * sum(k > 0 for k in counts))
    count = live.sum().clamp_min(1)
    # tokens so near a border that the fp32 clip constants may put them on its other side change the share, not the gain
    borders = torch.tensor([1 - cfg.clip_low, 1 + cfg.clip_high, cfg.dual_clip or 1 + cfg.clip_high], dtype=torch.float64).log()
    near = (live[:, None] & ((d[:, None] - borders).abs() < 1e-7)).any(1).sum()
    off = [12 * U * (w * size).sum(), 16 * U * (w * kl).sum(), 2 * U * (w * entropy).sum(), near / count,
           12 * U * (live * r).sum() / count, 16 * U * (live * (torch.expm1(d) - d)).sum() / count, torch.zeros(())]
    off = torch.stack([x.double() for x in off])
    loss_off = off[0] + cfg.kl_coef * (off[1] + U * stats[1].abs()) + cfg.entropy_coef * (off[2] + U * stats[2].abs())
    return (lp, old, a, mask, ref, h, bounds if layout else None), cfg, want, stats, loss_off + U * want.abs(), off + U * stats.abs()


CASES = [(n, aggregate, layout, number) for n in (1000, 4096, 4097, 70001) for aggregate in ("token", "sequence", "sum")
         for layout in (None, "empty ones", "padded tail") for number in range(4)]


@pytest.mark.gpu
@pytest.mark.parametrize("n, aggregate, layout, number", CASES)
def test_loss_and_statistics(n, aggregate, layout, number):
    from climbing_gym_amd import ops
    (lp, old, a, mask, ref, h, bounds), cfg, want, stats, loss_off, off = _case(n, aggregate, layout, number)
    dev = lambda t: None if t is None else t.to(DEV)
    got = ops.policy_loss_forward(dev(lp), dev(old), dev(a), mask=dev(mask), ref_logprobs=dev(ref), entropy=dev(h), config=cfg,
                                  cu_seqlens=None if bounds is None else torch.tensor(bounds, dtype=torch.int32, device=DEV))
    assert abs(got[0].double().cpu() - want) <= loss_off, (got[0].item(), want.item(), loss_off.item())
    error = (got[1].double().cpu() - stats).abs()
    assert (error <= off).all(), (error / off, error)


@pytest.mark.parametrize("n, aggregate, layout, number", [c for c in CASES if c[0] != 1000])
def test_the_bounds_notice_a_missing_workgroup(n, aggregate, layout, number):
    """The definition without the last 1024 tokens is outside of them, in the loss and in every statistic that sums."""
    (lp, old, a, mask, ref, h, bounds), cfg, want, stats, loss_off, off = _case(n, aggregate, layout, number)
    wide = lambda t: None if t is None else t.double()
    m = torch.ones(n, dtype=torch.bool) if mask is None else mask.clone()
    last = bounds[-1] if bounds else n
    m[last - 1024:last] = False
    other, other_stats = _definition(wide(lp), wide(old), wide(a), m, wide(ref), wide(h), bounds or [0, n], cfg)
    assert abs(other - want) > loss_off
    assert ((other_stats - stats).abs() > off)[[0, 3, 4, 5, 6]].all()
