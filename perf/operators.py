"""Operators of a grouped rollout and of the policy step that follows it, as workloads: what each call takes, a plain
torch form of it, the same call on this package's kernels, the work it cannot do without, and its value in 64 bits.

  attend_shared     one decode step's attention for rows in groups that share the first part of their history
  token_logprobs    log-probabilities (and entropies) of given tokens from the logits, and the gradient
  policy_loss       clipped policy loss with a KL term over packed sequences, with its gradient
  policy_gradient   the same loss straight from the logits, with the gradient of the logits
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
E4M3_MAX = 448.0


# ------------------------------------------------------------------------------------------------ cases
def _attention(name, **kw):
    base = dict(name=name, op="attend_shared", groups=16, rows=16, even=True, prefix_low=256, prefix_high=2048, own_low=1,
                own_high=1024, query_heads=32, kv_heads=8, head_dim=64, dtype="bf16", history="same", page=0, layers=1,
                finished=0.0, lengths=1)
    return {**base, **kw}


def _logprobs(name, **kw):
    base = dict(name=name, op="token_logprobs", rows=1024, vocab=65536, dtype="bf16", temperature=1.0, per_row=False,
                entropy=False, backward=False, pad=0, ignored=0.0)
    return {**base, **kw}


def _loss(name, **kw):
    base = dict(name=name, op="policy_loss", sequences=64, low=64, high=1024, aggregate="token", kl="k3", kl_coef=0.05,
                clip_low=0.2, clip_high=0.28, dual_clip=0.0, entropy_coef=0.0, per_sequence=True, masked=0.1, lengths=1)
    return {**base, **kw}


def _gradient(name, **kw):
    base = dict(name=name, op="policy_gradient", sequences=8, low=64, high=512, vocab=65536, dtype="bf16", temperature=1.0,
                aggregate="token", kl="k3", kl_coef=0.05, clip_low=0.2, clip_high=0.28, dual_clip=0.0, entropy_coef=0.0,
                masked=0.3, pad=0, lengths=1)
    return {**base, **kw}


def listed():
    return [
        # the first steps of one prompt's eight rollouts: few rows, nothing generated yet, latency counts
        _attention("shared-1x8-start", groups=1, rows=8, prefix_low=1024, prefix_high=1024, own_low=1, own_high=16, lengths=11),
        # the 256-row decode batch of the engine as 16 prompts with 16 rollouts each, e4m3 history, mid-job, all six
        # attention layers of a step
        _attention("shared-16x16-e4m3", own_high=900, history="e4m3", layers=6, lengths=12),
        # a paged model-dtype history with wide heads and a ragged batch: groups of 1 to 13 rows, some rows finished
        _attention("shared-paged-ragged", groups=7, rows=13, even=False, prefix_low=33, prefix_high=1777, own_low=1,
                   own_high=601, query_heads=24, kv_heads=4, head_dim=128, page=16, finished=0.15, lengths=13),
        # long shared prompts, 512 rows: the largest decode batch of the engine's benchmark
        _attention("shared-32x16-long", groups=32, rows=16, history="e4m3", prefix_low=4096, prefix_high=7000, own_high=512,
                   lengths=14),
        # scoring the first step of a handful of completions: a few rows, the temperature of each row its own
        _logprobs("score-few", rows=8, per_row=True),
        # scoring a prefill chunk of completions with entropies
        _logprobs("score-chunk", rows=4096, entropy=True, ignored=0.1),
        # a trainer's fp32 logits, odd vocabulary, rows inside a wider padded matrix, forward and backward
        _logprobs("train-odd-f32", rows=777, vocab=32003, dtype="f32", temperature=0.8, entropy=True, backward=True, pad=29,
                  ignored=0.25),
        # forward and backward over a chunk of the model's own logits
        _logprobs("train-chunk", rows=4096, backward=True, ignored=0.1),
        # the loss of one small group of completions: latency counts
        _loss("loss-group", sequences=8, low=16, high=256, lengths=15),
        # the loss of a whole rollout batch: 256 completions of up to 4096 tokens, means per sequence
        _loss("loss-batch", sequences=256, low=256, high=4096, aggregate="sequence", dual_clip=3.0, entropy_coef=0.01,
              per_sequence=False, lengths=16),
        # a small policy step in fp16 on a small vocabulary
        _gradient("step-small-f16", sequences=4, low=5, high=61, vocab=4096, dtype="f16", entropy_coef=0.01, lengths=17),
        # a policy step over a micro-batch of completions with the model's vocabulary
        _gradient("step-chunk", sequences=16, low=256, high=768, temperature=0.9, aggregate="sequence", lengths=18),
    ]


def _between(rng, low, high):
    """A whole number from low to high, spread over the logarithm where the range spans more than a factor of ten."""
    if high <= 10 * low:
        return rng.randint(low, high)
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(("attend_shared", "attend_shared", "token_logprobs", "policy_loss", "policy_gradient"))
    seed = rng.randint(1, 1 << 30)
    if kind == "attend_shared":
        kv_heads = rng.choice((1, 2, 4, 8))
        groups, rows = _between(rng, 1, 32), _between(rng, 1, 16)
        low = _between(rng, 16, 3000)
        case = _attention(None, groups=groups, rows=rows, even=rng.random() < 0.5, prefix_low=low,
                          prefix_high=_between(rng, low, 4000), own_high=_between(rng, 1, 500), kv_heads=kv_heads,
                          query_heads=kv_heads * rng.choice((1, 3, 4, 8)), head_dim=rng.choice((64, 64, 128, 32)),
                          dtype=rng.choice(("bf16", "bf16", "f16")), history=rng.choice(("same", "e4m3")),
                          page=rng.choice((0, 0, 16, 48)), layers=rng.choice((1, 2)), finished=rng.choice((0.0, 0.2)), lengths=seed)
    elif kind == "token_logprobs":
        vocab = _between(rng, 300, 65536)
        dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
        case = _logprobs(None, rows=_between(rng, 1, 2048), vocab=vocab, dtype=dtype, temperature=rng.choice((1.0, 0.7, 1.3)),
                         per_row=rng.random() < 0.3, entropy=rng.random() < 0.5, backward=rng.random() < 0.6,
                         pad=rng.choice((0, 0, 5, 64)), ignored=rng.choice((0.0, 0.2)))
    elif kind == "policy_loss":
        low = _between(rng, 1, 512)
        case = _loss(None, sequences=_between(rng, 1, 256), low=low, high=_between(rng, low, 4000),
                     aggregate=rng.choice(("token", "sequence", "sum")), kl=rng.choice(("k1", "k2", "k3")),
                     kl_coef=rng.choice((0.0, 0.1)), dual_clip=rng.choice((0.0, 3.0)), entropy_coef=rng.choice((0.0, 0.01)),
                     per_sequence=rng.random() < 0.5, masked=rng.choice((0.0, 0.3)), lengths=seed)
    else:
        low = _between(rng, 1, 64)
        case = _gradient(None, sequences=_between(rng, 1, 12), low=low, high=_between(rng, low, 512),
                         vocab=_between(rng, 300, 65536), dtype=rng.choice(("bf16", "bf16", "f16", "f32")),
                         temperature=rng.choice((1.0, 0.8)), aggregate=rng.choice(("token", "sequence", "sum")),
                         kl=rng.choice(("k1", "k2", "k3")), kl_coef=rng.choice((0.0, 0.1)), dual_clip=rng.choice((0.0, 3.0)),
                         entropy_coef=rng.choice((0.0, 0.01)), masked=rng.choice((0.0, 0.4)), pad=rng.choice((0, 0, 3)),
                         lengths=seed)
    case.pop("name")
    return case


# ------------------------------------------------------------------------------------------------ lengths of a case
def _groups(case):
    """(first row of every group and the row count, prefix lengths, own lengths per row, activity per row)"""
    rng = random.Random(case["lengths"])
    starts, prefix, own_tokens, active = [0], [], [], []
    for _ in range(case["groups"]):
        count = case["rows"] if case["even"] else rng.randint(1, case["rows"])
        starts.append(starts[-1] + count)
        prefix.append(rng.randint(case["prefix_low"], case["prefix_high"]))
        for _ in range(count):
            own_tokens.append(rng.randint(case["own_low"], case["own_high"]))
            active.append(rng.random() >= case["finished"])
    return starts, prefix, own_tokens, active


def _packed(case):
    rng = random.Random(case["lengths"])
    lengths = [_between(rng, case["low"], case["high"]) for _ in range(case["sequences"])]
    bounds = [0]
    for n in lengths:
        bounds.append(bounds[-1] + n)
    return bounds


# ------------------------------------------------------------------------------------------------ inputs
def _e4m3_rows(x):
    """Rows of the last dimension as (e4m3 codes, fp32 scale): the storage of the engine's e4m3 history."""
    scale = (x.float().abs().amax(-1) / E4M3_MAX).clamp_min(1e-12)
    return (x.float() / scale[..., None]).to(torch.float8_e4m3fn), scale


def _history(case, gen, pools, positions):
    """One tensor of keys or values, [slots or pages, positions, KV heads, dim], and its scales or None."""
    heads, dim, dtype = case["kv_heads"], case["head_dim"], DTYPES[case["dtype"]]
    paged = case["page"] > 0
    shape = (pools, positions, heads, dim) if paged else (pools, heads, positions, dim)   # dense: head-major storage
    e4m3 = case["history"] == "e4m3"
    out = torch.empty(shape, device="cuda", dtype=torch.float8_e4m3fn if e4m3 else dtype)
    scales = torch.empty(shape[:-1], device="cuda", dtype=torch.float32) if e4m3 else None
    step = max(1, (1 << 26) // max(1, positions * heads * dim))
    for a in range(0, pools, step):
        b = min(pools, a + step)
        x = torch.randn((b - a, *shape[1:]), device="cuda", generator=gen).to(dtype)
        if e4m3:
            codes, s = _e4m3_rows(x)
            out[a:b].view(torch.uint8).copy_(codes.view(torch.uint8))
            scales[a:b] = s
        else:
            out[a:b] = x
    if paged:
        return out, scales
    return out.permute(0, 2, 1, 3), None if scales is None else scales.permute(0, 2, 1)


def _prepare_attention(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    starts, prefix, own_tokens, active = _groups(case)
    rows = starts[-1]
    total = [prefix[g] + own_tokens[b] for g in range(case["groups"]) for b in range(starts[g], starts[g + 1])]
    table = None
    if case["page"]:
        page = case["page"]
        blocks = -(-max(total) // page)
        entries, used = [[0] * blocks for _ in range(rows)], 0
        for g in range(case["groups"]):
            whole = prefix[g] // page             # pages that hold prefix positions only are the group's
            for b in range(starts[g], starts[g + 1]):
                for i in range(-(-total[b] // page)):
                    if i < whole and b > starts[g]:
                        entries[b][i] = entries[starts[g]][i]
                    else:
                        entries[b][i] = used
                        used += 1
        order = list(range(used))
        random.Random(seed).shuffle(order)
        table = torch.tensor([[order[e] for e in row] for row in entries], dtype=torch.int32).cuda()
        pools, positions = used, page
    else:
        pools, positions = rows, -(-max(total) // 64) * 64
    layers = []
    for _ in range(case["layers"]):
        k, ks = _history(case, gen, pools, positions)
        v, vs = _history(case, gen, pools, positions)
        q = (2.0 * torch.randn((rows, 1, case["query_heads"], case["head_dim"]), device="cuda", generator=gen)).to(DTYPES[case["dtype"]])
        layers.append((q, k, v, ks, vs))
    ints = lambda x: torch.tensor(x, dtype=torch.int32).cuda()
    state = dict(case=case, layers=layers, table=table, positions=ints([n - 1 for n in total]),
                 active=torch.tensor(active).cuda() if case["finished"] else None, starts=ints(starts),
                 leaders=ints(starts[:-1]), prefix=ints(prefix), host=(starts, prefix, total, active))
    return state


def _logits(case, gen, rows):
    """Logits as a trained model makes them: a broad background and a few likely tokens; rows may be part of a wider,
    padded matrix."""
    wide = torch.randn((rows, case["vocab"] + case["pad"]), device="cuda", generator=gen)
    wide.mul_(2.0)
    likely = torch.randint(0, case["vocab"], (rows, 4), device="cuda", generator=gen)
    wide.scatter_add_(1, likely, 6.0 + 3.0 * torch.rand((rows, 4), device="cuda", generator=gen))
    logits = wide.to(DTYPES[case["dtype"]])[:, :case["vocab"]]
    pick = torch.randint(0, 5, (rows, 1), device="cuda", generator=gen)
    other = torch.randint(0, case["vocab"], (rows, 1), device="cuda", generator=gen)
    return logits, torch.where(pick < 4, likely.gather(1, pick.clamp_max(3)), other)[:, 0].contiguous()


def _prepare_logprobs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rows = case["rows"]
    logits, targets = _logits(case, gen, rows)
    uniform = lambda: torch.rand(rows, device="cuda", generator=gen)
    if case["ignored"]:
        targets = torch.where(uniform() < case["ignored"], torch.full_like(targets, -100), targets)
    temperature = 0.5 + uniform() if case["per_row"] else case["temperature"]
    state = dict(case=case, logits=logits, targets=targets, temperature=temperature)
    if case["backward"]:
        state["grad_logprobs"] = (uniform() - 0.5) / rows
        state["grad_entropy"] = uniform() / rows if case["entropy"] else None
    return state


def _prepare_loss(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    bounds = _packed(case)
    tokens, sequences = bounds[-1], case["sequences"]
    normal = lambda n: torch.randn(n, device="cuda", generator=gen)
    uniform = lambda n: torch.rand(n, device="cuda", generator=gen)
    old = -2.0 * uniform(tokens) ** 2 - 1e-3
    state = dict(case=case, cu=torch.tensor(bounds, dtype=torch.int32).cuda(), bounds=bounds, old=old,
                 logprobs=old + 0.15 * normal(tokens),
                 ref=old + 0.2 * normal(tokens) if case["kl_coef"] else None,
                 advantages=0.3 + normal(sequences if case["per_sequence"] else tokens),
                 mask=(uniform(tokens) >= case["masked"]) if case["masked"] else None,
                 entropy=0.2 + uniform(tokens) if case["entropy_coef"] else None)
    return state


def _prepare_gradient(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    bounds = _packed(case)
    tokens = bounds[-1]
    logits, targets = _logits(case, gen, tokens)
    normal = lambda n: torch.randn(n, device="cuda", generator=gen)
    now = torch.empty(tokens, device="cuda")
    for a in range(0, tokens, 512):   # what the tokens' log-probabilities are, for behaviour and reference policies nearby
        z = logits[a:a + 512].float() / case["temperature"]
        now[a:a + 512] = z.gather(1, targets[a:a + 512, None])[:, 0] - z.logsumexp(1)
    state = dict(case=case, logits=logits, targets=targets, cu=torch.tensor(bounds, dtype=torch.int32).cuda(), bounds=bounds,
                 old=now + 0.15 * normal(tokens), ref=now + 0.2 * normal(tokens) if case["kl_coef"] else None,
                 advantages=0.3 + normal(case["sequences"]),
                 mask=(torch.rand(tokens, device="cuda", generator=gen) >= case["masked"]) if case["masked"] else None)
    return state


PREPARE = {"attend_shared": _prepare_attention, "token_logprobs": _prepare_logprobs, "policy_loss": _prepare_loss,
           "policy_gradient": _prepare_gradient}


def prepare(case, seed):
    return PREPARE[case["op"]](case, seed)


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    op = state["case"]["op"]
    return (OWN if own else PLAIN)[op](state)


def _config(case):
    from climbing_gym_amd import ops
    return ops.PolicyLossConfig(clip_low=case["clip_low"], clip_high=case["clip_high"], dual_clip=case["dual_clip"] or None,
                                kl=case["kl"], kl_coef=case["kl_coef"], entropy_coef=case["entropy_coef"],
                                aggregate=case["aggregate"])


def _own_attention(state):
    """One decode step's calls: the work list once, then the attention of every layer."""
    from climbing_gym_amd import ops
    case = state["case"]
    prefix = ops.SharedPrefix(state["starts"], state["leaders"], state["prefix"])
    q, k = state["layers"][0][:2]
    capacity = state["table"].size(1) * case["page"] if case["page"] else k.size(1)
    schedule = ops.shared_schedule(state["positions"], prefix, state["active"], capacity=capacity,
                                   query_heads=case["query_heads"], kv_heads=case["kv_heads"], head_dim=case["head_dim"])
    return [ops.attend_shared(q, k, v, ks, vs, state["positions"], prefix, active=state["active"], block_table=state["table"],
                              page=case["page"] or 16, schedule=schedule) for q, k, v, ks, vs in state["layers"]]


def _own_logprobs(state):
    from climbing_gym_amd import ops
    case = state["case"]
    logprobs, entropy, stats = ops.token_logprobs_forward(state["logits"], state["targets"], temperature=state["temperature"],
                                                          entropy=case["entropy"])
    out = [logprobs] + ([entropy] if case["entropy"] else [])
    if case["backward"]:
        out.append(ops.token_logprobs_backward(state["logits"], state["targets"], stats, state["grad_logprobs"],
                                               state["grad_entropy"], temperature=state["temperature"]))
    return out


def _own_loss(state):
    from climbing_gym_amd import ops
    loss, stats, grad_logprobs, grad_entropy = ops.policy_loss_forward(
        state["logprobs"], state["old"], state["advantages"], mask=state["mask"], ref_logprobs=state["ref"],
        entropy=state["entropy"], cu_seqlens=state["cu"], per_sequence=state["case"]["per_sequence"], config=_config(state["case"]))
    return [loss, stats, grad_logprobs] + ([grad_entropy] if state["entropy"] is not None else [])


def _own_gradient(state):
    from climbing_gym_amd import ops
    loss, stats, logprobs, grad_logits = ops.policy_gradient(
        state["logits"], state["targets"], state["old"], state["advantages"], mask=state["mask"], ref_logprobs=state["ref"],
        cu_seqlens=state["cu"], per_sequence=True, temperature=state["case"]["temperature"], config=_config(state["case"]))
    return [loss, stats, logprobs, grad_logits]


OWN = {"attend_shared": _own_attention, "token_logprobs": _own_logprobs, "policy_loss": _own_loss, "policy_gradient": _own_gradient}


def _gather_history(cache, scales, table, rows, positions, page):
    """History of cache slots, or block-table rows, `rows` [n] at `positions` [n, m], in fp32: [n, m, KV heads, dim]."""
    pools, inside = rows[:, None].expand_as(positions), positions
    if table is not None:
        pools, inside = table[pools, positions // page].long(), positions % page
    raw = cache.view(torch.uint8) if cache.element_size() == 1 else cache
    x = raw[pools, inside].view(cache.dtype).float()
    return x if scales is None else x * scales[pools, inside, :, None]


def _plain_attention(state):
    """Group by group: scores of all rows against the shared positions in one product, scores of every row against its
    own (padded to the longest of the group), one softmax over both."""
    case = state["case"]
    starts, prefix, total, active = state["host"]
    kv, dim = case["kv_heads"], case["head_dim"]
    per = case["query_heads"] // kv
    outputs = []
    for q, k, v, ks, vs in state["layers"]:
        out = torch.zeros_like(q)
        for g in range(case["groups"]):
            live = [b for b in range(starts[g], starts[g + 1]) if active[b]]
            if not live:
                continue
            n, shared, longest = len(live), prefix[g], max(total[b] for b in live) - prefix[g]
            rows = torch.tensor(live, device=q.device)
            leader = rows.new_tensor([starts[g]])
            own_positions = (shared + torch.arange(longest, device=q.device)).expand(n, longest)
            lengths = state["positions"][rows] + 1
            hidden = own_positions >= lengths[:, None]
            own_positions = torch.minimum(own_positions, lengths[:, None] - 1)
            first = torch.arange(shared, device=q.device)[None]
            k0, v0 = [_gather_history(c, s, state["table"], leader, first, case["page"])[0].permute(1, 0, 2).contiguous()
                      for c, s in ((k, ks), (v, vs))]                                      # [KV heads, shared, dim]
            k1, v1 = [_gather_history(c, s, state["table"], rows, own_positions, case["page"]).permute(0, 2, 1, 3).contiguous()
                      for c, s in ((k, ks), (v, vs))]                                      # [rows, KV heads, own, dim]
            queries = q[rows, 0].float().view(n, kv, per, dim) * dim ** -0.5
            flat = queries.permute(1, 0, 2, 3).reshape(kv, n * per, dim)
            together = torch.matmul(flat, k0.transpose(1, 2).contiguous()).view(kv, n, per, shared).permute(1, 0, 2, 3)
            alone = torch.matmul(queries, k1.transpose(2, 3).contiguous())
            alone = alone.masked_fill(hidden[:, None, None, :], float("-inf"))
            scores = torch.cat((together, alone), -1)
            weights = torch.exp(scores - scores.amax(-1, keepdim=True))
            weights = weights / weights.sum(-1, keepdim=True)
            value = torch.matmul(weights[..., :shared].permute(1, 0, 2, 3).reshape(kv, n * per, shared), v0)
            value = value.view(kv, n, per, dim).permute(1, 0, 2, 3) + torch.matmul(weights[..., shared:].contiguous(), v1)
            out[rows, 0] = value.reshape(n, kv * per, dim).to(q.dtype)
        outputs.append(out)
    return outputs


def _temperature_column(temperature):
    return temperature[:, None] if isinstance(temperature, torch.Tensor) else temperature


def _plain_logprobs(state):
    case, targets = state["case"], state["targets"]
    t = _temperature_column(state["temperature"])
    z = state["logits"].float() / t
    z = z - z.amax(1, keepdim=True)
    e = torch.exp(z)
    s = e.sum(1, keepdim=True)
    live = targets >= 0
    index = targets.clamp_min(0)[:, None]
    logprobs = torch.where(live, (z.gather(1, index) - torch.log(s))[:, 0], 0.0)
    out = [logprobs]
    if case["entropy"]:
        entropy = torch.log(s) - (e * z).sum(1, keepdim=True) / s
        out.append(torch.where(live, entropy[:, 0], 0.0))
    if case["backward"]:
        p = e / s
        g = torch.where(live, state["grad_logprobs"], 0.0)[:, None]
        grad = -g * p
        grad.scatter_add_(1, index, g)
        if state["grad_entropy"] is not None:
            h = torch.where(live, state["grad_entropy"], 0.0)[:, None]
            grad = grad - h * p * (z - torch.log(s) + entropy)
        out.append((grad / t).to(state["logits"].dtype))
    return out


def _plain_weights(case, live, bounds, sequence):
    """Weight of every token: its share of the mean the loss takes (64 bits: the counts divide long sums)."""
    if case["aggregate"] == "sum":
        return live.double()
    if case["aggregate"] == "token":
        return live.double() / live.sum().clamp_min(1)
    counts = torch.zeros(len(bounds) - 1, device=live.device, dtype=torch.float64).index_add_(0, sequence, live.double())
    return live.double() / (counts.clamp_min(1)[sequence] * (counts > 0).sum().clamp_min(1))


def _plain_objective(case, state, logprobs, live, advantages, entropy):
    """(loss, statistics, d loss / d logprobs, d loss / d entropy); 64 bits, since a ratio next to the clip border is cut
    or not by its last bits and the loss is a long sum of terms of both signs."""
    bounds = state["bounds"]
    device = logprobs.device
    sequence = torch.repeat_interleave(torch.arange(len(bounds) - 1, device=device), state["cu"].long().diff(),
                                       output_size=bounds[-1])
    w = _plain_weights(case, live, bounds, sequence)
    zero = torch.zeros((), device=device, dtype=torch.float64)
    delta = torch.where(live, logprobs.double() - state["old"].double(), zero)
    a = advantages.double()
    a = torch.where(live, a[sequence] if case.get("per_sequence", True) else a, zero)
    ratio = torch.exp(delta)
    cut = ((a > 0) & (delta > math.log1p(case["clip_high"]))) | ((a < 0) & (delta < math.log1p(-case["clip_low"])))
    limit = torch.where(a > 0, 1.0 + case["clip_high"], 1.0 - case["clip_low"]).double()
    gain = torch.where(cut, limit, ratio) * a
    if case["dual_clip"]:
        floor = (a < 0) & (delta > math.log(case["dual_clip"]))
        gain = torch.where(floor, case["dual_clip"] * a, gain)
        cut = cut | floor
    grad = torch.where(cut, zero, -ratio * a)
    kl = torch.zeros_like(delta)
    if state["ref"] is not None:
        x = torch.where(live, state["ref"].double() - logprobs.double(), zero)
        kl = {"k1": -x, "k2": 0.5 * x * x, "k3": torch.expm1(x) - x}[case["kl"]]
        slope = {"k1": torch.ones_like(x), "k2": -x, "k3": -torch.expm1(x)}[case["kl"]]
        grad = grad + case["kl_coef"] * slope
    h = torch.where(live, entropy.double(), zero) if entropy is not None else torch.zeros_like(delta)
    count = live.sum().double()
    share = live.double() / count.clamp_min(1)
    policy, kl_mean, entropy_mean = -(w * gain).sum(), (w * kl).sum(), (w * h).sum()
    loss = policy + case["kl_coef"] * kl_mean - case["entropy_coef"] * entropy_mean
    stats = torch.stack((policy, kl_mean, entropy_mean, (share * (cut & live)).sum(), (share * ratio).sum(),
                         (share * (torch.expm1(delta) - delta)).sum(), count))
    return loss, stats, w * grad, -case["entropy_coef"] * w


def _plain_loss(state):
    case = state["case"]
    live = state["mask"] if state["mask"] is not None else torch.ones_like(state["logprobs"], dtype=torch.bool)
    loss, stats, grad, grad_entropy = _plain_objective(case, state, state["logprobs"], live, state["advantages"], state["entropy"])
    return [loss.float(), stats.float(), grad.float()] + ([grad_entropy.float()] if state["entropy"] is not None else [])


def _plain_gradient(state):
    case, targets = state["case"], state["targets"]
    live = targets >= 0
    if state["mask"] is not None:
        live = live & state["mask"]
    z = state["logits"].float() / case["temperature"]
    z = z - z.amax(1, keepdim=True)
    e = torch.exp(z)
    s = e.sum(1, keepdim=True)
    log_s = torch.log(s)
    index = targets.clamp_min(0)[:, None]
    logprobs = torch.where(live, (z.gather(1, index) - log_s)[:, 0], 0.0)
    entropy = (log_s - (e * z).sum(1, keepdim=True) / s) if case["entropy_coef"] else None
    loss, stats, grad, grad_entropy = _plain_objective(case, state, logprobs, live, state["advantages"],
                                                       None if entropy is None else entropy[:, 0])
    p = e / s
    g = grad.float()[:, None]
    out = -g * p
    out.scatter_add_(1, index, g)
    if entropy is not None:
        out = out - grad_entropy.float()[:, None] * p * (z - log_s + entropy)
    return [loss.float(), stats.float(), logprobs, (out / case["temperature"]).to(state["logits"].dtype)]


PLAIN = {"attend_shared": _plain_attention, "token_logprobs": _plain_logprobs, "policy_loss": _plain_loss,
         "policy_gradient": _plain_gradient}


# ------------------------------------------------------------------------------------------------ work of one pass
def work(case):
    if case["op"] == "attend_shared":
        starts, prefix, own_tokens, active = _groups(case)
        element = 1 if case["history"] == "e4m3" else 2
        token = 2 * case["kv_heads"] * (case["head_dim"] * element + (4 if case["history"] == "e4m3" else 0))
        tokens = pairs = 0
        for g in range(case["groups"]):
            live = [b for b in range(starts[g], starts[g + 1]) if active[b]]
            tokens += (prefix[g] if live else 0) + sum(own_tokens[b] for b in live)
            pairs += sum(prefix[g] + own_tokens[b] for b in live)
        rows = 2 * 2 * starts[-1] * case["query_heads"] * case["head_dim"]     # queries in, outputs out
        return {"bytes": case["layers"] * (tokens * token + rows),
                "flops": case["layers"] * 4 * case["query_heads"] * case["head_dim"] * pairs}
    if case["op"] == "policy_loss":
        n = _packed(case)[-1]
        per_token = 4 * (3 + (case["kl_coef"] > 0) + (case["entropy_coef"] > 0) * 2 + (not case["per_sequence"])) + (case["masked"] > 0)
        return {"bytes": n * per_token, "flops": 40 * n}
    element = {"bf16": 2, "f16": 2, "f32": 4}[case["dtype"]]
    if case["op"] == "token_logprobs":
        live = round(case["rows"] * (1 - case["ignored"]))
        values = live * case["vocab"]
        moved = values * element + 16 * case["rows"]
        if case["backward"]:   # the gradient needs the sums of the whole row: the logits once more, the gradient out
            moved += values * element + case["rows"] * case["vocab"] * element
        return {"bytes": moved, "flops": values * (4 + 4 * case["backward"] + 2 * case["entropy"])}
    n = _packed(case)[-1]
    live = round(n * (1 - case["masked"]))
    return {"bytes": (live + n) * case["vocab"] * element + 24 * n, "flops": 8 * live * case["vocab"]}


# ------------------------------------------------------------------------------------------------ values in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    return EXACT[case["op"]](state)


def _exact_attention(state):
    """Row by row from the definition: the row's whole history put together, softmax, weighted sum."""
    case = state["case"]
    starts, prefix, total, active = state["host"]
    group_of = [g for g in range(case["groups"]) for _ in range(starts[g], starts[g + 1])]
    kv, dim, page, table = case["kv_heads"], case["head_dim"], case["page"], state["table"]
    outputs = []
    for q, k, v, ks, vs in state["layers"]:
        def positions_of(cache, scales, row, a, b):
            if table is None:
                x = cache[row, a:b].to(torch.float64)
                return x if scales is None else x * scales[row, a:b].double().unsqueeze(-1)
            parts = []
            where = torch.arange(a, b, device="cuda")
            flat = cache.reshape(-1, kv, dim) if cache.element_size() > 1 else cache.view(torch.uint8).reshape(-1, kv, dim)
            at = table[row].long()[where // page] * page + where % page
            x = flat.index_select(0, at).view(cache.dtype).to(torch.float64)
            parts.append(x if scales is None else x * scales.reshape(-1, kv).index_select(0, at).double().unsqueeze(-1))
            return parts[0]

        result = torch.zeros(q.shape, device="cuda", dtype=torch.float64)
        shared = {}
        for b, n in enumerate(total):
            if not active[b]:
                continue
            g = group_of[b]
            if g not in shared:
                shared = {g: [positions_of(c, s, starts[g], 0, prefix[g]) for c, s in ((k, ks), (v, vs))]}
            keys, values = [torch.cat((head, positions_of(c, s, b, prefix[g], n))) for head, (c, s) in zip(shared[g], ((k, ks), (v, vs)))]
            queries = q[b, 0].double().reshape(kv, -1, dim)
            scores = torch.bmm(queries, keys.permute(1, 2, 0).contiguous()) / math.sqrt(dim)
            result[b, 0] = torch.bmm(torch.softmax(scores, -1), values.permute(1, 0, 2).contiguous()).reshape(-1, dim)
        outputs.append(result)
    return outputs


def _exact_rows(state, temperature, want_entropy, coefficients):
    """Log-probabilities, entropies and logit gradients in 64 bits, some rows at a time; `coefficients(logprobs, entropy)`
    gives d loss / d logprobs and d loss / d entropy (or None) once all rows' values are known."""
    logits, targets = state["logits"], state["targets"]
    n, vocab = logits.shape
    step = max(1, (1 << 27) // vocab)
    t = temperature.double() if isinstance(temperature, torch.Tensor) else torch.full((n,), float(temperature), device="cuda", dtype=torch.float64)
    live = targets >= 0
    logprobs, entropy = torch.zeros(n, device="cuda", dtype=torch.float64), torch.zeros(n, device="cuda", dtype=torch.float64)
    for a in range(0, n, step):
        logp = torch.log_softmax(logits[a:a + step].double() / t[a:a + step, None], 1)
        logprobs[a:a + step] = logp.gather(1, targets[a:a + step].clamp_min(0)[:, None])[:, 0]
        if want_entropy:
            entropy[a:a + step] = -(logp.exp() * logp).sum(1)
    logprobs, entropy = logprobs.masked_fill(~live, 0.0), entropy.masked_fill(~live, 0.0)
    if coefficients is None:
        return logprobs, entropy, None
    g, h = coefficients(logprobs, entropy)
    g = g.masked_fill(~live, 0.0)
    grad = torch.empty((n, vocab), device="cuda", dtype=torch.float64)
    for a in range(0, n, step):
        logp = torch.log_softmax(logits[a:a + step].double() / t[a:a + step, None], 1)
        hot = torch.zeros_like(logp).scatter_(1, targets[a:a + step].clamp_min(0)[:, None], 1.0)
        part = g[a:a + step, None] * (hot - logp.exp())
        if h is not None:
            plogp = logp.exp() * (logp + entropy[a:a + step, None])
            part = part - h.masked_fill(~live, 0.0)[a:a + step, None] * plogp
        grad[a:a + step] = part / t[a:a + step, None]
    return logprobs, entropy, grad


def _exact_logprobs(state):
    case = state["case"]
    coefficients = None
    if case["backward"]:
        coefficients = lambda logprobs, entropy: (state["grad_logprobs"].double(),
                                                  None if state["grad_entropy"] is None else state["grad_entropy"].double())
    logprobs, entropy, grad = _exact_rows(state, state["temperature"], case["entropy"], coefficients)
    return [logprobs] + ([entropy] if case["entropy"] else []) + ([grad] if case["backward"] else [])


def _exact_objective(case, state, logprobs, live, advantages, entropy):
    """The loss term by term on the host in 64 bits, its gradient by torch's own differentiation of the definition."""
    host = lambda x: None if x is None else x.detach().to("cpu", torch.float64)
    bounds, live = state["bounds"], live.cpu()
    n = bounds[-1]
    sequence = torch.zeros(n, dtype=torch.long)
    for i, (a, b) in enumerate(zip(bounds[:-1], bounds[1:])):
        sequence[a:b] = i
    index = live.nonzero()[:, 0]
    seq = sequence[index]
    logp = host(logprobs)[index].requires_grad_()
    h = host(entropy)[index].requires_grad_() if entropy is not None else torch.zeros(len(index), dtype=torch.float64, requires_grad=True)
    a = host(advantages)
    a = a[seq] if case.get("per_sequence", True) else a[index]
    old, ref = host(state["old"])[index], None if state["ref"] is None else host(state["ref"])[index]
    if case["aggregate"] == "sum":
        w = torch.ones(len(index), dtype=torch.float64)
    elif case["aggregate"] == "token":
        w = torch.full((len(index),), 1.0 / max(1, len(index)), dtype=torch.float64)
    else:
        counts = torch.bincount(seq, minlength=len(bounds) - 1)
        w = 1.0 / (counts[seq].double() * max(1, int((counts > 0).sum())))
    ratio = torch.exp(logp - old)
    bounded = torch.clamp(ratio, 1.0 - case["clip_low"], 1.0 + case["clip_high"])
    gain = torch.minimum(ratio * a, bounded * a)
    clipped = (bounded.detach() * a) < (ratio.detach() * a)
    if case["dual_clip"]:
        lower = case["dual_clip"] * a
        clipped = clipped | ((a < 0) & (lower > gain.detach()))
        gain = torch.where(a < 0, torch.maximum(gain, lower), gain)
    kl = torch.zeros(len(index), dtype=torch.float64)
    if ref is not None:
        x = ref - logp
        kl = -x if case["kl"] == "k1" else x * x / 2 if case["kl"] == "k2" else torch.expm1(x) - x
    policy, kl_mean, entropy_mean = -(w * gain).sum(), (w * kl).sum(), (w * h).sum()
    loss = policy + case["kl_coef"] * kl_mean - case["entropy_coef"] * entropy_mean
    g, gh = torch.autograd.grad(loss, (logp, h), allow_unused=True)
    spread = lambda x: torch.zeros(n, dtype=torch.float64).index_copy_(0, index, x).cuda()
    delta, count = (logp - old).detach(), max(1, len(index))
    stats = torch.tensor([policy.item(), kl_mean.item(), entropy_mean.item() if entropy is not None else 0.0,
                          clipped.double().sum().item() / count, ratio.sum().item() / count,
                          (torch.expm1(delta) - delta).sum().item() / count, float(len(index))], dtype=torch.float64)
    return loss.detach().cuda(), stats.cuda(), spread(g), None if entropy is None else spread(gh)


def _exact_loss(state):
    case = state["case"]
    live = state["mask"] if state["mask"] is not None else torch.ones(state["bounds"][-1], dtype=torch.bool)
    loss, stats, grad, grad_entropy = _exact_objective(case, state, state["logprobs"], live, state["advantages"], state["entropy"])
    return [loss, stats, grad] + ([grad_entropy] if state["entropy"] is not None else [])


def _exact_gradient(state):
    case = state["case"]
    kept = {}
    live = state["targets"] >= 0
    if state["mask"] is not None:
        live = live & state["mask"]
    masked = dict(state, targets=torch.where(live, state["targets"], torch.full_like(state["targets"], -1)))

    def coefficients(logprobs, entropy):
        used = entropy if case["entropy_coef"] else None
        kept["loss"], kept["stats"], g, h = _exact_objective(case, state, logprobs, live, state["advantages"], used)
        return g, h

    logprobs, _, grad = _exact_rows(masked, case["temperature"], bool(case["entropy_coef"]), coefficients)
    return [kept["loss"], kept["stats"], logprobs, grad]


EXACT = {"attend_shared": _exact_attention, "token_logprobs": _exact_logprobs, "policy_loss": _exact_loss,
         "policy_gradient": _exact_gradient}
