"""What the scoring and policy-loss calls refuse, without a GPU: the configuration's checks, the Python checks that come
before any launch, and the argument checks at the C boundary."""
import ctypes

import pytest
import torch

from climbing_gym_amd import _lib, build, ops


@pytest.fixture(scope="module")
def library():
    import os
    if not os.path.exists(_lib.LIBRARY_PATH):
        build.build()
    return _lib.load()


@pytest.mark.parametrize("kw, text", [
    (dict(clip_low=1.0), "clip_low"), (dict(clip_low=-0.1), "clip_low"), (dict(clip_low=float("nan")), "clip_low"),
    (dict(clip_high=-1.0), "clip_high"), (dict(clip_high=float("inf")), "clip_high"),
    (dict(dual_clip=1.0), "dual_clip"), (dict(dual_clip=float("nan")), "dual_clip"),
    (dict(kl="k4"), "kl must"), (dict(aggregate="mean"), "aggregate"), (dict(kl_coef=float("nan")), "coefficients"),
    (dict(entropy_coef=float("inf")), "coefficients")])
def test_policy_loss_config_refuses(kw, text):
    with pytest.raises(ValueError, match=text):
        ops.PolicyLossConfig(**kw)


def test_cpu_tensors_are_refused():
    logits, targets = torch.zeros(2, 8), torch.zeros(2, dtype=torch.long)
    row = torch.zeros(2)
    with pytest.raises(ValueError, match="GPU"):
        ops.token_logprobs(logits, targets)
    with pytest.raises(ValueError, match="GPU"):
        ops.token_logprobs_backward(logits, targets, torch.zeros(2, 4), row)
    with pytest.raises(ValueError, match="GPU"):
        ops.policy_loss(row, row, row)
    with pytest.raises(ValueError, match="GPU"):
        ops.policy_gradient(logits, targets, row, row)


def test_token_arguments_are_checked_before_the_device():
    row, longs = torch.zeros(4), torch.zeros(4, dtype=torch.long)
    bounds = torch.tensor([0, 4], dtype=torch.int32)
    loss = lambda **kw: ops.policy_loss_forward(**{**dict(logprobs=row, old_logprobs=row, advantages=row), **kw})
    for kw, text in ((dict(old_logprobs=torch.zeros(3)), "old_logprobs"), (dict(old_logprobs=row.double()), "old_logprobs"),
                     (dict(old_logprobs=torch.zeros(8)[::2]), "old_logprobs"), (dict(ref_logprobs=torch.zeros(5)), "ref_logprobs"),
                     (dict(config=ops.PolicyLossConfig(kl_coef=0.1)), "ref_logprobs"),
                     (dict(config=ops.PolicyLossConfig(entropy_coef=0.1)), "entropies"),
                     (dict(mask=longs), "mask"), (dict(mask=torch.ones(3, dtype=torch.bool)), "mask"),
                     (dict(cu_seqlens=bounds.long()), "cu_seqlens"), (dict(cu_seqlens=bounds[:1]), "cu_seqlens"),
                     (dict(cu_seqlens=bounds, per_sequence=True), "advantages"), (dict(per_sequence=True), "advantages"),
                     (dict(logprobs=torch.zeros(2, 2)), "logprobs")):
        with pytest.raises(ValueError, match=text):
            loss(**kw)


def test_c_boundary_refuses(library):
    buffer = ctypes.create_string_buffer(4096)
    p = ctypes.addressof(buffer)
    message = lambda: library.lfm2_last_error().decode()
    score = lambda **kw: library.lfm2_token_logprobs(p, None, p, p, kw.get("stride", 8), p, None, kw.get("t", 1.0), kw.get("n", 2), kw.get("v", 8), kw.get("dtype", 0), None)
    for kw, status, text in ((dict(n=0), -1, "empty"), (dict(v=0), -1, "empty"), (dict(stride=7), -1, "overlap"), (dict(t=0.0), -1, "temperature"),
                             (dict(t=float("nan")), -1, "temperature"), (dict(dtype=9), -3, "dtype"), (dict(n=1 << 31), -1, "2^31")):
        assert score(**kw) == status and text in message(), kw
    def loss(n=4, s=1, cu=None, old=p, aggregate=0, kl=3, low=0.2, high=0.2, dual=0.0, ws=p):
        return library.lfm2_policy_loss(p, p, p, None, p, old, p, None, None, None, cu, ws, n, s, 0, aggregate, kl, low, high, dual, 0.0, 0.0, None)
    for kw, text in ((dict(n=0), "tokens"), (dict(cu=p, s=0), "sequence"), (dict(old=None), "required"), (dict(aggregate=3), "aggregate"),
                     (dict(kl=0), "KL"), (dict(low=1.0), "clip"), (dict(high=float("nan")), "clip"), (dict(dual=0.5), "dual_clip"), (dict(ws=None), "null")):
        assert loss(**kw) == -1 and text in message(), kw
    assert library.lfm2_policy_workspace(0, 1, 0) == 0
    assert library.lfm2_policy_workspace(1, 1, 1) >= 15


def test_shared_attention_refuses_at_the_c_boundary(library):
    buffer = ctypes.create_string_buffer(4096 + 16)
    p = (ctypes.addressof(buffer) + 15) // 16 * 16
    message = lambda: library.lfm2_last_error().decode()
    def schedule(b=4, groups=1, capacity=64, qh=8, kh=2, d=64, at=p, starts=p):
        return library.lfm2_shared_schedule(at, p, None, None, starts, p, p, b, groups, capacity, qh, kh, d, None)
    for kw, text in ((dict(b=0), "empty"), (dict(b=5000), "rows"), (dict(groups=0), "groups"), (dict(groups=5000), "groups"), (dict(capacity=0), "empty"),
                     (dict(capacity=1 << 29), "positions"), (dict(kh=3), "divisible"), (dict(d=80), "head_dim"), (dict(at=p + 4), "unaligned"),
                     (dict(starts=None), "bounds"), (dict(qh=2048), "query heads")):
        assert schedule(**kw) == -1 and text in message(), (kw, message())
    def attend(b=4, d=64, q=p, c1=64, fp8=0, table=None, page=16, blocks=0, pools=4, dtype=0, scales=None, ws=p):
        return library.lfm2_shared_attention(p, q, p, p, scales, scales, p, table, blocks, page, ws, b, 8, 2, d, 64, pools, 64 * 128, c1, 64, 0.125, fp8, dtype, None)
    for kw, status, text in ((dict(b=0), -1, "empty"), (dict(q=p + 2), -1, "aligned"), (dict(c1=65), -1, "strides"), (dict(c1=16, fp8=1, scales=p), -1, "strides"),
                             (dict(fp8=1), -1, "scales"), (dict(table=p, blocks=3), -1, "page"), (dict(pools=0), -1, "cache"),
                             (dict(dtype=2), -3, "dtype"), (dict(ws=None), -1, "null")):
        assert attend(**kw) == status and text in message(), (kw, message())
    assert library.lfm2_shared_schedule_size(0, 64, 8, 2, 64) == 0 and library.lfm2_shared_attention_workspace(4, 64, 8, 3, 64) == 0
    assert library.lfm2_shared_schedule_size(4, 64, 8, 2, 64) >= 16 + 4 * 4 + 8 * 8


def test_binding_signatures_match_the_header():
    """Kinds and number of the arguments the binding passes, against the declarations."""
    import os
    import re
    text = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "lfm2_hip.h")).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    kind = lambda arg: "p" if "*" in arg else "l" if "int64_t" in arg else "f" if "float" in arg else "i"
    declared = {name: "".join(kind(a) for a in args.split(",") if a.strip() not in ("", "void"))
                for name, args in re.findall(r"\b(?:int|int64_t)\s+(lfm2_\w+)\s*\(([^)]*)\)", text)}
    for name, signature in {**_lib._SIGNATURES, **_lib._INT64_RESULT}.items():
        assert declared[name] == signature, name


def test_refuses_more_rows_or_sequences_than_a_launch_counts(library):
    buffer = ctypes.create_string_buffer(4096)
    p = ctypes.addressof(buffer)
    many = (1 << 22) + 1
    assert library.lfm2_token_logprobs(p, None, p, p, 8, p, None, 1.0, many, 8, 0, None) == -1 and b"2^22 rows" in library.lfm2_last_error()
    assert library.lfm2_policy_loss(p, p, p, None, p, p, p, None, None, None, p, p, 4, many, 0, 0, 3, 0.2, 0.2, 0.0, 0.0, 0.0, None) == -1
    assert b"2^22 sequences" in library.lfm2_last_error()
