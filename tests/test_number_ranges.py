"""Numbers that a 64-bit float holds and the kernels' fp32 does not: refused, without a GPU."""
import ctypes
import math
import os

import pytest

from climbing_gym_amd import _lib, build, ops


@pytest.fixture(scope="module")
def library():
    if not os.path.exists(_lib.LIBRARY_PATH):
        build.build()
    return _lib.load()


@pytest.mark.parametrize("kw, text", [(dict(kl_coef=1e39), "coefficients"), (dict(entropy_coef=-1e39), "coefficients"), (dict(clip_high=1e39), "clip_high"),
                                      (dict(dual_clip=1e39), "dual_clip"), (dict(kl_coef=3.41e38), "coefficients")])
def test_coefficients_beyond_fp32(kw, text):
    with pytest.raises(ValueError, match=text):
        ops.PolicyLossConfig(**kw)


@pytest.mark.parametrize("temperature", (1e39, 1e-39, 1e-50, 5e-324, math.inf, math.nan, 0.0, -1.0))
def test_temperatures_beyond_fp32(temperature):
    with pytest.raises(ValueError, match="temperature"):
        ops._temperature_number(temperature)


def test_the_largest_and_smallest_numbers_of_fp32_pass():
    assert ops._temperature_number(3.4e38) == 3.4e38 and ops._temperature_number(1.2e-38) == 1.2e-38
    ops.PolicyLossConfig(kl_coef=3.4e38, entropy_coef=-3.4e38, clip_high=3.0e38, dual_clip=3.4e38)


def test_the_c_boundary(library):
    buffer = ctypes.create_string_buffer(4096)
    p = ctypes.addressof(buffer)
    message = lambda: library.lfm2_last_error().decode()
    for t in (math.inf, math.nan, 1e-39, 1e39):
        assert library.lfm2_token_logprobs(p, None, p, p, 8, p, None, t, 2, 8, 9, None) == -1 and "temperature" in message(), t
        assert library.lfm2_token_logprobs_backward(p, 8, p, 8, p, p, p, None, None, t, 2, 8, 9, None) == -1 and "temperature" in message(), t
    def gradient(t=1.0, kl=0.0, entropy=0.0, scale=1.0):
        return library.lfm2_policy_gradient(p, p, p, p, p, 8, p, 8, p, p, p, p, None, None, None, t, p, 2, 8, 1, 0, 0, 3, 0.2, 0.2, 0.0, kl, entropy, scale, 9, None)
    for kw, text in ((dict(t=math.inf), "temperature"), (dict(t=1e-39), "temperature"), (dict(kl=math.inf), "coefficients"), (dict(entropy=math.nan), "coefficients"),
                     (dict(scale=math.inf), "grad_scale"), (dict(scale=math.nan), "grad_scale")):
        assert gradient(**kw) == -1 and text in message(), (kw, message())
    assert library.lfm2_policy_loss(p, p, p, None, p, p, p, p, None, None, None, p, 4, 1, 0, 0, 3, 0.2, 0.2, 0.0, math.inf, 0.0, None) == -1
    assert "coefficients" in message()


def test_attention_scales_beyond_fp32(library):
    """The kernels multiply by scale log2(e): 2.4e38 is a number of fp32, 2.4e38 x 1.44 is not."""
    buffer = ctypes.create_string_buffer(4096 + 16)
    p = (ctypes.addressof(buffer) + 15) // 16 * 16
    for scale in (2.4e38, 3.4e38, math.inf, math.nan, 0.0, -1.0):
        assert library.lfm2_shared_attention(p, p, p, p, None, None, p, None, 0, 16, p, 4, 8, 2, 64, 64, 4, 8192, 64, 64, scale, 0, 2, None) == -1, scale
        assert "scale" in library.lfm2_last_error().decode()
