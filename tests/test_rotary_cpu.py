"""Frequencies of the rotation, scaled and unscaled, against formulas in numpy, and what is refused."""

import math

import numpy as np
import pytest
import torch

from async_llm_amd import native
from async_llm_amd.rotary import RotaryEmbedding


def made(rotary=64, base=1e6, **scaling):
    return RotaryEmbedding(128, rotary, base, scaling=scaling or None, device="cpu")


def plain(rotary=64, base=1e6):
    return base ** (-np.arange(0, rotary, 2) / rotary)


def test_unscaled_and_linear():
    np.testing.assert_allclose(made().inv_freq.numpy(), plain(), rtol=1e-15)
    np.testing.assert_allclose(made(rope_type="default").inv_freq.numpy(), plain(), rtol=1e-15)
    np.testing.assert_allclose(made(rope_type="linear", factor=4.0).inv_freq.numpy(), plain() / 4, rtol=1e-15)
    assert made().attention_factor == 1.0 and made().inv_freq.dtype == torch.float64
    np.testing.assert_allclose(made(type="linear", factor=2).inv_freq.numpy(), plain() / 2, rtol=1e-15)


def test_llama3_stretches_long_waves_and_blends():
    got = made(128, 5e5, rope_type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0,
               original_max_position_embeddings=8192).inv_freq.numpy()
    f = plain(128, 5e5)
    wave = 2 * math.pi / f
    want = np.where(wave > 8192, f / 8, f)
    between = (wave <= 8192) & (wave >= 2048)
    share = (8192 / wave - 1) / 3
    want[between] = ((1 - share) * f / 8 + share * f)[between]
    np.testing.assert_allclose(got, want, rtol=1e-14)
    assert between.any() and (wave > 8192).any() and (wave < 2048).any()


def test_yarn_ramps_over_pairs():
    r = made(64, 1e6, rope_type="yarn", factor=4.0, original_max_position_embeddings=32768)
    f = plain()
    at = lambda t: 64 * math.log(32768 / (t * 2 * math.pi)) / (2 * math.log(1e6))  # noqa: E731
    low, high = math.floor(at(32)), math.ceil(at(1))
    ramp = np.clip((np.arange(32) - low) / (high - low), 0, 1)
    np.testing.assert_allclose(r.inv_freq.numpy(), f / 4 * ramp + f * (1 - ramp), rtol=1e-14)
    assert r.attention_factor == pytest.approx(0.1 * math.log(4) + 1, rel=1e-15)
    assert made(64, 1e6, rope_type="yarn", factor=4.0, original_max_position_embeddings=32768,
                attention_factor=1.5).attention_factor == 1.5


@pytest.mark.parametrize("scaling", [
    dict(rope_type="spiral", factor=2.0), dict(rope_type="linear"), dict(rope_type="linear", factor=-1.0),
    dict(rope_type="linear", factor=float("nan")), dict(rope_type="linear", factor=2.0, beta=1.0), dict(factor=2.0),
    dict(rope_type="llama3", factor=8.0, low_freq_factor=4.0, high_freq_factor=4.0, original_max_position_embeddings=8192),
    dict(rope_type="yarn", factor=2.0), dict(rope_type="linear", factor=True),
])
def test_scalings_that_are_refused(scaling):
    with pytest.raises(ValueError):
        made(**scaling)


@pytest.mark.parametrize("dims", [(128, 130), (128, 63), (128, 0), (127, None), (8192, 4096), (0, None)])
def test_widths_that_are_refused(dims):
    with pytest.raises(ValueError, match="must be even"):
        RotaryEmbedding(dims[0], dims[1], device="cpu")


def test_calls_without_a_gpu_are_refused():
    r = made()
    with pytest.raises(native.ViewAttnError, match="GPU only"):
        r(torch.zeros(1, dtype=torch.int64), torch.zeros(1, 128))
    with pytest.raises(native.ViewAttnError, match="GPU only"):
        r.cos_sin_cache(16)
    with pytest.raises(ValueError, match="interleaved"):
        RotaryEmbedding(64, interleaved=True, device="cpu").cos_sin_cache(16)


def test_entry_refuses():
    turns = native.VaTurns(64, 0, 1.0, None)
    call = lambda n, dim, hq, stride, dtype=native.VA_BF16: native.lib.va_rotate_qk(  # noqa: E731
        None, stride, hq, None, stride, None, 0, 0, None, 0, None, 1, n, dim, dtype, turns, None)
    assert call(0, 64, 4, 256) == 0 and call(4, 64, 0, 256) == 0
    assert call(4, 64, 4, 256) == native.VA_ERR_ARG and b"null pointer" in native.lib.va_last_error()
    assert call(4, 32, 4, 256) == native.VA_ERR_ARG and b"within head_dim" in native.lib.va_last_error()
    assert call(-1, 64, 4, 256) == native.VA_ERR_ARG and call(4, 65, 4, 256) == native.VA_ERR_ARG
    assert native.lib.va_rotary_table(turns, 0, 4, None, None) == native.VA_ERR_ARG
    assert native.lib.va_rotary_table(turns, 0, 0, None, None) == 0
