"""Rotary tables (host arithmetic) and the refusals of the paged-cache entry points that need no device."""
import ctypes as C
import math

import numpy as np
import pytest

from ferrum_gpu_b200 import CudaError, RopeScaling, _ffi, rope_tables


def _angles(s: RopeScaling, positions: int):
    half = s.rope_dim // 2
    i = np.arange(half, dtype=np.float64)
    freq = np.float64(np.float32(s.base)) ** (-2 * i / s.rope_dim) / np.float64(np.float32(s.linear_factor))
    if s.freq_factors is not None:
        freq = freq / np.asarray(s.freq_factors, dtype=np.float32).astype(np.float64)
    mag = 1.0
    if s.original_ctx:
        def pair(beta):  # base^(-2i / d) * ctx / (2 pi) = beta solved for i
            return s.rope_dim * math.log(s.original_ctx / (beta * 2 * math.pi)) / (2 * math.log(s.base))
        low, high = max(math.floor(pair(s.beta_fast)), 0), min(math.ceil(pair(s.beta_slow)), s.rope_dim - 1)
        slow = np.clip((i - low) / max(high - low, 1e-3), 0, 1)
        freq = freq * (1 - slow) + freq / s.factor * slow
        mag = s.attn_factor or 0.1 * math.log(s.factor) + 1
    return np.arange(positions, dtype=np.float64)[:, None] * freq[None, :], mag


@pytest.mark.parametrize("s", [
    RopeScaling(64), RopeScaling(64, base=1e6), RopeScaling(2), RopeScaling(96, linear_factor=4.0), RopeScaling(128, base=5e5, original_ctx=8192, factor=8.0),
    RopeScaling(64, base=1e4, original_ctx=2048, factor=16.0, beta_fast=24.0, beta_slow=2.0, attn_factor=1.25),
    RopeScaling(32, freq_factors=np.linspace(1, 8, 16)),
])
def test_tables_are_the_formula_in_64_bits(s):
    # one rounding to f32 of values up to `mag`, and at most one more unit where both sides' 64-bit results straddle a tie
    angle, mag = _angles(s, 3000)
    cos, sin = rope_tables(s, 3000)
    assert cos.shape == sin.shape == (3000, s.rope_dim // 2)
    assert np.abs(cos - np.cos(angle) * mag).max() <= mag * 2 ** -24 + 1e-9
    assert np.abs(sin - np.sin(angle) * mag).max() <= mag * 2 ** -24 + 1e-9


def test_long_positions_keep_their_angles():
    """At position 10^6 an angle formed in f32 is off by hundredths; formed in 64 bits it is not."""
    cos, _ = rope_tables(RopeScaling(8, base=10000.0), 1_000_001)
    for p in (999_983, 1_000_000):
        want = np.cos(p * 10000.0 ** (-2 * np.arange(4) / 8))
        assert np.abs(cos[p] - want).max() < 1e-6


@pytest.mark.parametrize("s,match", [
    (RopeScaling(7), "must be even"), (RopeScaling(0), "must be even"), (RopeScaling(8, base=0.0), "finite and positive"),
    (RopeScaling(8, linear_factor=float("nan")), "finite and positive"), (RopeScaling(8, freq_factors=np.ones(3)), "3 frequency factors for 4"),
    (RopeScaling(8, freq_factors=np.array([1, 0, 1, 1])), "frequency factor 1"), (RopeScaling(8, original_ctx=64, factor=-1.0), "finite and positive"),
])
def test_tables_refuse_what_is_no_scaling(s, match):
    with pytest.raises(CudaError, match=match):
        rope_tables(s, 4)


def test_null_device_is_refused():
    lib, view = _ffi.load(), _ffi.FcPagedCache()
    assert lib.fc_paged_extend_dev(None, C.byref(view), None, None, 0, 0, None, None, None, None, None, None, None) == _ffi.FC_ERR_ARG
    assert lib.fc_paged_release_dev(None, C.byref(view), None, 0, None, None, None) == _ffi.FC_ERR_ARG
    assert lib.fc_paged_append_dev(None, C.byref(view), None, None, 0, 0, 0, 0, None, None, None, 0) == _ffi.FC_ERR_ARG
    assert lib.fc_paged_attend_dev(None, C.byref(view), None, 0, 0, 0, 0, None, None, 0.0, None, 0) == _ffi.FC_ERR_ARG
    assert lib.fc_logprobs_dev(None, None, 0, 0, 0, 1, None, 0, None, None, None, None, None) == _ffi.FC_ERR_ARG
    assert lib.fc_rope_tables(None, 0, None, None) == _ffi.FC_ERR_ARG
