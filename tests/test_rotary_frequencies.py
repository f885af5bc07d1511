"""The frequencies of scaled rotations against the published formulas, pair by pair in Python floats (no device)."""
import math

import pytest

from adaptq_b200.rotary import _inverse_frequencies


def wavelength(dim, base, i):
    return 2 * math.pi * base ** (2 * i / dim)


def plain(dim, base, i, **_):
    return 1.0 / base ** (2 * i / dim)


def linear(dim, base, i, factor):
    """Position interpolation (Chen et al. 2023): positions divided by the factor."""
    return plain(dim, base, i) / factor


def ntk(dim, base, i, factor):
    """A larger base, under which the slowest pair turns `factor` times as slowly and the fastest as before."""
    return plain(dim, base * factor ** (dim / (dim - 2)), i)


def yarn(dim, base, i, factor, original_max_position, beta_fast=32.0, beta_slow=1.0):
    """YaRN (Peng et al. 2023), section 3.2 "NTK-by-parts", with the ramp over pair numbers between the pairs that turn beta_fast
    and beta_slow times within the original context."""
    pair = lambda turns: dim * math.log(original_max_position / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
    low, high = max(math.floor(pair(beta_fast)), 0), min(math.ceil(pair(beta_slow)), dim - 1)
    gamma = 1.0 - min(1.0, max(0.0, (i - low) / (high - low)))   # 1: extrapolated (kept), 0: interpolated
    w = plain(dim, base, i)
    return gamma * w + (1 - gamma) * w / factor


def llama3(dim, base, i, factor, original_max_position, low_freq_factor=1.0, high_freq_factor=4.0):
    """Long wavelengths divided, short ones kept, a ramp in turns per original context between."""
    w, turns = plain(dim, base, i), original_max_position / wavelength(dim, base, i)
    if turns < low_freq_factor:
        return w / factor
    if turns > high_freq_factor:
        return w
    s = (turns - low_freq_factor) / (high_freq_factor - low_freq_factor)
    return w * ((1 - s) / factor + s)


@pytest.mark.parametrize("dim,base", [(128, 10000.0), (64, 500000.0), (40, 10000.0), (96, 1e6)])
@pytest.mark.parametrize("formula,scaling", [
    (plain, None), (linear, dict(factor=4.0)), (ntk, dict(factor=2.5)), (yarn, dict(factor=8.0, original_max_position=4096)),
    (yarn, dict(factor=4.0, original_max_position=8192, beta_fast=16.0, beta_slow=2.0)),
    (llama3, dict(factor=8.0, original_max_position=8192)),
    (llama3, dict(factor=32.0, original_max_position=8192, low_freq_factor=2.0, high_freq_factor=6.0))])
def test_frequencies(dim, base, formula, scaling):
    given = None if scaling is None else dict(scaling, type=formula.__name__)
    w, factor = _inverse_frequencies(dim, base, given)
    assert len(w) == dim // 2
    for i, got in enumerate(w.tolist()):
        want = formula(dim, base, i, **(scaling or {}))
        assert abs(got - want) <= 1e-13 * want
    # the rotated vector is multiplied by YaRN's 0.1 ln(s) + 1 (its equation 22 as a square root of 1/t), else by one
    assert factor == (0.1 * math.log(scaling["factor"]) + 1.0 if formula is yarn else 1.0)


def test_fixed_points():
    """Values worked out by hand: base 10000, 4 coordinates, pairs at 1 and 1/100 radians a token."""
    assert _inverse_frequencies(4, 10000.0, None)[0].tolist() == [1.0, 0.01]
    assert _inverse_frequencies(4, 10000.0, {"type": "linear", "factor": 2.0})[0].tolist() == [0.5, 0.005]
    w, _ = _inverse_frequencies(4, 10000.0, {"type": "ntk", "factor": 3.0})   # base 90000: the slow pair three times slower
    assert w[0] == 1.0 and abs(float(w[1]) - 0.01 / 3) < 1e-15
    # llama3 over 1000 tokens: pair 0 turns 159 times (kept), pair 1 1.59 times: a ramp from 1 to 4 turns, s = 0.1972
    w, _ = _inverse_frequencies(4, 10000.0, {"type": "llama3", "factor": 8.0, "original_max_position": 1000})
    s = (10 / (2 * math.pi) - 1) / 3
    assert w[0] == 1.0 and abs(float(w[1]) - 0.01 * ((1 - s) / 8 + s)) < 1e-15
    assert _inverse_frequencies(64, 10000.0, {"type": "yarn", "factor": 2.0, "original_max_position": 4096, "attention_factor": 1.5})[1] == 1.5
