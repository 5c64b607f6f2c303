"""The scaled frequencies of rotary positions, pair by pair against their formulas, ramps included."""

from __future__ import annotations

import math

import pytest
import torch

CASES = [(64, 10000.0, 4.0, 4096, None, 1.0), (128, 1e6, 8.0, 32768, None, 1.0), (20, 500000.0, 2.5, 8192, None, 1.0), (64, 10000.0, 40.0, 4096, 16.0, 2.0), (128, 10000.0, 4.0, 100, None, 1.0)]


@pytest.mark.parametrize("width, base, factor, length, fast, slow", CASES)
def test_a_ramp_over_the_index(width, base, factor, length, fast, slow):
    from rl_engine.ops.attention import rotary_frequencies

    got = rotary_frequencies(width, base, factor=factor, scaling="bands", original_length=length, fast_turns=fast, slow_turns=slow, device="cpu")
    index_of = lambda turns: width * math.log(length / (turns * 2 * math.pi)) / (2 * math.log(base))  # where a pair makes that many turns  # noqa: E731
    first, last = max(math.floor(index_of(fast or 32.0)), 0), min(math.ceil(index_of(slow)), width - 1)
    inside = 0
    for i in range(width // 2):
        f = base ** (-2 * i / width)
        along = min(max((i - first) / (last - first), 0.0), 1.0)
        inside += 0.0 < along < 1.0
        want = (1 - along) * f + along * f / factor
        assert abs(float(got[i]) / want - 1) < 1e-13, i
    assert inside >= 2


@pytest.mark.parametrize("width, base, factor, length, fast, slow", CASES)
def test_a_ramp_over_the_turns(width, base, factor, length, fast, slow):
    from rl_engine.ops.attention import rotary_frequencies

    got = rotary_frequencies(width, base, factor=factor, scaling="wavelengths", original_length=length, fast_turns=fast, slow_turns=slow, device="cpu")
    inside = 0
    for i in range(width // 2):
        f = base ** (-2 * i / width)
        wavelength = 2 * math.pi / f
        if wavelength < length / (fast or 4.0):
            want = f
        elif wavelength > length / slow:
            want = f / factor
        else:
            smooth = (length / wavelength - slow) / ((fast or 4.0) - slow)
            inside += 1
            want = (1 - smooth) * f / factor + smooth * f
        assert abs(float(got[i]) / want - 1) < 1e-13, i
    assert inside >= 1 and got.dtype == torch.float64
