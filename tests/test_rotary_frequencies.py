"""rotary_frequencies' "yarn" scaling on both sides of the pair that turns once.

Pair i makes original_length * base^(-2 i / rotary_dim) / (2 pi) turns over the original length.
From the definition: at least `fast_turns`, the frequency is kept; at most `slow_turns`, it is
divided by the factor; between, it lies on a ramp, so it is divided by less than the factor. The
ramp's ends are whole pairs, 0 at the least and rotary_dim - 1 at the most, which is past the last
of the rotary_dim / 2 pairs. Frequencies are float64: a handful of operations, 2^-53 each.
"""

from __future__ import annotations

import math

import pytest
import torch

from tklab.kernels.rotary import rotary_frequencies

CASES = [(dim, base, length)
         for dim, base in ((2, 1e4), (4, 1e4), (16, 1e4), (64, 1e4), (128, 1e4), (128, 5e5))
         for length in (1, 3, 6, 7, 64, 2048, 8192, 32768, 65536, 131072, 1048576)]


@pytest.mark.parametrize("factor", [4.0, 40.0])
@pytest.mark.parametrize("dim,base,length", CASES)
def test_each_pair_is_divided_by_its_turns(dim, base, length, factor) -> None:
    plain, _ = rotary_frequencies(dim, base=base)
    scaled, magnitude = rotary_frequencies(dim, base=base, scaling="yarn", factor=factor,
                                           original_length=length)
    assert magnitude == pytest.approx(0.1 * math.log(factor) + 1)
    ratio = (plain / scaled).tolist()
    for i, r in enumerate(ratio):
        turns = length * base ** (-2 * i / dim) / (2 * math.pi)
        if turns >= 32:
            assert r == 1.0, i
        elif turns <= 1:
            assert r == pytest.approx(factor, rel=1e-14), i
        else:
            assert 1.0 <= r < factor * (1 - 1e-6), (i, turns)
    assert ratio == sorted(ratio)


@pytest.mark.parametrize("dim,base,length", [c for c in CASES if c[2] >= 64])
def test_the_ramp_is_linear_between_whole_pairs(dim, base, length) -> None:
    factor = 8.0
    scaled, _ = rotary_frequencies(dim, base=base, scaling="yarn", factor=factor,
                                   original_length=length)

    def pair(turns):
        return dim * math.log(length / (2 * math.pi * turns)) / (2 * math.log(base))

    low, high = max(math.floor(pair(32)), 0), min(math.ceil(pair(1)), dim - 1)
    want = []
    for i in range(dim // 2):
        t = min(max((i - low) / (high - low), 0.0), 1.0) if high > low else 0.0
        want.append(base ** (-2 * i / dim) * (1 - t + t / factor))
    torch.testing.assert_close(scaled, torch.tensor(want, dtype=torch.float64), rtol=1e-13, atol=0)


@pytest.mark.parametrize("dim,length,slowest", [(128, 131072, 2.17), (128, 65536, 3.23),
                                                (16, 32768, 2.29)])
def test_the_slowest_pair_of_long_contexts(dim, length, slowest) -> None:
    """Worked out by hand: (128, 131072): ramp from pair 45 to 70, the last pair is 18 / 25 along."""
    plain, _ = rotary_frequencies(dim)
    scaled, _ = rotary_frequencies(dim, scaling="yarn", factor=4.0, original_length=length)
    assert float(plain[-1] / scaled[-1]) == pytest.approx(slowest, abs=0.01)
