"""Rotary frequencies for longer contexts, pair by pair, from their definitions in 64 bits."""

import math

import numpy as np
import pytest

from aegaeon_amd import ops


@pytest.mark.parametrize("factor,want", [(0.25, 1.0), (0.99, 1.0), (1.0, 1.0),
                                         (4.0, 1 + 0.1 * math.log(4))])
def test_shorter_contexts_are_not_damped(factor, want):
    """A ramp's amplitude makes up for contexts that are longer; shorter ones keep 1."""
    _, amplitude = ops.rotary_frequencies(64, scaling="ramp", factor=factor, length=4096)
    assert amplitude == pytest.approx(want, rel=1e-15)


def pairs(dim, base):
    return [base ** (-2 * i / dim) for i in range(dim // 2)]


@pytest.mark.parametrize("dim,base,length", [(64, 1e4, 2048), (128, 1e4, 4096), (128, 1e6, 32768),
                                             (256, 5e5, 8192), (96, 1e4, 4096)])
@pytest.mark.parametrize("factor", [2.0, 8.0, 32.0])
def test_smooth_frequencies_pair_by_pair(dim, base, length, factor):
    """By wavelengths: up to a quarter of the length a pair keeps its frequency, from the length
    on it turns `factor` times slower, and the two are mixed between."""
    want, mixed = [], 0
    for f in pairs(dim, base):
        wave = 2 * math.pi / f
        if wave <= length / 4:
            want.append(f)
        elif wave >= length:
            want.append(f / factor)
        else:
            share = (length / wave - 1) / (4 - 1)
            want.append(share * f + (1 - share) * f / factor)
            mixed += 1
    got, amplitude = ops.rotary_frequencies(dim, base=base, scaling="smooth", factor=factor,
                                            length=length)
    assert mixed >= 2 and amplitude == 1.0
    assert np.allclose(got, want, rtol=1e-13)


@pytest.mark.parametrize("dim,base,length", [(64, 1e4, 2048), (128, 1e4, 4096), (128, 1e6, 32768),
                                             (256, 5e5, 8192), (96, 1e4, 4096)])
@pytest.mark.parametrize("factor", [2.0, 8.0, 32.0])
def test_ramp_frequencies_pair_by_pair(dim, base, length, factor):
    """From the last pair that turns 32 times over the length to the first that turns once,
    the share of the slower frequency grows by equal steps."""
    plain = pairs(dim, base)
    turns = [length * f / (2 * math.pi) for f in plain]
    first = max(i for i, t in enumerate(turns) if t >= 32)
    last = min(i for i, t in enumerate(turns) if t <= 1)
    want = []
    for i, f in enumerate(plain):
        slow = min(max((i - first) / (last - first), 0.0), 1.0)
        want.append(f * (1 - slow) + f / factor * slow)
    got, amplitude = ops.rotary_frequencies(dim, base=base, scaling="ramp", factor=factor,
                                            length=length)
    assert last - first > 4 and amplitude == pytest.approx(1 + 0.1 * math.log(factor), rel=1e-14)
    assert np.allclose(got, want, rtol=1e-12)
