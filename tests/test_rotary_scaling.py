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
