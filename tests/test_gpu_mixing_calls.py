"""Calls of a mixing layer's operators that their descriptions allow, one test each."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("trained", [1, 4, 6, 7, 300])
def test_yarn_slows_every_pair_that_turns_too_seldom(trained):
    """The first one too: 6 positions turn it by 6 radians, less than once."""
    import cumo_amd as m
    plain = 1e4 ** (-np.arange(8) / 8.0)
    f = m.Fused.rotary_frequencies(16, 1e4, "yarn", 4.0, trained=trained)[0].to_numpy()
    turns = trained * plain / (2 * math.pi)
    assert (np.abs(f[turns <= 1] * 4 / plain[turns <= 1] - 1) <= 1e-14).all()
    assert (f[turns >= 32] == plain[turns >= 32]).all() and (np.diff(f / plain) <= 1e-14).all()
