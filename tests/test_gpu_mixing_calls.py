"""Calls of a mixing layer's operators that their descriptions allow, one test each."""
import math

import numpy as np
import pytest

from test_gpu_rotary import cls_of, close, reference

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


@pytest.mark.parametrize("dt", [np.float32, np.float64])
@pytest.mark.parametrize("power", [43, 44, 45, 47, 49])
def test_rotary_by_angles_up_to_the_last(dt, power):
    """Pairs that the turn brings next to an axis: what is left of one of them shows the sine's and cosine's own error, which is below 8e-12 in SFloat at
    every angle."""
    import cumo_amd as m
    cls, n = cls_of(m, dt), 4000
    rng = np.random.default_rng(power)
    f = np.ldexp(1 + rng.random(n), power)
    x = np.zeros((2, 1, 2 * n), dt)
    x[0, 0, :n], x[0, 0, n:] = np.sin(f), np.cos(f)
    x[1, 0, :n], x[1, 0, n:] = -np.cos(f), np.sin(f)
    p = np.array([1, -1], np.int32)
    for inverse in (False, True):
        y = m.Fused.rotary(cls.cast(x), m.Int32.cast(p), m.DFloat.cast(f), inverse=inverse)
        close(y.to_numpy(), *reference(x, p, f, inverse=inverse))
