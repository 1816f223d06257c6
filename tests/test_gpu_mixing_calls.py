"""Calls of a mixing layer's operators that their descriptions allow, one test each."""
import math

import numpy as np
import pytest

from test_gpu_matmul_q8 import check, product
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


@pytest.mark.parametrize("dt", [np.float32, np.float64])
@pytest.mark.parametrize("rows,inner,cols", [(1990, 136, 3097), (2041, 257, 3081), (2050, 640, 2100), (700, 1025, 2500), (3900, 33, 3200)])
def test_matmul_in_tiles_of_each_size(dt, rows, inner, cols):
    """Results that go through the caches, in enough tiles of 128 that they are taken, in too few, and in enough of 256 (DFloat: past the caches)."""
    import cumo_amd as m
    cls = cls_of(m, dt)
    rng = np.random.default_rng(rows)
    x, w = (rng.integers(-128, 128, s).astype(np.int8) for s in ((rows, inner), (cols, inner)))
    xs, ws = (np.exp(rng.standard_normal((n, 1))).astype(dt) for n in (rows, cols))
    bias = rng.standard_normal(cols).astype(dt)
    y = m.Fused.matmul_q8(m.Int8.cast(x), cls.cast(xs), m.Int8.cast(w), cls.cast(ws), cls.cast(bias))
    check(y.to_numpy(), *product(x, xs, w, ws, bias, dt))
