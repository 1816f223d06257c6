"""Rotary positions against the formula in 64 bits and more, for every layout of pairs, and as a turn that can be taken back.

Tolerances: everything up to the result's one rounding (half a step of its type) is in double. The angle is a product in double, the same one in the
reference; SFloat sines and cosines leave out less than 8e-12, DFloat ones are within 4 half steps of 64 bits, and three operations follow."""
import ctypes as C
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

TYPES = [np.float32, np.float64]


def cls_of(m, dt):
    return m.SFloat if dt == np.float32 else m.DFloat


def reference(x, positions, f, interleaved=False, inverse=False, amplitude=1.0):
    """In long double; the angle's product in double."""
    n = len(f)
    angle = (positions.astype(np.float64)[..., None] * f)[..., None, :].astype(np.longdouble)
    c, s = np.cos(angle) * amplitude, np.sin(angle) * (-amplitude if inverse else amplitude)
    y, size = x.astype(np.longdouble), np.abs(x.astype(np.longdouble))
    one, two = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    u, v = y[..., one].copy(), y[..., two].copy()
    y[..., one], y[..., two] = u * c - v * s, v * c + u * s
    size[..., one] = size[..., two] = (np.abs(u) + np.abs(v)) * abs(amplitude)
    return y, size


def close(got, want, size):
    dt = got.dtype
    lost = 8e-12 + 8 * 2.0 ** -53 if dt == np.float32 else 8 * 2.0 ** -53
    assert got.shape == want.shape
    bad = ~(np.abs(got - want) <= np.finfo(dt).eps / 2 * np.abs(want) + lost * size)
    assert not bad.any(), (bad.sum(), np.argwhere(bad)[0], got[bad][0], want[bad][0])


CASES = [((1, 2), 1), ((3, 8), 2), ((5, 3, 16), 8), ((7, 1, 10), 5), ((2, 3, 4, 64), 32), ((2, 5, 3, 64), 16), ((3, 4, 5, 33), 11), ((2, 3, 2, 96), 30), ((64, 1, 32, 128), 64),
         ((2, 300, 9, 128), 64), ((2, 2, 3, 2, 40), 12), ((4, 6, 7, 9), 0), ((1, 9, 2, 260), 130), ((1, 4000, 33, 20), 10)]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("shape,pairs", CASES)
@pytest.mark.parametrize("interleaved", [False, True])
def test_matches_the_formula(dt, shape, pairs, interleaved):
    import cumo_amd as m
    cls = cls_of(m, dt)
    rng = np.random.default_rng(sum(shape) + pairs)
    x = rng.standard_normal(shape).astype(dt)
    positions = rng.integers(-5, 200000, shape[:-2]).astype(np.int32)
    f = 10000.0 ** (-2.0 * np.arange(pairs) / max(2 * pairs, 1))
    dx, df = cls.cast(x), m.DFloat.cast(f)
    dp = m.Int32.cast(positions if positions.ndim else positions.reshape(1))
    for inverse, amplitude in ((False, 1.0), (True, 1.2)):
        y = m.Fused.rotary(dx, dp, df, interleaved, inverse, amplitude)
        assert type(y) is cls
        close(y.to_numpy(), *reference(x, positions, f, interleaved, inverse, amplitude))


@pytest.mark.parametrize("dt", TYPES)
def test_far_positions_and_wide_angles(dt):
    """Positions up to the ends of their type, frequencies over a hundred powers of two; quarter turns; angles of 2^50 and more are NaN."""
    import cumo_amd as m
    cls = cls_of(m, dt)
    rng = np.random.default_rng(2)
    positions = np.concatenate([np.array([0, 1, -1, 2 ** 31 - 1, -2 ** 31, 12345678]), rng.integers(-2 ** 31, 2 ** 31, 60)]).astype(np.int32)
    f = np.concatenate([2.0 ** np.arange(-80, 18, 3), [math.pi / 2, math.pi, math.pi / 4]])
    x = rng.standard_normal((66, 3, 2 * len(f))).astype(dt)
    y = m.Fused.rotary(cls.cast(x), m.Int32.cast(positions), m.DFloat.cast(f))
    close(y.to_numpy(), *reference(x, positions, f))
    far = m.Fused.rotary(cls.cast(x[:2, :, :6]), m.Int32.cast(np.array([1, 3], np.int32)), m.DFloat.cast(np.array([2.0 ** 50, np.inf, np.nan]))).to_numpy()
    assert np.isnan(far).all()


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
def test_the_inverse_is_the_gradient(dt, interleaved):
    """<g, turn x> = <turn back g, x>, each side a sum of n products off by n half steps of its magnitudes; and turning back answers x."""
    import cumo_amd as m
    cls = cls_of(m, dt)
    rng = np.random.default_rng(3)
    x, g = (rng.standard_normal((2, 30, 4, 48)).astype(dt) for _ in range(2))
    p, (f, _) = m.Int32.cast(rng.integers(0, 1000, (2, 30)).astype(np.int32)), m.Fused.rotary_frequencies(40)
    y = m.Fused.rotary(cls.cast(x), p, f, interleaved, amplitude=1.5).to_numpy().astype(np.float64)
    gx = m.Fused.rotary(cls.cast(g), p, f, interleaved, inverse=True, amplitude=1.5).to_numpy().astype(np.float64)
    # every product has two rounded factors; 1.5 * 2 of u and v
    size = 2 * 3 * (np.abs(x).max() * np.abs(g).max()) * x.size
    assert abs((g * y).sum() - (gx * x).sum()) <= np.finfo(dt).eps * size
    back = m.Fused.rotary(m.Fused.rotary(cls.cast(x), p, f, interleaved), p, f, interleaved, inverse=True).to_numpy()
    assert (np.abs(back - x) <= 4 * np.finfo(dt).eps * np.abs(x).max()).all()


@pytest.mark.parametrize("dt", TYPES)
def test_layouts(dt):
    """Heads in front of time, a window of a packed array, backwards, every other element; results into windows and on top of x."""
    import cumo_amd as m
    from cumo_amd import _lib
    cls = cls_of(m, dt)
    rng = np.random.default_rng(4)
    b, t, h, d = 3, 5, 4, 24
    x = rng.standard_normal((b, t, h, d)).astype(dt)
    p, f = m.Int32.cast(rng.integers(0, 1000, (b, t)).astype(np.int32)), m.DFloat.cast(rng.random(9))
    want = m.Fused.rotary(cls.cast(x), p, f).to_numpy()
    wide = np.zeros((b, t, h, 2 * d + 3), dt)
    wide[..., 3::2] = x
    packed = np.zeros((b, t, 3 * h, d), dt)
    packed[:, :, h:2 * h] = x
    for view in (cls.cast(np.ascontiguousarray(x.transpose(0, 2, 1, 3))).transpose(0, 2, 1, 3), cls.cast(packed)[:, :, h:2 * h],
                 cls.cast(np.ascontiguousarray(x[::-1, ::-1, ::-1]))[::-1, ::-1, ::-1], cls.cast(wide)[:, :, :, 3::2], cls.cast(np.ascontiguousarray(x.transpose())).transpose()):
        assert (m.Fused.rotary(view, p, f).to_numpy() == want).all()
    ref = lambda z: C.byref(z._desc())  # noqa: E731
    dx = cls.cast(x)
    buf = cls(b, t, 3 * h, d + 5).fill(7)
    part = buf[:, :, h:2 * h, 2:d + 2]
    _lib.call(_lib.lib.cumo_hip_na_rotary, ref(dx), ref(p), ref(f), 0, 0, 1.0, ref(part))
    got = buf.to_numpy()
    assert (got[:, :, h:2 * h, 2:d + 2] == want).all()
    got[:, :, h:2 * h, 2:d + 2] = 7
    assert (got == 7).all()
    _lib.call(_lib.lib.cumo_hip_na_rotary, ref(dx), ref(p), ref(f), 0, 0, 1.0, ref(dx))
    assert (dx.to_numpy() == want).all()


def test_nothing_to_do():
    import cumo_amd as m
    f = m.DFloat.cast(np.ones(2))
    assert m.Fused.rotary(m.SFloat(0, 3, 8), m.Int32(0), f).shape == (0, 3, 8)
    assert m.Fused.rotary(m.SFloat(4, 0, 8), m.Int32(4), f).shape == (4, 0, 8)
    x = m.SFloat.cast(np.arange(10, dtype=np.float32).reshape(2, 5))
    assert (m.Fused.rotary(x, m.Int32.cast(np.array([3], np.int32)), m.DFloat(0)).to_numpy() == x.to_numpy()).all()


def test_frequencies():
    """What the three ways of reaching further do, from their descriptions."""
    import cumo_amd as m
    plain, one = m.Fused.rotary_frequencies(64, 1e4)
    plain = plain.to_numpy()
    assert one == 1.0 and (np.abs(plain - 1e4 ** (-np.arange(32) / 32.0)) <= 1e-15).all()
    linear, one = m.Fused.rotary_frequencies(64, 1e4, "linear", 4.0)
    assert one == 1.0 and (np.abs(linear.to_numpy() - plain / 4) <= 1e-15).all()
    based, one = m.Fused.rotary_frequencies(64, 1e4, "base", 4.0)
    based = based.to_numpy()
    assert one == 1.0 and based[0] == 1 and abs(based[-1] * 4 / plain[-1] - 1) <= 1e-12 and (np.diff(based / plain) < 0).all()
    yarn, up = m.Fused.rotary_frequencies(64, 1e4, "yarn", 4.0, trained=4096)
    yarn = yarn.to_numpy()
    turns = 4096 * plain / (2 * math.pi)
    assert abs(up - (1 + 0.1 * math.log(4.0))) <= 1e-15
    # those of 32 turns and more stay, those of one and less go by the factor, but for the pairs at the two borders
    assert (yarn[:np.sum(turns >= 32)] == plain[:np.sum(turns >= 32)]).all()
    slow = np.sum(turns > 1) + 1
    assert (np.abs(yarn[slow:] * 4 / plain[slow:] - 1) <= 1e-15).all() and (np.diff(yarn / plain) <= 0).all()
    for bad in (dict(dims=7), dict(dims=0), dict(dims=8, base=1.0), dict(dims=8, factor=0.5), dict(dims=8, scaling="other"), dict(dims=8, scaling="yarn", factor=2.0),
                dict(dims=8, scaling="yarn", trained=100, fast=1.0, slow=2.0)):
        with pytest.raises(ValueError):
            m.Fused.rotary_frequencies(**bad)
