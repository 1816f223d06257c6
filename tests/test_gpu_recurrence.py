"""The gated linear recurrence and its gradients against one step after the other in 64 bits and more.

Tolerances: with u half a step of the type, a step adds at most u times the state's magnitude (one fused rounding) and
carries the error before it on by |a|. Where an axis is cut, the parts start from zero and are joined by products of
a, whose roundings and the join's are of the same kind, each bounded by u times the same recurrence of magnitudes
H[t] = |a| H[t-1] + |b|. So E[t] = |a| E[t-1] + u H[t], twice for the two kinds; the gradient's steps round twice."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

TYPES = [np.float32, np.float64]


def cls_of(m, dt):
    return m.SFloat if dt == np.float32 else m.DFloat


def steps(a, b, h0, u):
    """States, and the bound E, along axis 0."""
    wide = np.float64 if u > 2.0 ** -30 else np.longdouble
    h, e, size = np.empty(b.shape, wide), np.empty(b.shape), np.empty(b.shape)
    state = np.zeros(b.shape[1:], wide) if h0 is None else h0.astype(wide)
    big, err = np.abs(state).astype(np.float64), np.zeros(b.shape[1:])
    for t in range(b.shape[0]):
        state = a[t].astype(wide) * state + b[t].astype(wide)
        big = np.abs(a[t]) * big + np.abs(b[t])
        err = np.abs(a[t]) * err + u * big
        h[t], e[t], size[t] = state, err, big
    return h, e, size


def make(rng, shape, dt, resets=True):
    a = rng.uniform(-0.2, 1.0, shape)
    if resets:
        a[rng.random(shape) < 0.02] = 0.0
        a[rng.random(shape) < 0.02] = 1.0
    return a.astype(dt), rng.standard_normal(shape).astype(dt)


def check(m, a, b, h0, axis, dt, arrays=None):
    """Forward and gradients of host arrays; `arrays`: device views of the same values."""
    cls, u = cls_of(m, dt), np.finfo(dt).eps / 2
    da, db = arrays or (cls.cast(a), cls.cast(b))
    d0 = None if h0 is None else cls.cast(h0)
    h = m.Fused.recurrence(da, db, d0, axis=axis)
    assert type(h) is cls and h.shape == a.shape
    front = lambda v: np.moveaxis(v, axis, 0)  # noqa: E731
    want, tol, _ = steps(front(a), front(b), h0, u)
    got = front(h.to_numpy())
    assert (np.abs(got - want) <= 2 * tol).all(), float((np.abs(got - want) / np.maximum(tol, 1e-300)).max())
    # gradients, with g = b and the states just checked
    out = m.Fused.recurrence_grad(db, da, h, d0, axis=axis)
    ga, gb = (front(v.to_numpy()) for v in out[:2])
    fa = front(a)
    n = fa.shape[0]
    after = np.concatenate([fa[1:], np.zeros_like(fa[:1])]) if n else fa
    want, tol, _ = steps(after[::-1], front(b)[::-1], None, u)
    want, tol = want[::-1], tol[::-1]
    assert (np.abs(gb - want) <= 4 * tol).all()
    zero = np.zeros(fa.shape[1:], dt) if h0 is None else h0
    before = np.concatenate([zero[None], got[:-1]]) if n else got
    assert (np.abs(ga - want * before) <= (4 * tol + u * np.abs(want)) * np.abs(before) * (1 + 1e-6)).all()
    if h0 is not None:
        w0 = fa[0] * want[0] if n else np.zeros_like(zero)
        t0 = np.abs(fa[0]) * (4 * tol[0] + u * np.abs(want[0])) * (1 + 1e-6) if n else 0
        assert out[2].shape == d0.shape and (np.abs(out[2].to_numpy() - w0) <= t0).all()
    else:
        assert len(out) == 2


# one step, a few, around the lengths that lanes, waves and blocks hold; few and many columns, an odd number; long with few columns
AXIS1 = [(1, 1, 1), (2, 1, 5), (64, 1, 1000), (3, 2, 64), (2, 7, 65), (1, 31, 63), (5, 32, 33), (2, 33, 128), (1, 64, 1), (1, 100, 300), (3, 257, 17),
         (2, 1000, 70), (1, 4097, 3), (1, 5000, 129), (700, 40, 64), (40, 3, 2000), (1, 2, 70000), (1, 30011, 2), (4, 520, 4100)]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("shape", AXIS1)
def test_along_a_middle_axis(dt, shape):
    import cumo_amd as m
    rng = np.random.default_rng(shape[1])
    a, b = make(rng, shape, dt)
    h0 = rng.standard_normal((shape[0], shape[2])).astype(dt)
    check(m, a, b, None, 1, dt)
    check(m, a, b, h0, 1, dt)


ROWS = [(1,), (5,), (64,), (1000,), (20001,), (100003,), (3, 1), (7, 2), (1000, 3), (65, 16), (33, 31), (500, 64), (40, 65), (7, 255), (9, 1024), (3, 4097),
        (300, 1000), (2, 3, 515), (2000, 129), (5, 40000)]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("shape", ROWS)
def test_along_rows(dt, shape):
    import cumo_amd as m
    rng = np.random.default_rng(shape[-1])
    a, b = make(rng, shape, dt)
    h0 = np.asarray(rng.standard_normal(shape[:-1]), dt)
    check(m, a, b, None, len(shape) - 1, dt)
    check(m, a, b, h0, len(shape) - 1, dt)


@pytest.mark.parametrize("dt", TYPES)
def test_first_axis_negative_axis_and_four_dimensions(dt):
    import cumo_amd as m
    rng = np.random.default_rng(1)
    a, b = make(rng, (50, 6, 7), dt)
    check(m, a, b, rng.standard_normal((6, 7)).astype(dt), 0, dt)
    a, b = make(rng, (3, 4, 20, 5), dt)
    check(m, a, b, rng.standard_normal((3, 4, 5)).astype(dt), 2, dt)
    cls = cls_of(m, dt)
    assert (m.Fused.recurrence(cls.cast(a), cls.cast(b), axis=-2).to_numpy() == m.Fused.recurrence(cls.cast(a), cls.cast(b), axis=2).to_numpy()).all()
    assert (m.Fused.recurrence(cls.cast(a), cls.cast(b)).to_numpy() == m.Fused.recurrence(cls.cast(a), cls.cast(b), axis=3).to_numpy()).all()


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("n", [9, 70, 700])
def test_views(dt, n):
    """Windows of time and of channels, time backwards, every other channel, a transposed array: the results of copies."""
    import cumo_amd as m
    cls = cls_of(m, dt)
    rng = np.random.default_rng(n)
    wide = make(rng, (3, n + 5, 40), dt)
    da, db = (cls.cast(v) for v in wide)
    every = slice(None)
    for key in [(every, slice(2, n + 2), every), (every, slice(0, n), slice(3, 36)), (every, slice(None, None, -1), every), (slice(None, None, 2), slice(0, n), every),
                (every, slice(0, n), slice(1, None, 2)), (every, slice(0, n, 3), slice(None, None, -1)), (slice(1, 2), slice(4, n), slice(5, 6))]:
        a, b = (np.ascontiguousarray(v[key]) for v in wide)
        h0 = rng.standard_normal((a.shape[0], a.shape[2])).astype(dt)
        check(m, a, b, h0, 1, dt, (da[key], db[key]))
    for perm in [(1, 0, 2), (2, 0, 1), (0, 2, 1), (2, 1, 0)]:
        a, b = (np.ascontiguousarray(v.transpose(perm)) for v in wide)
        for axis in range(3):
            check(m, a, b, None, axis, dt, (da.transpose(*perm), db.transpose(*perm)))


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("shape,axis", [((2, 3000, 33), 1), ((4, 5000), 1), ((700, 300), 0)])
def test_one_step_at_a_time_is_the_whole(dt, shape, axis):
    """Generation: the state of a prompt carried on token by token; both roundings are the same fused one, so a state
    that was reached is continued to the bit of the step's formula."""
    import cumo_amd as m
    cls = cls_of(m, dt)
    rng = np.random.default_rng(2)
    a, b = make(rng, shape, dt)
    da, db = cls.cast(a), cls.cast(b)
    h = m.Fused.recurrence(da, db, axis=axis)
    cut = shape[axis] - 3
    pick = lambda v, k: v[(slice(None),) * axis + (k,)]  # noqa: E731
    state = pick(h, cut - 1)
    for t in range(cut, shape[axis]):
        one = m.Fused.recurrence(pick(da, slice(t, t + 1)), pick(db, slice(t, t + 1)), state, axis=axis)
        state = pick(one, 0)
        want = np.float64(pick(a, t)) * pick(h, t - 1).to_numpy() + pick(b, t)
        assert np.abs(state.to_numpy() - want).max() <= 4 * np.finfo(dt).eps * np.abs(want).max()
    # the same in two parts, the second from the first's last state
    first = m.Fused.recurrence(pick(da, slice(0, 7)), pick(db, slice(0, 7)), axis=axis)
    rest = m.Fused.recurrence(pick(da, slice(7, None)), pick(db, slice(7, None)), pick(first, 6), axis=axis)
    got = np.concatenate([first.to_numpy(), rest.to_numpy()], axis=axis)
    f = lambda v: np.moveaxis(v, axis, 0)  # noqa: E731
    want, tol, _ = steps(f(a), f(b), None, np.finfo(dt).eps / 2)
    assert (np.abs(f(got) - want) <= 2 * tol).all()


# down columns in one pass and cut, along rows held by a wave and cut
LONG = [((1, 3000, 8), 1), ((1, 40000, 64), 1), ((2, 60001), 1), ((3, 500), 1), ((600, 700), 1), ((1, 100, 40000), 1)]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("shape,axis", LONG)
def test_nan_infinity_and_products_beyond_the_type(dt, shape, axis):
    import cumo_amd as m
    cls = cls_of(m, dt)
    rng = np.random.default_rng(6)
    n = shape[axis]
    f = lambda v: np.moveaxis(v, axis, 0)  # noqa: E731
    # a NaN and an infinity reach what comes after them, until a gate of 0 (0 * NaN is NaN: nothing ends it but the end)
    a, b = (np.full(shape, v, dt) for v in (0.5, 1.0))
    f(b)[n // 3].flat[0] = np.nan
    got = f(m.Fused.recurrence(cls.cast(a), cls.cast(b), axis=axis).to_numpy()).reshape(n, -1)
    assert np.isnan(got[n // 3:, 0]).all() and np.isfinite(got[:n // 3, 0]).all() and np.isfinite(got[:, 1:]).all()
    f(b)[n // 3].flat[0] = np.inf
    got = f(m.Fused.recurrence(cls.cast(a), cls.cast(b), axis=axis).to_numpy()).reshape(n, -1)
    assert (got[n // 3:, 0] == np.inf).all() and np.isfinite(got[:n // 3, 0]).all() and np.isfinite(got[:, 1:]).all()
    # a state of zero meets gates whose products are beyond the type, and stays zero; one input comes last
    a, b = np.full(shape, 2.0, dt), np.zeros(shape, dt)
    f(b)[n - 1] = 3.0
    got = f(m.Fused.recurrence(cls.cast(a), cls.cast(b), axis=axis).to_numpy())
    assert (got[:n - 1] == 0).all() and (got[n - 1] == 3).all()
    gb = f(m.Fused.recurrence_grad(cls.cast(b[..., ::-1] if axis == len(shape) - 1 else b[:, ::-1]), cls.cast(a), cls.cast(b), axis=axis)[1].to_numpy())
    assert (gb[0] == 3).all() and (gb[1:] == 0).all()
    # gates of zero forget whatever came before, to the bit
    a = rng.uniform(0, 1, shape).astype(dt)
    b = rng.standard_normal(shape).astype(dt)
    f(a)[n // 2] = 0
    got = f(m.Fused.recurrence(cls.cast(a), cls.cast(b), axis=axis).to_numpy())
    assert (got[n // 2] == f(b)[n // 2]).all()
    # products that vanish and grow back within the type: 2^-60 (SFloat), 2^-500 (DFloat) and back, twice over
    k = 60 if dt == np.float32 else 500
    a, b = np.ones(shape, dt), np.zeros(shape, dt)
    for at in range(0, n - 2 * k, 2 * k):
        f(a)[at:at + k], f(a)[at + k:at + 2 * k] = 0.5, 2.0
    h0 = np.full(f(a).shape[1:], 3.0, dt)
    got = f(m.Fused.recurrence(cls.cast(a), cls.cast(b), cls.cast(h0), axis=axis).to_numpy())
    assert (got[n - 1] == 3).all()
    # products that vanish beyond any type and grow back as far: a state that is left, or none, but nothing larger than it
    a[:] = 0.5
    f(a)[n // 2:] = 2.0
    got = f(m.Fused.recurrence(cls.cast(a), cls.cast(b), cls.cast(h0), axis=axis).to_numpy())
    assert (got >= 0).all() and (got <= 3).all() and np.abs(got[0] - 1.5).max() == 0
    # an infinite state stays so through such a product, with its sign
    f(a)[:] = -0.5
    got = f(m.Fused.recurrence(cls.cast(a), cls.cast(b), cls.cast(np.full(h0.shape, np.inf, dt)), axis=axis).to_numpy())
    assert (got[0::2] == -np.inf).all() and (got[1::2] == np.inf).all()


@pytest.mark.parametrize("dt", TYPES)
def test_of_nothing(dt):
    import cumo_amd as m
    cls = cls_of(m, dt)
    for shape, axis in [((0,), 0), ((3, 0, 4), 1), ((0, 5), 1), ((2, 5, 0), 1)]:
        x = cls.cast(np.zeros(shape, dt))
        h0 = cls.cast(np.ones([n for d, n in enumerate(shape) if d != axis], dt))
        assert m.Fused.recurrence(x, x, h0, axis=axis).shape == shape
        ga, gb, g0 = m.Fused.recurrence_grad(x, x, x, h0, axis=axis)
        assert ga.shape == gb.shape == shape and g0.shape == h0.shape and (g0.to_numpy() == 0).all()


def test_gradients_match_differences():
    """Central differences in double of sum(g h): every entry is linear in each input apart from the products."""
    import cumo_amd as m
    rng = np.random.default_rng(7)
    a, b = make(rng, (2, 40, 3), np.float64, resets=False)
    g, h0 = rng.standard_normal(a.shape), rng.standard_normal((2, 3))
    d = m.DFloat.cast

    def loss(a, b, h0):
        return float((m.Fused.recurrence(d(a), d(b), d(h0), axis=1).to_numpy() * g).sum())

    h = m.Fused.recurrence(d(a), d(b), d(h0), axis=1)
    grads = [v.to_numpy() for v in m.Fused.recurrence_grad(d(g), d(a), h, d(h0), axis=1)]
    step = 1e-6
    for k, (v, grad) in enumerate(zip((a, b, h0), grads)):
        for at in [tuple(rng.integers(0, n) for n in v.shape) for _ in range(6)] + [(0,) * v.ndim]:
            e = np.zeros_like(v)
            e[at] = step
            up, down = [a, b, h0], [a, b, h0]
            up[k], down[k] = v + e, v - e
            assert abs((loss(*up) - loss(*down)) / (2 * step) - grad[at]) < 1e-7 * (1 + abs(grad[at]))


@pytest.mark.parametrize("shape,axis", [((2, 1, 500), 1), ((1, 5000, 33), 1), ((2, 4000, 700), 1), ((3, 30000), 1), ((400, 100), 1)])
def test_captured_and_replayed(shape, axis):
    import cumo_amd as m
    from cumo_amd import _lib
    from test_gpu_rmsnorm import replayed
    rng = np.random.default_rng(3)
    a, b = (m.SFloat.cast(v) for v in make(rng, shape, np.float32))
    h0 = m.SFloat.cast(rng.standard_normal([n for d, n in enumerate(shape) if d != axis]).astype(np.float32))
    h = m.Fused.recurrence(a, b, h0, axis=axis)
    fixed = h.copy()
    results = [h] + list(m.Fused.recurrence_grad(b, a, fixed, h0, axis=axis))
    wants = [v.to_numpy() for v in results]
    da, db, d0, df = (C.byref(v._desc()) for v in (a, b, h0, fixed))
    oh, oa, ob, o0 = (C.byref(v._desc()) for v in results)

    def call():
        _lib.call(_lib.lib.cumo_hip_na_recurrence, da, db, d0, axis, oh)
        _lib.call(_lib.lib.cumo_hip_na_recurrence_grad, db, da, df, d0, axis, oa, ob, o0)

    replayed(m, call, results, wants)


@pytest.mark.parametrize("shape,axis", [((3, 200, 40), 1), ((1, 9000, 5), 1), ((5, 3000), 1)])
def test_into_given_arrays(shape, axis):
    """Over an operand, into a window with steps, one element along: copies' results, and nothing beside them changes."""
    import cumo_amd as m
    from cumo_amd import _lib
    rng = np.random.default_rng(4)
    a, b = make(rng, shape, np.float32)
    want = m.Fused.recurrence(m.SFloat.cast(a), m.SFloat.cast(b), axis=axis)
    grads = [v.to_numpy() for v in m.Fused.recurrence_grad(m.SFloat.cast(b), m.SFloat.cast(a), want, axis=axis)]
    want = want.to_numpy()

    def call(x, y, z):
        d = [v._desc() for v in (x, y, z)]
        _lib.call(_lib.lib.cumo_hip_na_recurrence, C.byref(d[0]), C.byref(d[1]), None, axis, C.byref(d[2]))

    for over in (0, 1):
        ops = [m.SFloat.cast(a), m.SFloat.cast(b)]
        call(ops[0], ops[1], ops[over])
        assert (ops[over].to_numpy() == want).all()
    wide = m.SFloat(*[2 * n + 3 for n in shape]).fill(9)
    key = tuple(slice(1, 2 * n + 1, 2) for n in shape)
    call(m.SFloat.cast(a), m.SFloat.cast(b), wide[key])
    got = wide.to_numpy()
    assert (got[key] == want).all()
    got[key] = 9
    assert (got == 9).all()
    # gradients over their operands
    g, x, h = m.SFloat.cast(b), m.SFloat.cast(a), m.SFloat.cast(want)
    d = [v._desc() for v in (g, x, h)]
    _lib.call(_lib.lib.cumo_hip_na_recurrence_grad, C.byref(d[0]), C.byref(d[1]), C.byref(d[2]), None, axis, C.byref(d[1]), C.byref(d[0]), None)
    assert (x.to_numpy() == grads[0]).all() and (g.to_numpy() == grads[1]).all()


def test_columns_further_apart_than_32_bits_reach():
    """Every 2^19th element of rows of 2^25: 40 columns 128 MiB apart, 5 GiB in all, time in steps of 2 MiB."""
    import cumo_amd as m
    rng = np.random.default_rng(8)
    a, b = make(rng, (64, 40), np.float32)
    wide = [m.SFloat(40, 1 << 25) for _ in range(2)]
    views = [w.transpose()[::1 << 19] for w in wide]
    for view, h in zip(views, (a, b)):
        view.store(m.SFloat.cast(h))
    check(m, a, b, rng.standard_normal(40).astype(np.float32), 0, np.float32, views)


GIVING_UP = """
import ctypes as C
import cumo_amd as m
from cumo_amd import _lib
L = _lib.lib
L.cumo_hip_wait_give_ups.restype = C.c_int
L.cumo_hip_wait_give_ups.argtypes = [C.POINTER(C.c_uint32 * 4)]
for shape, axis in (((1, 60000, 64), 1), ((1, 1 << 22), 1)):
    a, b = m.SFloat(*shape).fill(0.5), m.SFloat(*shape).fill(1.0)
    m.synchronize()
    said = None
    try:
        for _ in range(5):
            h = m.Fused.recurrence(a, b, axis=axis)
            g = m.Fused.recurrence_grad(b, a, b, axis=axis)
        m.synchronize()
    except m.RuntimeError as e:
        said = str(e)
    counts = (C.c_uint32 * 4)()
    assert L.cumo_hip_wait_give_ups(C.byref(counts)) == 0
    assert said and "gave up" in said and counts[1] > 0, (shape, said, list(counts))
print("reported")
"""


def test_waits_that_give_up_are_reported():
    """With no looks allowed (the knob of tests/test_gpu_wait_give_up.py) tiles do not wait for those before them; every
    kernel ends, and the next wait for the device says so."""
    import os
    import subprocess
    import sys
    env = dict(os.environ, PYTHONPATH=os.path.dirname(os.path.dirname(os.path.abspath(__file__))), CUMO_HIP_WAIT_LIMIT="0")
    p = subprocess.run([sys.executable, "-c", GIVING_UP], env=env, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=100)
    assert p.returncode == 0 and "reported" in p.stdout, p.stdout[-2000:]


def test_more_columns_than_a_launch_has_lanes():
    """2^32 columns and some: operands of one number each, broadcast; results looked at around the launches' borders."""
    import cumo_amd as m
    from cumo_amd import _lib
    n = (1 << 32) + 777
    one = [m.SFloat.cast(np.full((1, 1), v, np.float32)) for v in (0.5, 3.0, -2.0)]
    wide = [v._desc() for v in one]
    for d in wide:
        d.shape[0], d.shape[1] = 2, n
        d.stride[0] = d.stride[1] = 0
    a, b, h = wide
    out = m.SFloat(2, n).fill(9)
    do = out._desc()
    _lib.call(_lib.lib.cumo_hip_na_recurrence, C.byref(a), C.byref(b), None, 0, C.byref(do))
    ends = [slice(0, 100), slice((1 << 31) - 100, (1 << 31) + 100), slice((1 << 32) - 100, (1 << 32) + 100), slice(n - 100, n)]
    for s in ends:
        got = out[:, s].to_numpy()
        assert (got[0] == 3.0).all() and (got[1] == 4.5).all()
    ga = m.SFloat(2, n).fill(9)
    dg = ga._desc()
    _lib.call(_lib.lib.cumo_hip_na_recurrence_grad, C.byref(b), C.byref(a), C.byref(h), None, 0, C.byref(dg), C.byref(do), None)
    for s in ends:
        got, gb = ga[:, s].to_numpy(), out[:, s].to_numpy()
        assert (gb[1] == 3.0).all() and (gb[0] == 4.5).all()
        assert (got[1] == -6.0).all() and (got[0] == 0.0).all()


def one_by_one(a, b, h0):
    """States along axis 0 in the arrays' own type."""
    h, state = np.empty_like(b), h0
    with np.errstate(over="ignore", invalid="ignore"):
        for t in range(len(b)):
            state = h[t] = a[t] * state + b[t]
    return h


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("shape,axis", LONG + [((1, 1200, 12800), 1), ((300, 3000), 1)])
def test_gates_of_zero_beside_products_beyond_double(dt, shape, axis):
    """What a gate of 0 forgets does not come back, however large the products of the gates after it, or before it; steps'
    own values are finite all along. They are exact, too: every product here is one of powers of two, or with 0."""
    import cumo_amd as m
    cls = cls_of(m, dt)
    n = shape[axis]
    f = lambda v: np.moveaxis(v, axis, 0)  # noqa: E731
    h0 = np.ones(f(np.empty(shape, dt)).shape[1:], dt)
    for gate in (4.0, 16.0, -16.0):
        for at in (0, 5, 31):
            a, b = np.full(shape, gate, dt), np.zeros(shape, dt)
            f(a)[at] = 0
            want = one_by_one(f(a), f(b), h0)
            assert np.isfinite(want).all()
            assert (f(m.Fused.recurrence(cls.cast(a), cls.cast(b), cls.cast(h0), axis=axis).to_numpy()) == want).all(), (gate, at)
            # backwards: a gradient at the last step alone, and a gate of 0 a few steps before it
            f(a)[at], f(a)[n - 1 - at] = gate, 0
            f(b)[n - 1] = 1
            h = np.ones(shape, dt)
            ga, gb, g0 = m.Fused.recurrence_grad(cls.cast(b), cls.cast(a), cls.cast(h), cls.cast(h0), axis=axis)
            after = np.concatenate([f(a)[1:], np.zeros_like(f(a)[:1])])
            want = one_by_one(after[::-1], f(b)[::-1], np.zeros_like(h0))[::-1]
            assert np.isfinite(want).all() and (f(gb.to_numpy()) == want).all() and (f(ga.to_numpy()) == want).all(), (gate, at)
            assert (g0.to_numpy() == (0 if n > at + 1 else f(a)[0] * want[0])).all()
    if dt == np.float64:
        # a small state through gates whose product is beyond double, and forgotten after that
        for first, second, last in ((1, 2, 3), (1, 40, 70), (40, 41, 90)):
            a, b = np.ones(shape, dt), np.zeros(shape, dt)
            f(a)[first] = f(a)[second] = 2.0 ** 660
            f(a)[last] = 0
            f(b)[n - 1] = 5
            h0[...] = 2.0 ** -990
            want = one_by_one(f(a), f(b), h0)
            got = f(m.Fused.recurrence(cls.cast(a), cls.cast(b), cls.cast(h0), axis=axis).to_numpy())
            assert np.isfinite(want).all() and (got[last:] == want[last:]).all() and (got[:first] == want[:first]).all(), (first, second, last)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("shape,axis", LONG)
def test_largest_numbers_as_gates(dt, shape, axis):
    """A gate of the type's largest number is a number like any other; an infinite one leaves nothing finite behind."""
    import cumo_amd as m
    cls = cls_of(m, dt)
    n = shape[axis]
    f = lambda v: np.moveaxis(v, axis, 0)  # noqa: E731
    a, b = np.ones(shape, dt), np.zeros(shape, dt)
    h0 = np.full(f(a).shape[1:], 2.0 ** -100, dt)
    f(a)[n // 2] = np.finfo(dt).max
    want = one_by_one(f(a), f(b), h0)
    got = f(m.Fused.recurrence(cls.cast(a), cls.cast(b), cls.cast(h0), axis=axis).to_numpy())
    assert (np.abs(got - want) <= 2 * np.finfo(dt).eps * want).all()
    f(a)[n // 2] = np.inf
    got = f(m.Fused.recurrence(cls.cast(a), cls.cast(b), cls.cast(h0), axis=axis).to_numpy())
    assert (got[: n // 2] == h0).all() and not np.isfinite(got[n // 2:]).any()


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("shape,axis", LONG + [((1, 2500, 12800), 1), ((300, 5000), 1)])
def test_products_beyond_the_type_of_states_within_it(dt, shape, axis):
    """A large state halved until it is nearly the smallest number and doubled again, a small one the other way, over and
    over: exact steps, however far their products reach."""
    import cumo_amd as m
    cls = cls_of(m, dt)
    n = shape[axis]
    f = lambda v: np.moveaxis(v, axis, 0)  # noqa: E731
    large, small, k = (2.0 ** 110, 2.0 ** -120, 240) if dt == np.float32 else (2.0 ** 1000, 2.0 ** -1010, 2030)
    for h0, first, second in ((large, 0.5, 2.0), (small, 2.0, 0.5), (-large, -0.5, 2.0)):
        a, b = np.ones(shape, dt), np.zeros(shape, dt)
        for at in range(0, n, 2 * k):
            f(a)[at:at + k], f(a)[at + k:at + 2 * k] = first, second
        start = np.full(f(a).shape[1:], h0, dt)
        want = one_by_one(f(a), f(b), start)
        assert np.isfinite(want).all() and (want != 0).all()
        got = f(m.Fused.recurrence(cls.cast(a), cls.cast(b), cls.cast(start), axis=axis).to_numpy())
        assert (got == want).all(), (h0, first)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("shape,axis", LONG + [((1, 1200, 12800), 1), ((300, 3000), 1)])
def test_gates_of_every_size(dt, shape, axis):
    """Powers of two from the type's smallest to its largest, at random but for the states that they lead through: those stay
    within the type, so every step is exact, and so are the products of any of them that a state goes through."""
    import cumo_amd as m
    cls = cls_of(m, dt)
    rng = np.random.default_rng(9)
    n = shape[axis]
    f = lambda v: np.moveaxis(v, axis, 0)  # noqa: E731
    reach, least, most = (120, -149, 127) if dt == np.float32 else (1000, -1074, 1023)
    lead = f(np.empty(shape, bool)).shape[1:]
    at = np.zeros(lead, np.int64)
    a, b = np.empty(shape, dt), np.zeros(shape, dt)
    # each column's states: a walk over the exponents, the same for all but for where it starts
    to = rng.integers(-reach, reach + 1, n)
    start = rng.integers(-reach, reach + 1, lead)
    at = start
    want = np.empty(f(a).shape, dt)
    for t in range(n):
        step = np.clip(to[t] - at, least, most)
        at = at + step
        f(a)[t] = np.ldexp(dt(1), step)
        want[t] = np.ldexp(dt(1), at)
    h0 = np.ldexp(dt(1), start).astype(dt)
    got = f(m.Fused.recurrence(cls.cast(a), cls.cast(b), cls.cast(h0), axis=axis).to_numpy())
    assert (got == want).all()
    # backwards the gradient of the last step walks the other way: gb[t] = a[t+1] ... a[n-1] = want[n-1] / want[t], where that stays in the type
    g = np.zeros(shape, dt)
    f(g)[n - 1] = 1
    back = np.empty_like(want)
    back[n - 1] = 1
    with np.errstate(over="ignore", under="ignore"):
        for t in range(n - 2, -1, -1):
            back[t] = f(a)[t + 1] * back[t + 1]
    gb = f(m.Fused.recurrence_grad(cls.cast(g), cls.cast(a), cls.cast(b), axis=axis)[1].to_numpy())
    # (exact until a first gradient leaves the normal numbers of the type)
    tiny, big = np.finfo(dt).tiny, np.finfo(dt).max
    fine = np.logical_and.accumulate(((back >= tiny) & (back <= big))[::-1], axis=0)[::-1]
    assert (gb[fine] == back[fine]).all() and fine[-1].all()
