"""Tokens chosen by given numbers, against the definition by sorting in 64 bits.

A weight is within 2^-39 of itself and half a unit (2^-45 for rows of 2^18) of exp; the fixed inputs here lie further than
that from every border, unless a border is meant, and then the weights are exact (equal logits)."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

TYPES = [np.float32, np.float64]


def cls_of(m, dt):
    return m.SFloat if dt == np.float32 else m.DFloat


def chosen(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """The definition, a row at a time."""
    rows, n = x.shape
    each = lambda v: np.broadcast_to(np.asarray(v, np.float64), (rows,))  # noqa: E731
    u, temperature, top_k, top_p, min_p = (each(v) for v in (u, temperature, top_k, top_p, min_p))
    out = np.empty(rows, np.int32)
    for r in range(rows):
        row = x[r].astype(np.float64)
        if n == 0 or np.isnan(row).any() or row.max() == -np.inf:
            out[r] = -1
            continue
        order = np.argsort(-row, kind="stable")
        row = row[order]
        if not temperature[r] > 0:
            out[r] = order[0]
            continue
        with np.errstate(invalid="ignore"):
            w = np.exp(np.where(row == row[0], 0.0, (row - row[0]) / temperature[r]))
        if 0 < top_k[r] < n:
            w[int(top_k[r]):] = 0
        if top_p[r] < 1:
            before = np.cumsum(w) - w
            keep = before < max(top_p[r], 0) * w.sum()
            keep[0] = True
            w = np.where(keep, w, 0)
        if min_p[r] > 0:
            w = np.where(w >= min(min_p[r], 1.0), w, 0)
        run = np.cumsum(w)
        at = int((run <= u[r] * run[-1]).sum())
        out[r] = order[min(at, int((w > 0).sum()) - 1)]
    return out


def take(m, x, u, dt, **settings):
    cls = cls_of(m, dt)
    given = {}
    for name, v in settings.items():
        if isinstance(v, np.ndarray):
            given[name] = m.Int32.cast(v) if name == "top_k" else cls.cast(v)
        else:
            given[name] = v
    out = m.Fused.sample(cls.cast(x), cls.cast(u), **given)
    assert type(out) is m.Int32
    return out.to_numpy()


SETTINGS = [{}, {"temperature": 0.7}, {"temperature": 30.0}, {"top_k": 1}, {"top_k": 5}, {"top_k": 40}, {"top_p": 0.9}, {"top_p": 0.1}, {"top_p": 0.0}, {"min_p": 0.05},
            {"min_p": 1.0}, {"temperature": 1.5, "top_k": 300, "top_p": 0.97, "min_p": 0.01}, {"temperature": 0.0}, {"top_k": 1 << 20}]
SHAPES = [(1, 1), (4, 2), (7, 3), (33, 64), (20, 65), (9, 1000), (5, 1024), (3, 1025), (6, 4099), (2, 20001), (3, 50001), (1, 131072), (300, 777)]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_matches_the_definition(dt, shape):
    import cumo_amd as m
    rng = np.random.default_rng(shape[1])
    x = (rng.standard_normal(shape) * 3).astype(dt)
    u = rng.random(shape[0]).astype(dt)
    for settings in SETTINGS:
        assert (take(m, x, u, dt, **settings) == chosen(x, u, **settings)).all(), settings


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("shape", [(8, 50), (4, 3000), (3, 40000), (2, 131072)])
def test_flat_rows_peaked_rows_and_many_equal_logits(dt, shape):
    import cumo_amd as m
    rng = np.random.default_rng(shape[0])
    u = rng.random(shape[0]).astype(dt)
    flat = (rng.standard_normal(shape) * 0.01).astype(dt)
    peaked = (rng.standard_normal(shape) * 2).astype(dt)
    peaked[:, 7] += 25
    coarse = (np.round(rng.standard_normal(shape) * 3 * 8) / 8).astype(dt)   # steps of 1/8: many of a kind
    two = np.where(rng.random(shape) < 0.5, 1.0, 0.0).astype(dt)
    for x in (flat, peaked, coarse, two):
        for settings in SETTINGS:
            assert (take(m, x, u, dt, **settings) == chosen(x, u, **settings)).all(), settings
    # settings that keep part of the equal ones
    for k in (1, 2, shape[1] // 3, shape[1] - 1):
        assert (take(m, two, u, dt, top_k=k) == chosen(two, u, top_k=k)).all(), k


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("n", [4, 64, 4096, 65536])
def test_equal_logits_are_taken_by_index_exactly(dt, n):
    """n equal weights (a power of two): the answer is floor(u n), at every border."""
    import cumo_amd as m
    k = np.unique(np.concatenate([np.arange(4), np.arange(n - 4, n), np.linspace(0, n - 1, 9).astype(int)]))
    at = np.concatenate([k / n, np.nextafter((k + 1) / n, 0)]).astype(np.float64)
    x = np.full((len(at), n), -2.5, dt)
    u = m.DFloat.cast(at)   # (u may be of the other type)
    got = m.Fused.sample(cls_of(m, dt).cast(x), u).to_numpy()
    assert (got == np.concatenate([k, k])).all()
    # the first half by top_k, then by top_p: a half exactly
    for settings in ({"top_k": n // 2}, {"top_p": 0.5}):
        got = m.Fused.sample(cls_of(m, dt).cast(x), u, **settings).to_numpy()
        assert (got == np.floor(at * (n // 2))).all(), settings


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("n", [3, 100, 5000, 70000])
def test_masked_infinite_and_nan_logits(dt, n):
    import cumo_amd as m
    rng = np.random.default_rng(n)
    x = rng.standard_normal((10, n)).astype(dt)
    x[0] = -np.inf                       # nothing to choose
    x[1] = -np.inf
    x[1, n // 2] = -1e30                 # one left
    x[2, 0] = np.nan
    x[3, n - 1] = np.inf                 # one that outweighs all
    x[4, [0, n - 1]] = np.inf            # two of those
    x[5, : n - 2] = -np.inf
    x[6] = np.finfo(dt).min              # the type's lowest value, everywhere
    x[7, 1:] = np.finfo(dt).min
    x[8] = 0.0
    x[8, ::2] = -0.0                     # the zeros are equal
    x[9] = rng.integers(0, 3, n) * np.finfo(dt).smallest_subnormal   # three numbers next to each other
    for u in (0.0, 0.3, 0.75, 1 - 2.0 ** -24):
        us = np.full(10, u, dt)
        for settings in SETTINGS + [{"top_k": 2}, {"top_k": n - 1}]:
            got = take(m, x, us, dt, **settings)
            want = chosen(x, us, **settings)
            assert (got == want).all(), (u, settings)
        assert got[0] == -1 and got[2] == -1 and got[1] == n // 2 and got[3] == n - 1


def test_u_outside_its_range_and_settings_at_their_limits():
    import cumo_amd as m
    x = np.log(np.array([[0.5, 0.25, 0.125, 0.125]], np.float64))
    for u, want in ((-1.0, 0), (np.nan, 0), (1.0, 3), (7.0, 3), (np.inf, 3)):
        assert take(m, x, np.array([u]), np.float64)[0] == want, u
    one = np.array([0.999])
    f = lambda **s: take(m, x, one, np.float64, **s)[0]  # noqa: E731
    d = lambda v: np.array([v], np.float64)  # noqa: E731
    # settings of rows are not refused but brought into their range
    assert f(temperature=d(-1.0)) == 0 and f(temperature=d(np.nan)) == 0 and f(temperature=d(np.inf)) == 3
    assert f(top_k=np.array([-3], np.int32)) == 3 and f(top_k=np.array([0], np.int32)) == 3 and f(top_k=np.array([2], np.int32)) == 1
    assert f(top_p=d(-0.5)) == 0 and f(top_p=d(np.nan)) == 3 and f(top_p=d(2.0)) == 3
    assert f(min_p=d(-1.0)) == 3 and f(min_p=d(np.nan)) == 3 and f(min_p=d(5.0)) == 0 and f(min_p=d(0.4)) == 1
    # numbers far from zero, an infinite one, at any temperature
    for shift in (1e6, -3e7, 1e30):
        for dt in TYPES:
            y = (np.array([[3.0, 2.0, 1.0, 0.0]]) * (1 if abs(shift) < 1e20 else 1e24) + shift).astype(dt)
            for t in (0.5, 1.0, 1e24, float("inf")):
                for u in (0.1, 0.6, 0.99):
                    assert take(m, y, np.array([u], dt), dt, temperature=t)[0] == chosen(y, np.array([u], dt), temperature=t)[0], (shift, dt, t, u)
    y = np.array([[1.0, np.inf, 2.0, np.inf]])
    assert take(m, y, np.array([0.3]), np.float64, temperature=float("inf"))[0] == 1 and take(m, y, np.array([0.7]), np.float64, temperature=2.0)[0] == 3
    assert f(temperature=1e-30) == 0 and f(temperature=1e300) == 3 and f(temperature=float("inf")) == 3


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("shape", [(40, 300), (64, 9001), (5, 60000)])
def test_a_row_of_its_own_settings_each(dt, shape):
    import cumo_amd as m
    rng = np.random.default_rng(12)
    rows = shape[0]
    x = (rng.standard_normal(shape) * 2).astype(dt)
    settings = {"temperature": np.where(rng.random(rows) < 0.2, 0, rng.uniform(0.3, 2, rows)).astype(dt), "top_k": rng.integers(0, 100, rows).astype(np.int32),
                "top_p": rng.uniform(0.2, 1, rows).astype(dt), "min_p": rng.uniform(0, 0.1, rows).astype(dt)}
    u = rng.random(rows).astype(dt)
    want = chosen(x, u, **settings)
    assert (take(m, x, u, dt, **settings) == want).all()
    # each row's answer does not depend on the rows beside it, nor on how many there are
    for r in range(0, rows, 7):
        one = {k: v[r:r + 1] for k, v in settings.items()}
        assert take(m, x[r:r + 1], u[r:r + 1], dt, **one)[0] == want[r]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("n", [300, 9000, 140000])
def test_few_tokens_left_by_a_mask_and_large_limits(dt, n):
    """A top_k beyond what a mask leaves, and top_k of every size around what lists hold."""
    import cumo_amd as m
    rng = np.random.default_rng(n)
    x = np.full((6, n), -np.inf, dt)
    for r, left in enumerate((1, 2, 17, 120, 200, 250)):
        x[r, rng.choice(n, left, replace=False)] = rng.standard_normal(left) * 2
    u = rng.random(6).astype(dt)
    full = (rng.standard_normal((6, n)) * 2).astype(dt)
    coarse = np.round(full * 4) / 4
    for k in (2, 17, 50, 255, 256, 257, 511, 512, 513, 1023, 1025, 5000, n - 1):
        for rows in (x, full, coarse):
            for more in ({}, {"top_p": 0.9}, {"min_p": 0.2, "temperature": 2.0}, {"top_p": 0.7, "min_p": 0.1}):
                assert (take(m, rows, u, dt, top_k=k, **more) == chosen(rows, u, top_k=k, **more)).all(), (k, more)


def test_more_rows_than_one_round_takes():
    import cumo_amd as m
    rng = np.random.default_rng(21)
    x = (rng.standard_normal((9001, 40)) * 2).astype(np.float32)
    u = rng.random(9001).astype(np.float32)
    k = rng.integers(0, 20, 9001).astype(np.int32)
    p = rng.uniform(0.3, 1, 9001).astype(np.float32)
    assert (take(m, x, u, np.float32, top_k=k, top_p=p) == chosen(x, u, top_k=k, top_p=p)).all()


@pytest.mark.parametrize("dt", TYPES)
def test_views_dimensions_and_nothing(dt):
    import cumo_amd as m
    cls = cls_of(m, dt)
    rng = np.random.default_rng(13)
    h = (rng.standard_normal((4, 6, 210)) * 2).astype(dt)
    u = rng.random((4, 6)).astype(dt)
    x, du = cls.cast(h), cls.cast(u)
    flat = lambda a: np.ascontiguousarray(a).reshape(-1, a.shape[-1])  # noqa: E731
    for key in [slice(None), (slice(None), slice(None), slice(3, 200)), (slice(None), slice(None), slice(None, None, 2)), (slice(None, None, -1), slice(1, 5)),
                (slice(None), slice(None), slice(None, None, -1))]:
        want = chosen(flat(h[key]), u[key[:2] if isinstance(key, tuple) else key].reshape(-1), top_p=0.8)
        got = m.Fused.sample(x[key], du[key[:2] if isinstance(key, tuple) else key], top_p=0.8)
        assert got.shape == h[key].shape[:-1] and (got.to_numpy().reshape(-1) == want).all(), key
    t = np.ascontiguousarray(h[0].T)   # [210, 6]
    assert (m.Fused.sample(cls.cast(t).transpose(), du[0]).to_numpy() == chosen(h[0], u[0])).all()
    one = m.Fused.sample(cls.cast(h[0, 0]), cls.cast(u[0, 0]))   # a row: no dimensions are left
    assert one.shape == () and int(one) == chosen(h[0, :1], u[0, :1])[0]
    assert (m.Fused.sample(cls(5, 0), cls.cast(np.zeros(5, dt))).to_numpy() == -1).all()
    assert m.Fused.sample(cls(0, 5), cls(0)).shape == (0,)


@pytest.mark.parametrize("dt", TYPES)
def test_shares_are_those_of_the_weights(dt):
    """Numbers evenly over [0, 1): every token has its share of them, within one."""
    import cumo_amd as m
    cls = cls_of(m, dt)
    rng = np.random.default_rng(14)
    n, rows = 12, 4000
    row = rng.standard_normal(n).astype(dt)
    x = np.broadcast_to(row, (rows, n))
    u = (np.arange(rows) + 0.5) / rows
    got = m.Fused.sample(cls.cast(x), m.DFloat.cast(u), 0.9).to_numpy()
    p = np.exp(row.astype(np.float64) / 0.9)
    p /= p.sum()
    assert (np.abs(np.bincount(got, minlength=n) - p * rows) <= 1).all()


@pytest.mark.parametrize("shape", [(1, 131072), (3, 900), (200, 5000)])
def test_captured_and_replayed(shape):
    import cumo_amd as m
    from cumo_amd import _lib
    from test_gpu_rmsnorm import replayed
    rng = np.random.default_rng(3)
    x = m.SFloat.cast((rng.standard_normal(shape) * 2).astype(np.float32))
    u = m.SFloat.cast(rng.random(shape[0]).astype(np.float32))
    results = [m.Fused.sample(x, u, 0.8, 40, 0.95, 0.01), m.Fused.sample(x, u, 1.0, 0, 0.99)]
    wants = [v.to_numpy() for v in results]
    dx, du, o1, o2 = (C.byref(v._desc()) for v in (x, u, *results))

    def call():
        _lib.call(_lib.lib.cumo_hip_na_sample, dx, du, 0.8, None, 40, None, 0.95, None, 0.01, None, o1)
        _lib.call(_lib.lib.cumo_hip_na_sample, dx, du, 1.0, None, 0, None, 0.99, None, 0.0, None, o2)

    replayed(m, call, results, wants)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("n", [6000, 70001])
def test_more_numbers_together_than_are_put_in_order(dt, n):
    """A crowd far below its row's largest number: of many different numbers, of few, of two with infinities above."""
    import cumo_amd as m
    rng = np.random.default_rng(n)
    x = np.empty((8, n), dt)
    x[0] = rng.standard_normal(n) * 1e-3
    x[1] = 100 + rng.standard_normal(n) * 1e-3
    x[2] = np.round(rng.standard_normal(n) * 8) / 4096
    x[3] = np.where(rng.random(n) < 0.5, 0.0, np.finfo(dt).eps)
    x[4] = rng.standard_normal(n) * 3
    x[5] = np.where(rng.random(n) < 0.7, -1e30, 1e30)
    x[6] = -np.exp(rng.uniform(-80, 80, n))
    x[7] = rng.standard_normal(n)
    x[:4, n // 3] += 9                       # (70001 exp(-9): 8.6, next to the largest's 1)
    x[7, : n // 2] = np.inf
    for u in (0.02, 0.4, 0.999):
        us = np.full(8, u, dt)
        for settings in ({}, {"top_k": 5}, {"top_k": 300}, {"top_k": 300, "min_p": 1e-5}, {"top_k": n // 2}, {"top_p": 0.9}, {"top_k": n // 3, "top_p": 0.7},
                         {"top_k": 400, "top_p": 0.8, "min_p": 1e-4}, {"min_p": 1e-5}, {"top_k": n // 2 + 40}):
            assert (take(m, x, us, dt, **settings) == chosen(x, us, **settings)).all(), (u, settings)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("n", [2, 70, 5000, 70001])
def test_logits_further_apart_than_their_type_reaches(dt, n):
    """Differences beyond the type's largest number, at temperatures at which such logits still have weights. Logits and
    temperature are a quarter of themselves for the definition, which goes by their quotients alone."""
    import cumo_amd as m
    rng = np.random.default_rng(n)
    top = float(np.finfo(dt).max)
    x = np.empty((5, n), dt)
    x[0] = np.where(np.arange(n) % 2, -0.9, 0.9) * top
    x[1] = -top
    x[1, n // 2] = 0.3 * top
    x[2] = rng.uniform(-1, 1, n) * top
    x[3] = -top
    x[3, ::3] = top
    x[4] = rng.standard_normal(n)
    x[4, n // 3] = -top
    x[4, n - 1] = top
    for u in (0.02, 0.4, 0.75, 0.999):
        us = np.full(5, u, dt)
        for temperature in (float("inf"), top, top / 3, top / 60, 1.0):
            for settings in ({}, {"top_k": 1 << 20}, {"top_k": 600}, {"top_k": 300}, {"top_p": 0.9}, {"top_p": 0.3}, {"min_p": 0.2}, {"top_k": n - 1, "top_p": 0.7, "min_p": 0.01}):
                got = take(m, x, us, dt, temperature=temperature, **settings)
                want = chosen(x.astype(np.float64) / 4, us, temperature=temperature / 4, **settings)
                assert (got == want).all(), (u, temperature, settings, got, want)


@pytest.mark.parametrize("n", [2, 900, 20001])
def test_logits_of_the_size_of_the_smallest_normal_numbers(n):
    """Temperatures so small that a bin for each 48th of one is more bins a unit than SFloat counts."""
    import cumo_amd as m
    rng = np.random.default_rng(n)
    x = (rng.standard_normal((4, n)) * 1e-36).astype(np.float32)
    x[3, 0] = 7.0
    for u in (0.1, 0.6, 0.95):
        us = np.full(4, u, np.float32)
        for settings in ({}, {"top_k": 700}, {"top_k": 40}, {"top_p": 0.8}, {"min_p": 0.05}):
            for temperature in (1e-37, 1e-36, 1e-38):
                assert (take(m, x, us, np.float32, temperature=temperature, **settings) == chosen(x, us, temperature=temperature, **settings)).all(), (u, settings)


@pytest.mark.parametrize("dt,margin", [(np.float32, 2.0 ** -37), (np.float64, 2.0 ** -46)])
def test_weights_are_as_exact_as_the_type(dt, margin):
    """Two tokens, numbers next to either side of their border. A weight is off by half a unit (2^-51), by what its exponent has been
    rounded (|z| e^z 2^-52 for z = (x - max) / temperature: 2^-53 at most) and by its exponential: 2^-39 for SFloat, less
    than 2^-51 for DFloat."""
    import cumo_amd as m
    rng = np.random.default_rng(31)
    x = np.zeros((3000, 2), dt)
    x[:, 1] = -rng.uniform(0.01, 6, 3000)
    for temperature in (1.0, 0.37, 2.5):
        w = np.exp(x[:, 1].astype(np.longdouble) / np.longdouble(temperature))
        border = 1 / (1 + w)
        for side, want in ((-1, 0), (1, 1)):
            u = (border + side * np.longdouble(margin)).astype(np.float64)
            got = m.Fused.sample(cls_of(m, dt).cast(x), m.DFloat.cast(u), temperature).to_numpy()
            assert (got == want).all(), (temperature, side, int((got != want).sum()))


def broadcast_row(m, x, u, **settings):
    """One row of logits for every number of u, without copies of it."""
    from cumo_amd import _lib
    x, u = cls_of(m, x.dtype).cast(x), m.DFloat.cast(u)
    d, du = x._desc(), u._desc()
    d.ndim = 2
    d.shape[0], d.shape[1], d.stride[0], d.stride[1] = u.shape[0], x.shape[0], 0, d.stride[0]
    z = m.Int32(u.shape[0]).fill(-9)
    dz = z._desc()
    _lib.call(_lib.lib.cumo_hip_na_sample, C.byref(d), C.byref(du), settings.get("temperature", 1.0), None, settings.get("top_k", 0), None, settings.get("top_p", 1.0), None,
              settings.get("min_p", 0.0), None, C.byref(dz))
    return z.to_numpy()


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("n,low", [((1 << 18) + 1, -32.0), (1 << 20, -30.0), ((1 << 24) + 5, -30.0)])
def test_long_rows_keep_what_a_flat_tail_holds(dt, n, low):
    """One token and a flat tail far below it. Either sum that an answer compares is off by n / 2 units at most, the unit being 2^-50 of the
    largest weight where the row's sum allows it, and by 2^-39 of the tail: so answers are those of numbers that far from u."""
    import cumo_amd as m
    x = np.full(n, low, dt)
    top = n // 3
    x[top] = 0
    w = np.exp(np.float64(low))
    tail = w * (n - 1)
    u = np.concatenate([[0.0, 0.5, 1 - 2 * tail], 1 - tail * np.array([0.9, 0.5, 0.25, 0.1, 1e-3])])
    got = broadcast_row(m, x, u)
    place = np.where(got == top, 0, np.where(got < top, got + 1, got)).astype(np.float64)   # in order of falling x
    total = 1 + tail
    begin, end = np.where(place == 0, 0, 1 + (place - 1) * w) / total, (1 + place * w) / total
    off = 2 * n * 2.0 ** -51 + 2.0 ** -38 * tail
    assert ((got >= 0) & (begin - off <= u) & (u <= end + off)).all(), (got, begin - u, end - u)
    assert (got[:2] == top).all() and (got[3:] != top).all()


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("n", [(1 << 18) + 1, 1 << 20, (1 << 22) + 77])
def test_long_rows(dt, n):
    """Every answer's stretch of the running sum holds u, but for n 2^-51 of the sum and 2^-39 of the weights, either way."""
    import cumo_amd as m
    rng = np.random.default_rng(n)
    x = (rng.standard_normal(n) * 3).astype(dt)
    u = np.concatenate([rng.random(20), [0.0, 0.999999]])
    order = np.argsort(-x, kind="stable")
    rank = np.empty(n, np.int64)
    rank[order] = np.arange(n)
    every = np.exp(x[order].astype(np.float64) - np.float64(x[order[0]]))
    for settings in ({}, {"top_k": n // 2}, {"top_p": 0.9}, {"min_p": 1e-4}, {"top_k": 700}, {"top_k": 40}):
        w = every.copy()
        w[settings.get("top_k") or n:] = 0
        w[w < settings.get("min_p", 0.0)] = 0
        run = np.cumsum(w)
        off = 2.0 ** -37 + 2 * n * 2.0 ** -51
        if "top_p" in settings:
            w[1:][run[:-1] >= settings["top_p"] * run[-1]] = 0
            off += off + w[w > 0].min() / w.sum()   # (the limit may be a token off)
            run = np.cumsum(w)
        at = rank[broadcast_row(m, x, u, **settings)]
        assert ((run[at] - w[at]) / run[-1] - off <= u).all() and (u <= run[at] / run[-1] + off).all(), settings
    flat = np.full(1 << 20, 2.0, dt)
    at = np.arange(0, 1 << 20, 99991)
    assert (broadcast_row(m, flat, at / 2.0 ** 20) == at).all() and (broadcast_row(m, flat, np.nextafter((at + 1) / 2.0 ** 20, 0)) == at).all()
